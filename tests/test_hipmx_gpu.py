"""GPU tests of microscaled 4-bit quantisation and product (ops/hipmx.py).

The kernels' codes have to be those of the definition, bit for bit. Products
of codes are exact in float32, so a result is off by what its sum in float32
and its one rounding cost.
"""

import sys
from pathlib import Path

import numpy as np
import pytest

OPS_DIR = Path(__file__).resolve().parent.parent / "code_interpreter_amd" / "ops"
sys.path.insert(0, str(OPS_DIR))
sys.path.insert(0, str(Path(__file__).resolve().parent))

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "bfloat16", "float16"]


@pytest.fixture(scope="module")
def mx():
    torch = pytest.importorskip("torch")
    if not torch.cuda.is_available():
        pytest.skip("torch sees no GPU")
    import hipmx

    return torch, hipmx


def values(torch, q):
    """What codes stand for, in 64 bits, on the host."""
    import lm_oracle as oracle

    return oracle.values(q.codes.cpu().numpy(), q.scales.cpu().numpy(),
                         q.shape[-1])


def same_codes(torch, hipmx, x):
    """The kernel's codes of x against those of the plain form on the host,
    which is tested against the definition element by element."""
    q, want = hipmx.quantize(x), hipmx.quantize(x.cpu())
    assert torch.equal(q.scales.cpu(), want.scales)
    # a negative number that rounds to 0 may keep its sign or not
    a, b = q.codes.cpu(), want.codes
    for shift in (0, 4):
        p, r = (a >> shift) & 15, (b >> shift) & 15
        assert torch.equal(torch.where(p == 8, 0, p), torch.where(r == 8, 0, r))
    return q


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 32), (3, 31), (5, 33),
                                   (7, 100), (64, 4096), (333, 1000),
                                   (2, 3, 65), (70000, 8)])
def test_quantize_codes(mx, dtype, shape):
    torch, hipmx = mx
    g = torch.Generator().manual_seed(sum(shape))
    x = torch.randn(*shape, generator=g) * torch.exp(
        4 * torch.randn(*shape, generator=g))
    x = x.clamp(-6e4, 6e4).to(getattr(torch, dtype)).cuda()
    q = same_codes(torch, hipmx, x)
    for out in DTYPES:
        v = q.dequantize(getattr(torch, out))
        want = torch.from_numpy(values(torch, q)).to(getattr(torch, out))
        assert torch.equal(v.cpu(), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_every_16_bit_pattern(mx, dtype):
    torch, hipmx = mx
    bits = torch.arange(65536, dtype=torch.int32)
    if dtype == "float32":
        x = (bits << 16).view(torch.float32)
    else:
        x = torch.where(bits > 32767, bits - 65536, bits).to(
            torch.int16).view(getattr(torch, dtype))
    g = torch.Generator().manual_seed(5)
    # in order (blocks of near values) and mixed (blocks of far ones, most
    # with a NaN among them), and mixed without NaN
    fine = x[torch.isfinite(x.float())]
    for t in (x, x[torch.randperm(65536, generator=g)],
              fine[torch.randperm(fine.numel(), generator=g)]):
        same_codes(torch, hipmx, t.reshape(1, -1).cuda())


def test_quantize_strided(mx):
    torch, hipmx = mx
    base = torch.randn(40, 200, device="cuda", dtype=torch.bfloat16)
    for x in (base[:, 3:103], base[::3], base.t(), base[:, ::2], base[5:6],
              base[0].expand(4, 200), base[:, 7]):
        same_codes(torch, hipmx, x)


def test_empty(mx):
    torch, hipmx = mx
    q = hipmx.quantize(torch.zeros(0, 40, device="cuda"))
    assert q.dequantize().shape == (0, 40)
    w = hipmx.quantize(torch.randn(5, 40, device="cuda"))
    assert hipmx.linear(torch.zeros(2, 0, 40, device="cuda"), w).shape == (2, 0, 5)


def operands(torch, hipmx, m, n, k, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g) * torch.exp(
        torch.randn(1, k, generator=g))
    w = torch.randn(n, k, generator=g) * 0.05
    bias = torch.randn(n, generator=g)
    dt = getattr(torch, dtype)
    return (x.to(dt).cuda(), hipmx.quantize(w.cuda()), bias.to(dt).cuda())


def check_linear(torch, hipmx, y, x, w, bias):
    """y against the product of the values in 64 bits. In float32 a sum of k
    products in any order is off by at most k 2^-24 of the sum of their
    magnitudes; the result is off by half a step more."""
    q = x if isinstance(x, hipmx.MXFP4Tensor) else hipmx.quantize(x)
    a = torch.from_numpy(values(torch, q)).cuda()
    b = torch.from_numpy(values(torch, w)).cuda()
    want, size = a @ b.T, a.abs() @ b.abs().T
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    k = a.shape[-1]
    info = torch.finfo(y.dtype)
    slack = ((k + 2) * 2.0 ** -24 * size * (1 + info.eps)
             + info.eps / 2 * want.abs() + info.smallest_normal * info.eps)
    err = (y.double() - want).abs()
    assert (err <= slack).all(), (err - slack).max().item()


SHAPES = [
    (1, 1, 1), (1, 16, 32), (1, 17, 33), (1, 512, 4096), (2, 100, 2056),
    (15, 64, 512), (16, 64, 544), (17, 65, 1000), (33, 48, 96), (48, 33, 64),
    (49, 128, 16384), (64, 1000, 777), (64, 16, 8192), (65, 64, 32),
    (65, 200, 1056), (127, 129, 255), (128, 128, 256), (129, 300, 300),
    (300, 257, 480), (1000, 96, 2048), (513, 4097, 288), (2049, 2050, 520),
    # few tokens, quantised in a launch of their own, and long rows
    (16, 64, 8192), (3, 40, 20001), (16, 8200, 4200),
    # tiles of 32 x 64, with and without a rest of k
    (96, 8200, 300), (65, 8192, 512), (33, 8191, 2080),
    # tiles of 64 x 128, 64 x 64 and 128 x 128 with a rest of k
    (333, 5001, 296), (130, 5600, 544), (1600, 2000, 1000),
    # a step of k more or less than the loads under way
    (40, 64, 1536), (40, 64, 1537), (40, 64, 1280), (200, 8200, 768),
]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear(mx, m, n, k, dtype):
    torch, hipmx = mx
    x, w, bias = operands(torch, hipmx, m, n, k, dtype, m + n + k)
    y = hipmx.linear(x, w, bias)
    assert y.shape == (m, n) and y.dtype == x.dtype
    check_linear(torch, hipmx, y, x, w, bias)
    check_linear(torch, hipmx, hipmx.linear(x, w), x, w, None)
    # an operand that comes quantised gives the same sums
    p = hipmx.linear(hipmx.quantize(x), w, bias, dtype=x.dtype)
    check_linear(torch, hipmx, p, x, w, bias)
    # and the same call the same bits
    assert torch.equal(hipmx.linear(x, w, bias), y)


@pytest.mark.parametrize("m,n,k", [(4096, 4096, 512), (4100, 4200, 264),
                                   (256, 16384, 1024)])
def test_linear_large(mx, m, n, k):
    torch, hipmx = mx
    x, w, bias = operands(torch, hipmx, m, n, k, "bfloat16", 1)
    check_linear(torch, hipmx, hipmx.linear(x, w, bias), x, w, bias)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_linear_tells_rows_and_columns_apart(mx, m):
    torch, hipmx = mx
    # a weight of one element a row, each of another size and place
    n = k = 320
    w = torch.zeros(n, k, device="cuda")
    at = (torch.arange(n, device="cuda") * 7) % k
    w[torch.arange(n), at] = 2.0 ** (torch.arange(n, device="cuda") % 9 - 4)
    x = torch.zeros(m, k, device="cuda")
    x[torch.arange(m), (torch.arange(m) * 11) % k] = 3.0
    y = hipmx.linear(x, hipmx.quantize(w))
    assert torch.equal(y, (x.double() @ w.double().T).float())


@pytest.mark.parametrize("m", [1, 20, 100])
def test_linear_nan_stays_in_its_row(mx, m):
    torch, hipmx = mx
    x, w, _ = operands(torch, hipmx, m, 100, 96, "float32")
    x[m // 2, 40] = float("inf")
    y = hipmx.linear(x, w)
    bad = y.isnan()
    assert bad[m // 2].all() and bad.sum() == 100
    w.scales[7, 2] = 255
    x[m // 2, 40] = 0.0
    bad = hipmx.linear(x, w).isnan()
    assert bad[:, 7].all() and bad.sum() == m


@pytest.mark.parametrize("m", [1, 24, 200])
def test_linear_scales_at_the_ends(mx, m):
    torch, hipmx = mx
    # large weights against small activations: the products are ordinary
    g = torch.Generator().manual_seed(2)
    x = (torch.randn(m, 128, generator=g) * 2.0 ** -100).cuda()
    w = hipmx.quantize((torch.randn(70, 128, generator=g) * 2.0 ** 100).cuda())
    y = hipmx.linear(x, w)
    check_linear(torch, hipmx, y, x, w, None)
    assert hipmx.linear(torch.zeros_like(x), w).abs().max() == 0


def test_linear_inputs_of_other_strides(mx):
    torch, hipmx = mx
    base = torch.randn(90, 400, device="cuda", dtype=torch.bfloat16)
    w = hipmx.quantize(torch.randn(50, 90, device="cuda"))
    for x in (base.t(), base.t()[:3], base.t()[::7], base.t()[3]):
        y = hipmx.linear(x, w)
        assert torch.equal(y, hipmx.linear(x.contiguous(), w))
    wide = torch.randn(30, 200, device="cuda")
    for x in (wide[:, 5:95], wide[:2, 1:91]):
        assert torch.equal(hipmx.linear(x, w),
                           hipmx.linear(x.contiguous(), w))
    bias = torch.randn(100, device="cuda")[::2]
    y = hipmx.linear(wide[:, :90], w, bias)
    assert torch.equal(y, hipmx.linear(wide[:, :90], w, bias.contiguous()))


@pytest.mark.parametrize("m,n,k", [(1, 5, 40), (3, 17, 64), (40, 37, 100),
                                   (70, 37, 64), (129, 131, 288),
                                   (2049, 2055, 32), (4097, 4101, 32)])
def test_results_end_where_they_end(mx, m, n, k):
    torch, hipmx = mx
    import lm_oracle as oracle

    x, w, _ = operands(torch, hipmx, m, n, k, "bfloat16")
    nb = -(-k // 32)
    bias = torch.zeros(n, device="cuda", dtype=torch.bfloat16)

    def ends(call):  # one call's results, looked at before the next
        oracle.fill_free_blocks(torch, 2 * m * n, 2 * m * k, m * nb * 16,
                                m * nb)
        out = call()
        torch.cuda.synchronize()
        for t in out:
            assert (oracle.behind(torch, t) == 0xA5).all()

    q = hipmx.quantize(x)
    ends(lambda: [hipmx.linear(x, w, bias)])
    ends(lambda: [hipmx.linear(q, w)])
    ends(lambda: (lambda p: [p.codes, p.scales])(hipmx.quantize(x)))
    ends(lambda: [q.dequantize()])


@pytest.mark.parametrize("m", [1, 16, 40, 200])
def test_linear_in_a_graph(mx, m):
    torch, hipmx = mx
    x, w, bias = operands(torch, hipmx, m, 300, 16384, "bfloat16")
    other = operands(torch, hipmx, m, 300, 16384, "bfloat16", 9)[0]
    want = [hipmx.linear(t, w, bias) for t in (x, other)]
    still = x.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        hipmx.linear(still, w, bias)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs, alive together
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = hipmx.linear(still, w, bias)
        graphs.append((g, y))
    for i in (0, 1, 0, 1):
        still.copy_((x, other)[i])
        for g, _ in graphs:
            g.replay()
        hipmx.linear(other, w, bias)  # eager work in between
        torch.cuda.synchronize()
        for _, y in graphs:
            assert torch.equal(y, want[i])


def test_linear_on_another_stream(mx):
    torch, hipmx = mx
    x, w, bias = operands(torch, hipmx, 130, 300, 512, "bfloat16")
    want = hipmx.linear(x, w, bias)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = hipmx.linear(x, w, bias)
        b = hipmx.linear(a[:, :256], hipmx.quantize(a[:40, :256]))
    side.synchronize()
    assert torch.equal(a, want)
    c = hipmx.linear(want[:, :256], hipmx.quantize(want[:40, :256]))
    assert torch.equal(b, c)


def test_torch_linear_dispatches(mx):
    torch, hipmx = mx
    import hiptorch

    x, w, bias = operands(torch, hipmx, 5, 64, 96, "bfloat16")
    want = hipmx.linear(x, w, bias)
    before = hipmx.STATS["linear"]
    assert torch.equal(torch.nn.functional.linear(x, w, bias), want)
    assert hiptorch.install(mode="require")
    try:
        assert torch.equal(torch.nn.functional.linear(x, w, bias), want)
    finally:
        hiptorch.uninstall()
    assert hipmx.STATS["linear"] == before + 2


def test_mixed_devices_are_refused(mx):
    torch, hipmx = mx
    x, w, bias = operands(torch, hipmx, 5, 64, 96, "bfloat16")
    with pytest.raises(ValueError, match="weight on"):
        hipmx.linear(x.cpu(), w)
    with pytest.raises(ValueError, match="bias must be"):
        hipmx.linear(x, w, bias.cpu())
    with pytest.raises(ValueError, match="different devices"):
        hipmx.MXFP4Tensor(w.codes, w.scales.cpu(), 96)
    moved = w.to("cpu")
    assert torch.equal(moved.dequantize(), w.dequantize().cpu())


def test_far_offsets(mx):
    """Tensors whose later rows stand behind 2^32 bytes and elements."""
    torch, hipmx = mx
    rows, k = 140_000, 32_768  # 4.6e9 elements, 2.3e9 bytes of codes
    x = torch.empty(rows, k, dtype=torch.bfloat16, device="cuda")
    last = torch.randn(64, k, device="cuda").bfloat16()
    x[:64] = last.flip(0)
    x[-64:] = last
    q, want = hipmx.quantize(x), hipmx.quantize(last)
    assert torch.equal(q.codes[-64:], want.codes)
    assert torch.equal(q.scales[-64:], want.scales)
    del x
    v = q.dequantize()
    assert torch.equal(v[-64:], want.dequantize())
    del v
    # as a weight, twice as long: the last rows' codes are behind 4 GB
    w = hipmx.MXFP4Tensor(torch.cat([q.codes, q.codes]),
                          torch.cat([q.scales, q.scales]), k)
    del q
    for m in (2, 20, 300):
        t = torch.randn(m, k, device="cuda").bfloat16()
        y = hipmx.linear(t, w)
        near = hipmx.linear(t, want)
        torch.testing.assert_close(y[:, -64:], near, rtol=0.02, atol=0.5)
        torch.testing.assert_close(y[:, :64], near.flip(1), rtol=0.02,
                                   atol=0.5)
    # as tokens: the rows of the result too
    y = hipmx.linear(w, want)
    near = hipmx.linear(want, want)
    torch.testing.assert_close(y[-64:], near, rtol=0.02, atol=0.5)


def test_long_rows(mx):
    torch, hipmx = mx
    k = hipmx.MAX_K
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(2, k, generator=g, device="cuda").sign()
    w = hipmx.quantize(torch.randn(3, k, generator=g, device="cuda").sign())
    want = x.double() @ w.dequantize(torch.float32).double().T
    # sums of ones: whole numbers below 2^24, exact in any order
    assert torch.equal(hipmx.linear(x, w).double(), want)
    assert torch.equal(hipmx.linear(x.repeat(20, 1), w).double(),
                       want.repeat(20, 1))


@pytest.mark.parametrize("m", [3, 40])
def test_views_that_negate(mx, m):
    """torch keeps a conjugate's imaginary part as a view with a mark; the
    kernels get its values."""
    torch, hipmx = mx
    g = torch.Generator(device="cuda").manual_seed(2)
    z = torch.randn(m, 100, 2, generator=g, device="cuda")
    x = torch.view_as_complex(z).conj().imag
    assert x.is_neg()
    q, want = hipmx.quantize(x), hipmx.quantize(x.resolve_neg())
    assert torch.equal(q.codes, want.codes)
    assert torch.equal(q.scales, want.scales)
    w = hipmx.quantize(torch.randn(m, 100, generator=g, device="cuda"))
    bias = x[:, 0]
    assert bias.is_neg()
    assert torch.equal(hipmx.linear(x, w, bias),
                       hipmx.linear(x.resolve_neg(), w, bias.resolve_neg()))


@pytest.mark.parametrize("m,n,k", [
    # 17 to 64 tokens that every block quantises, and just more than it does
    (17, 4095, 1900), (31, 33, 1000), (32, 100, 1024), (32, 100, 1025),
    (33, 40, 992), (47, 4096, 690), (63, 4095, 520), (64, 17, 31),
    (64, 4097, 100), (64, 1, 1), (50, 15, 600),
    # few tokens and many outputs
    (3, 20001, 4096), (8, 40000, 700), (16, 33000, 1030), (2, 9000, 8200),
])
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_few_tokens(mx, m, n, k, dtype):
    torch, hipmx = mx
    x, w, bias = operands(torch, hipmx, m, n, k, dtype, m + n + k)
    y = hipmx.linear(x, w, bias)
    check_linear(torch, hipmx, y, x, w, bias)
    check_linear(torch, hipmx, hipmx.linear(hipmx.quantize(x), w, dtype=x.dtype),
                 x, w, None)
    wide = torch.full((m, k + 3), 9.0, dtype=x.dtype, device="cuda")
    wide[:, 1:k + 1] = x
    assert torch.equal(hipmx.linear(wide[:, 1:k + 1], w, bias), y)


@pytest.mark.parametrize("m,n,k", [
    # low and wide: tiles by their height, scales laid out in many blocks
    (33, 40001, 300), (64, 33000, 1100), (65, 40001, 520), (128, 33000, 300),
    (129, 40001, 264), (70, 2049, 2500), (250, 40001, 1100), (1100, 9000, 1060),
])
def test_linear_wide(mx, m, n, k):
    torch, hipmx = mx
    x, w, bias = operands(torch, hipmx, m, n, k, "bfloat16", m + n + k)
    check_linear(torch, hipmx, hipmx.linear(x, w, bias), x, w, bias)
    check_linear(torch, hipmx, hipmx.linear(hipmx.quantize(x), w), x, w, None)


@pytest.mark.parametrize("m,n", [(333, 5001), (200, 4096), (100, 4096),
                                 (40, 100)])
@pytest.mark.parametrize("k", [8192, 8288])
def test_linear_rings_go_round(mx, m, n, k):
    """Each of the small tiles, long enough that its buffers are filled many
    times over what was read before."""
    torch, hipmx = mx
    x, w, bias = operands(torch, hipmx, m, n, k, "bfloat16", m)
    y = hipmx.linear(x, w, bias)
    check_linear(torch, hipmx, y, x, w, bias)
    q = hipmx.quantize(x)
    for _ in range(8):
        assert torch.equal(hipmx.linear(x, w, bias), y)
        check_linear(torch, hipmx, hipmx.linear(q, w, bias), x, w, bias)


def test_parts_that_were_changed_in_place(mx):
    """Codes and scales are a program's to change, but not to resize, move or
    turn around: refused before a kernel reads them."""
    torch, hipmx = mx
    x = torch.randn(40, 96, device="cuda")
    byte = torch.zeros(10000, dtype=torch.uint8, device="cuda")
    changes = [
        lambda t: t.resize_(1, t.shape[1]),
        lambda t: t.resize_(t.shape[0], 1),
        lambda t: t.resize_(t.numel()),
        lambda t: t.t_(),
        lambda t: t.unsqueeze_(0),
        lambda t: t.set_(byte[:1]),
        lambda t: t.set_(byte.as_strided(t.shape, (1, 1))),
        lambda t: setattr(t, "data", t.cpu()),
        lambda t: setattr(t, "data", t.int()),
    ]
    for change in changes:
        for part in ("codes", "scales"):
            q = hipmx.quantize(x)
            change(getattr(q, part))
            w = hipmx.quantize(x)
            calls = [lambda: hipmx.linear(x, q), lambda: hipmx.linear(q, w)]
            if part == "scales" or q.codes.is_cuda:
                calls.append(q.dequantize)
            for call in calls:
                with pytest.raises((ValueError, RuntimeError, TypeError)):
                    call()
    # one that is not a multiple of 16 bytes into memory
    q = hipmx.quantize(x)
    codes = byte[1:1 + q.codes.numel()].view(q.codes.shape)
    codes.copy_(q.codes)
    q.codes.set_(codes)
    with pytest.raises(ValueError, match="fit each other"):
        q.dequantize()
    # changed values are what counts
    q = hipmx.quantize(x)
    q.codes.zero_()
    assert (q.dequantize() == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_dequantize_every_code_and_scale(mx, dtype):
    """Every code under every scale byte, to each type: also what float16 and
    bfloat16 round, lose or make an infinity of, as torch rounds it."""
    torch, hipmx = mx
    pair = torch.arange(256, dtype=torch.uint8)
    codes = pair.reshape(1, 16, 16).expand(256, 16, 16).reshape(4096, 16)
    scales = pair.repeat_interleave(16)[:, None].contiguous()
    q = hipmx.MXFP4Tensor(codes.contiguous(), scales, 32)
    want = torch.from_numpy(values(torch, q)).to(getattr(torch, dtype))
    got = q.to("cuda").dequantize(getattr(torch, dtype)).cpu()
    assert got.dtype == want.dtype
    same = (got == want) | (got.isnan() & want.isnan())
    assert same.all(), (got[~same][:5], want[~same][:5])
    host = q.dequantize(getattr(torch, dtype))
    assert ((host == want) | (host.isnan() & want.isnan())).all()


def test_vmap_is_refused(mx):
    torch, hipmx = mx
    import hiplm

    x = torch.randn(2, 3, 64, device="cuda")
    ids = torch.zeros(3, 2, dtype=torch.long, device="cuda")
    w = hipmx.quantize(x[0])
    for call in (
        lambda a: hipmx.quantize(a).scales,
        lambda a: hipmx.linear(a, w),
        lambda a: hipmx.linear(x[0], w, a[:, 0]),
        lambda a: hiplm.token_logprobs(a, ids[:, 0]).logprobs,
        lambda a: hiplm.token_logprobs(x[0], ids[:, 0] + (a[:, 0] > 0)
                                       ).logprobs,
        lambda a: hiplm.topk_distill_loss(x[0], a[:, :2], ids),
    ):
        with pytest.raises((TypeError, RuntimeError)):
            torch.vmap(call)(x)
    with pytest.raises((TypeError, RuntimeError)):
        torch.func.grad(lambda a: hiplm.topk_distill_loss(
            a, x[0, :, :2], ids))(x[0])
