"""GPU tests of the scoring operators (ops/hiplm.py): the kernels against the
definitions in 64 bits.

Slack. The kernels work in float32 on the logits' own values. A term e of a
row's sum is off by its exponent's rounding (3 steps of the exponent y) and
its own (2 steps), a thread's sum of a row of v elements by v / 256 steps at
most, their union by 20: relative to the sum at most STEP (v / 256 + 64 + 3
|y|), y <= 40 where e counts. What is added to or multiplied with that is a
few steps more.
"""

import math
import sys
from pathlib import Path

import numpy as np
import pytest

OPS_DIR = Path(__file__).resolve().parent.parent / "code_interpreter_amd" / "ops"
sys.path.insert(0, str(OPS_DIR))
sys.path.insert(0, str(Path(__file__).resolve().parent))

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "bfloat16", "float16"]
STEP = 2.0 ** -24
INF = math.inf


@pytest.fixture(scope="module")
def lm():
    torch = pytest.importorskip("torch")
    if not torch.cuda.is_available():
        pytest.skip("torch sees no GPU")
    import hiplm

    return torch, hiplm


def relative(v):
    return STEP * (v / 256 + 200)


def host(t):
    return t.detach().double().cpu().numpy()


def near(got, want, slack):
    got = host(got)
    most = np.finfo(np.float32).max  # results are float32
    want = np.where(np.abs(want) > most, np.copysign(INF, want), want)
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        err = np.where(same, 0, np.abs(got - want) - slack)
    assert (err <= 0).all(), np.argwhere(~(err <= 0))[:5]


def trouble(torch, v, dtype, seed=0):
    """Rows that are plain, tied, sharp, masked in part or as a whole (by -inf
    and by the type's lowest value), rising, falling, with a NaN or an
    infinity; their tokens."""
    g = torch.Generator().manual_seed(seed + v)
    dt = getattr(torch, dtype)
    low = torch.finfo(dt).min
    x = (torch.randn(18, v, generator=g) * 3).to(dt)
    x[1] = 2.5
    x[2, v // 2] = 60
    x[3, ::2] = -INF
    x[4, 1:] = -INF
    x[5] = -INF
    x[6, : v - v // 5] = low
    x[7] = low
    x[8, v // 3] = math.nan
    x[9, v // 3] = INF
    x[12] = torch.linspace(-8, 8, v).to(dt)
    x[13] = torch.linspace(8, -8, v).to(dt)
    x[14] = (torch.arange(v) % 3).to(dt)
    x[15] = 0.0
    x[15, 1::2] = -0.0
    x[16, : v - v // 7] = -INF
    x[17] = (x[17].float() * 1000).to(dt)
    tokens = torch.randint(v, (18,), generator=g)
    tokens[4] = 0
    tokens[10] = -100
    tokens[11] = v
    return x.cuda(), tokens.cuda()


def check_logprobs(torch, hiplm, x, tokens, top, t):
    import lm_oracle as oracle

    v = x.shape[-1]
    r = hiplm.token_logprobs(x, tokens, top=top, temperature=t)
    lp, h, top_lp, top_ids = oracle.token_logprobs(
        host(x), host(tokens).astype(np.int64), top, t)
    def slack(a):
        return relative(v) + 4 * STEP * np.abs(np.where(np.isfinite(a), a, 0))

    near(r.logprobs, lp, slack(lp))
    # H = ln S - U / S: U's terms are at most 40 S in sum
    near(r.entropy, h, 42 * relative(v))
    rows = ~np.isnan(top_lp).any(-1) if top else slice(0)
    assert np.array_equal(r.top_tokens.cpu().numpy()[rows], top_ids[rows])
    near(r.top_logprobs, top_lp, slack(top_lp))
    return r


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v,top", [
    (1, 1), (2, 2), (5, 3), (63, 20), (256, 128), (1000, 1), (2047, 5),
    (2049, 64), (8192, 20), (10007, 128), (50001, 20), (131072, 64),
])
def test_token_logprobs(lm, dtype, v, top):
    torch, hiplm = lm
    x, tokens = trouble(torch, v, dtype)
    check_logprobs(torch, hiplm, x, tokens, top, 1.0)


@pytest.mark.parametrize("t", [0.25, 0.9, 4.0])
def test_token_logprobs_temperature(lm, t):
    torch, hiplm = lm
    for dtype in DTYPES:
        x, tokens = trouble(torch, 1001, dtype)
        check_logprobs(torch, hiplm, x, tokens, 7, t)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows", [300, 1100])
@pytest.mark.parametrize("v,top", [(777, 9), (40000, 33)])
def test_token_logprobs_many_rows(lm, dtype, rows, v, top):
    """Enough rows that each is one block's: compared with the same rows a
    few at a time, which are split, and a few of them with the definition."""
    torch, hiplm = lm
    x, tokens = trouble(torch, v, dtype)
    keep = torch.arange(rows) % 18
    many = hiplm.token_logprobs(x[keep], tokens[keep], top=top)
    few = check_logprobs(torch, hiplm, x, tokens, top, 1.0)
    good = [r for r in range(18) if r not in (8, 9)]
    for i in good:
        at = torch.nonzero(keep == i)[:, 0].cuda()
        assert torch.equal(many.top_tokens[at],
                           few.top_tokens[i].expand(len(at), top))
        for a, b in ((many.logprobs, few.logprobs),
                     (many.entropy, few.entropy)):
            # the same sums in another order
            wide = 84 * relative(v) + 8 * STEP * abs(host(b[i]))
            near(a[at], np.broadcast_to(host(b[i]), (len(at),)),
                 np.where(np.isfinite(wide), wide, 0))


def test_top_of_hard_rows(lm):
    """Rows that make the choice of alternatives work: all values equal but
    few, the best in one thread's place, the best in the last part, rising in
    steps, one cluster."""
    torch, hiplm = lm
    v = 70001
    x = torch.full((7, v), -1.0)
    x[0, v - 3:] = torch.tensor([1.0, 2.0, 3.0])
    x[1, 40000:40008] = torch.arange(8).float()
    x[2, 65000:] = torch.rand(v - 65000)
    x[3] = torch.div(torch.arange(v), 500, rounding_mode="floor").float()
    x[4, 1024:1024 + 3000] = 5 + torch.rand(3000)
    x[5] = (torch.arange(v) * 7919 % v).float()
    x[6] = torch.finfo(torch.float32).min
    x[6, ::1000] = 0.5
    tokens = torch.zeros(7, dtype=torch.long)
    for dtype in DTYPES:
        for top in (1, 20, 64, 128):
            few = x.to(getattr(torch, dtype)).cuda()
            check_logprobs(torch, hiplm, few, tokens.cuda(), top, 1.0)
            many = hiplm.token_logprobs(few.repeat(150, 1),
                                        tokens.repeat(150).cuda(), top=top)
            one = hiplm.token_logprobs(few, tokens.cuda(), top=top)
            assert torch.equal(many.top_tokens,
                               one.top_tokens.repeat(150, 1))


@pytest.mark.parametrize("rows", [1, 500])
@pytest.mark.parametrize("v", [300, 1000, 2100, 40007])
def test_top_of_narrow_rows(lm, rows, v):
    """What is left of a row stands where few of a block's threads see it, or
    is so close that the candidates are many: rows shorter than a chunk, a
    window in a masked row, falling and rising values, values that differ in
    the last bits of a float32, rows of one value."""
    torch, hiplm = lm
    g = torch.Generator().manual_seed(v)
    x = torch.full((7, v), -math.inf)
    x[0] = torch.randn(v, generator=g)
    x[1, v // 3: v // 3 + 1300] = torch.randn(
        len(range(v)[v // 3: v // 3 + 1300]), generator=g)
    x[2, ::97] = 1.0
    x[3] = torch.arange(v) / 64.0
    x[4] = -torch.arange(v) / 64.0
    x[5] = 1 + torch.rand(v, generator=g) * 2.0 ** -13
    x[6] = 0
    tokens = torch.zeros(rows, dtype=torch.long, device="cuda")
    for dtype in DTYPES:
        few = x.to(getattr(torch, dtype))
        many = few.repeat(-(-rows // 7), 1)[:max(rows, 7)]
        values, ids = few.float().sort(dim=-1, descending=True, stable=True)
        ids[values == -math.inf] = -1
        for top in (1, 13, 64, 128):
            if rows == 1:
                got = torch.cat([hiplm.token_logprobs(
                    row[None].cuda(), tokens, top=top).top_tokens
                    for row in many])
            else:
                got = hiplm.token_logprobs(many.cuda(), tokens,
                                           top=top).top_tokens
            want = ids[:, :top].repeat(-(-rows // 7), 1)[:max(rows, 7)]
            assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("value", [-7.5, 0.0, 3.0])
def test_top_of_rows_of_few_values(lm, value):
    """Rows in parts whose lists all end in the same value: of equal ones the
    first by index, below and above 0."""
    torch, hiplm = lm
    g = torch.Generator().manual_seed(4)
    x = torch.full((3, 131072), value)
    x[1, torch.randint(131072, (70,), generator=g)] = value + 1
    x[2] += torch.randint(0, 2, (131072,), generator=g)
    tokens = torch.zeros(3, dtype=torch.long, device="cuda")
    want = x.sort(dim=-1, descending=True, stable=True)[1]
    for dtype in DTYPES:
        for top in (1, 20, 100, 128):
            r = hiplm.token_logprobs(x.to(getattr(torch, dtype)).cuda(),
                                     tokens, top=top)
            assert torch.equal(r.top_tokens.cpu(), want[:, :top])


@pytest.mark.parametrize("rows", [1, 500])
def test_top_of_rows_with_nan(lm, rows):
    """Numbers are chosen from what is one, also where some of a block's
    threads see nothing but NaN; all log probabilities of the row are NaN."""
    torch, hiplm = lm
    g = torch.Generator().manual_seed(8)
    x = torch.randn(rows, 30011, generator=g)
    x[:, :600] = math.nan     # what a block's first threads take
    x[:, 9000:20000] = math.nan
    x[0, 25000] = math.inf
    tokens = torch.full((rows,), 700)
    for dtype in DTYPES:
        few = x.to(getattr(torch, dtype))
        for top in (1, 7, 40, 128):
            r = hiplm.token_logprobs(few.cuda(), tokens.cuda(), top=top)
            want = few.float().nan_to_num(-math.inf, math.inf).sort(
                dim=-1, descending=True, stable=True)[1][:, :top]
            assert torch.equal(r.top_tokens.cpu(), want)
            for part in (r.logprobs, r.entropy, r.top_logprobs):
                assert part.isnan().all()


def check_grad(torch, got, want, size, v, dtype):
    """One rounding to the logits' type, and the error of p: of its exponent,
    and of the row's sum. The hardware's exponential has no subnormal
    results: a p below 2^-126 is 0. What it is multiplied with is at most
    (|g_lp| + |g_h| (|ln p| + H)) / t with |g| < 5, H < 12 and t > 0.6, and p
    |ln p| is at most 88 * 2^-126 there: below 2^-116 in all."""
    info = torch.finfo(getattr(torch, dtype))
    slack = (2.0 ** -116 + info.eps / 2 * (np.abs(want) + 50 * relative(v) * size)
             + 50 * relative(v) * size + info.smallest_normal * info.eps)
    near(got, want, slack)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [1, 7, 64, 2049, 10007, 65536])
def test_token_logprobs_gradient(lm, dtype, v):
    torch, hiplm = lm
    import lm_oracle as oracle

    x, tokens = trouble(torch, v, dtype)
    x.requires_grad_(True)
    g = torch.Generator().manual_seed(v)
    for t, use in ((1.0, "both"), (0.7, "lp"), (1.3, "h")):
        r = hiplm.token_logprobs(x, tokens, temperature=t)
        g_lp, g_h = (torch.randn(18, generator=g).cuda() for _ in range(2))
        outs, gs = [r.logprobs, r.entropy], [g_lp, g_h]
        if use == "lp":
            outs, gs, g_h = outs[:1], gs[:1], torch.zeros(18)
        if use == "h":
            outs, gs, g_lp = outs[1:], gs[1:], torch.zeros(18)
        (got,) = torch.autograd.grad(outs, [x], gs)
        assert got.dtype == x.dtype and got.shape == x.shape
        want, size = oracle.token_logprobs_grad(
            host(x), host(tokens).astype(np.int64), t, host(g_lp), host(g_h))
        rows = [i for i in range(18) if i not in (8, 9)]
        check_grad(torch, got[rows], want[rows], size[rows], v, dtype)
        assert got[8].isnan().any() and got[11].isnan().all()


def test_gradient_against_differences(lm):
    torch, hiplm = lm
    g = torch.Generator().manual_seed(0)
    x = torch.randn(3, 50, generator=g).cuda()
    tokens = torch.tensor([4, 0, 49]).cuda()
    teacher = torch.randn(3, 6, generator=g).cuda()
    ids = torch.stack([torch.randperm(50, generator=g)[:6]
                       for _ in range(3)]).cuda()

    def scores(z):
        r = hiplm.token_logprobs(z, tokens, temperature=0.8)
        loss = hiplm.topk_distill_loss(z, teacher, ids, temperature=1.5)
        return (r.logprobs * 0.3 - r.entropy * 0.7).sum() + loss

    z = x.clone().requires_grad_(True)
    (grad,) = torch.autograd.grad(scores(z), [z])
    step = 2.0 ** -6
    for i, j in ((0, 4), (0, 5), (1, 0), (2, 49), (2, 17)):
        d = torch.zeros_like(x)
        d[i, j] = step
        with torch.no_grad():
            got = ((scores(x + d) - scores(x - d)) / (2 * step)).item()
        # the third derivative is below 8, a score is off by some 2^-20
        assert abs(got - grad[i, j].item()) < 8 * step ** 2 / 6 + 2.0 ** -13


@pytest.mark.parametrize("v", [1000, 9001])
def test_strided_logits(lm, v):
    torch, hiplm = lm
    wide = torch.randn(6, 4, v + 24, device="cuda", dtype=torch.bfloat16)
    tokens = torch.randint(v, (6, 4), device="cuda")
    views = [wide[..., :v], wide[..., 5:v + 5], wide[..., 1:v + 1]]
    views.append(wide[..., :v].transpose(0, 1).contiguous().transpose(0, 1))
    views.append(wide[..., :v].permute(2, 0, 1).contiguous().permute(1, 2, 0))
    views.append(wide[:1, :, 3:v + 3].expand(6, 4, v))
    for x in views:
        a = x.detach().requires_grad_(True)
        b = x.detach().contiguous().requires_grad_(True)
        outs = []
        for z in (a, b):
            r = hiplm.token_logprobs(z, tokens, top=9)
            loss = hiplm.topk_distill_loss(z, r.top_logprobs.flip(-1),
                                           r.top_tokens)
            total = loss + r.logprobs.mean() + r.entropy.sum()
            (grad,) = torch.autograd.grad(total, [z])
            outs.append([*[o.detach() for o in r], loss.detach(), grad])
        for p, q in zip(*outs):
            assert torch.equal(p, q)


def records(torch, v, k, rows, dtype):
    g = torch.Generator().manual_seed(100 * v + k)
    teacher = (torch.randn(rows, k, generator=g) * 2).to(getattr(torch, dtype))
    ids = torch.randint(v, (rows, k), generator=g)  # repeated ones too
    ids[1, k // 2:] = -1
    teacher[2, k // 2:] = -INF
    ids[3] = -1
    teacher[4] = -INF
    ids[7] = ids[7, 0]
    ids[10] = torch.arange(k) % v
    ids[12] = v - 1 - torch.arange(k) % v
    teacher[13] = torch.finfo(teacher.dtype).min
    ids[11, 0] = v
    teacher[14, 0] = math.nan
    return teacher.cuda(), ids.cuda()


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("dtype,t_dtype", [
    ("float32", "float32"), ("bfloat16", "float32"), ("float16", "bfloat16"),
    ("bfloat16", "float16")])
@pytest.mark.parametrize("v,k", [(1, 1), (9, 4), (2049, 64), (10007, 256),
                                 (65536, 20)])
def test_distill(lm, dtype, t_dtype, v, k, reduction):
    torch, hiplm = lm
    import lm_oracle as oracle

    t = 1.5
    x, _ = trouble(torch, v, dtype)
    teacher, ids = records(torch, v, k, 18, t_dtype)
    keep = [0, 1, 2, 3, 4, 6, 7, 10, 12, 13, 14, 15, 17]
    if reduction != "none":  # the one with a NaN in its record
        keep.remove(14)
    else:
        keep += [5, 8, 9, 11, 16]
    x = x[keep].requires_grad_(True)
    loss = hiplm.topk_distill_loss(x, teacher[keep], ids[keep],
                                   temperature=t, reduction=reduction)
    want, grad, size = oracle.distill(
        host(x), host(teacher[keep]), host(ids[keep]).astype(np.int64), t,
        reduction)
    with np.errstate(invalid="ignore"):
        spread = (relative(v) + 64 * STEP) * (
            1 + np.abs(host(x)).max(initial=0, where=host(x) > -1e30)) * 4
    scale = t * t + np.abs(np.where(np.isfinite(want), want, 0))
    near(loss, want, spread * scale)
    (got,) = torch.autograd.grad(loss.sum(), [x])
    rows = np.isfinite(np.broadcast_to(want, (len(keep),)))
    check_grad(torch, got[rows], grad[rows], size[rows], v, dtype)
    # a masked entry in the record: an infinite loss, a finite gradient
    if reduction == "none":
        for i, r in enumerate(keep):
            if want[i] == INF:
                assert got[i].isfinite().all()


@pytest.mark.parametrize("rows", [16, 17, 64, 65, 390])
@pytest.mark.parametrize("v", [600, 17003])
def test_distill_by_the_number_of_rows(lm, rows, v):
    """What finishes a call's rows goes by their number and length."""
    torch, hiplm = lm
    import lm_oracle as oracle

    g = torch.Generator().manual_seed(rows + v)
    x = torch.randn(rows, v, generator=g)
    teacher = torch.randn(rows, 30, generator=g)
    ids = torch.randint(v, (rows, 30), generator=g)
    ids[::5, 20:] = -1
    ids[3] = -1
    ids[4, 7] = ids[4, 2]
    for reduction in ("mean", "sum"):
        leaf = x.cuda().requires_grad_(True)
        loss = hiplm.topk_distill_loss(leaf, teacher.cuda(), ids.cuda(),
                                       reduction=reduction)
        want, grad, size = oracle.distill(
            x.numpy(), teacher.numpy(), ids.numpy(), 1.0, reduction)
        spread = (relative(v) + 64 * STEP) * 24
        near(loss, want, spread * (1 + abs(want)) * (
            rows if reduction == "sum" else 1))
        (got,) = torch.autograd.grad(loss, [leaf])
        check_grad(torch, got, grad, size, v, "float32")


def test_distill_weights_rows(lm):
    torch, hiplm = lm
    x = torch.randn(5, 300, device="cuda", requires_grad=True)
    teacher, ids = torch.randn(5, 8).cuda(), torch.randint(300, (5, 8)).cuda()
    rows = hiplm.topk_distill_loss(x, teacher, ids, reduction="none")
    g = torch.randn(5, device="cuda")
    (a,) = torch.autograd.grad(rows, [x], g, retain_graph=True)
    (b,) = torch.autograd.grad(rows.sum(), [x])  # a gradient of no stride
    s = hiplm.topk_distill_loss(x, teacher, ids, reduction="sum")
    (c,) = torch.autograd.grad(s, [x])
    assert torch.equal(b, c)
    torch.testing.assert_close(a, b * g[:, None], rtol=1e-6, atol=1e-9)
    m = hiplm.topk_distill_loss(x, teacher, ids)
    torch.testing.assert_close(m * 5, s)


def test_empty(lm):
    torch, hiplm = lm
    x = torch.zeros(0, 3, 9, device="cuda", requires_grad=True)
    ids = torch.zeros(0, 3, dtype=torch.long, device="cuda")
    r = hiplm.token_logprobs(x, ids, top=2)
    assert r.logprobs.shape == (0, 3) and r.top_tokens.shape == (0, 3, 2)
    (g,) = torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), [x])
    assert g.shape == x.shape
    loss = hiplm.topk_distill_loss(
        x, torch.zeros(0, 3, 2).cuda(),
        torch.zeros(0, 3, 2, dtype=torch.long).cuda())
    assert loss.item() == 0
    (g,) = torch.autograd.grad(loss, [x])
    assert g.shape == x.shape
    none = torch.full((4, 3), -1, device="cuda")
    z = torch.randn(4, 9, device="cuda", requires_grad=True)
    loss = hiplm.topk_distill_loss(z, torch.zeros(4, 3).cuda(), none)
    (g,) = torch.autograd.grad(loss, [z])
    assert loss.item() == 0 and (g == 0).all()


def test_second_derivatives_are_refused(lm):
    torch, hiplm = lm
    x = torch.randn(2, 9, device="cuda", requires_grad=True)
    r = hiplm.token_logprobs(x, torch.zeros(2, dtype=torch.long).cuda())
    (g,) = torch.autograd.grad(r.logprobs.sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_same_bits(lm):
    torch, hiplm = lm
    x, tokens = trouble(torch, 50001, "bfloat16")
    x.requires_grad_(True)
    outs = []
    for _ in range(3):
        r = hiplm.token_logprobs(x, tokens, top=20)
        loss = hiplm.topk_distill_loss(x[:3], r.top_logprobs[:3],
                                       r.top_tokens[:3])
        (g,) = torch.autograd.grad(r.logprobs[:8].sum() + loss, [x])
        outs.append([o.detach().nan_to_num(nan=7.0)
                     for o in (*r, loss, g)])
    for other in outs[1:]:
        for a, b in zip(outs[0], other):
            assert torch.equal(a, b)


@pytest.mark.parametrize("rows", [2, 700])
def test_forward_and_backward_in_a_graph(lm, rows):
    torch, hiplm = lm
    v, k = 5003, 12
    g = torch.Generator(device="cuda").manual_seed(3)

    def inputs():
        x = torch.randn(rows, v, generator=g, device="cuda")
        return (x.bfloat16(),
                torch.randint(v, (rows,), generator=g, device="cuda"))

    def step(x, tokens):
        r = hiplm.token_logprobs(x, tokens, top=k)
        loss = hiplm.topk_distill_loss(x, r.top_logprobs.sqrt().nan_to_num(),
                                       r.top_tokens, temperature=2.0)
        total = loss + r.entropy.mean() - r.logprobs.mean()
        return [*r, loss, *torch.autograd.grad(total, [x])]

    sets = [inputs() for _ in range(2)]
    want = []
    for x, tokens in sets:
        out = step(x.clone().requires_grad_(True), tokens)
        want.append([o.detach().clone() for o in out])
        del out
    x, tokens = sets[0][0].clone().requires_grad_(True), sets[0][1].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, tokens)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x, tokens)
    got = [o.detach() for o in got]
    for i in (0, 1, 0, 1):
        with torch.no_grad():
            x.copy_(sets[i][0])
        tokens.copy_(sets[i][1])
        graph.replay()
        step(sets[1][0].clone().requires_grad_(True), sets[1][1])  # eager
        torch.cuda.synchronize()
        for a, b in zip(got, want[i]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("rows,v,top", [(1, 9, 3), (3, 2049, 128),
                                        (5, 50001, 20), (1030, 333, 1)])
def test_results_end_where_they_end(lm, rows, v, top):
    torch, hiplm = lm
    import lm_oracle as oracle

    x = torch.randn(rows, v, device="cuda").bfloat16().requires_grad_(True)
    tokens = torch.randint(v, (rows,), device="cuda")
    g, one = torch.ones(rows, device="cuda"), torch.ones((), device="cuda")

    def ends(call):  # one call's results, looked at before the next
        oracle.fill_free_blocks(torch, 4 * rows, 4 * rows * top,
                                8 * rows * top, 2 * rows * v, 4)
        out = call()
        torch.cuda.synchronize()
        for t in out:
            assert (oracle.behind(torch, t) == 0xA5).all()
        return out

    r = ends(lambda: hiplm.token_logprobs(x, tokens, top=top))
    ends(lambda: torch.autograd.grad([r.logprobs, r.entropy], [x], [g, g]))
    (loss,) = ends(lambda: [hiplm.topk_distill_loss(x, r.top_logprobs,
                                                    r.top_tokens)])
    ends(lambda: torch.autograd.grad(loss, [x], one))


def test_on_another_stream(lm):
    torch, hiplm = lm
    x = torch.randn(40, 3001, device="cuda", requires_grad=True)
    tokens = torch.randint(3001, (40,), device="cuda")

    def step():
        r = hiplm.token_logprobs(x, tokens, top=5)
        return [*r, *torch.autograd.grad(r.logprobs.sum(), [x])]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_a_head_records_and_a_student_learns(lm):
    """The operators in a row, as they would be used."""
    torch, hiplm = lm
    import hipmx
    import lm_oracle as oracle

    g = torch.Generator().manual_seed(4)
    hidden, vocab, rows = 512, 5003, 70
    head = hipmx.quantize((torch.randn(vocab, hidden, generator=g) * 0.2)
                          .bfloat16().cuda())
    x = torch.randn(rows, hidden, generator=g).bfloat16().cuda()
    with torch.no_grad():
        logits = torch.nn.functional.linear(x, head)
    said = check_logprobs(torch, hiplm, logits, logits.argmax(-1), 16, 1.0)
    student = torch.randn(rows, vocab, generator=g).cuda().requires_grad_(True)
    loss = hiplm.topk_distill_loss(student, said.top_logprobs,
                                   said.top_tokens)
    (got,) = torch.autograd.grad(loss, [student])
    want, grad, size = oracle.distill(
        host(student), host(said.top_logprobs),
        host(said.top_tokens).astype(np.int64), 1.0, "mean")
    near(loss, want, 64 * relative(vocab))
    check_grad(torch, got, grad, size, vocab, "float32")
    # a student that says what the teacher says loses nothing
    same = hiplm.topk_distill_loss(
        torch.full((rows, vocab), -INF).cuda().scatter(
            1, said.top_tokens, said.top_logprobs),
        said.top_logprobs, said.top_tokens)
    assert abs(same.item()) < 64 * relative(vocab)


def test_far_offsets(lm):
    """Logits whose later rows stand behind 2^32 bytes and elements."""
    torch, hiplm = lm
    rows, v = 70_000, 65_537  # 4.6e9 elements
    x = torch.zeros(rows, v, dtype=torch.bfloat16, device="cuda")
    x[-30:] = torch.randn(30, v, device="cuda").bfloat16()
    tokens = torch.randint(v, (rows,), device="cuda")
    teacher = torch.randn(rows, 5, device="cuda")
    ids = torch.randint(v, (rows, 5), device="cuda")
    outs = []
    for cut in (slice(None), slice(rows - 400, None)):
        z = x[cut].detach().requires_grad_(True)
        r = hiplm.token_logprobs(z, tokens[cut], top=3)
        loss = hiplm.topk_distill_loss(z, teacher[cut], ids[cut],
                                       reduction="none")
        (dx,) = torch.autograd.grad(r.logprobs, [z], torch.ones_like(loss))
        (dz,) = torch.autograd.grad(loss, [z], torch.ones_like(loss))
        outs.append([t[-400:].detach().clone() for t in (*r, loss, dx, dz)])
        del dx, dz, z, r, loss
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_views_that_negate(lm):
    """torch keeps a conjugate's imaginary part as a view with a mark; the
    kernels get its values."""
    torch, hiplm = lm
    g = torch.Generator(device="cuda").manual_seed(2)
    z = torch.randn(3, 1000, 2, generator=g, device="cuda")
    x = torch.view_as_complex(z).conj().imag
    assert x.is_neg()
    record = torch.view_as_complex(z).conj().imag[:, 5:9]
    tokens = torch.tensor([1, 2, 3], device="cuda")
    ids = torch.arange(12, device="cuda").reshape(3, 4)
    results = []
    for a, b in ((x, record), (x.resolve_neg(), record.resolve_neg())):
        a = a.detach().requires_grad_(True)
        r = hiplm.token_logprobs(a, tokens, top=3)
        loss = hiplm.topk_distill_loss(a, b, ids)
        weight = torch.view_as_complex(z[:, :1]).conj().imag[:, 0]
        grad, = torch.autograd.grad([r.logprobs, loss], [a],
                                    [weight, torch.ones((), device="cuda")])
        results.append([*r, loss, grad])
    for one, other in zip(*results):
        assert torch.equal(one, other)


def test_as_many_rows_as_a_launch_has(lm):
    torch, hiplm = lm
    rows = (1 << 24) - 1
    x = torch.ones(rows + 1, 1, dtype=torch.bfloat16, device="cuda")
    tokens = torch.zeros(rows + 1, dtype=torch.long, device="cuda")
    few = x[:rows].requires_grad_(True)
    r = hiplm.token_logprobs(few, tokens[:rows])
    grad, = torch.autograd.grad(r.logprobs.sum(), [few])
    for part in (r.logprobs, r.entropy, grad):
        assert not part.any()
    with pytest.raises(RuntimeError, match="too many rows"):
        hiplm.token_logprobs(x, tokens)


def test_forward_mode_is_refused(lm):
    torch, hiplm = lm
    import hipmx
    from torch.autograd import forward_ad

    x = torch.randn(2, 64, device="cuda")
    ids = torch.zeros(2, 1, dtype=torch.long, device="cuda")
    w = hipmx.quantize(x)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: hiplm.token_logprobs(dual, ids[:, 0]),
                     lambda: hiplm.topk_distill_loss(dual, x[:, :1], ids),
                     lambda: hipmx.linear(dual, w)):
            with pytest.raises(RuntimeError, match="jvp|forward-mode"):
                call()


@pytest.mark.parametrize("op", ["logprobs", "entropy", "distill"])
@pytest.mark.parametrize("leaf", [True, False])
def test_a_gradient_penalty_is_refused(lm, op, leaf):
    """A second derivative, also where the first one's incoming gradient is a
    constant and the rest of the loss has a graph of its own: an error, no
    gradient that lacks a term. The first derivative is the same as ever."""
    torch, hiplm = lm
    g = torch.Generator(device="cuda").manual_seed(6)
    h = torch.randn(4, 8, generator=g, device="cuda", requires_grad=True)
    w = torch.randn(8, 50, generator=g, device="cuda")
    ids = torch.arange(8, device="cuda").reshape(4, 2)
    teacher = torch.randn(4, 2, generator=g, device="cuda")

    def loss_of(z):
        if op == "distill":
            return hiplm.topk_distill_loss(z, teacher, ids)
        return getattr(hiplm.token_logprobs(z, ids[:, 0]), op).sum()

    x = (h @ w).detach().requires_grad_(True) if leaf else h
    logits = x if leaf else h @ w
    loss = loss_of(logits)
    (grad,) = torch.autograd.grad(loss, [x], create_graph=True)
    first = loss_of(x if leaf else h @ w)
    (plain,) = torch.autograd.grad(first, [x])
    assert torch.equal(grad.detach(), plain)
    with pytest.raises(RuntimeError, match="no second derivative"):
        (loss + grad.pow(2).sum()).backward(retain_graph=True)
    # by some of the leaves only: torch runs what is on the way to them
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(loss + grad.pow(2).sum(), [x])
    # an incoming gradient that has a graph itself
    weight = torch.ones((), device="cuda", requires_grad=True)
    loss = loss_of(x if leaf else h @ w)
    (grad,) = torch.autograd.grad(loss, [x], weight, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(grad.sum(), [weight])


def test_gradients_without_memory_are_refused(lm):
    """An incoming gradient that wraps others, as a distributed tensor's."""
    torch, hiplm = lm

    class Wrapper(torch.Tensor):
        @staticmethod
        def __new__(cls, like):
            return torch.Tensor._make_wrapper_subclass(
                cls, like.shape, dtype=like.dtype, device=like.device)

        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            raise TypeError(str(func))

    x = torch.randn(3, 64, device="cuda", requires_grad=True)
    ids = torch.zeros(3, 2, dtype=torch.long, device="cuda")
    outs = [*hiplm.token_logprobs(x, ids[:, 0])[:2],
            hiplm.topk_distill_loss(x, torch.zeros(3, 2, device="cuda"), ids)]
    for out in outs:
        with pytest.raises((TypeError, RuntimeError)):
            torch.autograd.grad(out, [x], Wrapper(out))
    with pytest.raises(TypeError, match="memory of its own"):
        hiplm.token_logprobs(Wrapper(x), ids[:, 0])


@pytest.mark.parametrize("v", [1, 7, 300, 20000])
def test_kernels_and_host_agree_on_wrong_rows(lm, v):
    """Padding that holds NaN, tokens outside of the vocabulary, bad records,
    rows that are masked as a whole: what is NaN, 0 and infinite is so on GPU
    and CPU tensors alike, in results and gradients."""
    torch, hiplm = lm
    import test_hiplm as on_host

    x, tokens = on_host.garbage(v)
    k = min(v, 4)
    teacher, ids = on_host.records(v, k, rows=18)
    ids[[8, 12, 14]] = -1
    teacher[[9, 13]] = -INF
    ids[16, k - 1] = v + 5
    teacher[17] = math.nan
    results = []
    for device in ("cpu", "cuda"):
        z = x.to(device).requires_grad_(True)
        r = hiplm.token_logprobs(z, tokens.to(device), top=min(v, 3))
        (g,) = torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), [z])
        loss = hiplm.topk_distill_loss(z, teacher.to(device), ids.to(device),
                                       reduction="none")
        (d,) = torch.autograd.grad(loss, [z], torch.ones_like(loss))
        results.append([t.detach().cpu() for t in (*r, g, loss, d)])
    for a, b in zip(*results):
        # NaN where the other has one, infinities and exact zeros of rows too
        torch.testing.assert_close(a, b, rtol=1e-3, atol=1e-3, equal_nan=True)
    for i in (3, 6):  # the gradients
        none = [(t[i] == 0).all(-1) for t in results]
        assert torch.equal(*none)


@pytest.mark.parametrize("t", [0.3, 0.5, 1.0, 1.5])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("v", [50, 70001])
def test_distill_of_lowest_logits_is_finite(lm, dtype, t, v):
    torch, hiplm = lm
    import lm_oracle as oracle
    import test_hiplm as on_host

    x, teacher, ids = on_host.lowest_in_record(v, getattr(torch, dtype))
    loss = hiplm.topk_distill_loss(x.cuda(), teacher.cuda(), ids.cuda(),
                                   temperature=t, reduction="none")
    want, _, _ = oracle.distill(
        x.double().numpy(), teacher.double().numpy(), ids.numpy(), t, "none")
    near(loss, want, (on_host.LOWEST + relative(v)) * (1 + np.abs(want)))


def test_saved_tensors_through_hooks(lm):
    """What is kept for the backward may go to the host and back. What comes
    back as something else is refused before the kernels read it."""
    torch, hiplm = lm
    hooks = torch.autograd.graph
    x = torch.randn(5, 700, device="cuda", requires_grad=True)
    ids = torch.arange(15, device="cuda").reshape(5, 3)
    teacher = torch.randn(5, 3, device="cuda")
    calls = [
        lambda: hiplm.token_logprobs(x, ids[:, 0], top=2).logprobs.sum(),
        lambda: hiplm.token_logprobs(x, ids[:, 0], top=2).entropy.sum(),
        lambda: hiplm.topk_distill_loss(x, teacher, ids),
        lambda: hiplm.topk_distill_loss(x, teacher, ids,
                                        reduction="none").sum(),
    ]
    changes = [
        lambda t: t.cpu(),
        lambda t: t.half() if t.is_floating_point() else t,
        lambda t: t.int() if t.dtype == torch.int64 else t,
        lambda t: t[:3],
        lambda t: t[..., :2],
        lambda t: t.flatten()[:1],
        lambda t: t[None],
    ]
    for call in calls:
        (want,) = torch.autograd.grad(call(), [x])
        with hooks.save_on_cpu():
            out = call()
        (got,) = torch.autograd.grad(out, [x])
        assert torch.equal(got, want)
        # packed with a stride of their own
        with hooks.saved_tensors_hooks(
                lambda t: torch.stack([t, t], -1), lambda t: t[..., 0]):
            out = call()
        (got,) = torch.autograd.grad(out, [x])
        assert torch.equal(got, want)
        for change in changes:
            for which in range(3):  # of what an operator keeps
                count = iter(range(100))
                with hooks.saved_tensors_hooks(
                        lambda t: (next(count), t),
                        lambda p: change(p[1]) if p[0] == which else p[1]):
                    out = call()
                kept = next(count)
                assert kept >= 3
                try:
                    (got,) = torch.autograd.grad(out, [x])
                except RuntimeError as e:
                    # logits of another vocabulary: their own gradient is
                    # computed, which torch does not take
                    assert "came back" in str(e) or "invalid gradient" in str(e)
                else:  # a change that changed nothing
                    assert torch.equal(got, want)


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("t", [0.3, 0.9])
@pytest.mark.parametrize("k", [1, 2, 7, 100])
def test_distill_of_nothing_but_lowest_logits(lm, k, t, reduction):
    torch, hiplm = lm
    import lm_oracle as oracle
    import test_hiplm as on_host

    x, teacher, ids = on_host.all_lowest(k)
    loss = hiplm.topk_distill_loss(x.cuda(), teacher.cuda(), ids.cuda(),
                                   temperature=t, reduction=reduction)
    want, _, _ = oracle.distill(x.double().numpy(), teacher.double().numpy(),
                                ids.numpy(), t, reduction)
    assert np.isfinite(want).all()
    near(loss, want, (on_host.LOWEST + relative(400)) * (1 + np.abs(want)))
