"""CPU tests of microscaled 4-bit quantisation and product (ops/hipmx.py):
the format against its definition, the refusals, and the dispatch from
torch's own linear."""

import copy
import sys
from pathlib import Path

import numpy as np
import pytest

torch = pytest.importorskip("torch")

OPS_DIR = Path(__file__).resolve().parent.parent / "code_interpreter_amd" / "ops"
sys.path.insert(0, str(OPS_DIR))
sys.path.insert(0, str(Path(__file__).resolve().parent))

import hipmx  # noqa: E402
import hiptorch  # noqa: E402
import lm_oracle as oracle  # noqa: E402


def edges(dtype):
    """Rows of every border between two codes, under several scales, and of
    the type's own limits."""
    half = [0, 0.25, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6,
            7, 7.9]
    row = torch.tensor(half + [-v for v in half[:15]], dtype=torch.float64)
    rows = [row * 2.0 ** s for s in (-160, -127, -126, -24, -14, 0, 1, 12,
                                     100, 124)]
    rows = torch.stack([r.to(dtype) for r in rows])
    rows[~torch.isfinite(rows)] = 1.0
    more = torch.zeros(4, 32, dtype=dtype)
    more[1, 3] = torch.finfo(dtype).max
    more[2, 7] = torch.finfo(dtype).tiny
    more[2, 8] = torch.finfo(dtype).smallest_normal / 4  # subnormal
    more[3] = torch.finfo(dtype).smallest_normal / 4
    return torch.cat([rows, more])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16,
                                   torch.float16])
def test_quantize_is_the_format(dtype):
    x = edges(dtype)
    q = hipmx.quantize(x)
    codes, scales = oracle.quantize(x.double().numpy())
    assert np.array_equal(q.codes.numpy(), codes)
    assert np.array_equal(q.scales.numpy(), scales)
    want = oracle.values(codes, scales, 32)
    got = q.dequantize(torch.float32).double().numpy()
    assert np.array_equal(got, want)


@pytest.mark.parametrize("k", [1, 2, 31, 32, 33, 100])
def test_odd_lengths_and_shapes(k):
    torch.manual_seed(k)
    x = torch.randn(2, 3, k)
    q = hipmx.quantize(x)
    assert q.shape == (2, 3, k) and q.dim() == 3 and q.size(-1) == k
    codes, scales = oracle.quantize(x.reshape(6, k).double().numpy())
    assert np.array_equal(q.codes.reshape(6, -1).numpy(), codes)
    assert np.array_equal(q.scales.reshape(6, -1).numpy(), scales)
    assert q.dequantize().shape == x.shape
    assert q.dequantize().dtype == torch.bfloat16
    # strides do not matter
    t = hipmx.quantize(x.transpose(0, 1).contiguous().transpose(0, 1))
    assert torch.equal(t.codes, q.codes)


def test_a_block_with_nan_or_inf_is_nan():
    x = torch.ones(3, 64)
    x[1, 5] = float("nan")
    x[2, 40] = float("inf")
    q = hipmx.quantize(x)
    assert q.scales.tolist() == [[125, 125], [255, 125], [125, 255]]
    assert (q.codes[1, :16] == 0).all()
    v = q.dequantize(torch.float32)
    assert v[1, :32].isnan().all() and v[2, 32:].isnan().all()
    assert torch.equal(v[0], x[0]) and torch.equal(v[1, 32:], x[1, 32:])


def test_empty_tensors():
    q = hipmx.quantize(torch.zeros(0, 40))
    assert q.shape == (0, 40) and q.dequantize().shape == (0, 40)
    w = hipmx.quantize(torch.randn(5, 40))
    assert hipmx.linear(torch.zeros(0, 40), w).shape == (0, 5)


def test_linear_matches_its_definition():
    torch.manual_seed(0)
    x, w = torch.randn(2, 3, 70), torch.randn(9, 70)
    bias = torch.randn(9)
    qw = hipmx.quantize(w)
    y = hipmx.linear(x, qw, bias)
    xv = oracle.values(*oracle.quantize(x.reshape(6, 70).numpy()), 70)
    wv = oracle.values(*oracle.quantize(w.numpy()), 70)
    want = (xv @ wv.T + bias.double().numpy()).reshape(2, 3, 9)
    # 70 products added in 24 bits, in any order
    slack = 72 * 2.0 ** -24 * (
        np.abs(xv) @ np.abs(wv).T + bias.abs().double().numpy()
    ).reshape(2, 3, 9)
    assert (np.abs(y.double().numpy() - want) <= slack).all()
    # an operand that is quantised already, a row alone
    p = hipmx.linear(hipmx.quantize(x), qw, bias, dtype=torch.float32)
    assert torch.equal(p, y)
    assert hipmx.linear(x[0, 0], qw, bias).shape == (9,)


def test_torch_linear_dispatches():
    import torch.nn.functional as F

    torch.manual_seed(1)
    x, w = torch.randn(4, 64), hipmx.quantize(torch.randn(8, 64))
    bias = torch.randn(8)
    want = hipmx.linear(x, w, bias)
    assert torch.equal(F.linear(x, w, bias), want)
    assert torch.equal(F.linear(x, w, bias=bias), want)
    with hiptorch._make_mode(torch):  # under the matmul routing too
        assert torch.equal(F.linear(x, w, bias), want)
    with pytest.raises(TypeError):
        torch.matmul(x, w)


def test_refusals():
    w = hipmx.quantize(torch.randn(8, 64))
    x = torch.randn(4, 64)
    with pytest.raises(TypeError, match="x must be a tensor"):
        hipmx.quantize([1.0])
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        hipmx.quantize(torch.zeros(4, dtype=torch.float64))
    with pytest.raises(ValueError, match="last axis"):
        hipmx.quantize(torch.tensor(1.0))
    with pytest.raises(ValueError, match="last axis"):
        hipmx.quantize(torch.zeros(3, 0))
    with pytest.raises(TypeError, match="strided"):
        hipmx.quantize(torch.zeros(3, 32).to_sparse())
    with pytest.raises(TypeError, match="MXFP4Tensor"):
        hipmx.linear(x, torch.randn(8, 64))
    with pytest.raises(TypeError, match="input"):
        hipmx.linear(x.long(), w)
    with pytest.raises(ValueError, match="differ in their last axis"):
        hipmx.linear(x[:, :32], w)
    with pytest.raises(ValueError, match=r"\[n, k\]"):
        hipmx.linear(x, hipmx.quantize(torch.randn(2, 8, 64)))
    with pytest.raises(ValueError, match="is the most"):
        long = hipmx.quantize(torch.zeros(1, 1 << 24))
        hipmx.linear(torch.zeros(1, 1 << 24), long)
    with pytest.raises(ValueError, match="bias must be"):
        hipmx.linear(x, w, torch.zeros(7))
    with pytest.raises(ValueError, match="bias must be"):
        hipmx.linear(x, w, torch.zeros(8, dtype=torch.bfloat16))
    with pytest.raises(TypeError, match="dtype"):
        hipmx.linear(x, w, dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="dtype"):
        hipmx.linear(hipmx.quantize(x), w, dtype=torch.int32)
    with pytest.raises(TypeError, match="dtype"):
        w.dequantize(torch.float64)


def test_products_refuse_gradients():
    w = hipmx.quantize(torch.nn.Parameter(torch.randn(8, 64)))
    x = torch.randn(4, 64, requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward"):
        hipmx.linear(x, w)
    with pytest.raises(RuntimeError, match="no backward"):
        hipmx.linear(x.detach(), w, torch.zeros(8, requires_grad=True))
    with torch.no_grad():
        assert not hipmx.linear(x, w).requires_grad


def test_parts_are_checked_and_shared():
    q = hipmx.quantize(torch.randn(3, 40))
    t = hipmx.MXFP4Tensor(q.codes, q.scales, 40)
    assert t.codes.data_ptr() == q.codes.data_ptr()
    assert torch.equal(t.dequantize(), q.dequantize())
    for bad in (
        (q.codes, q.scales, 65), (q.codes, q.scales, 32), (q.codes, q.scales, 0),
        (q.codes[:2], q.scales, 40), (q.codes[:, :16], q.scales, 40),
    ):
        with pytest.raises(ValueError, match="codes are"):
            hipmx.MXFP4Tensor(*bad)
    with pytest.raises(TypeError, match="uint8"):
        hipmx.MXFP4Tensor(q.codes.int(), q.scales, 40)
    with pytest.raises(TypeError, match="codes must be a tensor"):
        hipmx.MXFP4Tensor(q.codes.numpy(), q.scales, 40)
    # parts cut out of larger ones
    big = torch.zeros(3, 64, dtype=torch.uint8)
    big[:, 5:37] = q.codes
    t = hipmx.MXFP4Tensor(big[:, 5:37], q.scales, 40)
    assert torch.equal(t.dequantize(), q.dequantize())


def test_parts_are_not_replaced():
    q = hipmx.quantize(torch.ones(2, 40))
    for name in ("codes", "scales", "shape"):
        with pytest.raises(AttributeError):
            setattr(q, name, getattr(q, name))
    again = copy.deepcopy(q)
    assert torch.equal(again.codes, q.codes) and again.shape == q.shape


def test_another_default_device_and_type():
    """torch's defaults are for tensors that a program makes, not for these
    operators' tables."""
    x = edges(torch.float32)
    w = hipmx.quantize(x)
    y = hipmx.linear(x, w)
    torch.set_default_device("meta")
    torch.set_default_dtype(torch.float16)
    try:
        q = hipmx.quantize(x)
        v, z = q.dequantize(torch.float32), hipmx.linear(x, w)
    finally:
        torch.set_default_device(None)
        torch.set_default_dtype(torch.float32)
    assert torch.equal(q.codes, w.codes) and torch.equal(q.scales, w.scales)
    assert torch.equal(v, w.dequantize(torch.float32))
    assert torch.equal(z, y)


def test_the_kernels_take_no_parts_of_the_host():
    module = pytest.importorskip("_hiplm")
    q = hipmx.quantize(torch.randn(3, 40))
    for call in (
        lambda: module.mx_dequantize(q.codes, q.scales, 40, 0),
        lambda: module.mx_linear(torch.randn(2, 40), None, q.codes, q.scales,
                                 None, 40, 0),
    ):
        with pytest.raises(ValueError, match="fit each other"):
            call()
