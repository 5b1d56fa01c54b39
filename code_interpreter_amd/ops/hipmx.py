"""Microscaled 4-bit floating point for sandboxed user code: quantisation and
the product of quantised operands, on the gfx950 scaled matrix instructions.

Importable standalone inside the sandbox (APP_OPS_DIR is on sys.path), next
to torch:

    import hipmx, torch
    w = hipmx.quantize(layer.weight)            # 4.25 bits an element
    y = hipmx.linear(x, w, layer.bias)          # x quantised on the way in
    y = torch.nn.functional.linear(x, w)        # the same

The format: along the last axis 32 elements share a scale, a power of two
whose exponent + 127 is held in a byte; an element is one of 0, 0.5, 1, 1.5,
2, 3, 4, 6 and a sign (e2m1), two a byte, the earlier in the low half. The
scale of a block is 2^(floor(log2 max|x|) - 2), at least 2^-127; elements are
rounded to nearest, ties to even, and saturate at 6 scales. A block with a
NaN or an infinity becomes NaN as a whole (scale byte 255).

GPU tensors run on the kernels, on torch's current stream of their device,
and raise where the extension is missing; CPU tensors are computed in plain
torch, to the same codes. Products have no backward.
"""

from operator import attrgetter

import hiptorch

BLOCK = 32
MAX_K = (1 << 24) - 32  # of a product

STATS = {"quantize": 0, "dequantize": 0, "linear": 0}


def _blocks(k: int) -> int:
    return -(-k // BLOCK)


class MXFP4Tensor:
    """A tensor of microscaled 4-bit elements.

    ``codes``: uint8 [..., blocks * 16], ``scales``: uint8 [..., blocks], of
    equal leading sizes; ``k``: the last axis' length, blocks =
    ceil(k / 32). Wraps given parts without a copy where they are contiguous
    (and the codes' address is a multiple of 16); codes behind ``k`` have to
    be 0.
    """

    __slots__ = ("_codes", "_scales", "_shape")

    # not to be replaced one by one: the kernels rely on their fitting
    codes = property(attrgetter("_codes"))
    scales = property(attrgetter("_scales"))
    shape = property(attrgetter("_shape"))

    def __init__(self, codes, scales, k: int):
        torch = hiptorch.lm_torch()
        hiptorch.check_tensor("codes", codes)
        hiptorch.check_tensor("scales", scales)
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError("codes and scales must be uint8, got "
                            f"{codes.dtype} and {scales.dtype}")
        if codes.device != scales.device:
            raise ValueError("codes and scales are on different devices")
        k = int(k)
        nb = _blocks(k)
        lead = scales.shape[:-1]
        if (k < 1 or codes.dim() < 1 or scales.dim() < 1
                or codes.shape[:-1] != lead or scales.shape[-1] != nb
                or codes.shape[-1] != nb * 16):
            raise ValueError(
                f"for a last axis of {k} codes are [..., {nb * 16}] and "
                f"scales [..., {nb}], got {list(codes.shape)} and "
                f"{list(scales.shape)}")
        codes = codes.contiguous()
        if codes.data_ptr() % 16:
            codes = codes.clone()
        self._set(codes, scales.contiguous(), torch.Size((*lead, k)))

    def _set(self, codes, scales, shape):
        self._codes, self._scales, self._shape = codes, scales, shape
        return self

    @property
    def device(self):
        return self.codes.device

    def dim(self) -> int:
        return len(self.shape)

    def size(self, axis=None):
        return self.shape if axis is None else self.shape[axis]

    def to(self, device):
        return MXFP4Tensor(self.codes.to(device), self.scales.to(device),
                           self.shape[-1])

    def dequantize(self, dtype=None):
        """The values that the codes stand for, in float32, bfloat16 (the
        default) or float16; rounded where float16 does not hold them."""
        return _dequantize(self, dtype)

    def __repr__(self):
        return (f"MXFP4Tensor(shape={list(self.shape)}, "
                f"device={str(self.device)!r})")

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        import torch

        if func is torch.nn.functional.linear:
            return linear(*args, **(kwargs or {}))
        return NotImplemented


def quantize(x) -> MXFP4Tensor:
    """x ([..., k], float32, bfloat16 or float16) in microscaled 4-bit form.
    The result is data: it carries no gradient."""
    torch = hiptorch.lm_torch()
    hiptorch.check_tensor("x", x)
    code = hiptorch.check_dtype("x", x.dtype)
    shape = x.shape
    if not shape or not shape[-1]:
        raise ValueError(f"x needs a last axis, got {list(shape)}")
    if not x.is_cuda:
        return MXFP4Tensor(*_cpu_quantize(torch, x.detach()), shape[-1])
    codes, scales = hiptorch.ensure_hiplm().mx_quantize(x, code)
    STATS["quantize"] += 1
    return MXFP4Tensor.__new__(MXFP4Tensor)._set(codes, scales, shape)


def _dequantize(q: MXFP4Tensor, dtype=None):
    torch = hiptorch.lm_torch()
    dtype = torch.bfloat16 if dtype is None else dtype
    code = hiptorch.check_dtype("dtype", dtype)
    if not q.codes.is_cuda:
        return _cpu_dequantize(torch, q).to(dtype)
    STATS["dequantize"] += 1
    return hiptorch.ensure_hiplm().mx_dequantize(q.codes, q.scales,
                                                 q.shape[-1], code)


def linear(input, weight: MXFP4Tensor, bias=None, *, dtype=None):
    """``input @ weight.T + bias`` of microscaled 4-bit operands.

    input: a tensor [..., k] (float32, bfloat16, float16), which is quantised
    as by ``quantize`` on the way in and gives the result its type, or an
    MXFP4Tensor, with the result's type in ``dtype`` (bfloat16 if not given).
    weight: [n, k], k below 2^24. bias: [n], of the result's type. Sums are
    float32; the result is rounded once. There is no backward: tensors that
    require a gradient are refused while gradients are enabled.
    """
    torch = hiptorch.lm_torch()
    if not isinstance(weight, MXFP4Tensor):
        raise TypeError("weight must be an MXFP4Tensor, got "
                        f"{type(weight).__name__}")
    if len(weight.shape) != 2:
        raise ValueError(f"weight must be [n, k], got {list(weight.shape)}")
    n, k = weight.shape
    if k > MAX_K:
        raise ValueError(f"the last axis is {k} long, {MAX_K} is the most")
    wcodes = weight.codes
    packed = isinstance(input, MXFP4Tensor)
    if packed:
        dtype = torch.bfloat16 if dtype is None else dtype
        code = hiptorch.check_dtype("dtype", dtype)
        data = input.codes
    else:
        hiptorch.check_tensor("input", input)
        code = hiptorch.check_dtype("input", input.dtype)
        if dtype is not None and dtype != input.dtype:
            raise TypeError("dtype is for an MXFP4Tensor input: a tensor's "
                            "own type is the result's")
        dtype = input.dtype
        data = input
    shape = input.shape
    if not shape or shape[-1] != k:
        raise ValueError(f"input {list(shape)} and weight "
                         f"{list(weight.shape)} differ in their last axis")
    if data.device != wcodes.device:
        raise ValueError(f"input is on {data.device}, weight on "
                         f"{wcodes.device}")
    if bias is not None:
        hiptorch.check_tensor("bias", bias)
        if (bias.dtype != dtype or bias.shape != (n,)
                or bias.device != wcodes.device):
            raise ValueError(
                f"bias must be [{n}], {dtype}, on {wcodes.device}, got "
                f"{list(bias.shape)}, {bias.dtype}, on {bias.device}")
    if ((not packed and input.requires_grad)
            or (bias is not None and bias.requires_grad)):
        if torch.is_grad_enabled():
            raise RuntimeError("hipmx.linear has no backward: call it under "
                               "torch.no_grad(), or detach its inputs")
    if not wcodes.is_cuda:
        q = input if packed else quantize(input)
        y = _cpu_dequantize(torch, q) @ _cpu_dequantize(torch, weight).T
        if bias is not None:
            y = y + bias.detach().float()
        return y.to(dtype)
    STATS["linear"] += 1
    return hiptorch.ensure_hiplm().mx_linear(
        data, input.scales if packed else None, wcodes, weight.scales, bias,
        k, code)


# ---------------------------------------------------------------------------
# CPU tensors
# ---------------------------------------------------------------------------
_VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _cpu_quantize(torch, x):
    lead, k = x.shape[:-1], x.shape[-1]
    v = torch.nn.functional.pad(x.float(), (0, -k % BLOCK))
    v = v.reshape(*lead, _blocks(k), BLOCK)
    a = v.abs()
    top = a.amax(-1, keepdim=True)
    good = torch.isfinite(top)
    # frexp's mantissa is in [1/2, 1)
    shift = (torch.frexp(torch.where(good, top, 1.0)).exponent - 3)
    shift = torch.where(top == 0, -127, shift.clamp(min=-127))
    a = torch.ldexp(torch.where(good, a, 0.0).double(), -shift)
    # a code is its place among the values; the border between two codes
    # falls to the even one
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0],
                           dtype=a.dtype, device=a.device)
    even_above = torch.tensor([False, True] * 3 + [False], device=a.device)
    code = ((a[..., None] > borders)
            | ((a[..., None] == borders) & even_above)).sum(-1)
    code = code + 8 * (torch.signbit(v) & good)
    code = code.to(torch.uint8).reshape(*lead, _blocks(k) * BLOCK)
    codes = code[..., 0::2] | (code[..., 1::2] << 4)
    scales = torch.where(good, shift + 127, 255)[..., 0].to(torch.uint8)
    return codes, scales


def _cpu_dequantize(torch, q):
    table = torch.tensor(_VALUES + [-f for f in _VALUES],
                         dtype=torch.float32, device=q.device)
    v = torch.stack([table[(q.codes & 15).long()],
                     table[(q.codes >> 4).long()]], -1)
    v = v.reshape(*q.scales.shape, BLOCK)
    s = q.scales.int()[..., None]
    v = torch.where(s == 255, float("nan"),
                    torch.ldexp(v.double(), s - 127).float())
    lead, nb = q.scales.shape[:-1], q.scales.shape[-1]
    return v.reshape(*lead, nb * BLOCK)[..., :q.shape[-1]]
