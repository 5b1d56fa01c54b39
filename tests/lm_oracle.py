"""The language-model operators' definitions in 64 bits, for the tests of
hipmx and hiplm: plain numpy on host copies, row by row, written from the
formulas."""

import math

import numpy as np

VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _nearest(a):
    """The code whose value is nearest to a in [0, inf), ties to even."""
    best = min(range(8), key=lambda i: (abs(VALUES[i] - a), i & 1))
    return best


def quantize_block(block):
    """(codes, scale byte) of up to 32 numbers."""
    block = [float(v) for v in block] + [0.0] * (32 - len(block))
    if not all(math.isfinite(v) for v in block):
        return [0] * 32, 255
    top = max(abs(v) for v in block)
    shift = -127
    if top > 0:
        shift = max(math.frexp(top)[1] - 3, -127)
    codes = []
    for v in block:
        code = _nearest(math.ldexp(abs(v), -shift))
        codes.append(code + (8 if math.copysign(1, v) < 0 else 0))
    return codes, shift + 127


def quantize(x):
    """(packed codes, scale bytes) of [rows, k] numbers."""
    rows, k = x.shape
    nb = -(-k // 32)
    codes = np.zeros((rows, nb * 16), np.uint8)
    scales = np.zeros((rows, nb), np.uint8)
    for r in range(rows):
        for b in range(nb):
            c, s = quantize_block(x[r, 32 * b: 32 * b + 32])
            codes[r, 16 * b: 16 * b + 16] = (
                np.array(c[0::2]) | np.array(c[1::2]) << 4)
            scales[r, b] = s
    return codes, scales


def values(codes, scales, k):
    """What packed codes and scale bytes stand for, in 64 bits."""
    table = np.array(VALUES + [-v for v in VALUES])
    v = np.stack([table[codes & 15], table[codes >> 4]], -1)
    v = v.reshape(*scales.shape, 32)
    unit = np.ldexp(1.0, scales.astype(np.int64) - 127)
    unit = np.where(scales == 255, np.nan, unit)
    return (v * unit[..., None]).reshape(*scales.shape[:-1], -1)[..., :k]


def log_softmax(row, t):
    """ln softmax of a row; None where everything is masked."""
    row = np.asarray(row, np.float64)
    if np.all(row == -np.inf):
        return None
    if not np.all(row < np.inf):  # a NaN or +inf
        return np.full(row.shape, np.nan)
    z = (row - row.max()) / t
    return z - math.log(np.exp(z).sum())


def token_logprobs(x, tokens, top, t, ignore=-100):
    rows, v = x.shape
    lp, h = np.zeros(rows), np.zeros(rows)
    top_lp = np.full((rows, top), -np.inf)
    top_ids = np.full((rows, top), -1, np.int64)
    for r in range(rows):
        if tokens[r] == ignore:
            continue
        ls = log_softmax(x[r], t)
        if ls is not None:
            order = [j for j in np.argsort(-x[r], kind="stable")
                     if x[r][j] > -np.inf][:top]
            top_ids[r, :len(order)] = order
            top_lp[r, :len(order)] = ls[order]
        if not 0 <= tokens[r] < v:
            lp[r] = h[r] = np.nan
        elif ls is None:
            lp[r] = -np.inf
        else:
            lp[r] = ls[tokens[r]]
            p = np.exp(ls)
            h[r] = -np.sum(np.where(p == 0, 0.0, p) * np.where(
                p == 0, 0.0, ls))
    return lp, h, top_lp, top_ids


def token_logprobs_grad(x, tokens, t, g_lp, g_h, ignore=-100):
    """(gradient, what its terms add up to in magnitude)."""
    rows, v = x.shape
    grad, size = np.zeros((rows, v)), np.zeros((rows, v))
    for r in range(rows):
        ls = log_softmax(x[r], t)
        if tokens[r] == ignore:
            continue
        if not 0 <= tokens[r] < v:
            grad[r] = np.nan
            continue
        if ls is None:
            continue
        p = np.exp(ls)
        safe = np.where(p == 0, 0.0, ls)
        h = -np.sum(p * safe)
        grad[r] = -p * (g_lp[r] + g_h[r] * (safe + h)) / t
        size[r] = p * (abs(g_lp[r]) + abs(g_h[r]) * (abs(safe) + h)) / t
        grad[r, tokens[r]] += g_lp[r] / t
        size[r, tokens[r]] += abs(g_lp[r]) / t
    return grad, size


def distill(x, teacher, ids, t, reduction):
    """(loss, gradient of the sum of its elements, magnitude of the
    gradient's terms)."""
    rows, v = x.shape
    loss, grad = np.zeros(rows), np.zeros((rows, v))
    size, count = np.zeros((rows, v)), 0
    for r in range(rows):
        there = [j for j in range(ids.shape[1])
                 if ids[r, j] != -1 and teacher[r, j] != -np.inf]
        if not there:
            continue
        count += 1
        z = np.array([teacher[r, j] for j in there], np.float64) / t
        at = [int(ids[r, j]) for j in there]
        if not np.all(z < np.inf) or any(not 0 <= i < v for i in at):
            loss[r] = np.nan
            grad[r] = np.nan
            continue
        lq = z - z.max()
        lq = lq - math.log(np.exp(lq).sum())
        q = np.exp(lq)
        ls = log_softmax(x[r], t)
        if ls is None:
            loss[r] = np.inf
            continue
        loss[r] = t * t * sum(
            q[j] * (lq[j] - ls[i]) for j, i in enumerate(at) if q[j] > 0)
        grad[r] = size[r] = t * np.exp(ls)
        for j, i in enumerate(at):
            grad[r, i] -= t * q[j]
            size[r, i] += t * q[j]
    # a row's loss is a float32: an infinity where it is out of that range
    loss = np.where(loss > np.finfo(np.float32).max, np.inf, loss)
    if reduction == "none":
        return loss, grad, size
    by = max(count, 1) if reduction == "mean" else 1
    return loss.sum() / by, grad / by, size / by


# ---------------------------------------------------------------------------
# writes behind a tensor's end
# ---------------------------------------------------------------------------
# The caching allocator hands out blocks of whole 512 bytes, the best fitting
# free one first. Free blocks of a result's size are filled with a pattern
# beforehand; what stands between the result's end and its block's has to be
# there still.
def fill_free_blocks(torch, *sizes):
    for size in sizes:
        whole = -(-size // 512) * 512
        blocks = [torch.full((whole,), 0xA5, dtype=torch.uint8, device="cuda")
                  for _ in range(12)]
        del blocks


def behind(torch, t):
    """The bytes between a tensor's end and its block's."""
    size = t.numel() * t.element_size()
    whole = -(-size // 512) * 512
    storage = torch._C._construct_storage_from_data_pointer(
        t.data_ptr(), t.device, whole)
    every = torch.empty(0, dtype=torch.uint8, device=t.device).set_(storage)
    return every[size:].cpu()
