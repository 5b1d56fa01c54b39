"""Scoring rows of logits for sandboxed user code: log probabilities of given
tokens with entropies and top alternatives, and distillation from a teacher's
recorded top logits, with their backward passes, on gfx950 kernels.

Importable standalone inside the sandbox (APP_OPS_DIR is on sys.path), next
to torch:

    import hiplm
    r = hiplm.token_logprobs(logits, tokens, top=20)
    r.logprobs, r.entropy, r.top_logprobs, r.top_tokens
    loss = hiplm.topk_distill_loss(student_logits, r.top_logprobs,
                                   r.top_tokens)

A row of logits is read once in a forward and once in a backward pass, in
its own type (float32, bfloat16, float16); sums are float32. Masked entries
are -inf (or very low) logits.

GPU tensors run on the kernels, on torch's current stream of their device,
and raise where the extension is missing; CPU tensors are computed in plain
torch. Kernels have no second derivative: differentiating a gradient raises a
RuntimeError.
"""

from collections import namedtuple
import math

import hiptorch

MAX_TOP = 128      # alternatives of a row
MAX_RECORD = 256   # recorded teacher entries of a row

STATS = {"token_logprobs": 0, "topk_distill_loss": 0}

TokenLogprobs = namedtuple(
    "TokenLogprobs", ["logprobs", "entropy", "top_logprobs", "top_tokens"])

_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def _check_logits(logits) -> int:
    hiptorch.check_tensor("logits", logits)
    code = hiptorch.check_dtype("logits", logits.dtype)
    shape = logits.shape
    if not shape or not shape[-1]:
        raise ValueError(f"logits need a last axis, got {list(shape)}")
    if shape[-1] >= 1 << 31:
        raise ValueError("the last axis of logits is too long")
    return code


def _check_temperature(temperature) -> float:
    t = float(temperature)
    if not 1e-4 <= t <= 1e4:
        raise ValueError(f"temperature must be in [1e-4, 1e4], got {t}")
    return t


def _check_ids(torch, name, ids, shape, device):
    hiptorch.check_tensor(name, ids)
    if ids.dtype != torch.int64:
        if ids.dtype != torch.int32:
            raise TypeError(f"{name} must be int64 or int32, got {ids.dtype}")
        ids = ids.long()
    if ids.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got "
                         f"{list(ids.shape)}")
    if ids.device != device:
        raise ValueError(f"{name} are on {ids.device}, logits on {device}")
    return ids


def token_logprobs(logits, tokens, *, top: int = 0, temperature=1.0,
                   ignore_index: int = -100) -> TokenLogprobs:
    """ln p(token), the entropy and the ``top`` most likely tokens of rows of
    logits, p = softmax(logits / temperature).

    logits: [..., v]; tokens: [...] (int64, int32). Returns ``logprobs`` and
    ``entropy`` [...] in float32, both differentiable, ``top_logprobs``
    [..., top] in float32 and ``top_tokens`` [..., top] in int64, largest
    first, of equal logits the lowest token first; neither carries a
    gradient. top: 0 to 128, at most v.

    A masked token (-inf) is no alternative: a row with fewer than ``top``
    others ends in (-inf, -1). A row that is masked as a whole has no
    distribution: ln p is -inf, the entropy 0, the gradient 0. A row whose
    token is ``ignore_index`` is padding: 0, 0, (-inf, -1) and no gradient.
    A token outside of [0, v), or a NaN or +inf among the logits, gives NaN.
    """
    torch = hiptorch.lm_torch()
    code = _check_logits(logits)
    t = _check_temperature(temperature)
    shape = logits.shape
    top = int(top)
    if not 0 <= top <= MAX_TOP or top > shape[-1]:
        raise ValueError(f"top must be in [0, {min(MAX_TOP, shape[-1])}], got "
                         f"{top}")
    tokens = _check_ids(torch, "tokens", tokens, shape[:-1], logits.device)
    if not logits.is_cuda:
        return _cpu_token_logprobs(torch, logits, tokens, top, t,
                                   int(ignore_index))
    STATS["token_logprobs"] += 1
    return TokenLogprobs._make(hiptorch.ensure_hiplm().token_logprobs(
        logits, tokens, code, top, 1.0 / t, int(ignore_index)))


def topk_distill_loss(logits, teacher_logits, teacher_tokens, *,
                      temperature=1.0, reduction: str = "mean"):
    """The divergence of a student from a teacher's recorded top logits,
    T^2 sum_k q_k (ln q_k - ln p[token_k]), with q the softmax of the
    recorded entries over each other and p the student's softmax over the
    whole vocabulary, both at temperature T.

    logits: the student's, [..., v]. teacher_logits: [..., k] (float32,
    bfloat16, float16), logits or log probabilities, k from 1 to 256, without
    a gradient. teacher_tokens: [..., k] (int64, int32). A row with fewer
    entries is filled with tokens of -1 or logits of -inf; one with none
    has no loss and no gradient. A token that is recorded twice counts
    twice.

    reduction: "mean" (over rows with a record; 0 if there are none), "sum"
    or "none" ([...]); rows' losses and the result are float32. An entry that
    the student masks (-inf) gives an infinite loss, with the finite gradient
    T (p - q) / rows; a share q below the smallest normal float32 may count
    as 0.
    A token outside of [0, v) but -1, or a NaN or +inf on either side, gives
    NaN.
    """
    torch = hiptorch.lm_torch()
    code = _check_logits(logits)
    t = _check_temperature(temperature)
    lead = logits.shape[:-1]
    hiptorch.check_tensor("teacher_logits", teacher_logits)
    t_code = hiptorch.check_dtype("teacher_logits", teacher_logits.dtype)
    t_shape = teacher_logits.shape
    if (len(t_shape) != len(lead) + 1 or t_shape[:-1] != lead
            or not 1 <= t_shape[-1] <= MAX_RECORD):
        raise ValueError(
            f"teacher_logits must be [{', '.join(map(str, lead))}, k] with k "
            f"from 1 to {MAX_RECORD}, got {list(t_shape)}")
    if teacher_logits.device != logits.device:
        raise ValueError(f"teacher_logits are on {teacher_logits.device}, "
                         f"logits on {logits.device}")
    if teacher_logits.requires_grad:
        if torch.is_grad_enabled():
            raise ValueError("the teacher gets no gradient: detach its logits")
        teacher_logits = teacher_logits.detach()
    ids = _check_ids(torch, "teacher_tokens", teacher_tokens, t_shape,
                     logits.device)
    how = _REDUCTIONS.get(reduction)
    if how is None:
        raise ValueError("reduction must be 'mean', 'sum' or 'none', got "
                         f"{reduction!r}")
    if not logits.is_cuda:
        return _cpu_distill(torch, logits, teacher_logits, ids, t, reduction)
    STATS["topk_distill_loss"] += 1
    return hiptorch.ensure_hiplm().distill(
        logits, teacher_logits, ids, code, t_code, 1.0 / t, how)


# ---------------------------------------------------------------------------
# CPU tensors
# ---------------------------------------------------------------------------
def _cpu_shifted(torch, logits, without):
    """Rows in float32 less their largest logit: divided by a temperature
    before that, a lowest value would be an infinity. Of rows `without` a
    result the numbers are of no use, but no NaN either."""
    z = torch.where(without[..., None], 0.0, logits.float())
    return z - z.detach().amax(-1, keepdim=True)


def _cpu_empty(logits):
    """Rows that are masked as a whole."""
    return (logits.detach() == -math.inf).all(-1)


def _cpu_wrong(torch, rows, o):
    """o, with NaN in the given rows, and in their gradients."""
    return o * torch.where(rows, math.nan, 1.0)


def _cpu_token_logprobs(torch, logits, tokens, top, t, ignore):
    v = logits.shape[-1]
    ignored = tokens == ignore
    outside = ~ignored & ((tokens < 0) | (tokens >= v))
    empty = _cpu_empty(logits) & ~outside
    lp = torch.log_softmax(
        _cpu_shifted(torch, logits, empty | ignored) / t, -1)
    at = tokens.clamp(0, v - 1)[..., None]
    zero = 0.0
    logprobs = lp.gather(-1, at)[..., 0]
    logprobs = torch.where(empty, -math.inf, logprobs)
    entropy = -(lp.exp() * lp.clamp(min=-1e4)).sum(-1)
    entropy = torch.where(empty, zero, entropy)
    logprobs, entropy = (
        torch.where(ignored, zero, _cpu_wrong(torch, outside, o))
        for o in (logprobs, entropy))
    with torch.no_grad():
        z = logits.float()
        z = torch.where(z.isnan() | ignored[..., None], -math.inf, z)
        values, ids = torch.sort(z, dim=-1, descending=True, stable=True)
        values, ids = values[..., :top], ids[..., :top]
        there = values > -math.inf
        top_lp = torch.where(there, lp.gather(-1, ids), -math.inf)
        top_ids = torch.where(there, ids, -1)
    return TokenLogprobs(logprobs, entropy, top_lp, top_ids)


def _cpu_distill(torch, logits, teacher, ids, t, reduction):
    v = logits.shape[-1]
    z = teacher.float()
    there = (ids != -1) & (z != -math.inf)
    bad = there & (z.isnan() | (z == math.inf) | (ids < 0) | (ids >= v))
    absent = ~there.any(-1)
    wrong = bad.any(-1)
    empty = _cpu_empty(logits) & ~wrong
    # logarithms in units of 1 / t, and sums of them in quarters, so that
    # recorded lowest values overflow only where the loss does
    x = _cpu_shifted(torch, logits, empty | absent)
    lse = torch.logsumexp(x / t, -1, keepdim=True) * t
    z = torch.where(there & ~bad, z, -math.inf)
    z = _cpu_shifted(torch, z, _cpu_empty(z))
    q = torch.softmax(z / t, -1)
    lq = z - torch.logsumexp(z / t, -1, keepdim=True) * t
    # a share of 0 adds nothing, whatever the student gives it
    there = there & (q > 0)
    mine = x.gather(-1, ids.clamp(0, v - 1)) - lse
    mine = torch.where(empty[..., None], -math.inf, mine)
    mine = torch.where(there, mine, 0.0)
    loss = torch.where(there, q * ((lq - mine) * 0.25), 0.0).sum(-1) * (4 * t)
    loss = torch.where(absent, 0.0, _cpu_wrong(torch, wrong, loss))
    if reduction == "none":
        return loss
    total = loss.double().sum()
    if reduction == "mean":
        total = total / (~absent).sum().clamp(min=1)
    return total.float()
