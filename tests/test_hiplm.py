"""CPU tests of the scoring operators (ops/hiplm.py): values and gradients
against their definitions in 64 bits, masks, padding, and the refusals."""

import math
import sys
from pathlib import Path

import numpy as np
import pytest

torch = pytest.importorskip("torch")

OPS_DIR = Path(__file__).resolve().parent.parent / "code_interpreter_amd" / "ops"
sys.path.insert(0, str(OPS_DIR))
sys.path.insert(0, str(Path(__file__).resolve().parent))

import hiplm  # noqa: E402
import hipmx  # noqa: E402
import lm_oracle as oracle  # noqa: E402

INF, NAN = math.inf, math.nan


def rows_with_trouble(v, dtype=torch.float32):
    """Rows that are plain, sharp, tied, partly and wholly masked (by -inf and
    by the type's lowest value), and that hold a NaN or an infinity; tokens
    for them."""
    g = torch.Generator().manual_seed(v)
    low = torch.finfo(dtype).min
    x = (torch.randn(12, v, generator=g) * 3).to(dtype)
    x[1] = 2.5
    x[2, v // 2] = 60
    x[3, ::2] = -INF
    x[4, 1:] = -INF
    x[5] = -INF
    x[6, ::2] = low
    x[7] = low
    x[8, v // 3] = NAN
    x[9, v // 3] = INF
    tokens = torch.randint(v, (12,), generator=g)
    tokens[4] = 0
    tokens[10] = -100
    tokens[11] = v
    return x, tokens


def check(got, want, slack):
    got = got.detach().double().cpu().numpy()
    # results are float32: what lies outside of its range is an infinity
    most = np.finfo(np.float32).max
    want = np.where(np.abs(want) > most, np.copysign(INF, want), want)
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        assert (same | (np.abs(got - want) <= slack)).all()


@pytest.mark.parametrize("t", [1.0, 0.5, 3.0])
@pytest.mark.parametrize("v", [1, 2, 7, 300])
def test_token_logprobs_values(v, t):
    x, tokens = rows_with_trouble(v)
    top = min(5, v)
    r = hiplm.token_logprobs(x, tokens, top=top, temperature=t)
    lp, h, top_lp, top_ids = oracle.token_logprobs(
        x.double().numpy(), tokens.numpy(), top, t)
    slack = 2.0 ** -18 * (1 + np.abs(np.where(np.isfinite(lp), lp, 0)))
    check(r.logprobs, lp, slack)
    check(r.entropy, h, 2.0 ** -18 * (1 + math.log(v)))
    good = ~np.isnan(top_lp)
    assert np.array_equal(r.top_tokens.numpy()[good], top_ids[good])
    big = np.abs(np.where(np.isfinite(top_lp), top_lp, 0))
    check(r.top_logprobs, top_lp, 2.0 ** -18 * (1 + big))


def test_token_logprobs_gradient():
    v, t = 300, 0.7
    x, tokens = rows_with_trouble(v)
    x = x.requires_grad_(True)
    r = hiplm.token_logprobs(x, tokens, temperature=t)
    g_lp, g_h = torch.randn(12), torch.randn(12)
    (grad,) = torch.autograd.grad([r.logprobs, r.entropy], [x], [g_lp, g_h])
    want, size = oracle.token_logprobs_grad(
        x.detach().double().numpy(), tokens.numpy(), t,
        g_lp.double().numpy(), g_h.double().numpy())
    rows = [0, 1, 2, 3, 4, 5, 6, 7, 10]  # those without NaN
    check(grad[rows], want[rows], 2.0 ** -17 * size[rows] + 1e-30)
    assert not r.top_logprobs.requires_grad


def test_shapes_and_ids():
    x = torch.randn(2, 3, 17)
    tokens = torch.randint(17, (2, 3), dtype=torch.int32)
    r = hiplm.token_logprobs(x, tokens, top=4)
    assert r.logprobs.shape == r.entropy.shape == (2, 3)
    assert r.top_logprobs.shape == r.top_tokens.shape == (2, 3, 4)
    assert r.top_tokens.dtype == torch.int64
    one = hiplm.token_logprobs(x[1, 2], tokens[1, 2], top=4)
    assert one.logprobs.shape == () and one.top_tokens.shape == (4,)
    torch.testing.assert_close(one.logprobs, r.logprobs[1, 2])
    none = hiplm.token_logprobs(x[:0], tokens[:0], top=4)
    assert none.logprobs.shape == (0, 3) and none.top_tokens.shape == (0, 3, 4)
    pad = hiplm.token_logprobs(x, torch.full((2, 3), 7), ignore_index=7)
    assert (pad.logprobs == 0).all() and (pad.entropy == 0).all()


def records(v, k, rows=12):
    """Teacher records: full, short, empty, repeated, and wrong ones."""
    g = torch.Generator().manual_seed(100 * v + k)
    teacher = torch.randn(rows, k, generator=g) * 2
    ids = torch.stack([torch.randperm(v, generator=g)[:k] if k <= v else
                       torch.randint(v, (k,), generator=g)
                       for _ in range(rows)])
    ids[1, k // 2:] = -1
    teacher[2, k // 2:] = -INF
    ids[3] = -1
    teacher[4] = -INF
    ids[7] = ids[7, 0]
    ids[9, 0] = v
    teacher[10, 0] = NAN
    return teacher, ids


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("v,k", [(1, 1), (9, 4), (300, 8), (300, 256)])
def test_distill(v, k, reduction):
    t = 1.5
    x, _ = rows_with_trouble(v)
    teacher, ids = records(v, k)
    keep = [0, 1, 2, 3, 4, 6, 7]
    if reduction == "none":  # rows of NaN and of an infinite loss too
        keep = list(range(12))
    x = x[keep].requires_grad_(True)
    loss = hiplm.topk_distill_loss(x, teacher[keep], ids[keep],
                                   temperature=t, reduction=reduction)
    want, grad, size = oracle.distill(
        x.detach().double().numpy(), teacher[keep].double().numpy(),
        ids[keep].numpy(), t, reduction)
    scale = 1 + np.abs(np.where(np.isfinite(want), want, 0))
    check(loss, want, 2.0 ** -16 * scale)
    (got,) = torch.autograd.grad(loss.sum(), [x])
    # what is not finite in a row's loss says nothing of its gradient here
    rows = np.isfinite(np.broadcast_to(want, (len(keep),)))
    check(got[rows], grad[rows], 2.0 ** -16 * size[rows] + 1e-30)


def test_distill_without_any_record():
    x = torch.randn(2, 9, requires_grad=True)
    loss = hiplm.topk_distill_loss(x, torch.zeros(2, 3),
                                   torch.full((2, 3), -1))
    assert loss.item() == 0
    (grad,) = torch.autograd.grad(loss, [x])
    assert (grad == 0).all()
    assert hiplm.topk_distill_loss(
        x[:0], torch.zeros(0, 3), torch.zeros(0, 3, dtype=torch.long)
    ).item() == 0


def test_token_logprobs_refusals():
    x, tokens = torch.randn(3, 20), torch.zeros(3, dtype=torch.long)
    with pytest.raises(TypeError, match="logits must be a tensor"):
        hiplm.token_logprobs(x.numpy(), tokens)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        hiplm.token_logprobs(x.double(), tokens)
    with pytest.raises(ValueError, match="last axis"):
        hiplm.token_logprobs(torch.zeros(3, 0), tokens)
    with pytest.raises(TypeError, match="int64 or int32"):
        hiplm.token_logprobs(x, tokens.float())
    with pytest.raises(ValueError, match="tokens must be"):
        hiplm.token_logprobs(x, tokens[:2])
    for top in (-1, 21, 129):
        with pytest.raises(ValueError, match="top must be"):
            hiplm.token_logprobs(x, tokens, top=top)
    for t in (0, -1.0, 1e-5, INF, NAN):
        with pytest.raises(ValueError, match="temperature"):
            hiplm.token_logprobs(x, tokens, temperature=t)


def test_distill_refusals():
    x, teacher = torch.randn(3, 20), torch.randn(3, 4)
    ids = torch.zeros(3, 4, dtype=torch.long)
    loss = hiplm.topk_distill_loss
    with pytest.raises(ValueError, match="teacher_tokens must be"):
        loss(x, teacher, ids[:, :3])
    with pytest.raises(ValueError, match="teacher_logits must be"):
        loss(x, teacher[:2], ids[:2])
    with pytest.raises(ValueError, match="k from 1 to 256"):
        loss(x, torch.zeros(3, 257), torch.zeros(3, 257, dtype=torch.long))
    with pytest.raises(ValueError, match="k from 1 to 256"):
        loss(x, teacher[:, :0], ids[:, :0])
    with pytest.raises(ValueError, match="detach"):
        loss(x, teacher.requires_grad_(True), ids)
    teacher = teacher.detach()
    with pytest.raises(TypeError, match="int64 or int32"):
        loss(x, teacher, ids.float())
    with pytest.raises(TypeError, match="teacher_logits"):
        loss(x, teacher.double(), ids)
    with pytest.raises(ValueError, match="reduction"):
        loss(x, teacher, ids, reduction="batchmean")
    with pytest.raises(ValueError, match="temperature"):
        loss(x, teacher, ids, temperature=0)


def test_a_head_records_and_a_student_learns():
    """The operators in a row: a 4-bit teacher head answers, its top
    alternatives are recorded, a student's gradient is that of the record."""
    torch.manual_seed(3)
    hidden, vocab = 64, 200
    head = hipmx.quantize(torch.randn(vocab, hidden) * 0.2)
    x = torch.randn(5, hidden)
    with torch.no_grad():
        logits = torch.nn.functional.linear(x, head)
    said = hiplm.token_logprobs(logits, logits.argmax(-1), top=8)
    assert torch.equal(said.top_tokens[:, 0], logits.argmax(-1))
    assert torch.equal(said.top_logprobs[:, 0], said.logprobs)
    w = torch.randn(vocab, hidden, requires_grad=True)
    loss = hiplm.topk_distill_loss(x @ w.T, said.top_logprobs,
                                   said.top_tokens)
    (grad,) = torch.autograd.grad(loss, [w])
    _, dz, _ = oracle.distill(
        (x @ w.T).detach().double().numpy(),
        said.top_logprobs.double().numpy(), said.top_tokens.numpy(), 1.0,
        "mean")
    want = dz.T @ x.double().numpy()
    np.testing.assert_allclose(grad.numpy(), want, atol=1e-5)


class Wrapper(torch.Tensor):
    """Has a type, sizes and a device, and no memory, as distributed tensors
    have none."""

    @staticmethod
    def __new__(cls, like, device="cuda"):
        return torch.Tensor._make_wrapper_subclass(
            cls, like.shape, strides=like.stride(), storage_offset=8,
            dtype=like.dtype, device=device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise NotImplementedError(str(func))


def fake(like):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        return torch.empty(like.shape, dtype=like.dtype, device="cuda")


@pytest.mark.parametrize("make", [Wrapper, fake])
def test_tensors_without_memory_are_refused(make):
    """Before anything is launched: here no GPU is needed to see it."""
    pytest.importorskip("_hiplm")
    x, ids = make(torch.randn(3, 64)), make(torch.zeros(3, 2).long())
    one = make(torch.zeros(3).long())
    codes = make(torch.zeros(5, 32, dtype=torch.uint8))
    scales = make(torch.zeros(5, 2, dtype=torch.uint8))
    module = hiplm.hiptorch.ensure_hiplm()
    for call in (
        lambda: hiplm.token_logprobs(x, one, top=2),
        lambda: hiplm.topk_distill_loss(x, make(torch.zeros(3, 2)), ids),
        lambda: hipmx.quantize(x),
        lambda: module.mx_dequantize(codes, scales, 64, 0),
        lambda: module.mx_linear(x, None, codes, scales, None, 64, 0),
    ):
        with pytest.raises(TypeError, match="memory of its own"):
            call()


def test_batched_tensors_are_refused():
    """vmap's tensors have no memory either, at the kernels' entry."""
    module = pytest.importorskip("_hiplm")
    for call in (
        lambda x: module.mx_quantize(x, 0),
        lambda x: module.token_logprobs(x, torch.zeros(3).long(), 0, 0, 1.0,
                                        -100),
    ):
        with pytest.raises(TypeError, match="memory of its own"):
            torch.vmap(call)(torch.randn(2, 3, 64))


def garbage(v):
    """Rows of trouble, and padded rows and wholly masked ones that hold or
    are given what is wrong."""
    x, tokens = rows_with_trouble(v)
    more = x[:6].clone()
    more[0, v // 2] = NAN
    more[1, 0] = INF
    more[2] = NAN
    more[3] = -INF
    more[4] = -INF
    tokens = torch.cat([tokens, torch.tensor([-100, -100, -100, -100, v, -3])])
    return torch.cat([x, more]), tokens


@pytest.mark.parametrize("use", ["both", "logprobs", "entropy"])
@pytest.mark.parametrize("v", [1, 7, 300])
def test_gradients_of_wrong_and_padded_rows(v, use):
    """Padding gets no gradient, whatever stands in it; a token outside of
    the vocabulary and a NaN give NaN gradients, as on the kernels."""
    x, tokens = garbage(v)
    x = x.requires_grad_(True)
    r = hiplm.token_logprobs(x, tokens, temperature=0.7)
    g = torch.Generator().manual_seed(v)
    gs = {name: torch.randn(len(x), generator=g) * (use in ("both", name))
          for name in ("logprobs", "entropy")}
    (grad,) = torch.autograd.grad(
        [getattr(r, name) for name in gs], [x], list(gs.values()))
    want, size = oracle.token_logprobs_grad(
        x.detach().double().numpy(), tokens.numpy(), 0.7,
        *(o.double().numpy() for o in gs.values()))
    check(grad, want, 2.0 ** -17 * size + 1e-30)
    lp, h, _, _ = oracle.token_logprobs(
        x.detach().double().numpy(), tokens.numpy(), 0, 0.7)
    check(r.logprobs, lp, 2.0 ** -18 * (
        1 + np.abs(np.where(np.isfinite(lp), lp, 0))))
    check(r.entropy, h, 2.0 ** -18 * (1 + math.log(v)))


@pytest.mark.parametrize("v,k", [(1, 1), (9, 4), (300, 8)])
def test_distill_gradients_of_wrong_and_padded_rows(v, k):
    """The same of distillation: a row without a record has no gradient,
    whatever its logits; a bad entry gives its row NaN gradients."""
    x, _ = garbage(v)
    teacher, ids = records(v, k, rows=18)
    ids[[8, 12, 14]] = -1         # without a record: NaN in the logits,
    teacher[[9, 13]] = -INF       # and an infinity
    ids[16, k - 1] = v + 5        # bad: the row is masked as a whole,
    teacher[17] = NAN             # and all of its entries are
    x = x.requires_grad_(True)
    loss = hiplm.topk_distill_loss(x, teacher, ids, temperature=1.5,
                                   reduction="none")
    want, grad, size = oracle.distill(
        x.detach().double().numpy(), teacher.double().numpy(), ids.numpy(),
        1.5, "none")
    check(loss, want, 2.0 ** -16 * (
        1 + np.abs(np.where(np.isfinite(want), want, 0))))
    (got,) = torch.autograd.grad(loss.sum(), [x])
    rows = ~np.isposinf(want)  # those with a masked entry are tested elsewhere
    check(got[rows], grad[rows], 2.0 ** -16 * size[rows] + 1e-30)


def lowest_in_record(v, dtype):
    """A student that gives the type's lowest value to tokens with a share of
    the record, next to ordinary ones."""
    g = torch.Generator().manual_seed(v)
    x = torch.randn(6, v, generator=g).to(dtype)
    teacher = torch.randn(6, 4, generator=g)
    ids = torch.stack([torch.randperm(v, generator=g)[:4] for _ in range(6)])
    for i in range(1, 6):
        x[i, ids[i, :1 + i // 2]] = torch.finfo(dtype).min
    return x, teacher, ids


# a share is off by its exponent's rounding and scale, 5 steps of at most 16,
# and its own; what it is multiplied with and added to by a few steps: relative
# to a loss that these entries make up at most 128 steps
LOWEST = 128 * 2.0 ** -24


@pytest.mark.parametrize("t", [0.3, 0.5, 1.0, 1.5])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_distill_of_lowest_logits_is_finite(dtype, t):
    x, teacher, ids = lowest_in_record(50, dtype)
    x = x.requires_grad_(True)
    loss = hiplm.topk_distill_loss(x, teacher, ids, temperature=t,
                                   reduction="none")
    want, grad, size = oracle.distill(
        x.detach().double().numpy(), teacher.double().numpy(), ids.numpy(),
        t, "none")
    check(loss, want, LOWEST * (1 + np.abs(want)))
    (got,) = torch.autograd.grad(loss.sum(), [x])
    # one rounding to the type
    check(got, grad, 2.0 ** -16 * size + 1e-30
          + torch.finfo(dtype).eps / 2 * np.abs(grad))


def all_lowest(k):
    """Records all of whose tokens the student gives the type's lowest value:
    shares of 1 in sum, times the largest number that a float32 has."""
    g = torch.Generator().manual_seed(k)
    x = torch.randn(40, 400, generator=g)
    ids = torch.stack([torch.randperm(400, generator=g)[:k]
                       for _ in range(40)])
    x.scatter_(1, ids, torch.finfo(torch.float32).min)
    return x, torch.randn(40, k, generator=g), ids


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("t", [0.3, 0.9])
@pytest.mark.parametrize("k", [1, 2, 7, 100])
def test_distill_of_nothing_but_lowest_logits(k, t, reduction):
    x, teacher, ids = all_lowest(k)
    loss = hiplm.topk_distill_loss(x, teacher, ids, temperature=t,
                                   reduction=reduction)
    want, _, _ = oracle.distill(x.double().numpy(), teacher.double().numpy(),
                                ids.numpy(), t, reduction)
    assert np.isfinite(want).all()
    check(loss, want, LOWEST * (1 + np.abs(want)))


def test_second_derivatives_of_host_tensors():
    """A gradient penalty, against torch's own operations in 64 bits."""
    g = torch.Generator().manual_seed(9)
    x = torch.randn(3, 20, generator=g)
    teacher, ids = torch.randn(3, 4, generator=g), torch.arange(12).view(3, 4)

    def penalty(loss, z):
        (grad,) = torch.autograd.grad(loss, [z], create_graph=True)
        return torch.autograd.grad(loss + grad.pow(2).sum(), [z])[0]

    z = x.clone().requires_grad_(True)
    r = hiplm.token_logprobs(z, ids[:, 0])
    got = penalty(r.logprobs.sum() + r.entropy.sum()
                  + hiplm.topk_distill_loss(z, teacher, ids), z)
    z = x.double().requires_grad_(True)
    lp, lq = torch.log_softmax(z, -1), torch.log_softmax(teacher.double(), -1)
    at = lp.gather(-1, ids)
    want = penalty(at[:, 0].sum() - (lp.exp() * lp).sum()
                   + (lq.exp() * (lq - at)).sum() / 3, z)
    # sums of some ten terms of size 1 to 10, a few roundings each
    torch.testing.assert_close(got.double(), want, rtol=2e-5, atol=2e-5)
