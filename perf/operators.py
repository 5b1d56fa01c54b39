"""Language-model operators on the gfx950 kernels: what is measured.

Four operators, used one after the other by a program that serves a 4-bit
output head, records what it answers and trains a student on the record:

- ``quantize``: a tensor to microscaled 4-bit floating point (blocks of 32
  along the last axis, e2m1 elements, one power-of-two scale a block) and
  back to the values that the codes stand for;
- ``linear``: the product of an activation, quantised on the way in, with a
  weight that is held in that form;
- ``logprobs``: the log probabilities of given tokens under rows of logits,
  the rows' entropies and their top alternatives, and the backward pass;
- ``distill``: the divergence of a student's distribution from a teacher's
  recorded top logits, and the backward pass.

With ``own`` false, ``run`` computes them in plain torch operations in 32
bits; with it true, through the framework's entry points.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BLOCK = 32


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one request's hidden states on their way into a 4-bit product
        {"name": "quantize-tokens", "op": "quantize", "rows": 16, "k": 4096,
         "dtype": "bf16"},
        # a weight matrix converted once, when a model is loaded
        {"name": "quantize-weight", "op": "quantize", "rows": 8192,
         "k": 8192, "dtype": "bf16"},
        # a master weight whose rows end inside a block
        {"name": "quantize-ragged", "op": "quantize", "rows": 4097,
         "k": 1000, "dtype": "f32"},
        # decoding: one token through a square projection
        {"name": "linear-1", "op": "linear", "m": 1, "n": 8192, "k": 8192,
         "dtype": "bf16", "bias": False},
        # decoding: a batch of sequences, with a bias
        {"name": "linear-37", "op": "linear", "m": 37, "n": 4096, "k": 4096,
         "dtype": "f16", "bias": True},
        # a short prompt against sizes that no tile divides
        {"name": "linear-ragged", "op": "linear", "m": 333, "n": 5001,
         "k": 2056, "dtype": "bf16", "bias": True},
        # a batch of prompts
        {"name": "linear-8192", "op": "linear", "m": 8192, "n": 8192,
         "k": 8192, "dtype": "bf16", "bias": False},
        # one decoding step whose answer reports 20 alternatives
        {"name": "logprobs-step", "op": "logprobs", "rows": 1, "v": 131072,
         "dtype": "bf16", "top": 20, "grad": False, "mask": "none"},
        # a prompt's tokens scored under a constrained vocabulary of odd size
        {"name": "logprobs-prompt", "op": "logprobs", "rows": 509,
         "v": 50001, "dtype": "f32", "top": 5, "grad": False, "mask": "inf"},
        # policy training: log probabilities and entropies with gradients,
        # padded rows among them
        {"name": "logprobs-train", "op": "logprobs", "rows": 4096,
         "v": 131072, "dtype": "bf16", "top": 0, "grad": True,
         "mask": "none"},
        # a small student on a record of 8 alternatives
        {"name": "distill-small", "op": "distill", "rows": 61, "v": 10007,
         "dtype": "f16", "top": 8, "temperature": 2.0},
        # a training step on a record of 64 alternatives
        {"name": "distill-train", "op": "distill", "rows": 4096,
         "v": 65536, "dtype": "bf16", "top": 64, "temperature": 1.0},
    ]


def _spread(rng, low, high):
    return max(low, min(high, round(math.exp(
        rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "logprobs", "distill"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "quantize":
        return {"op": op, "rows": _spread(rng, 1, 8192),
                "k": _spread(rng, 32, 8192), "dtype": dtype}
    if op == "linear":
        n, k = _spread(rng, 64, 8192), _spread(rng, 64, 8192)
        if rng.random() < 0.5:
            n, k = n // 64 * 64, k // 64 * 64
        return {"op": op, "m": _spread(rng, 1, 8192), "n": n, "k": k,
                "dtype": dtype, "bias": rng.random() < 0.5}
    v = _spread(rng, 1000, 131072)
    if op == "logprobs":
        # rows of 32-bit logits are half as many, so that no drawn case
        # moves more bytes than the largest listed one
        rows = _spread(rng, 1, 2048 if dtype == "f32" else 4096)
        grad = rng.random() < 0.5
        return {"op": op, "rows": rows, "v": v, "dtype": dtype,
                "top": 0 if grad else rng.choice([0, 1, 5, 20, 64]),
                "grad": grad, "mask": rng.choice(["none", "inf", "lowest"])}
    return {"op": op, "rows": _spread(rng, 1, 2048), "v": v, "dtype": dtype,
            "top": rng.choice([1, 8, 16, 50, 64, 128]),
            "temperature": rng.choice([1.0, 2.0, 0.7])}


def _blocks(k):
    return -(-k // BLOCK)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "quantize":
        n = case["rows"] * case["k"]
        stored = case["rows"] * _blocks(case["k"]) * (BLOCK // 2 + 1)
        # x in, codes and scales out; codes and scales in, values out
        return {"bytes": 2 * n * size + 2 * stored, "flops": 0}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m * k + m * n + (n if case["bias"] else 0)) * size
                + n * _blocks(k) * (BLOCK // 2 + 1),
                "flops": 2 * m * n * k}
    rows, n = case["rows"], case["rows"] * case["v"]
    if case["op"] == "logprobs":
        small = rows * (8 + 4 + 4 + 12 * case["top"])
        if case["grad"]:  # the backward reads logits again, writes gradients
            return {"bytes": 3 * n * size + small + 8 * rows, "flops": 12 * n}
        return {"bytes": n * size + small, "flops": 6 * n}
    return {"bytes": 3 * n * size + rows * case["top"] * 12, "flops": 9 * n}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _logits(g, rows, v, dtype):
    """Rows of logits as a head makes them: most of the vocabulary far below
    a few likely tokens, another sharpness from row to row."""
    x = torch.randn(rows, v, generator=g, device="cuda")
    x *= 1.0 + 2.0 * torch.rand(rows, 1, generator=g, device="cuda")
    hot = torch.randint(v, (rows, 4), generator=g, device="cuda")
    lift = 6.0 + 8.0 * torch.rand(rows, 4, generator=g, device="cuda")
    x.scatter_(1, hot, lift)
    return x.to(dtype), hot


def prepare(case, seed):
    g = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "quantize":
        rows, k = case["rows"], case["k"]
        x = torch.randn(rows, k, generator=g, device="cuda")
        # a few channels far larger than the rest, as activations have them
        x *= 0.5 + 20.0 * (torch.rand(1, k, generator=g, device="cuda") > 0.99)
        return {"op": "quantize", "x": x.to(dtype)}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        x = torch.randn(m, k, generator=g, device="cuda").to(dtype)
        codes = torch.randint(256, (n, _blocks(k) * (BLOCK // 2)),
                              generator=g, device="cuda", dtype=torch.uint8)
        if k % BLOCK:  # elements behind the row's end are zeros
            at = torch.arange(codes.shape[1], device="cuda") * 2
            codes &= ((at < k) * 0x0F + (at + 1 < k) * 0xF0).to(torch.uint8)
        # weights of about 0.02: block scales of 2^-9 to 2^-6
        scales = torch.randint(118, 122, (n, _blocks(k)), generator=g,
                               device="cuda", dtype=torch.uint8)
        bias = None
        if case["bias"]:
            bias = torch.randn(n, generator=g, device="cuda").to(dtype)
        return {"op": "linear", "x": x, "codes": codes, "scales": scales,
                "k": k, "bias": bias}
    rows, v = case["rows"], case["v"]
    logits, hot = _logits(g, rows, v, dtype)
    if case["op"] == "logprobs":
        tokens = torch.randint(v, (rows,), generator=g, device="cuda")
        # half of the given tokens are likely ones, as an answer's own are
        likely = torch.rand(rows, generator=g, device="cuda") < 0.5
        tokens = torch.where(likely, hot[:, 0], tokens)
        if case["mask"] != "none":
            # a grammar that allows a fifth of the vocabulary, the given
            # tokens among it
            low = (-math.inf if case["mask"] == "inf"
                   else torch.finfo(dtype).min)
            keep = logits.gather(1, tokens[:, None])
            banned = torch.rand(1, v, generator=g, device="cuda") < 0.8
            logits.masked_fill_(banned, low)
            logits.scatter_(1, tokens[:, None], keep)
        state = {"op": "logprobs", "logits": logits, "tokens": tokens,
                 "top": case["top"], "grad": case["grad"]}
        if case["grad"]:
            pad = torch.rand(rows, generator=g, device="cuda") < 0.1
            tokens.masked_fill_(pad, -100)
            state["g_logprobs"] = torch.randn(rows, generator=g,
                                              device="cuda") / rows
            state["g_entropy"] = torch.full((rows,), -0.01 / rows,
                                            device="cuda")
            logits.requires_grad_(True)
        return state
    k = case["top"]
    teacher = torch.randn(rows, k, generator=g, device="cuda") * 2.0
    teacher = teacher.sort(-1, descending=True).values.contiguous()
    # a record names each alternative once; the first ones are the student's
    # likely ones too
    at = torch.arange(k, device="cuda") * (v // k)
    shift = torch.randint(v, (rows, 1), generator=g, device="cuda")
    ids = ((at + shift) % v).contiguous()
    return {"op": "distill", "logits": logits.requires_grad_(True),
            "teacher": teacher, "ids": ids,
            "temperature": case["temperature"]}


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _plain_round_trip(x):
    """The values in 32 bits that x's microscaled 4-bit form stands for."""
    rows, k = x.shape
    padded = _blocks(k) * BLOCK
    v = torch.zeros(rows, padded, device=x.device)
    v[:, :k] = x
    v = v.view(rows, -1, BLOCK)
    largest = v.abs().amax(-1, keepdim=True)
    # frexp's mantissa is in [1/2, 1): floor(log2) is its exponent less 1;
    # 2 more is the exponent of the largest element, 6 = 1.5 * 2^2
    shift = (torch.frexp(largest).exponent - 3).clamp(min=-127)
    a = torch.ldexp(v.abs(), -shift)
    step = 0.5 + 0.5 * (a >= 2) + 1.0 * (a >= 4)
    a = (torch.round(a / step) * step).clamp(max=6.0)
    v = torch.ldexp(torch.copysign(a, v), shift)
    v = torch.where(torch.isfinite(largest), v, math.nan)
    return v.view(rows, padded)[:, :k]


def _plain_values(codes, scales, k):
    """The values in 32 bits that stored codes and scales stand for."""
    half = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0],
                        device=codes.device)
    table = torch.cat([half, -half])
    v = torch.stack([table[(codes & 15).int()], table[(codes >> 4).int()]], -1)
    v = v.view(codes.shape[0], -1, BLOCK)
    v = torch.ldexp(v, scales.int()[..., None] - 127)
    return v.view(codes.shape[0], -1)[:, :k]


def _plain_softmax(z):
    """(exp(z - max), sum of them, z - max) of rows in 32 bits."""
    d = z - z.amax(-1, keepdim=True)
    e = torch.exp(d)
    return e, e.sum(-1, keepdim=True), d


def _plain_logprobs(s):
    z = s["logits"].detach().float()
    tokens = s["tokens"]
    live = tokens >= 0
    e, total, d = _plain_softmax(z)
    log_total = torch.log(total)
    at = tokens.clamp(min=0)[:, None]
    lp = (d.gather(1, at) - log_total)[:, 0]
    # a masked entry has no share: its 0 * -inf counts as 0
    d.clamp_(min=-1e4)
    entropy = (log_total - (e * d).sum(-1, keepdim=True) / total)[:, 0]
    out = [torch.where(live, lp, 0.0), torch.where(live, entropy, 0.0)]
    if s["top"]:
        values, ids = torch.sort(z, dim=-1, descending=True,
                                 stable=True)
        values, ids = values[:, :s["top"]], ids[:, :s["top"]]
        top = values - z.amax(-1, keepdim=True) - log_total
        out += [top, torch.where(values > -math.inf, ids, -1)]
    if s["grad"]:
        g_lp = torch.where(live, s["g_logprobs"], 0.0)[:, None]
        g_h = torch.where(live, s["g_entropy"], 0.0)[:, None]
        p = e / total
        grad = -p * (g_lp + g_h * (d - log_total + entropy[:, None]))
        grad.scatter_add_(1, at, g_lp)
        out.append(grad.to(s["logits"].dtype))
    return out


def _plain_distill(s):
    t, ids = s["temperature"], s["ids"]
    e, total, d = _plain_softmax(s["logits"].detach().float() / t)
    lp = d.gather(1, ids) - torch.log(total)
    te, t_total, td = _plain_softmax(s["teacher"].float() / t)
    q = te / t_total
    rows = ids.shape[0]
    loss = (q * (td - torch.log(t_total) - lp)).sum() * (t * t / rows)
    grad = (e / total).scatter_add_(1, ids, -q) * (t / rows)
    return [loss, grad.to(s["logits"].dtype)]


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _own_run(s):
    from code_interpreter_amd.ops import load_hiplm, load_hipmx

    if s["op"] == "quantize":
        return load_hipmx().quantize(s["x"]).dequantize(s["x"].dtype)
    if s["op"] == "linear":
        mx = load_hipmx()
        w = mx.MXFP4Tensor(s["codes"], s["scales"], s["k"])
        return mx.linear(s["x"], w, s["bias"])
    lm = load_hiplm()
    if s["op"] == "logprobs":
        r = lm.token_logprobs(s["logits"], s["tokens"], top=s["top"])
        out = [r.logprobs, r.entropy]
        if s["top"]:
            out += [r.top_logprobs, r.top_tokens]
        if s["grad"]:
            out += torch.autograd.grad(
                out[:2], [s["logits"]], [s["g_logprobs"], s["g_entropy"]])
        return out
    loss = lm.topk_distill_loss(s["logits"], s["teacher"], s["ids"],
                                temperature=s["temperature"])
    return [loss, torch.autograd.grad(loss, [s["logits"]])[0]]


def run(state):
    if own:
        return _own_run(state)
    if state["op"] == "quantize":
        return _plain_round_trip(state["x"]).to(state["x"].dtype)
    if state["op"] == "linear":
        w = _plain_values(state["codes"], state["scales"], state["k"])
        y = _plain_round_trip(state["x"]) @ w.T
        if state["bias"] is not None:
            y += state["bias"]
        return y.to(state["x"].dtype)
    if state["op"] == "logprobs":
        return _plain_logprobs(state)
    return _plain_distill(state)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_round_trip(x):
    rows, k = x.shape
    v = torch.nn.functional.pad(x.double(), (0, -k % BLOCK))
    v = v.reshape(rows, -1, BLOCK)
    largest = v.abs().amax(-1, keepdim=True)
    unit = torch.exp2(torch.floor(torch.log2(
        largest.clamp(min=2.0 ** -125))) - 2)
    a = v.abs() / unit
    # halfway points between neighbours, each rounded to the even code
    result = torch.zeros_like(a)
    for value, border, up in ((0.5, 0.25, False), (1.0, 0.75, True),
                              (1.5, 1.25, False), (2.0, 1.75, True),
                              (3.0, 2.5, False), (4.0, 3.5, True),
                              (6.0, 5.0, False)):
        result[(a >= border) if up else (a > border)] = value
    v = torch.sign(v) * result * unit
    return v.reshape(rows, -1)[:, :k]


def _exact_values(codes, scales, k):
    nibble = torch.stack([codes & 15, codes >> 4], -1).flatten(1).long()
    power, odd = (nibble >> 1) & 3, nibble & 1
    v = torch.where(power == 0, 0.5 * odd,
                    torch.exp2(power.double() - 1) * (1 + 0.5 * odd))
    v = torch.where(nibble >= 8, -v, v)
    unit = torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, 1)
    return (v * unit)[:, :k]


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "quantize":
        return _exact_round_trip(s["x"])
    if s["op"] == "linear":
        y = _exact_round_trip(s["x"]) @ _exact_values(
            s["codes"], s["scales"], s["k"]).T
        return y if s["bias"] is None else y + s["bias"].double()
    x = s["logits"].detach().double()
    if s["op"] == "logprobs":
        lp = torch.log_softmax(x, -1)
        p = lp.exp()
        entropy = -torch.where(p > 0, p * lp, 0.0).sum(-1)
        tokens = s["tokens"]
        live = tokens >= 0
        at = tokens.clamp(min=0)[:, None]
        out = [torch.where(live, lp.gather(1, at)[:, 0], 0.0),
               torch.where(live, entropy, 0.0)]
        if s["top"]:
            out += [lp.topk(s["top"], -1).values, None]
        if s["grad"]:
            g_lp, g_h = s["g_logprobs"].double(), s["g_entropy"].double()
            slope = torch.where(p > 0, lp + entropy[:, None], 0.0)
            grad = -p * g_lp[:, None] - p * slope * g_h[:, None]
            grad.scatter_add_(1, at, g_lp[:, None])
            out.append(grad * live[:, None])
        return out
    t = s["temperature"]
    lp = torch.log_softmax(x / t, -1)
    lq = torch.log_softmax(s["teacher"].double() / t, -1)
    q = lq.exp()
    rows = x.shape[0]
    loss = (q * (lq - lp.gather(1, s["ids"]))).sum(-1).mean() * t * t
    target = torch.zeros_like(lp).scatter_add_(1, s["ids"], q)
    return [loss, (lp.exp() - target) * (t / rows)]
