"""Top alternatives of a policy's next-token distribution, and distillation from a teacher's, as measurable cases.

Four operators, each a ``kind`` of case.  ``z`` are a token's logits over the vocabulary, ``q = softmax(z / T)``:

* ``topk``: from materialised logits, the log-probability of the token that was taken, the entropy of ``q``, and the ``k``
  most likely tokens with their log-probabilities (largest logit first, the lowest index among equals);
* ``distil``: from materialised logits, the divergence of ``q`` from a teacher's ``k`` most likely tokens, per token;
* ``head_topk``: as ``topk``, from the hidden states and the weight of the vocabulary projection;
* ``head_distil``: as ``distil``, from the hidden states and the weight.

With ``t`` the teacher's log-probabilities of its tokens, ``p = exp(t)`` and ``q`` the student's probabilities of the same
tokens, a token's loss is ``sum p (t - log q)`` (``forward_kl``), ``sum q (log q - t)`` (``reverse_kl``), or ``beta sum p (t -
log m) + (1 - beta) sum q (log q - log m)`` with ``m = beta p + (1 - beta) q`` (``jsd``).  Cases with ``backward`` return the
gradients too, for given upstream gradients.
"""
from __future__ import annotations

import math

import torch

own = False

# (hidden_size, vocab) of the benchmark's heads
HEADS = ((896, 151936), (3584, 152064), (4096, 128256))
BETA = 0.3


def listed():
    return [
        # one new token of a single request, with the 20 alternatives a serving interface offers at most
        _rows("topk_one_token", "topk", 1, 151936, "bfloat16", 20),
        # one decoding step of a batch of requests; sampling temperature, fp32 logits as a sampler holds them
        _rows("topk_decoding_batch", "topk", 64, 128256, "float32", 5, 0.7),
        # the teacher's side of a distillation run without its fused head: a micro-batch of materialised logits
        _rows("topk_teacher_batch", "topk", 4096, 152064, "bfloat16", 64),
        # a loss on the alternatives of one response, through log-probs and entropy: an odd vocabulary, rows off 16 bytes
        _rows("topk_train_odd", "topk", 777, 50257, "float16", 8, backward=True),
        # an update of the student on a micro-batch of materialised logits
        _rows("distil_batch", "distil", 2048, 152064, "bfloat16", 64, backward=True),
        # the same for one response, fp32 logits, odd vocabulary, symmetric divergence
        _rows("distil_odd", "distil", 333, 151935, "float32", 100, 0.7, "jsd", backward=True),
        # validation loss of a small micro-batch: no gradient
        _rows("distil_validation", "distil", 200, 128256, "bfloat16", 32, divergence="reverse_kl"),
        # one decoding step of a teacher that scores what the student samples
        _head("head_topk_decoding", "head_topk", 64, HEADS[1], 20),
        # the teacher's pass over a micro-batch
        _head("head_topk_batch", "head_topk", 4096, HEADS[1], 64),
        # one short response of an update with a micro-batch of one, small model
        _head("head_distil_one_response", "head_distil", 93, HEADS[0], 64, backward=True),
        # an odd number of tokens, another divergence and temperature
        _head("head_distil_odd", "head_distil", 1301, HEADS[2], 32, 0.7, "reverse_kl", backward=True),
        # an update of the student on a full micro-batch
        _head("head_distil_batch", "head_distil", 8192, HEADS[1], 64, backward=True),
    ]


def _rows(name, kind, tokens, vocab, dtype, k, temperature=1.0, divergence="forward_kl", backward=False):
    return {"name": name, "kind": kind, "tokens": tokens, "vocab": vocab, "hidden": 0, "dtype": dtype, "k": k,
            "temperature": temperature, "divergence": divergence if kind == "distil" else "", "backward": backward}


def _head(name, kind, tokens, head, k, temperature=1.0, divergence="forward_kl", backward=False):
    return {"name": name, "kind": kind, "tokens": tokens, "vocab": head[1], "hidden": head[0], "dtype": "bfloat16", "k": k,
            "temperature": temperature, "divergence": divergence if kind == "head_distil" else "", "backward": backward}


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("topk", "distil", "head_topk", "head_distil"))
    divergence, temperature = rng.choice(("forward_kl", "reverse_kl", "jsd")), rng.choice((1.0, 1.0, 0.7))
    if kind in ("topk", "distil"):
        dtype = rng.choice(("bfloat16", "bfloat16", "float16", "float32"))
        vocab = rng.choice((32000, 50257, 65536, 128256, 151935, 151936, 152064))
        backward = rng.random() < (0.4 if kind == "topk" else 0.7)
        tokens = _log_int(rng, 1, 2000 if backward or dtype == "float32" else 4000)
        case = _rows("", kind, tokens, vocab, dtype, _log_int(rng, 1, 128), temperature, divergence, backward)
    else:
        hidden, vocab = rng.choice(HEADS)
        if rng.random() < 0.3:
            vocab -= rng.randint(1, 999)
        backward = kind == "head_distil" and rng.random() < 0.8
        case = _head("", kind, _log_int(rng, 1, 4000), (hidden, vocab), _log_int(rng, 1, 128), temperature, divergence,
                     backward)
    del case["name"]
    return case


# ---- inputs -----------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, v, k = case["tokens"], case["vocab"], case["k"]
    f32 = dict(generator=g, device="cuda", dtype=torch.float32)
    state = {"case": case}
    if case["hidden"]:
        h = case["hidden"]
        # Hidden states in eighths and weights in 512ths, so that every sum of their products is exact in fp32 and the order of
        # the alternatives is the same in whatever order it is summed.  A token's state leans towards its next token's weight.
        weight = _steps(torch.randn(v, h, **f32) * 0.02, 512, 100)
        lean = torch.randint(v, (n,), generator=g, device="cuda")
        strength = torch.rand(n, 1, **f32) * 12.0
        hidden = _steps(torch.randn(n, h, **f32) + strength * weight[lean], 8, 31)
        state["hidden"], state["weight"] = hidden.bfloat16(), weight.bfloat16()
        del weight, hidden
        logits_of = lambda rows: state["hidden"][rows].float() @ _f32(state["weight"]).t()
        if case["backward"]:
            # tokens of the prompt carry no gradient
            state["upstream"] = torch.rand(n, **f32) / n * (torch.arange(n, device="cuda") >= n // 8)
    else:
        dtype = getattr(torch, case["dtype"])
        logits = torch.empty(n, v, device="cuda", dtype=dtype)
        frequency = -1.2 * torch.log1p(torch.arange(v, device="cuda") / 500.0)   # common tokens have low ids
        for rows in _pieces(n):
            m = rows.stop - rows.start
            x = torch.randn(m, v, **f32) * 2.0 + frequency
            x.scatter_add_(1, torch.randint(v, (m, 1), generator=g, device="cuda"), torch.rand(m, 1, **f32) * 24.0)
            logits[rows] = x.to(dtype)
        state["logits"] = logits
        logits_of = lambda rows: state["logits"][rows].float()
        if case["backward"]:
            state["upstream"] = torch.rand(n, **f32) / n
    if case["kind"].endswith("topk"):
        state["labels"] = torch.empty(n, device="cuda", dtype=torch.int64)
        for rows in _pieces(n):   # the token taken: a sample
            x = logits_of(rows) / case["temperature"]
            state["labels"][rows] = (x - torch.rand(x.shape, **f32).clamp_(min=1e-20).log_().neg_().log_()).argmax(1)
        if case["backward"]:
            state["d_entropy"] = torch.full((n,), -0.01 / n, device="cuda")
            state["d_top"] = torch.randn(n, k, **f32) / n
    else:
        # the teacher: the student with its logits disturbed
        state["teacher_logprobs"] = torch.empty(n, k, device="cuda")
        state["teacher_indices"] = torch.empty(n, k, device="cuda", dtype=torch.int64)
        for rows in _pieces(n):
            x = logits_of(rows)
            x = ((x + torch.randn(x.shape, **f32)) / case["temperature"]).log_softmax(1)
            state["teacher_logprobs"][rows], state["teacher_indices"][rows] = x.topk(k, 1)
    return state


def _pieces(n, size=1024):
    return [slice(a, min(n, a + size)) for a in range(0, n, size)]


def _f32(x):
    return x.to(torch.float32)


def _steps(x, per_unit, most):
    return (x * per_unit).round_().clamp_(-most, most) / per_unit


# ---- one pass ---------------------------------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from verl_amd.utils.kernel.linear_topk import linear_topk_distillation, linear_topk_logprobs
    from verl_amd.utils.torch_functional import topk_distillation_from_logits, topk_logprobs_from_logits

    c = s["case"]
    kind, k, temperature, divergence = c["kind"], c["k"], c["temperature"], c["divergence"]
    if kind == "topk":
        logits = s["logits"].detach().requires_grad_(c["backward"])
        lp, entropy, top, index = topk_logprobs_from_logits(logits, s["labels"], k, temperature)
        out = {"logprobs": lp, "entropy": entropy, "top": top, "index": index}
        if c["backward"]:
            out["d_logits"], = torch.autograd.grad((lp, entropy, top), logits, (s["upstream"], s["d_entropy"], s["d_top"]))
        return out
    if kind == "head_topk":
        lp, entropy, top, index = linear_topk_logprobs(s["hidden"], s["weight"], s["labels"], k, temperature)
        return {"logprobs": lp, "entropy": entropy, "top": top, "index": index}
    if kind == "distil":
        logits = s["logits"].detach().requires_grad_(c["backward"])
        loss = topk_distillation_from_logits(logits, s["teacher_logprobs"], s["teacher_indices"], divergence, BETA, temperature)
        out = {"loss": loss}
        if c["backward"]:
            out["d_logits"], = torch.autograd.grad(loss, logits, s["upstream"])
        return out
    hidden, weight = (s[x].detach().requires_grad_(c["backward"]) for x in ("hidden", "weight"))
    loss = linear_topk_distillation(hidden, weight, s["teacher_logprobs"], s["teacher_indices"], divergence, BETA, temperature)
    out = {"loss": loss}
    if c["backward"]:
        out["d_hidden"], out["d_weight"] = torch.autograd.grad(loss, (hidden, weight), s["upstream"])
    return out


def _run_plain(s):
    c = s["case"]
    raw = _f32(s["hidden"]) @ _f32(s["weight"]).t() if c["hidden"] else _f32(s["logits"])
    z = raw / c["temperature"]
    highest = z.amax(1, keepdim=True)
    e = torch.exp(z - highest)
    total = e.sum(1, keepdim=True)
    lse = (highest + torch.log(total))[:, 0]
    q = e / total
    del e
    if c["kind"].endswith("topk"):
        out, d_z = _plain_topk(s, c, raw, z, lse, q)
    else:
        out, d_z = _plain_distil(s, c, z, lse, q)
    if not c["backward"]:
        return out
    d_logits = d_z / c["temperature"]
    if c["hidden"]:
        out["d_hidden"] = (d_logits @ _f32(s["weight"])).to(torch.bfloat16)
        out["d_weight"] = (d_logits.t() @ _f32(s["hidden"])).to(torch.bfloat16)
    else:
        out["d_logits"] = d_logits.to(s["logits"].dtype)
    return out


def _plain_topk(s, c, raw, z, lse, q):
    # one whole number per logit: its order in the high half, the place from the end in the low half, so that none are equal
    bits = (raw + 0.0).view(torch.int32).to(torch.int64)
    order = torch.where(bits < 0, -2147483648 - bits - 1, bits)
    place = torch.arange(raw.shape[1] - 1, -1, -1, device=raw.device)
    index = raw.shape[1] - 1 - (torch.topk(order * 2**32 + place, c["k"], 1).values % 2**32)
    del bits, order
    top = z.gather(1, index) - lse[:, None]
    lp = z.gather(1, s["labels"][:, None])[:, 0] - lse
    mean = (q * z).sum(1)
    out = {"logprobs": lp, "entropy": lse - mean, "top": top, "index": index}
    if not c["backward"]:
        return out, None
    given = s["upstream"] + s["d_top"].sum(1)
    d_z = -q * (given[:, None] + s["d_entropy"][:, None] * (z - mean[:, None]))
    d_z.scatter_add_(1, s["labels"][:, None], s["upstream"][:, None])
    d_z.scatter_add_(1, index, s["d_top"])
    return out, d_z


def _plain_distil(s, c, z, lse, q):
    t, index = s["teacher_logprobs"], s["teacher_indices"]
    log_q = z.gather(1, index) - lse[:, None]
    p, qk = torch.exp(t), torch.exp(log_q)
    if c["divergence"] == "forward_kl":
        terms, slope = p * (t - log_q), -p
    elif c["divergence"] == "reverse_kl":
        terms, slope = qk * (log_q - t), qk * (log_q - t + 1)
    else:
        log_m = torch.log(BETA * p + (1 - BETA) * qk)
        terms = BETA * p * (t - log_m) + (1 - BETA) * qk * (log_q - log_m)
        slope = (1 - BETA) * qk * (log_q - log_m)
    out = {"loss": terms.sum(1)}
    if not c["backward"]:
        return out, None
    slope = slope * s["upstream"][:, None]
    d_z = -q * slope.sum(1, keepdim=True)
    d_z.scatter_add_(1, index, slope)
    return out, d_z


# ---- what a pass cannot do without -------------------------------------------------------------------------------------
def work(case):
    n, v, h, k = case["tokens"], case["vocab"], case["hidden"], case["k"]
    size = 4 if case["dtype"] == "float32" else 2
    per_token = 8 * k + 4 * k + (16 if case["kind"].endswith("topk") else 4) + (4 if case["backward"] else 0)
    if case["backward"] and case["kind"] == "topk":
        per_token += 4 + 4 * k
    matrices = (n * h + v * h if h else n * v) * size
    products = (3 if case["backward"] else 1) * 2 * n * v * h
    return {"bytes": matrices * (2 if case["backward"] else 1) + n * per_token,
            "flops": products + (10 if case["backward"] else 5) * n * v}


# ---- the same from the definition, in 64 bits ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    n, temperature, backward = case["tokens"], case["temperature"], case["backward"]
    wide = {x: s[x].double() for x in ("weight", "upstream", "d_entropy", "d_top", "teacher_logprobs") if x in s}
    outs, d_rows, d_weight = [], [], None
    for rows in _pieces(n, 512):
        raw = s["hidden"][rows].double() @ wide["weight"].t() if case["hidden"] else s["logits"][rows].double()
        z = (raw / temperature).requires_grad_(backward)
        log_q = torch.log_softmax(z, 1)
        if case["kind"].endswith("topk"):
            index = torch.sort(raw, dim=1, descending=True, stable=True).indices[:, :case["k"]]
            found = [log_q.gather(1, s["labels"][rows, None])[:, 0], -(log_q.exp() * log_q).sum(1), log_q.gather(1, index)]
            given = [wide[x][rows] for x in ("upstream", "d_entropy", "d_top")] if backward else None
            piece = dict(zip(("logprobs", "entropy", "top"), found), index=index)
        else:
            found = [_divergence(case["divergence"], wide["teacher_logprobs"][rows], log_q.gather(1, s["teacher_indices"][rows]))]
            given = [wide["upstream"][rows]] if backward else None
            piece = {"loss": found[0]}
        if backward:
            d_logits = torch.autograd.grad(found, z, given)[0] / temperature
            if case["hidden"]:
                d_rows.append(d_logits @ wide["weight"])
                part = d_logits.t() @ s["hidden"][rows].double()
                d_weight = part if d_weight is None else d_weight.add_(part)
            else:
                d_rows.append(d_logits)
        outs.append({name: x.detach() for name, x in piece.items()})
        del raw, z, log_q, found
    out = {name: torch.cat([x[name] for x in outs]) for name in outs[0]}
    if backward:
        out["d_hidden" if case["hidden"] else "d_logits"] = torch.cat(d_rows)
        if case["hidden"]:
            out["d_weight"] = d_weight
    return out


def _divergence(kind, t, log_q):
    if kind == "forward_kl":
        return (t.exp() * (t - log_q)).sum(1)
    if kind == "reverse_kl":
        return (log_q.exp() * (log_q - t)).sum(1)
    log_m = torch.logaddexp(t + math.log(BETA), log_q + math.log(1 - BETA))
    return (BETA * t.exp() * (t - log_m) + (1 - BETA) * log_q.exp() * (log_q - log_m)).sum(1)
