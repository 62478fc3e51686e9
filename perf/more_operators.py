"""Measured cases of the operators at the ends of a training step and between its layers:
embedding lookup with its gradient by sorted tokens, layer norm with its weights'
gradients, activations kept in 8 bits for the backward, and log probabilities of given
tokens with entropy and top alternatives.

``own`` selects what :func:`run` computes: the plain forms below (elementary torch
operations in 32 bits, 8-bit codes in 64) or the framework's operators.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
GROUP = 128            # elements that share a step of 8 bits


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one prompt of a few tokens in the small plumbing model: the launch counts
        _embedding("embedding_prompt", tokens=37, vocab=1000, dim=256, train=False, scale=16.0),
        # a training batch of 8192 tokens against the widest vocabulary
        _embedding("embedding_train_152k", tokens=8192, vocab=152064, dim=3584, train=True, scale=1.0),
        # full training in fp32 over many tokens: padded batch, odd token count, odd width
        _embedding("embedding_train_fp32_odd", tokens=40013, vocab=50257, dim=1001, train=True,
                   dtype="fp32", scale=31.5, padded=1013),
        # a handful of rows in fp32, with gradients: launches
        _norm("norm_tiny", rows=61, dim=256, train=True, dtype="fp32", residual=False, saved="full"),
        # a training batch with the residual stream's addition
        _norm("norm_residual_train", rows=8192, dim=3584, train=True, residual=True, saved="full"),
        # a wide model's norm, its input kept in 8 bits
        _norm("norm_saved_8bit", rows=16384, dim=5120, train=True, residual=False, saved="8bit"),
        # a short ragged input of a checkpointed layer, kept and read back
        _act8("checkpoint_short", kind="checkpoint", rows=333, dim=1000, dtype="fp16"),
        # the input of a checkpointed layer of the 5120-wide model at 16384 tokens
        _act8("checkpoint_wide", kind="checkpoint", rows=16384, dim=5120),
        # the gated activation of one layer, its two inputs kept in 8 bits
        _act8("swiglu_saved_8bit", kind="swiglu", rows=8192, dim=18944),
        # scoring a few tokens of a small vocabulary with their top alternatives
        _logprobs("logprobs_tiny", rows=5, vocab=1000, k=5, train=False),
        # policy training on sampled answers: log probability and entropy, prompts ignored
        _logprobs("logprobs_policy_50k", rows=4096, vocab=50257, k=0, train=True, temperature=0.8,
                  ignored=512),
        # a teacher's entries for distillation at the widest vocabulary, with gradients
        _logprobs("logprobs_wide_152k", rows=8192, vocab=152064, k=32, train=True),
    ]


def _embedding(name, tokens, vocab, dim, train, scale, dtype="bf16", padded=0):
    return {"name": name, "op": "embedding", "tokens": tokens, "vocab": vocab, "dim": dim, "train": train,
            "scale": scale, "dtype": dtype, "padded": padded}


def _norm(name, rows, dim, train, residual, saved, dtype="bf16", bias=True, eps=1e-5):
    return {"name": name, "op": "norm", "rows": rows, "dim": dim, "train": train, "residual": residual,
            "saved": saved, "dtype": dtype, "bias": bias, "eps": eps}


def _act8(name, kind, rows, dim, dtype="bf16"):
    return {"name": name, "op": "act8", "kind": kind, "rows": rows, "dim": dim, "dtype": dtype}


def _logprobs(name, rows, vocab, k, train, temperature=1.0, dtype="bf16", ignored=0):
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "k": k, "train": train,
            "temperature": temperature, "dtype": dtype, "ignored": ignored}


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embedding", "norm", "act8", "logprobs"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "embedding":
        vocab = rng.choice([1000, 1024, 32003, 50257, 152064, _spread(rng, 300, 200000)])
        dim = min(_spread(rng, 64, 8192), (1 << 29) // vocab)
        dim = dim if rng.random() < 0.3 else (dim + 7) // 8 * 8
        tokens = min(_spread(rng, 1, 131072), (1 << 27) // dim)
        case = _embedding("", tokens=tokens, vocab=vocab, dim=dim, train=rng.random() < 0.7, dtype=dtype,
                          scale=rng.choice([1.0, math.sqrt(dim)]),
                          padded=rng.choice([0, 0, rng.randint(0, tokens // 2)]))
    elif op == "norm":
        dim = _spread(rng, 32, 12288)
        dim = dim if rng.random() < 0.3 else (dim + 7) // 8 * 8
        case = _norm("", rows=min(_spread(rng, 1, 131072), (1 << 26) // dim), dim=dim,
                     train=rng.random() < 0.75, residual=rng.random() < 0.5,
                     saved=rng.choice(["full", "8bit"]), dtype=dtype, bias=rng.random() < 0.8,
                     eps=rng.choice([1e-5, 1e-6]))
    elif op == "act8":
        kind = rng.choice(["checkpoint", "gelu", "swiglu"])
        dim = _spread(rng, 32, 32768)
        dim = dim if rng.random() < 0.3 else (dim + 7) // 8 * 8
        case = _act8("", kind=kind, rows=min(_spread(rng, 1, 131072), (1 << 26) // dim), dim=dim, dtype=dtype)
    else:
        vocab = rng.choice([1000, 1024, 32003, 50257, 152064, _spread(rng, 500, 200000)])
        rows = min(_spread(rng, 1, 16384), (1 << 29) // vocab)
        case = _logprobs("", rows=rows, vocab=vocab, k=rng.choice([0, 1, 5, 20, _spread(rng, 1, 128)]),
                         train=rng.random() < 0.6, temperature=rng.choice([1.0, 0.7, 1.3]), dtype=dtype,
                         ignored=rng.choice([0, rng.randint(0, rows // 3)]))
    del case["name"]
    return case


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    if case["op"] == "embedding":
        n = case["tokens"] * case["dim"]
        there = (case["tokens"] - case["padded"]) * case["dim"]
        # rows in, rows out; gradients of the rows in, the weight's gradient out
        back = there * size + case["vocab"] * case["dim"] * size if case["train"] else 0
        return {"bytes": (there + n) * size + 8 * case["tokens"] + back,
                "flops": n + (2 * there if case["train"] else 0)}
    if case["op"] == "norm":
        n = case["rows"] * case["dim"]
        streams = 2 + (2 if case["residual"] else 0)         # x -> y; and delta -> h
        if case["train"]:
            streams += 2 + (1 if case["residual"] else 0)    # dy -> dx; and dh
        return {"bytes": streams * n * size + case["dim"] * 16, "flops": n * (24 if case["train"] else 8)}
    if case["op"] == "act8":
        n = case["rows"] * case["dim"]
        kept = n + 4 * case["rows"] * ((case["dim"] + GROUP - 1) // GROUP)
        if case["kind"] == "checkpoint":                     # x -> kept; kept -> x
            return {"bytes": 2 * n * size + 2 * kept, "flops": 4 * n}
        inputs = 2 if case["kind"] == "swiglu" else 1
        # inputs -> y and kept; dy and kept -> gradients
        return {"bytes": (2 * inputs + 2) * n * size + 2 * inputs * kept, "flops": 40 * n}
    counted = (case["rows"] - case["ignored"]) * case["vocab"]
    # the logits once; their gradient once
    out = case["rows"] * case["vocab"] * size if case["train"] else 0
    return {"bytes": counted * size + out + case["rows"] * (16 + 12 * case["k"]),
            "flops": counted * (14 if case["train"] else 6)}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, kind=None):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).to(kind or dtype)

    state = {"case": case}
    if case["op"] == "embedding":
        T, V, D = case["tokens"], case["vocab"], case["dim"]
        state["weight"] = normal(V, D, std=0.02)
        # a few tokens are most of a text: ranks spread over their logarithm, ids all over the table
        rank = torch.rand(T, generator=g, device="cuda").mul_(math.log(V)).exp_().long().sub_(1).clamp_(0, V - 1)
        stride = next(s for s in range(7919 % V | 1, 4 * V + 9, 2) if math.gcd(s, V) == 1)
        ids = (rank * stride + 11) % V
        ids[T - case["padded"]:] = -100
        state["ids"] = ids
        if case["train"]:
            state["dy"] = normal(T, D)
            state["weight"].requires_grad_()
    elif case["op"] == "norm":
        M, D = case["rows"], case["dim"]
        # a residual stream: rows of various sizes, a few columns much larger than the others
        columns = normal(D, kind=torch.float32).mul_(0.5).exp_()
        columns[torch.randint(0, D, (max(1, D // 500),), generator=g, device="cuda")] *= 20.0
        sizes = normal(M, 1, kind=torch.float32).mul_(0.3).exp_()
        state["x"] = (normal(M, D, kind=torch.float32) * columns * sizes + 0.1).to(dtype)
        if case["residual"]:
            state["delta"] = normal(M, D, std=0.5)
        state["w"] = (1.0 + 0.2 * normal(D, kind=torch.float32))
        state["b"] = 0.1 * normal(D, kind=torch.float32) if case["bias"] else None
        if case["train"]:
            state["dy"] = normal(M, D)
            if case["residual"]:
                state["dh"] = normal(M, D)
            for n in ("x", "delta", "w", "b"):
                if state.get(n) is not None:
                    state[n].requires_grad_()
    elif case["op"] == "act8":
        M, D = case["rows"], case["dim"]
        sizes = normal(M, 1, kind=torch.float32).mul_(0.5).exp_()
        state["x"] = (normal(M, D, kind=torch.float32) * sizes).to(dtype)
        if case["kind"] == "swiglu":
            state["u"] = normal(M, D)
            state["u"].requires_grad_()
        if case["kind"] != "checkpoint":
            state["dy"] = normal(M, D)
            state["x"].requires_grad_()
    else:
        M, V, K = case["rows"], case["vocab"], case["k"]
        wide = (V + 127) // 128 * 128               # logits rows are padded to whole tiles
        logits = normal(M, wide, std=2.0)
        # a trained model: a few candidates stand out in a row, the sampled one is mostly among them
        n = 24
        stride = next(s for s in range(7919 % V | 1, 4 * V + 9, 2) if math.gcd(s, V) == 1)
        first = torch.randint(0, V, (M, 1), generator=g, device="cuda")
        ids = (first + stride * torch.arange(n, device="cuda")) % V
        falling = 13.0 - 3.0 * torch.arange(1, n + 1, device="cuda").float().log()
        logits.scatter_add_(1, ids, (falling + normal(M, n, kind=torch.float32)).to(dtype))
        pick = torch.rand(M, generator=g, device="cuda").pow_(2).mul_(n).long().clamp_(max=n - 1)
        targets = ids.gather(1, pick[:, None])[:, 0]
        targets[: case["ignored"]] = -100           # the prompts' tokens
        state.update(logits=logits, targets=targets)
        if case["train"]:
            state["gp"], state["gh"] = normal(M, kind=torch.float32), normal(M, std=0.01, kind=torch.float32)
            state["gt"] = normal(M, K, std=0.1, kind=torch.float32)
            state["logits"].requires_grad_()
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return {"embedding": _own_embedding, "norm": _own_norm, "act8": _own_act8,
                "logprobs": _own_logprobs}[case["op"]](state, case)
    with torch.no_grad():
        return {"embedding": _plain_embedding, "norm": _plain_norm, "act8": _plain_act8,
                "logprobs": _plain_logprobs}[case["op"]](state, case)


def _own_embedding(state, case):
    from zeroq_b200.ops import embedding

    y = embedding(state["ids"], state["weight"], scale=case["scale"])
    if not case["train"]:
        return y
    return (y,) + torch.autograd.grad(y, state["weight"], state["dy"])


def _own_norm(state, case):
    from zeroq_b200.ops import add_layer_norm, layer_norm

    x, w, b = state["x"], state["w"], state["b"]
    if case["residual"]:
        out = add_layer_norm(x, state["delta"], w, b, eps=case["eps"], saved=case["saved"])
    else:
        out = (layer_norm(x, w, b, eps=case["eps"], saved=case["saved"]),)
    if not case["train"]:
        return out
    leaves = (x, w) + ((b,) if b is not None else ())
    up = (state["dh"], state["dy"]) if case["residual"] else (state["dy"],)
    # (the gradient of delta is the one of x)
    return out + torch.autograd.grad(out, leaves, up)


def _own_act8(state, case):
    from zeroq_b200.ops import dequantize_activation, gelu, quantize_activation, swiglu

    if case["kind"] == "checkpoint":
        return dequantize_activation(quantize_activation(state["x"]))
    if case["kind"] == "gelu":
        y = gelu(state["x"], saved="8bit")
        return (y,) + torch.autograd.grad(y, state["x"], state["dy"])
    y = swiglu(state["x"], state["u"], saved="8bit")
    return (y,) + torch.autograd.grad(y, (state["x"], state["u"]), state["dy"])


def _own_logprobs(state, case):
    from zeroq_b200.ops import token_logprobs

    out = token_logprobs(state["logits"], state["targets"], top_k=case["k"], temperature=case["temperature"],
                         vocab=case["vocab"])
    if not case["train"]:
        return tuple(out)
    values, up = [out.logprobs, out.entropy], [state["gp"], state["gh"]]
    if case["k"]:
        values.append(out.top_logprobs)
        up.append(state["gt"])
    return tuple(out) + torch.autograd.grad(values, state["logits"], up)


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _plain_embedding(state, case):
    ids, w = state["ids"], state["weight"]
    there = (ids >= 0) & (ids < case["vocab"])
    at = torch.where(there, ids, 0)
    y = w[at].float() * case["scale"]
    y = torch.where(there[:, None], y, 0.0).to(w.dtype)
    if not case["train"]:
        return y
    dw = torch.zeros(w.shape, dtype=torch.float32, device=w.device)
    dw.index_add_(0, ids[there], state["dy"][there].float())
    return y, dw.mul_(case["scale"]).to(w.dtype)


def _plain_codes(x):
    """(codes, steps per element) of the rows of x, in groups of 128 columns."""
    M, D = x.shape
    pad = -D % GROUP
    groups = torch.nn.functional.pad(x.float(), (0, pad)).view(M, -1, GROUP)
    a = groups.abs().amax(-1, keepdim=True)
    zero = a < 2.0 ** -119
    a = torch.where(zero, torch.ones_like(a), a)
    inv = torch.full_like(a, 127.0) / a                              # one division, rounded once
    codes = (groups.double() * inv.double()).round_().float().masked_fill_(zero, 0.0)   # ties to even
    step = (a * torch.tensor(1.0 / 127.0, dtype=torch.float32, device=x.device)).masked_fill_(zero, 0.0)
    step = step.expand(groups.shape)
    return codes.view(M, -1)[:, :D], step.reshape(M, -1)[:, :D]


def _plain_kept(x):
    codes, step = _plain_codes(x)
    return codes * step


def _plain_norm(state, case):
    x, w, b = state["x"], state["w"], state["b"]
    h = x
    if case["residual"]:
        h = (x.float() + state["delta"].float()).to(x.dtype)
    hf = h.float()
    mu = hf.mean(-1, keepdim=True)
    r = ((hf - mu).square().mean(-1, keepdim=True) + case["eps"]).rsqrt()
    y = (hf - mu) * r * w
    if b is not None:
        y = y + b
    out = (h, y.to(x.dtype)) if case["residual"] else (y.to(x.dtype),)
    if not case["train"]:
        return out
    xh = ((_plain_kept(h) if case["saved"] == "8bit" else hf) - mu) * r
    dy = state["dy"].float()
    a = dy * w
    dx = r * (a - a.mean(-1, keepdim=True) - xh * (a * xh).mean(-1, keepdim=True))
    if case["residual"]:
        dx = dx + state["dh"].float()
    grads = (dx.to(x.dtype), (dy * xh).sum(0)) + ((dy.sum(0),) if b is not None else ())
    return out + grads


def _plain_act8(state, case):
    x = state["x"]
    if case["kind"] == "checkpoint":
        return _plain_kept(x).to(x.dtype)
    dy = state["dy"].float()
    if case["kind"] == "gelu":
        y = 0.5 * x.float() * (1.0 + torch.erf(x.float() * math.sqrt(0.5)))
        q = _plain_kept(x)
        slope = 0.5 * (1.0 + torch.erf(q * math.sqrt(0.5))) + q * torch.exp(-0.5 * q * q) / math.sqrt(2.0 * math.pi)
        return y.to(x.dtype), (dy * slope).to(x.dtype)
    u = state["u"]
    y = x.float() / (1.0 + torch.exp(-x.float())) * u.float()
    gq, uq = _plain_kept(x), _plain_kept(u)
    s = 1.0 / (1.0 + torch.exp(-gq))
    return y.to(x.dtype), (dy * uq * s * (1.0 + gq * (1.0 - s))).to(x.dtype), (dy * gq * s).to(x.dtype)


def _plain_top(z, k):
    """Ids of the k largest of each row, the lowest id first among equals (blocks of rows)."""
    V = z.shape[1]
    ids = []
    rows = max(1, (1 << 26) // V)
    for r in range(0, z.shape[0], rows):
        bits = (z[r: r + rows] + 0.0).view(torch.int32)              # -0 is 0
        bits = bits ^ ((bits >> 31) & 0x7FFFFFFF)                    # whole numbers in the values' order
        key = (bits.long() << 31) + (V - torch.arange(V, device=z.device))
        ids.append(key.topk(k, -1).indices)
    return torch.cat(ids)


def _plain_logprobs(state, case):
    V, K, T = case["vocab"], case["k"], case["temperature"]
    logits, targets = state["logits"], state["targets"]
    z = logits[:, :V].float()
    counted = (targets >= 0) & (targets < V)
    on = counted.float()
    ids = _plain_top(z, K) if K else torch.empty(len(z), 0, dtype=torch.long, device=z.device)
    high = z.amax(-1, keepdim=True)
    t = (z - high) / T
    e = t.exp()
    total = e.sum(-1, keepdim=True)
    log_total = total.log()
    e /= total                                                        # p
    t -= log_total                                                    # log p
    entropy = -(e * t).sum(-1, keepdim=True)
    label = torch.where(counted, targets, 0)[:, None]
    logp = t.gather(1, label)[:, 0] * on
    top = t.gather(1, ids) * on[:, None]
    out = (logp, entropy[:, 0] * on, top, torch.where(counted[:, None], ids, -1))
    if not case["train"]:
        return out
    gp, gh, gt = state["gp"], state["gh"][:, None], state["gt"]
    t += entropy
    t *= -gh
    t -= (gp + gt.sum(-1))[:, None]
    t *= e
    t.scatter_add_(1, label, gp[:, None])
    t.scatter_add_(1, ids, gt)
    t *= (on / T)[:, None]
    grad = torch.zeros_like(logits)
    grad[:, :V] = t.to(logits.dtype)
    return out + (grad,)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
@torch.no_grad()
def exact(case, seed):
    state = prepare(case, seed)
    return {"embedding": _exact_embedding, "norm": _exact_norm, "act8": _exact_act8,
            "logprobs": _exact_logprobs}[case["op"]](state, case)


def _exact_embedding(state, case):
    """The gradient over the ids that occur alone, laid out over the whole table at the end."""
    ids, w, s = state["ids"], state["weight"], case["scale"]
    real = torch.nonzero((ids >= 0) & (ids < case["vocab"]))[:, 0]
    y = torch.zeros(len(ids), case["dim"], dtype=torch.float64, device="cuda")
    y[real] = w.index_select(0, ids[real]).double() * s
    if not case["train"]:
        return y
    dw = torch.zeros(w.shape, dtype=torch.float64, device="cuda")
    kinds, where = torch.unique(ids[real], return_inverse=True)
    sums = torch.zeros(len(kinds), case["dim"], dtype=torch.float64, device="cuda")
    step = max(1, (1 << 26) // case["dim"])
    for r in range(0, len(real), step):
        sums.index_put_((where[r: r + step],), state["dy"][real[r: r + step]].double(), accumulate=True)
    dw[kinds] = sums * s
    return y, dw


def _exact_kept(x):
    """Column ranges of a group, one after another.  The step and its reciprocal are 32-bit numbers."""
    out = torch.empty(x.shape, dtype=torch.float64, device="cuda")
    for c in range(0, x.shape[1], GROUP):
        v = x[:, c: c + GROUP].double()
        a = v.abs().max(-1, keepdim=True).values
        tiny = a < 2.0 ** -119
        inv = (torch.full_like(a, 127.0) / a).float().double()
        step = (a * float(torch.tensor(1.0 / 127.0, dtype=torch.float32))).float().double()
        out[:, c: c + GROUP] = torch.where(tiny, 0.0, torch.round(v * inv) * step)
    return out


def _exact_norm(state, case):
    x, D = state["x"].double(), case["dim"]
    if case["residual"]:
        x = (x + state["delta"].double()).to(state["x"].dtype).double()
    var, mean = torch.var_mean(x, -1, keepdim=True, correction=0)
    sd = torch.sqrt(var + case["eps"])
    w = state["w"].double()
    y = torch.addcmul(torch.zeros_like(w) if state["b"] is None else state["b"].double(), (x - mean) / sd, w)
    out = (x, y) if case["residual"] else (y,)
    if not case["train"]:
        return out
    if case["saved"] == "8bit":
        rounded = (state["x"] if not case["residual"] else x.to(state["x"].dtype))
        x = _exact_kept(rounded)
    n = (x - mean) / sd
    dy = state["dy"].double()
    a = dy * w
    dx = (D * a - a.sum(-1, keepdim=True) - n * torch.einsum("md,md->m", a, n)[:, None]) / (D * sd)
    if case["residual"]:
        dx += state["dh"].double()
    grads = (dx, torch.einsum("md,md->d", dy, n))
    return out + grads + ((dy.sum(0),) if state["b"] is not None else ())


def _exact_act8(state, case):
    if case["kind"] == "checkpoint":
        return _exact_kept(state["x"])
    x, dy = state["x"].double(), state["dy"].double()
    if case["kind"] == "gelu":
        cdf = lambda v: torch.special.ndtr(v)  # noqa: E731
        q = _exact_kept(state["x"])
        return x * cdf(x), dy * (cdf(q) + q * torch.exp(-q * q / 2) / math.sqrt(2 * math.pi))
    q, u = _exact_kept(state["x"]), _exact_kept(state["u"])
    s = torch.sigmoid(q)
    return (x * torch.sigmoid(x) * state["u"].double(), dy * u * (s + q * s * torch.sigmoid(-q)), dy * q * s)


def _exact_logprobs(state, case):
    """Blocks of rows; the top alternatives by a stable sort."""
    V, K, T = case["vocab"], case["k"], case["temperature"]
    logits, targets = state["logits"], state["targets"]
    M = logits.shape[0]
    logp, entropy = (torch.zeros(M, dtype=torch.float64, device="cuda") for _ in range(2))
    top = torch.zeros(M, K, dtype=torch.float64, device="cuda")
    ids = torch.full((M, K), -1, dtype=torch.long, device="cuda")
    grad = torch.zeros(logits.shape, dtype=torch.float64, device="cuda") if case["train"] else None
    rows = torch.nonzero((targets >= 0) & (targets < V))[:, 0]
    for r in rows.split(max(1, (1 << 26) // V)):
        z = logits[r, :V].double()
        lp = torch.log_softmax(z / T, -1)
        p = lp.exp()
        y = targets[r][:, None]
        logp[r] = lp.gather(1, y)[:, 0]
        h = -(p * lp).sum(-1)
        entropy[r] = h
        best = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :K] if K else y[:, :0]
        ids[r], top[r] = best, lp.gather(1, best)
        if grad is not None:
            gp, gh, gt = (state[n][r].double() for n in ("gp", "gh", "gt"))
            d = -p * ((gp + gt.sum(-1))[:, None] + gh[:, None] * (lp + h[:, None]))
            d.scatter_add_(1, y, gp[:, None])
            d.scatter_add_(1, best, gt)
            grad[r, :V] = d / T
    return (logp, entropy, top, ids) + ((grad,) if grad is not None else ())
