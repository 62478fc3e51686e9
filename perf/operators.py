"""Measured cases of the operators for fine-tuning on packed documents: rotary
positions, attention over packed sequences, and distillation from a teacher's
top logits, each with its gradient.

``own`` selects what :func:`run` computes: the plain forms below (elementary torch
operations in 32 bits, angles in 64) or the framework's operators.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one prompt of a few tokens through a GQA layer: the launch counts
        _rotary("rotary_prompt", tokens=37, hq=28, hk=4, dim=128, rot=128, train=False),
        # a packed batch of 8192 tokens, one training step of one layer
        _rotary("rotary_packed_train", tokens=8192, hq=28, hk=4, dim=128, rot=128, train=True,
                theta=1e6, far=8192),
        # far positions under a stretched context, interleaved pairs, half of each head, odd token count
        _rotary("rotary_long_partial", tokens=65537, hq=16, hk=2, dim=128, rot=64, train=False,
                dtype="fp16", interleaved=True, scaling="yarn", factor=8.0, far=262144),
        # fp32 activations, linear interpolation, 64-wide heads (the small plumbing model)
        _rotary("rotary_fp32_linear", tokens=4099, hq=4, hk=4, dim=64, rot=64, train=True,
                dtype="fp32", scaling="linear", factor=4.0, far=32768),
        # a handful of short chat turns in one row, forward only
        _attention("attention_short_eval", "1,5,37,2,64,19", hq=4, hk=4, dim=64, train=False),
        # an instruction-tuning batch of the 28-head GQA layer: ragged documents, a padded tail
        _attention("attention_packed_gqa", "1999,517,1024,88,1311,640,293,1777,431", hq=28, hk=4,
                   dim=128, train=True, tail=112),
        # whole documents of 1024 tokens and odd ones next to them, no head sharing
        _attention("attention_docs_mha", "1024,1024,1001,1024,777,1024,130", hq=24, hk=24, dim=128,
                   train=True),
        # one long document with a short one behind it
        _attention("attention_long_doc", "8191,1037", hq=8, hk=2, dim=128, train=True),
        # bidirectional scoring of short texts in fp16 with 64-wide heads
        _attention("attention_bidirectional", "300,511,129,64,700,255,401,33", hq=12, hk=12, dim=64,
                   train=False, dtype="fp16", causal=False),
        # the plumbing model's vocabulary, a few rows, distillation alone
        _distill("distill_tiny", rows=61, vocab=1000, k=8, temperature=1.0, alpha=1.0, train=True),
        # a training batch mixed with the hard targets at temperature 2
        _distill("distill_mixed_50k", rows=4096, vocab=50257, k=32, temperature=2.0, alpha=0.5, train=True),
        # the widest vocabulary: the largest logits a step has
        _distill("distill_wide_152k", rows=8192, vocab=152064, k=64, temperature=1.0, alpha=0.7, train=True),
    ]


def _rotary(name, tokens, hq, hk, dim, rot, train, dtype="bf16", theta=10000.0, interleaved=False,
            scaling="none", factor=1.0, far=4096):
    return {"name": name, "op": "rotary", "tokens": tokens, "hq": hq, "hk": hk, "dim": dim, "rot": rot,
            "train": train, "dtype": dtype, "theta": theta, "interleaved": interleaved,
            "scaling": scaling, "factor": factor, "far": far}


def _attention(name, lengths, hq, hk, dim, train, dtype="bf16", causal=True, tail=0):
    return {"name": name, "op": "attention", "lengths": lengths, "hq": hq, "hk": hk, "dim": dim,
            "train": train, "dtype": dtype, "causal": causal, "tail": tail}


def _distill(name, rows, vocab, k, temperature, alpha, train, dtype="bf16"):
    return {"name": name, "op": "distill", "rows": rows, "vocab": vocab, "k": k, "dtype": dtype,
            "temperature": temperature, "alpha": alpha, "train": train}


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "attention", "distill"])
    if op == "rotary":
        dim = rng.choice([64, 80, 128])
        hk = rng.choice([1, 2, 4, 8])
        case = _rotary("", tokens=_spread(rng, 1, 32768), hq=hk * rng.choice([1, 3, 4, 7]), hk=hk, dim=dim,
                       rot=rng.choice([dim, dim, dim // 2]), train=rng.random() < 0.5,
                       dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                       theta=rng.choice([10000.0, 500000.0, 1e6]), interleaved=rng.random() < 0.4,
                       scaling=rng.choice(["none", "linear", "ntk", "yarn"]),
                       factor=rng.choice([2.0, 4.0, 8.0]), far=_spread(rng, 4096, 262144))
        case["tokens"] = min(case["tokens"], (1 << 27) // ((case["hq"] + case["hk"]) * dim))
    elif op == "attention":
        hk = rng.choice([1, 2, 4])
        hq = hk * rng.choice([1, 2, 4, 7])
        causal = rng.random() < 0.75
        # what the plain form can hold: documents x heads x longest x longest scores
        room = 2.0 ** (29 if causal else 28)
        longest = min(_spread(rng, 16, 8191), int(math.sqrt(room / hq)))
        count = max(1, min(64, int(room / (hq * longest * longest)), 32768 // longest))
        count = rng.randint(1, count)
        lengths = [longest] + [rng.randint(1, longest) for _ in range(count - 1)]
        rng.shuffle(lengths)
        case = _attention("", ",".join(map(str, lengths)), hq=hq, hk=hk, dim=rng.choice([64, 80, 128, 128]),
                          train=rng.random() < 0.6, dtype=rng.choice(["bf16", "bf16", "fp16"]),
                          causal=causal, tail=rng.choice([0, 0, rng.randint(1, 130)]))
    else:
        vocab = rng.choice([1000, 1024, 32003, 50257, 152064, _spread(rng, 500, 200000)])
        case = _distill("", rows=min(_spread(rng, 1, 16384), max(1, (1 << 30) // vocab)), vocab=vocab,
                        k=_spread(rng, 1, 256), temperature=rng.choice([1.0, 1.5, 2.0, 4.0]),
                        alpha=rng.choice([1.0, 0.5, 0.3]), train=rng.random() < 0.75,
                        dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    del case["name"]
    return case


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    if case["op"] == "rotary":
        n = case["tokens"] * (case["hq"] + case["hk"])
        passes = 2 if case["train"] else 1          # (x, y), and (dy, dx)
        return {"bytes": passes * 2 * n * case["dim"] * size + 8 * case["tokens"],
                "flops": passes * 3 * n * case["rot"]}
    if case["op"] == "attention":
        lengths = [int(x) for x in case["lengths"].split(",")]
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lengths)
        # two products forward; five backward, the recomputed scores among them
        flops = (14 if case["train"] else 4) * pairs * case["hq"] * case["dim"]
        tokens = sum(lengths) + case["tail"]
        q, kv = tokens * case["hq"] * case["dim"] * size, tokens * case["hk"] * case["dim"] * size
        # q, k, v -> o; and do -> dq, dk, dv
        return {"bytes": 2 * q + 2 * kv + (2 * q + 2 * kv if case["train"] else 0), "flops": flops}
    # the logits once, their gradient once, and the teacher's entries
    logits = case["rows"] * case["vocab"] * size
    return {"bytes": logits * (2 if case["train"] else 1) + case["rows"] * (case["k"] * 8 + 8),
            "flops": case["rows"] * case["vocab"] * (8 if case["train"] else 4)}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, kind=None):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).to(kind or dtype)

    state = {"case": case}
    if case["op"] == "rotary":
        T, hq, hk, D = case["tokens"], case["hq"], case["hk"], case["dim"]
        # q and k are column ranges of one projection's output, as a fused q/k/v product leaves them
        qkv = normal(T, (hq + 2 * hk) * D)
        state["q"] = qkv[:, : hq * D].view(T, hq, D)
        state["k"] = qkv[:, hq * D: (hq + hk) * D].view(T, hk, D)
        # documents that start at random places of the context: rising runs of positions
        start = torch.randint(0, max(1, case["far"] - T), (1,), generator=g, device="cuda")
        state["positions"] = (start + torch.arange(T, device="cuda")) % case["far"]
        if case["train"]:
            state["gq"], state["gk"] = normal(T, hq, D), normal(T, hk, D)
            state["q"].requires_grad_(), state["k"].requires_grad_()
    elif case["op"] == "attention":
        lengths = [int(x) for x in case["lengths"].split(",")]
        T, hq, hk, D = sum(lengths) + case["tail"], case["hq"], case["hk"], case["dim"]
        qkv = normal(T, (hq + 2 * hk) * D)
        state["q"] = qkv[:, : hq * D].view(T, hq, D)
        state["k"] = qkv[:, hq * D: (hq + hk) * D].view(T, hk, D)
        state["v"] = qkv[:, (hq + hk) * D:].view(T, hk, D)
        state["cu_seqlens"] = torch.tensor([0] + lengths, device="cuda").cumsum(0).to(torch.int32)
        if case["train"]:
            state["do"] = normal(T, hq, D)
            state["q"].requires_grad_(), state["k"].requires_grad_(), state["v"].requires_grad_()
    else:
        M, V, K = case["rows"], case["vocab"], case["k"]
        wide = (V + 127) // 128 * 128               # logits rows are padded to whole tiles
        logits = normal(M, wide, std=2.0)
        # distinct ids of a row: a random start and an odd stride that shares no factor with V
        stride = next(s for s in range(7919 % V | 1, 4 * V + 9, 2) if math.gcd(s, V) == 1)
        first = torch.randint(0, V, (M, 1), generator=g, device="cuda")
        ids = (first + stride * torch.arange(min(K, V), device="cuda")) % V
        # a teacher's logits fall off quickly; the student has learnt some of them
        falling = 12.0 - 2.5 * torch.arange(1, ids.shape[1] + 1, device="cuda").float().log()
        teacher = falling + normal(M, ids.shape[1], std=0.7, kind=torch.float32)
        logits.scatter_add_(1, ids, (0.7 * teacher).to(dtype))
        # some rows have fewer entries than K
        short = torch.rand(M, 1, generator=g, device="cuda") < 0.1
        ids = torch.where(short & (torch.arange(ids.shape[1], device="cuda") >= (K + 1) // 2), -1, ids)
        # the targets are mostly the teacher's first entry; prompt tokens are ignored
        targets = torch.where(torch.rand(M, generator=g, device="cuda") < 0.6, first[:, 0],
                              torch.randint(0, V, (M,), generator=g, device="cuda"))
        targets[torch.rand(M, generator=g, device="cuda") < 0.2] = -100
        state.update(logits=logits, ids=ids.to(torch.int32), teacher=teacher, targets=targets)
        if case["train"]:
            state["logits"].requires_grad_()
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return {"rotary": _own_rotary, "attention": _own_attention, "distill": _own_distill}[case["op"]](state, case)
    with torch.no_grad():
        return {"rotary": _plain_rotary, "attention": _plain_attention,
                "distill": _plain_distill}[case["op"]](state, case)


def _own_rotary(state, case):
    from zeroq_b200.ops import RopeScaling, rotary_embedding

    scaling = None
    if case["scaling"] != "none":
        scaling = RopeScaling(case["scaling"], case["factor"], original_max_position=4096)
    q, k = rotary_embedding(state["q"], state["k"], state["positions"], theta=case["theta"],
                            rotary_dim=case["rot"], interleaved=case["interleaved"], scaling=scaling)
    if not case["train"]:
        return q, k
    return (q, k) + torch.autograd.grad((q, k), (state["q"], state["k"]), (state["gq"], state["gk"]))


def _own_attention(state, case):
    from zeroq_b200.ops import flash_attention_varlen

    o = flash_attention_varlen(state["q"], state["k"], state["v"], state["cu_seqlens"], causal=case["causal"])
    if not case["train"]:
        return o
    return (o,) + torch.autograd.grad(o, (state["q"], state["k"], state["v"]), state["do"])


def _own_distill(state, case):
    from zeroq_b200.ops import distillation_loss

    loss = distillation_loss(state["logits"], state["ids"], state["teacher"], state["targets"],
                             temperature=case["temperature"], alpha=case["alpha"], vocab=case["vocab"],
                             reduction="mean" if case["train"] else "none")
    if not case["train"]:
        return loss
    return (loss,) + torch.autograd.grad(loss, state["logits"])


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _frequencies(case, device):
    """(64-bit angle per position of each pair, factor on cos and sin) of a case's scaling."""
    R, theta, s = case["rot"], case["theta"], case["factor"]
    i = torch.arange(R // 2, dtype=torch.float64, device=device)
    if case["scaling"] == "ntk":                     # a larger base: the slowest pair slows by s
        theta = theta * s ** (R / (R - 2)) if R > 2 else theta
    freq = theta ** (-2.0 * i / R)
    if case["scaling"] == "linear":
        return freq / s, 1.0
    if case["scaling"] != "yarn":
        return freq, 1.0
    # pairs that turn more than 32 times within 4096 positions stay, those that turn less
    # than once are interpolated, a ramp over the pair's index lies between
    low = max(0, math.floor(R * math.log(4096 / (32 * 2 * math.pi)) / (2 * math.log(theta))))
    high = min(R - 1, math.ceil(R * math.log(4096 / (1 * 2 * math.pi)) / (2 * math.log(theta))))
    ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
    return freq * (1 - ramp) + freq / s * ramp, 0.1 * math.log(s) + 1.0


def _plain_rotate(x, cos, sin, case):
    R, xf = case["rot"], x.float()
    if case["interleaved"]:
        a, b = xf[..., 0:R:2], xf[..., 1:R:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = xf[..., : R // 2], xf[..., R // 2: R]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, xf[..., R:]], dim=-1).to(x.dtype)


def _plain_rotary(state, case):
    freq, factor = _frequencies(case, state["q"].device)
    angle = state["positions"].double()[:, None, None] * freq
    cos, sin = (angle.cos() * factor).float(), (angle.sin() * factor).float()
    out = (_plain_rotate(state["q"], cos, sin, case), _plain_rotate(state["k"], cos, sin, case))
    if case["train"]:                                # the transposed rotation
        out += (_plain_rotate(state["gq"], cos, -sin, case), _plain_rotate(state["gk"], cos, -sin, case))
    return out


def _plain_attention(state, case):
    q, k, v, cu = state["q"], state["k"], state["v"], state["cu_seqlens"].long()
    T, hq, D = q.shape
    hk = k.shape[1]
    L = max(int(x) for x in case["lengths"].split(","))
    at = torch.arange(L, device=q.device)
    valid = at < (cu[1:] - cu[:-1])[:, None]                      # [documents, L]
    rows = torch.where(valid, cu[:-1, None] + at, T)               # row T: nothing
    share = hq // hk

    def padded(x, heads):
        x = torch.cat([x.float(), x.new_zeros(1, *x.shape[1:], dtype=torch.float32)])[rows].transpose(1, 2)
        return x.repeat_interleave(share, dim=1) if heads != hq else x

    def packed(x):
        out = torch.zeros(T + 1, x.shape[1], D, device=x.device)
        out[rows.reshape(-1)] = x.transpose(1, 2).reshape(-1, x.shape[1], D)
        return out[:T].to(q.dtype)

    scale = 1.0 / math.sqrt(D)
    qp, kp, vp = padded(q, hq), padded(k, hk), padded(v, hk)
    s = (qp * scale) @ kp.transpose(-1, -2)
    seen = valid[:, None, None, :]
    if case["causal"]:
        seen = seen & (at[None, :] <= at[:, None])
    s.masked_fill_(~seen, -math.inf)
    s -= s.amax(-1, keepdim=True)
    p = s.exp_()
    p /= p.sum(-1, keepdim=True)
    o = p @ vp
    if not case["train"]:
        return packed(o)
    do = padded(state["do"], hq)
    delta = (do * o).sum(-1, keepdim=True)
    dv = p.transpose(-1, -2) @ do
    ds = do @ vp.transpose(-1, -2)
    ds -= delta
    ds *= p
    dq = (ds @ kp) * scale
    dk = (ds.transpose(-1, -2) @ qp) * scale
    over = lambda x: x.unflatten(1, (hk, share)).sum(2)  # noqa: E731
    return packed(o), packed(dq), packed(over(dk)), packed(over(dv))


def _plain_distill(state, case):
    V, temp, alpha = case["vocab"], case["temperature"], case["alpha"]
    logits, ids, targets = state["logits"], state["ids"].long(), state["targets"]
    z = logits[:, :V].float()
    counted = ((targets >= 0) & (targets < V)).float()
    n = counted.sum().clamp_min(1.0)
    there = ids >= 0
    at = ids.clamp_min(0)
    t = (state["teacher"].float() / temp).masked_fill(~there, -math.inf)
    t = t - t.amax(-1, keepdim=True)
    p = t.exp()
    mass = p.sum(-1, keepdim=True)
    p = p / mass
    log_p = torch.where(p > 0, t - mass.log(), 0.0)
    high = z.amax(-1, keepdim=True)
    soft = ((z - high) / temp).exp_()
    soft_sum = soft.sum(-1, keepdim=True)
    log_q = (z.gather(1, at) - high) / temp - soft_sum.log()
    kl = (p * (log_p - torch.where(p > 0, log_q, 0.0))).sum(-1)
    hard = (z - high).exp_()
    hard_sum = hard.sum(-1, keepdim=True)
    label = targets.clamp(0, V - 1)[:, None]
    ce = (hard_sum.log() - (z.gather(1, label) - high))[:, 0]
    loss = counted * (alpha * temp * temp * kl + (1.0 - alpha) * ce)
    if not case["train"]:
        return loss
    soft *= alpha * temp / soft_sum
    hard *= (1.0 - alpha) / hard_sum
    soft += hard
    soft.scatter_add_(1, at, -alpha * temp * p)
    soft.scatter_add_(1, label, torch.full_like(counted, alpha - 1.0)[:, None])
    soft *= (counted / n)[:, None]
    grad = torch.zeros_like(logits)
    grad[:, :V] = soft.to(logits.dtype)
    return loss.sum() / n, grad


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
@torch.no_grad()
def exact(case, seed):
    state = prepare(case, seed)
    return {"rotary": _exact_rotary, "attention": _exact_attention, "distill": _exact_distill}[case["op"]](state, case)


def _exact_rotary(state, case):
    """Each pair is one complex number; a position multiplies it by factor · e^(i·angle)."""
    R, s, theta = case["rot"], case["factor"], case["theta"]
    if case["scaling"] == "ntk" and R > 2:
        theta = theta * s ** (R / (R - 2))
    freq = [theta ** (-2.0 * i / R) for i in range(R // 2)]
    factor = 1.0
    if case["scaling"] == "linear":
        freq = [f / s for f in freq]
    elif case["scaling"] == "yarn":
        factor = 0.1 * math.log(s) + 1.0
        turns = lambda n: R * math.log(4096 / (n * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        low, high = max(0, math.floor(turns(32))), min(R - 1, math.ceil(turns(1)))
        keep = [1.0 - min(1.0, max(0.0, (i - low) / max(high - low, 0.001))) for i in range(R // 2)]
        freq = [f * w + f / s * (1.0 - w) for f, w in zip(freq, keep)]
    angle = state["positions"].double()[:, None] * torch.tensor(freq, dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.full_like(angle, factor), angle)[:, None]

    def rotate(x, by):
        out = x.double().clone()
        first, second = (slice(0, R, 2), slice(1, R, 2)) if case["interleaved"] else (slice(0, R // 2), slice(R // 2, R))
        c = torch.complex(out[..., first].contiguous(), out[..., second].contiguous()) * by
        out[..., first], out[..., second] = c.real, c.imag
        return out

    out = [rotate(state["q"], turn), rotate(state["k"], turn)]
    if case["train"]:
        out += [rotate(state["gq"], turn.conj()), rotate(state["gk"], turn.conj())]
    return tuple(out)


def _exact_attention(state, case):
    """Document by document and head by head."""
    q, k, v = (state[n].double() for n in "qkv")
    T, hq, D = q.shape
    share = hq // k.shape[1]
    out = [torch.zeros_like(q)]
    if case["train"]:
        do = state["do"].double()
        out += [torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)]
    begin = 0
    for n in (int(x) for x in case["lengths"].split(",")):
        rows = slice(begin, begin + n)
        begin += n
        hidden = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1) if case["causal"] else None
        for h in range(hq):
            qh, kh, vh = q[rows, h], k[rows, h // share], v[rows, h // share]
            s = qh @ kh.T / math.sqrt(D)
            if hidden is not None:
                s = s.masked_fill(hidden, -math.inf)
            p = torch.softmax(s, -1)
            o = p @ vh
            out[0][rows, h] = o
            if case["train"]:
                g = do[rows, h]
                ds = p * (g @ vh.T - (g * o).sum(-1, keepdim=True)) / math.sqrt(D)
                out[1][rows, h] = ds @ kh
                out[2][rows, h // share] += ds.T @ qh
                out[3][rows, h // share] += p.T @ g
    return tuple(out) if case["train"] else out[0]


def _exact_distill(state, case):
    """Blocks of rows; the teacher's distribution is laid out over the whole vocabulary."""
    V, temp, alpha = case["vocab"], case["temperature"], case["alpha"]
    logits, targets = state["logits"], state["targets"]
    counted = (targets >= 0) & (targets < V)
    n = max(1, int(counted.sum()))
    losses = []
    grad = torch.zeros(logits.shape, dtype=torch.float64, device="cuda") if case["train"] else None
    step = max(1, (1 << 27) // V)
    for r in range(0, logits.shape[0], step):
        rows = slice(r, r + step)
        z = logits[rows, :V].double()
        ids, on = state["ids"][rows].long(), counted[rows].double()
        weights = torch.softmax(state["teacher"][rows].double().div(temp).masked_fill(ids < 0, -math.inf), -1)
        teacher = torch.zeros_like(z).scatter_add_(1, ids.clamp_min(0), weights)
        log_soft, log_hard = torch.log_softmax(z / temp, -1), torch.log_softmax(z, -1)
        kl = torch.special.xlogy(weights, weights).sum(-1) - (teacher * log_soft).sum(-1)
        label = targets[rows].clamp(0, V - 1)[:, None]
        losses.append(on * (alpha * temp ** 2 * kl - (1 - alpha) * log_hard.gather(1, label)[:, 0]))
        if case["train"]:
            d = alpha * temp * (log_soft.exp() - teacher)
            d += (1 - alpha) * log_hard.exp()
            d.scatter_add_(1, label, torch.full_like(on, alpha - 1)[:, None])
            grad[rows, :V] = d * (on / n)[:, None]
    loss = torch.cat(losses)
    return (loss.sum() / n, grad) if case["train"] else loss
