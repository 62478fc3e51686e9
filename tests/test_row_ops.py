"""embedding, layer_norm, 8-bit activations and token_logprobs against their formulas in 64
bits, on the CPU and on the GPU.

Tolerances: an output is rounded once to its type (half a step relative to the value; below
fp16's normal range half a step is 2^-25), next to the 32-bit error in front of it, which
each oracle bounds from the sizes of the terms: u = 2^-24 is one 32-bit rounding."""

import math

import pytest
import torch

from zeroq_b200.ops import (Activation8, add_layer_norm, dequantize_activation, embedding, gelu, layer_norm,
                            quantize_activation, swiglu, token_logprobs)

U = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float16, torch.float32]
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.fixture(params=DEVICES)
def device(request):
    if request.param == "cuda":
        request.getfixturevalue("cuda")
    return request.param


def near(got, want, more):
    """half a step of got's type, and `more`"""
    want = want.double().cpu()
    tol = torch.finfo(got.dtype).eps / 2 * want.abs() + more.double().cpu()
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    assert got.shape == want.shape
    beyond = want.abs() > torch.finfo(got.dtype).max * (1 + torch.finfo(got.dtype).eps)   # of the type's range
    got = got.detach().double().cpu()
    assert (got.isinf() & (got.sign() == want.sign()))[beyond].all()
    off = torch.where(beyond, 0.0, (got - want).abs())
    assert (off <= tol).all(), (float((off - tol).max()), int((off > tol).sum()))


def randn(*shape, seed=0, dtype=torch.float32, device="cpu"):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(device=device, dtype=dtype)


# ---------------------------------------------------------------------------
# embedding
# ---------------------------------------------------------------------------
def embedding_case(device, T, V, D, dtype, scale, ids=None, idtype=torch.int64, shape=None, strided=False):
    w = randn(V, 2 * D if strided else D, seed=T + D, dtype=dtype, device=device)[:, :D].requires_grad_()
    if ids is None:
        ids = torch.randint(-2, V + 2, (T,), generator=torch.Generator().manual_seed(T))
    ids = ids.to(device=device, dtype=idtype)
    y = embedding(ids.view(shape) if shape else ids, w, scale)
    i = ids.cpu().long()
    there = (i >= 0) & (i < V)
    W = w.detach().double().cpu()
    want = torch.where(there[:, None], W[i.clamp(0, V - 1)] * scale, 0.0)
    assert y.dtype == dtype and y.shape == ((*shape, D) if shape else (T, D))
    near(y.view(T, D), want, 4 * U * want.abs())
    assert (y.view(T, D)[~there.to(device)] == 0).all()
    dy = randn(T, D, seed=T + 1, dtype=dtype, device=device)
    (dw,) = torch.autograd.grad(y, w, dy.view(y.shape))
    g = dy.double().cpu()
    want, size = (torch.zeros(V, D, dtype=torch.float64).index_add_(0, i[there], x[there]) * abs(scale)
                  for x in (g, g.abs()))
    count = torch.zeros(V, dtype=torch.float64).index_add_(0, i[there], torch.ones(int(there.sum()), dtype=torch.float64))
    near(dw, want * math.copysign(1.0, scale), (count[:, None] + 4) * U * size)
    (again,) = torch.autograd.grad(embedding(ids, w, scale), w, dy)
    assert torch.equal(dw, again)
    return dw


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V,D", [(1, 1, 1), (1, 300, 256), (31, 5, 8), (33, 257, 264), (64, 1, 100), (200, 70000, 24),
                                   (1000, 255, 129)])
def test_embedding(device, T, V, D, dtype):
    embedding_case(device, T, V, D, dtype, 1.0 if T % 2 else -11.3)


@pytest.mark.gpu
@pytest.mark.parametrize("T,V,D", [(8191, 3, 40), (8192, 50257, 264), (8193, 65536, 72), (20011, 256, 33), (40000, 1000, 16),
                                   (100003, 1 << 17, 8)])
def test_embedding_long(cuda, T, V, D):
    embedding_case("cuda", T, V, D, torch.bfloat16, 2.0)


@pytest.mark.gpu
def test_embedding_one_id_only(cuda):
    """the longest run: every token is the same; with one other in the middle, and none at all"""
    for T in (32, 33, 64, 5000, 20000):
        ids = torch.full((T,), 7)
        embedding_case("cuda", T, 9, 300, torch.float32, 0.5, ids=ids)
        ids[T // 2] = 3
        embedding_case("cuda", T, 9, 300, torch.bfloat16, 1.0, ids=ids)
    assert (embedding_case("cuda", 100, 9, 300, torch.float16, 1.0, ids=torch.full((100,), -100)) == 0).all()


def test_embedding_shapes_and_strides(device):
    embedding_case(device, 24, 50, 40, torch.bfloat16, 3.0, idtype=torch.int32, shape=(2, 3, 4))
    embedding_case(device, 24, 50, 40, torch.float32, 3.0, strided=True)
    w = randn(10, 16, device=device, dtype=torch.bfloat16).requires_grad_()
    ids = torch.arange(10, device=device)
    y = embedding(ids, w)
    (dw,) = torch.autograd.grad(y, w, torch.ones(1, 1, device=device, dtype=w.dtype).expand(10, 16))   # strides of 0
    assert (dw == 1).all()
    assert embedding(ids[:0], w).shape == (0, 16)
    base = randn(10, 17, device=device, dtype=torch.bfloat16)
    odd = base[:, 1:]                                  # rows that start anywhere
    assert torch.equal(embedding(ids, odd), odd)
    wt = randn(16, 10, device=device).t()              # columns apart
    assert torch.equal(embedding(ids, wt), wt)


def test_embedding_refusals(device):
    w = randn(4, 8, device=device)
    ids = torch.zeros(3, dtype=torch.int64, device=device)
    with pytest.raises(TypeError, match="int32 or int64"):
        embedding(ids.float(), w)
    with pytest.raises(ValueError, match=r"\[V, D\]"):
        embedding(ids, w[0])
    with pytest.raises(ValueError, match="weight"):
        embedding(ids, w.long())
    with pytest.raises(TypeError):
        embedding([0, 1], w)
    x = w.clone().requires_grad_()
    if device == "cuda":
        with pytest.raises(ValueError, match="on cpu"):
            embedding(ids.cpu(), w)
        y = embedding(ids, x)
        with pytest.raises(RuntimeError, match="not differentiable"):
            torch.autograd.grad(y.sum(), x, create_graph=True)


# ---------------------------------------------------------------------------
# 8 bits
# ---------------------------------------------------------------------------
def kept64(x):
    """what 8 bits hold of x: the rounded product in 64 bits, the step in 32"""
    x = x.detach().cpu()
    D = x.shape[-1]
    out = torch.empty(x.shape, dtype=torch.float64)
    for c in range(0, D, 128):
        v = x[..., c:c + 128].double()
        a = v.abs().amax(-1, keepdim=True)
        f = a.float()
        inv = (torch.full_like(f, 127.0) / f).double()
        step = (f * torch.tensor(1.0 / 127.0)).double()
        q = torch.round(v * inv) * step
        q = torch.where(a < 2.0 ** -119, torch.zeros_like(q), q)
        out[..., c:c + 128] = torch.where(torch.isfinite(a), q, torch.full_like(q, float("nan")))
    return out


SHAPES = [(1, 1), (1, 127), (3, 128), (2, 129), (5, 200), (7, 256), (3, 1000), (4, 2049), (33, 640)]


def columns(M, D, dtype, device, seed=0):
    """rows of many sizes, some columns far larger"""
    x = randn(M, D, seed=seed) * torch.exp(1.5 * randn(M, 1, seed=seed + 1))   # (within fp16's range)
    x[:, :: 37] *= 30.0
    return x.to(device=device, dtype=dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,D", SHAPES)
def test_kept_values(device, M, D, dtype):
    x = columns(M, D, dtype, device)
    kept = quantize_activation(x)
    y = dequantize_activation(kept)
    assert y.dtype == dtype and y.shape == x.shape
    near(y, kept64(x), U * kept64(x).abs())            # (code * step is rounded to 32 bits, then to the type)
    assert kept.nbytes == M * ((D + 15) // 16 * 16) + 4 * M * ((D + 127) // 128)
    # codes themselves, to the unit
    a = torch.nn.functional.pad(x.float().cpu(), (0, -D % 128)).view(M, -1, 128)
    inv = (torch.full((M, a.shape[1], 1), 127.0) / a.abs().amax(-1, keepdim=True).clamp_min(1e-30)).double()
    codes = torch.round(a.double() * inv).view(M, -1)[:, :D]
    assert torch.equal(kept.codes[:, :D].cpu().double(), codes)
    # and no further off than half a step of the group's largest
    off = torch.nn.functional.pad((y.double() - x.double()).abs().cpu(), (0, -D % 128)).view(M, -1, 128)
    top = a.double().abs().amax(-1, keepdim=True)
    assert (off <= top / 254 * (1 + 2.0 ** -20) + torch.finfo(dtype).eps / 2 * top + 2.0 ** -25).all()


def test_kept_ties_and_extremes(device):
    # multiples of half a step: ties go to the even code
    half = (torch.arange(128) - 64.0) / 2 * 2.0
    x = torch.cat([half * 2, torch.tensor([254.0]), torch.zeros(127)])[None].to(device)
    x[0, 127] = 254.0
    assert torch.equal(dequantize_activation(quantize_activation(x)).cpu(), kept64(x).float())
    for v in (0.0, -0.0, 1e-38, 2.0 ** -119, 2.0 ** -120, 3.3e38, 1e-45):
        x = torch.full((2, 130), v, device=device)
        y = dequantize_activation(quantize_activation(x))
        assert torch.equal(y.cpu(), kept64(x).float()), v
    for bad in (float("nan"), float("inf"), float("-inf")):
        x = torch.ones(2, 300, device=device)
        x[0, 130] = bad
        y = dequantize_activation(quantize_activation(x))
        assert y[0, 128:256].isnan().all() and not y[0, :128].isnan().any() and not y[0, 256:].isnan().any()
        assert not y[1].isnan().any()


def test_kept_shapes_and_strides(device):
    x = randn(2, 3, 4, 200, device=device)
    assert torch.equal(dequantize_activation(quantize_activation(x)).cpu(), kept64(x).float())
    for v in (x[..., 1:190], x.transpose(0, 2), x[..., ::2], x[:, :1].expand(2, 5, 4, 200), x[:0], x[..., :0],
              randn(40, device=device)):
        assert torch.equal(dequantize_activation(quantize_activation(v)).cpu(), kept64(v).float())


def test_kept_refusals(device):
    x = randn(4, 40, device=device)
    for bad in (x.long(), x.double(), [1.0]):
        with pytest.raises(TypeError, match="quantize_activation"):
            quantize_activation(bad)
    with pytest.raises(ValueError, match="single number"):
        quantize_activation(x[0, 0])
    with pytest.raises(TypeError):
        dequantize_activation(x)
    k = quantize_activation(x)
    for bad in (Activation8(k.codes[:2], k.steps, k.shape, k.dtype), Activation8(k.codes, k.steps[:, :0], k.shape, k.dtype),
                Activation8(k.codes, k.steps, (4, 80), k.dtype), Activation8(k.codes.int(), k.steps, k.shape, k.dtype)):
        with pytest.raises(ValueError, match="do not belong"):
            dequantize_activation(bad)
    for f in (lambda s: gelu(x, saved=s), lambda s: swiglu(x, x, saved=s), lambda s: layer_norm(x, saved=s)):
        with pytest.raises(ValueError, match="'full' or '8bit'"):
            f("4bit")
    with pytest.raises(ValueError, match="one shape"):
        swiglu(x, x[:, :20], saved="8bit")
    with pytest.raises(TypeError, match="bf16, fp16 or fp32"):
        gelu(x.double(), saved="8bit")


# 16-bit kernels take a cdf that is off by at most 1e-6 and fast exponentials: 2 + 1.173 |x|
# units in the last place, 2^-18 up to |x| = 20 with the quotient's
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,D", SHAPES)
def test_gelu_kept(device, M, D, dtype):
    x = (2.0 * randn(M, D, seed=D)).to(device=device, dtype=dtype).requires_grad_()
    y = gelu(x, saved="8bit")
    v = x.detach().double().cpu()
    near(y, v * torch.special.ndtr(v), 1e-6 * v.abs())
    dy = randn(M, D, seed=D + 1, dtype=dtype, device=device)
    (dx,) = torch.autograd.grad(y, x, dy)
    q, g = kept64(x), dy.double().cpu()
    slope = torch.special.ndtr(q) + q * torch.exp(-q * q / 2) / math.sqrt(2 * math.pi)
    near(dx, g * slope, 4e-6 * g.abs())
    if dtype == torch.bfloat16 and x.numel() % 8 == 0:
        assert torch.equal(y, gelu(x))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,D", SHAPES)
def test_swiglu_kept(device, M, D, dtype):
    a = (3.0 * randn(M, D, seed=D)).to(device=device, dtype=dtype).requires_grad_()
    b = randn(M, D, seed=D + 1, dtype=dtype, device=device).requires_grad_()
    y = swiglu(a, b, saved="8bit")
    A, B = a.detach().double().cpu(), b.detach().double().cpu()
    want = A * torch.sigmoid(A) * B
    near(y, want, 2.0 ** -17 * want.abs())
    dy = randn(M, D, seed=D + 2, dtype=dtype, device=device)
    da, db = torch.autograd.grad(y, (a, b), dy)
    q, u, g = kept64(a), kept64(b), dy.double().cpu()
    s = torch.sigmoid(q)
    near(db, g * q * s, 2.0 ** -17 * (g * q * s).abs())
    near(da, g * u * s * (1 + q * (1 - s)), 2.0 ** -16 * (g * u).abs() * s * (1 + q.abs() * (1 - s)))
    if dtype == torch.bfloat16 and a.numel() % 8 == 0:
        assert torch.equal(y, swiglu(a, b))


def test_kept_activations_of_strided_inputs(device):
    both = randn(6, 400, seed=3, device=device, dtype=torch.bfloat16).requires_grad_()
    y = swiglu(both[:, :200], both[:, 200:], saved="8bit")     # two halves of one projection
    y.backward(torch.ones((), device=device, dtype=y.dtype).expand_as(y))
    a = both.detach()[:, :200].contiguous().requires_grad_()
    b = both.detach()[:, 200:].contiguous().requires_grad_()
    z = swiglu(a, b, saved="8bit")
    z.sum().backward()
    assert torch.equal(y, z) and torch.equal(both.grad, torch.cat([a.grad, b.grad], -1))
    with torch.no_grad():
        assert torch.equal(swiglu(a, b, saved="8bit"), swiglu(a, b))


# ---------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------
def norm_case(device, M, D, dtype, wtype=torch.float32, bias=True, weight=True, residual=False, saved="full", eps=1e-5,
              x=None):
    x = columns(M, D, dtype, device, seed=D) + 0.5 if x is None else x
    x = x.to(dtype).detach().requires_grad_()
    delta = randn(M, D, seed=7, dtype=dtype, device=device).requires_grad_() if residual else None
    w = (1 + 0.3 * randn(D, seed=8)).to(device=device, dtype=wtype).requires_grad_() if weight else None
    b = randn(D, seed=9, dtype=wtype, device=device).requires_grad_() if bias else None
    h, y = add_layer_norm(x, delta, w, b, eps=eps, saved=saved)
    X = x.detach().double().cpu()
    if residual:
        H = X + delta.detach().double().cpu()
        near(h, H, U * H.abs())
        X = h.detach().double().cpu()
    else:
        assert h is x
    W = torch.ones(D, dtype=torch.float64) if w is None else w.detach().double().cpu()
    B = torch.zeros(D, dtype=torch.float64) if b is None else b.detach().double().cpu()
    mu = X.mean(-1, keepdim=True)
    r = (X.var(-1, unbiased=False, keepdim=True) + eps).rsqrt()
    n = (X - mu) * r
    # sums of at most 128 roundings: the mean is off by 2^-17 of the mean size, r by 2^-17 of itself
    dn = 2.0 ** -17 * (r * X.abs().mean(-1, keepdim=True) + n.abs())
    near(y, n * W + B, W.abs() * dn + 4 * U * ((n * W).abs() + B.abs()))
    dy = randn(M, D, seed=10, dtype=dtype, device=device)
    dh = randn(M, D, seed=11, dtype=dtype, device=device) if residual else None
    outs, ups = ((h, y), (dh, dy)) if residual else ((y,), (dy,))
    leaves = [t for t in (x, delta, w, b) if t is not None]
    grads = list(torch.autograd.grad(outs, leaves, ups))
    if saved == "8bit":
        n = (kept64(h) - mu) * r
        dn = dn + 2.0 ** -17 * n.abs()
    g = dy.double().cpu()
    a = g * W
    m1, m2 = a.mean(-1, keepdim=True), (a * n).mean(-1, keepdim=True)
    want = r * (a - m1 - n * m2)
    s1, s2 = a.abs().mean(-1, keepdim=True), (a * n).abs().mean(-1, keepdim=True)
    more = 2.0 ** -16 * r * (a.abs() + s1 + n.abs() * s2)
    more = more + r * (dn * m2.abs() + n.abs() * (a.abs() * dn).mean(-1, keepdim=True)) + 2.0 ** -17 * want.abs()
    if residual:
        want = want + dh.double().cpu()
        more = more + 2 * U * want.abs()
    near(grads.pop(0), want, more)
    if residual:
        near(grads.pop(0), want, more)
    if weight:
        near(grads.pop(0), (g * n).sum(0), (g.abs() * dn).sum(0) + (M + 4) * U * (g * n).abs().sum(0))
    if bias:
        near(grads.pop(0), g.sum(0), (M + 4) * U * g.abs().sum(0))
    runs = [torch.autograd.grad(add_layer_norm(x, delta, w, b, eps=eps, saved=saved) if residual
                                else layer_norm(x, w, b, eps, saved), leaves, ups) for _ in range(2)]
    assert all(torch.equal(p, q) for p, q in zip(*runs))


NORMS = [(1, 1), (1, 8), (3, 33), (61, 256), (9, 257), (300, 512), (5, 1000), (17, 1001), (4, 2056), (3, 4096), (2, 5120)]


@pytest.mark.parametrize("residual,saved", [(False, "full"), (True, "full"), (False, "8bit"), (True, "8bit")])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,D", NORMS)
def test_layer_norm(device, M, D, dtype, residual, saved):
    norm_case(device, M, D, dtype, residual=residual, saved=saved)


@pytest.mark.gpu
@pytest.mark.parametrize("residual,saved", [(False, "full"), (True, "8bit")])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,D", [(2000, 640), (3000, 72), (700, 3584), (500, 8192), (3, 8200), (5, 12289), (2, 16384)])
def test_layer_norm_sizes(cuda, M, D, dtype, residual, saved):
    norm_case("cuda", M, D, dtype, residual=residual, saved=saved)


def test_layer_norm_parameters(device):
    for wtype in TYPES:
        norm_case(device, 40, 72, torch.bfloat16, wtype=wtype)
    norm_case(device, 40, 72, torch.float16, bias=False)
    norm_case(device, 40, 72, torch.float16, weight=False)
    norm_case(device, 40, 72, torch.float32, weight=False, bias=False, eps=1e-3, residual=True)


def test_layer_norm_far_from_zero(device):
    """the variance of rows with a large mean does not cancel"""
    norm_case(device, 12, 520, torch.float32, x=1000.0 + randn(12, 520, device=device))
    norm_case(device, 3, 4100, torch.float32, x=-3e5 + randn(3, 4100, device=device))
    norm_case(device, 2, 300, torch.bfloat16, x=torch.full((2, 300), 3.0, device=device), bias=False)   # no variance


def test_layer_norm_of_rows_with_nan(device):
    x = randn(3, 300, device=device)
    x[1, 5] = float("nan")
    x[2, 7] = float("inf")
    y = layer_norm(x)
    assert not y[0].isnan().any() and y[1].isnan().all() and y[2].isnan().any()


def test_layer_norm_gradients_alone(device):
    """one output's gradient alone, inputs of which some take none, strides of 0"""
    x, d = randn(5, 96, device=device).requires_grad_(), randn(5, 96, seed=1, device=device)
    w = torch.ones(96, device=device)
    h, y = add_layer_norm(x, d, w)
    (g,) = torch.autograd.grad(h, x, torch.ones_like(h), retain_graph=True)
    assert (g == 1).all()
    (g,) = torch.autograd.grad(y.sum(), x)           # a row's sum does not change
    assert g.abs().max() < 1e-4
    w.requires_grad_()
    (gw,) = torch.autograd.grad(layer_norm(x.detach(), w).sum(), w)
    assert torch.allclose(gw, layer_norm(x.detach()).sum(0), atol=1e-5)
    v = randn(4, 6, 200, device=device, dtype=torch.bfloat16)
    for z in (v[..., 1:150], v.transpose(0, 1), v[..., ::2], v[:, :1].expand(4, 3, 200)):
        assert torch.equal(layer_norm(z), layer_norm(z.contiguous()))
    assert layer_norm(v[:0]).shape == (0, 6, 200)
    one, w = randn(40, device=device).requires_grad_(), torch.ones(40, device=device, requires_grad=True)
    for saved in ("full", "8bit"):
        gx, gw = torch.autograd.grad(layer_norm(one, w, saved=saved), (one, w), torch.ones(40, device=device))
        assert gx.shape == (40,) and gw.shape == (40,)
    h, y = add_layer_norm(v[:, :, :0], v[:, :, :0])
    assert y.shape == (4, 6, 0)


def test_layer_norm_refusals(device):
    x, w = randn(3, 16, device=device), randn(16, device=device)
    with pytest.raises(ValueError, match="weight must be"):
        layer_norm(x, w[:8])
    with pytest.raises(ValueError, match="bias must be"):
        layer_norm(x, w, w.long())
    with pytest.raises(TypeError, match="one type"):
        layer_norm(x, w, w.bfloat16())
    with pytest.raises(ValueError, match="delta"):
        add_layer_norm(x, x.half(), w)
    with pytest.raises(ValueError, match="floating-point"):
        layer_norm(x.long())
    with pytest.raises(TypeError, match="8 bits"):
        layer_norm(x.double(), saved="8bit")
    if device == "cuda":
        with pytest.raises(ValueError, match="at most 16384"):
            layer_norm(randn(1, 16392, device=device))
        y = layer_norm(x.requires_grad_())
        with pytest.raises(RuntimeError, match="not differentiable"):
            torch.autograd.grad(y.sum(), x, create_graph=True)


def test_layer_norm_against_differences():
    x, w, b = randn(3, 10).double(), randn(10, seed=1).double(), randn(10, seed=2).double()
    for t in (x, w, b):
        t.requires_grad_()
    assert torch.autograd.gradcheck(lambda *a: layer_norm(*a), (x, w, b))


# ---------------------------------------------------------------------------
# token log probabilities
# ---------------------------------------------------------------------------
def logprob_case(device, z, vocab=None, k=0, temperature=1.0, targets="some", ignore=-100, want=("p", "h", "t")):
    z = z.detach().requires_grad_()
    M, V = z.shape[0], z.shape[1] if vocab is None else vocab
    gen = torch.Generator().manual_seed(M + V)
    if isinstance(targets, str):
        targets = torch.randint(0, V, (M,), generator=gen)
        targets[torch.rand(M, generator=gen) < 0.2] = ignore
        targets = targets.to(z.device)
    out = token_logprobs(z, targets, top_k=k, temperature=temperature, vocab=vocab, ignore_index=ignore)
    Z = z.detach()[:, :V].double().cpu()
    counted = (Z > -math.inf).any(-1)
    Y = torch.zeros(M, dtype=torch.int64)
    if targets is not None:
        Y = targets.long().cpu()
        counted &= (Y != ignore) & (Y >= 0) & (Y < V)
        Y = torch.where(counted, Y, 0)
    Z = torch.where(counted[:, None], Z, 0.0)
    high = Z.amax(-1, keepdim=True)
    l = torch.log_softmax((Z - high) / temperature, -1)
    p = l.exp()
    pl = torch.where(p > 0, p * l, 0.0)
    H = -pl.sum(-1)
    # S: V / 256 sums in a row and their joins, 2^-22 an exponential and its argument's error,
    # 3 u |t| with |t| 2^t < 1; the same for A, in units of the sum of p |t|
    es = (V / 256 + 64) * U
    spread = (torch.where(p > 0, p * ((Z - high) / temperature).abs(), 0.0)).sum(-1)
    near(out.entropy, torch.where(counted, H, 0.0), 2 * es * (1 + spread + H) + 0 * H)
    ids = torch.sort(Z, dim=-1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(out.top_ids.cpu(), torch.where(counted[:, None], ids, -1))
    # (what lies beyond 32 bits' range is -inf there)
    lo = lambda x: torch.where(x.float() == -math.inf, torch.zeros_like(x), x)  # noqa: E731
    top = torch.where(counted[:, None], l.gather(1, ids), 0.0)
    assert torch.equal(out.top_logprobs.cpu() == -math.inf, top.float() == -math.inf)
    near(lo(out.top_logprobs), lo(top), torch.full_like(top, es))
    lp = torch.where(counted, l.gather(1, Y[:, None])[:, 0], 0.0)
    outs, ups, g_p, g_h, g_t = [], [], torch.zeros(M), torch.zeros(M), torch.zeros(M, k)
    if targets is None:
        assert out.logprobs is None
    else:
        assert torch.equal(out.logprobs.cpu() == -math.inf, lp.float() == -math.inf)
        near(lo(out.logprobs), lo(lp), torch.full_like(lp, es))
        if "p" in want:
            g_p = torch.randn(M, generator=gen)
            outs, ups = outs + [out.logprobs], ups + [g_p.to(z.device)]
    if "h" in want:
        g_h = torch.randn(M, generator=gen)
        outs, ups = outs + [out.entropy], ups + [g_h.to(z.device)]
    if "t" in want and k:
        g_t = torch.randn(M, k, generator=gen)
        outs, ups = outs + [out.top_logprobs], ups + [g_t.to(z.device)]
    (dz,) = torch.autograd.grad(outs, z, ups)
    g_p, g_h, g_t = g_p.double(), g_h.double()[:, None], g_t.double()
    g = (g_p + g_t.sum(-1))[:, None]
    l0 = torch.where(p > 0, l, 0.0)
    hot = torch.zeros_like(Z).scatter_add_(1, ids, g_t).scatter_add_(1, Y[:, None], g_p[:, None])
    hots = torch.zeros_like(Z).scatter_add_(1, ids, g_t.abs()).scatter_add_(1, Y[:, None], g_p.abs()[:, None])
    exact = (hot - p * (g + g_h * (l0 + H[:, None]))) / temperature
    size = p * (g.abs() + g_t.abs().sum(-1, keepdim=True) * (k + 8) * U + g_h.abs() * (l0.abs() + H[:, None]))
    t = ((Z - high) / temperature).abs()
    rel = 2 * es + 2.0 ** -20 * (1 + torch.where(p > 0, t, 0.0))
    slack = p * g_h.abs() * 4 * es * (1 + spread + H)[:, None]
    more = (size * rel + slack + hots * 4 * U) / temperature
    on = counted[:, None]
    near(dz[:, :V], torch.where(on, exact, 0.0), torch.where(on, more + 2.0 ** -126, 0.0))
    assert (dz[:, V:] == 0).all() and (dz[~counted.to(z.device)] == 0).all()
    return out


def logits(M, W, dtype, device, seed=0):
    return (3.0 * randn(M, W, seed=seed)).to(device=device, dtype=dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,V,W,k,tau", [(1, 1, 1, 1, 1.0), (3, 7, 7, 7, 2.0), (5, 1000, 1024, 5, 1.0), (7, 1001, 1001, 20, 0.7),
                                         (40, 513, 640, 0, 1.3), (2, 300, 300, 256, 1.0), (2, 2100, 2104, 256, 1.0)])
def test_token_logprobs(device, M, V, W, k, tau, dtype):
    logprob_case(device, logits(M, W, dtype, device), V, k, tau)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,V,W,k", [(500, 2000, 2048, 3), (3, 50257, 50304, 128), (310, 33000, 33000, 9), (1, 65536, 65536, 256),
                                     (2, 65537, 65540, 256), (700, 1000, 1000, 20),
                                     (700, 301, 304, 0), (1300, 5000, 5056, 8), (3, 152064, 152064, 32), (1, 152063, 152063, 0), (20, 40000, 40000, 0)])
def test_token_logprobs_sizes(cuda, M, V, W, k, dtype):
    logprob_case("cuda", logits(M, W, dtype, "cuda"), V, k)


def test_token_logprobs_targets_and_rows(device):
    z = logits(6, 72, torch.float32, device)
    logprob_case(device, z, 70, 4, targets=None)
    logprob_case(device, z, 70, 0, targets=None, want=("h",))
    logprob_case(device, z, 70, 4, targets=torch.tensor([0, 69, 70, -1, -100, 5], device=device))
    logprob_case(device, z, 70, 4, targets=torch.tensor([0, 69, 70, -1, 1 << 40, 5], device=device))
    logprob_case(device, z, 70, 4, targets=torch.tensor([0, 69, 3, 3, 1, 5], device=device, dtype=torch.int32), ignore=3)
    logprob_case(device, z, 70, 4, want=("p",))
    logprob_case(device, z, 70, 4, want=("t",))
    out = token_logprobs(z, torch.full((6,), -100, device=device), top_k=2)
    assert (out.top_ids == -1).all() and (out.logprobs == 0).all() and (out.entropy == 0).all()
    empty = token_logprobs(z[:0], torch.zeros(0, dtype=torch.int64, device=device), top_k=2)
    assert empty.logprobs.shape == (0,) and empty.top_ids.shape == (0, 2)


@pytest.mark.parametrize("V,k", [(1000, 40), pytest.param(70000, 40, marks=pytest.mark.gpu),
                                 pytest.param(70000, 256, marks=pytest.mark.gpu)])
def test_token_logprobs_order(device, V, k):
    """equal logits go to the lowest id; rows whose best lie side by side; 0 and -0"""
    r = randn(8, V, seed=V)
    z = torch.stack([torch.zeros(V), torch.arange(V) / V * 8, -torch.arange(V) / V * 8, r[0].round(), (r[1] * 2).clamp(max=0.0),
                     torch.where(r[2] > 0, 0.0, -0.0), torch.arange(V).flip(0).div(300, rounding_mode="floor") * 0.01,
                     torch.full((V,), -7.0)])
    for dtype in TYPES:
        logprob_case(device, z.to(device=device, dtype=dtype), None, k, targets=torch.arange(8, device=device))


@pytest.mark.parametrize("V,k", [(600, 8), pytest.param(70001, 8, marks=pytest.mark.gpu)])
@pytest.mark.parametrize("dtype", TYPES)
def test_token_logprobs_masks(device, V, k, dtype):
    low = torch.finfo(dtype).min
    z = logits(10, V, dtype, device, seed=1)
    z[0] = -math.inf                        # nothing left
    z[1] = -math.inf
    z[1, V - 2] = 1.0                       # one left
    z[2, ::2] = -math.inf
    z[3, : V - 3] = -math.inf               # fewer than k
    z[4] = low                              # all equal, at the type's lowest
    z[5] = low
    z[5, 3:9] = -math.inf
    z[6, 5:] = low
    z[7, : V // 2] = -30000.0
    z[8, 0] = -math.inf                     # the target's
    z[9] = low
    z[9, 7] = torch.finfo(dtype).max / 4
    targets = torch.tensor([1, V - 2, 1, V - 1, 5, 0, 2, V - 1, 0, 7], device=device)
    logprob_case(device, z, None, k, targets=targets)
    z[2:4, 1] = 60000.0                     # masks and temperatures at the ends of their range
    for tau in (1e-6, 0.01, 300.0, 1e6):
        logprob_case(device, z, None, k, tau, targets=targets)


@pytest.mark.parametrize("V", [300, pytest.param(70000, marks=pytest.mark.gpu)])
def test_token_logprobs_nan_and_infinity(device, V):
    z = logits(5, V + 20, torch.float32, device)
    z[:, V:] = float("nan")                 # padding is not read
    z[1, 3] = float("nan")
    z[2, 4] = float("inf")
    z[3] = -math.inf
    z[3, 7] = float("nan")
    z.requires_grad_()
    out = token_logprobs(z, torch.arange(5, device=device), top_k=3, vocab=V)
    (dz,) = torch.autograd.grad(out.logprobs.sum() + out.entropy.sum(), z)
    for m in (1, 2, 3):
        assert out.logprobs[m].isnan() and out.entropy[m].isnan() and out.top_logprobs[m].isnan().all()
        assert ((out.top_ids[m] >= 0) & (out.top_ids[m] < V)).all()
    assert out.top_ids[1, 0] == 3 and out.top_ids[2, 0] == 4 and out.top_ids[3, 0] == 7
    for m in (0, 4):
        assert torch.isfinite(out.logprobs[m]) and torch.isfinite(out.entropy[m]) and torch.isfinite(dz[m]).all()
    assert (dz[:, V:] == 0).all() and dz[1, :V].isnan().all()


def test_token_logprobs_rows_of_any_alignment(device):
    for dtype in TYPES:
        base = logits(5, 203, dtype, device)
        for c in range(0, 9):
            logprob_case(device, base[:, c: c + 190], 189, 6)
        logprob_case(device, base.t()[:5], None, 3)
        logprob_case(device, base[:1].expand(4, 203), None, 3)
        logprob_case(device, base[:, ::2], None, 3)


def test_token_logprobs_refusals(device):
    z, y = logits(3, 16, torch.float32, device), torch.zeros(3, dtype=torch.int64, device=device)
    for kwargs in ({"top_k": 17}, {"top_k": -1}, {"vocab": 17}, {"vocab": 0}, {"temperature": 0.0},
                   {"temperature": float("inf")}, {"temperature": float("nan")}):
        with pytest.raises(ValueError, match="token_logprobs"):
            token_logprobs(z, y, **kwargs)
    with pytest.raises(ValueError, match="top_k"):
        token_logprobs(logits(1, 300, torch.float32, device), None, top_k=257)
    with pytest.raises(ValueError, match=r"\[M, V\]"):
        token_logprobs(z[0], y)
    with pytest.raises(ValueError, match="targets must be"):
        token_logprobs(z, y[:2])
    with pytest.raises(TypeError, match="int32 or int64"):
        token_logprobs(z, y.float())
    if device == "cuda":
        with pytest.raises(ValueError, match="on cpu"):
            token_logprobs(z, y.cpu())
        out = token_logprobs(z.requires_grad_(), y)
        with pytest.raises(RuntimeError, match="not differentiable"):
            torch.autograd.grad(out.logprobs.sum(), z, create_graph=True)


def test_token_logprobs_against_differences():
    z = logits(4, 12, torch.float64, "cpu").requires_grad_()
    y = torch.tensor([0, 3, -100, 11])
    f = lambda z: token_logprobs(z, y, top_k=3, temperature=1.7, vocab=11)[:3]  # noqa: E731
    assert torch.autograd.gradcheck(f, (z,))
