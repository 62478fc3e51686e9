"""Ends of the ranges of the row operators."""

import math

import pytest
import torch

from tests.test_row_ops import DEVICES, TYPES, U, near, norm_case, randn
from zeroq_b200.ops import add_layer_norm, embedding, layer_norm, token_logprobs


@pytest.fixture(params=DEVICES)
def device(request):
    if request.param == "cuda":
        request.getfixturevalue("cuda")
    return request.param


# ---------------------------------------------------------------------------
# token log probabilities
# ---------------------------------------------------------------------------
def entropy_gradient(z, tau, g):
    """dz of g . H against -g p (l + H) / tau in 64 bits; the bounds of the formula's other tests"""
    z = z.requires_grad_()
    M, V = z.shape
    out = token_logprobs(z, None, temperature=tau)
    (dz,) = torch.autograd.grad(out.entropy, z, g)
    Z, G = z.detach().double().cpu(), g.double().cpu()[:, None]
    high = Z.amax(-1, keepdim=True)
    t = (Z - high) / tau
    l = torch.log_softmax(t, -1)
    p = l.exp()
    l0, t0 = torch.where(p > 0, l, 0.0), torch.where(p > 0, t.abs(), 0.0)
    H = -(p * l0).sum(-1, keepdim=True)
    spread = (p * t0).sum(-1, keepdim=True)
    # S: V / 256 sums in a row and their joins, 2^-22 an exponential; its argument's error; H's
    es = (V / 256 + 64) * U
    more = p * G.abs() * ((l0.abs() + H) * (2 * es + 2.0 ** -20 * (1 + t0)) + 4 * es * (1 + spread + H)) / tau
    # a p below 32 bits' normal range, 2^-126, is 0 (with its error, from 2^-125 down it may be), times
    # the same factor
    more = more + 2.0 ** -125 * G.abs() * (l0.abs() + H) / tau
    want = -G * p * (l0 + H) / tau
    # (an entry whose bounds reach past the type's range may be there; near() takes the others)
    tol = torch.finfo(z.dtype).eps / 2 * want.abs() + more
    low, high, got = (want - tol).to(z.dtype), (want + tol).to(z.dtype), dz.cpu()
    edge = low.isinf() | high.isinf()
    assert ((low <= got) & (got <= high))[edge].all()
    near(torch.where(edge, 0.0, got), torch.where(edge, 0.0, want), more + 2.0 ** -126)


@pytest.mark.parametrize("V", [600, pytest.param(70001, marks=pytest.mark.gpu)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tau,g", [(0.01, 65536.0), (1e-3, 400.0), (1e-4, 10.0), (1e-5, 0.1), (1e-5, 1e5), (1e-6, 1.0)])
def test_entropy_gradient_of_masked_logits(device, tau, g, dtype, V):
    z = randn(9, V, seed=V) * tau            # several of a row weigh something
    z[5:] = randn(4, V, seed=1).clamp(max=0.5)
    z[5:, 7] = torch.tensor([0.6, 1.0, 3.0, 5.0])   # one has all the weight
    z = z.to(device=device, dtype=dtype)
    gone = torch.rand(9, V, generator=torch.Generator().manual_seed(2)) < 0.3
    gone[:, 7] = False
    for low in (-math.inf, torch.finfo(dtype).min, max(-1e9, torch.finfo(dtype).min)):
        entropy_gradient(torch.where(gone.to(device), low, z), tau, g * randn(9, seed=3, device=device))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [300, 5003, pytest.param(70000, marks=pytest.mark.gpu)])
def test_log_probabilities_are_at_most_0(device, V, dtype):
    """a certain token's: neither the exponential's error nor a sum's rounding shows above 0"""
    M = 400 if V < 60000 else 40
    z = randn(M, V, seed=V)
    z[torch.arange(M), torch.arange(M) % V] += torch.linspace(0, 30, M)
    z[: M // 4] = -math.inf                      # no other token at all
    z[torch.arange(M), torch.arange(M) % V] = z[torch.arange(M), torch.arange(M) % V].nan_to_num(neginf=3.3)
    z[: M // 4, :3] = z[: M // 4, :3].clamp(min=-30.0)
    for tau in (1.0, 0.7, 1e-3):
        out = token_logprobs(z.to(device=device, dtype=dtype), torch.arange(M, device=device) % V, top_k=3, temperature=tau)
        assert (out.logprobs <= 0).all() and (out.top_logprobs <= 0).all() and (out.entropy >= 0).all()


# ---------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [1, 8, 33, 256, 264, 1000, 1001, 1032, 3584, 5120, 8200, 12289, 16384])
def test_layer_norm_of_rows_of_one_value(cuda, D, dtype, residual):
    """differences from the mean are 0 to the bit: y is the bias, dw is 0"""
    c = torch.tensor([10000.0, 0.1, -777.7, 3.0, 1e-3, 60000.0], device=cuda)[:, None]
    x = c.expand(6, D).to(dtype).contiguous().requires_grad_()
    w, b = randn(D, seed=8, device=cuda).requires_grad_(), randn(D, seed=9, device=cuda)
    y = add_layer_norm(x, torch.zeros_like(x), w, b, eps=1e-5)[1] if residual else layer_norm(x, w, b, eps=1e-5)
    assert torch.equal(y, b.to(dtype).expand(6, D))
    dw, dx = torch.autograd.grad(y, [w, x], randn(6, D, seed=10, dtype=dtype, device=cuda))
    assert (dw == 0).all() and torch.isfinite(dx).all()


@pytest.mark.gpu
@pytest.mark.parametrize("first", [0.0, 50.0])
@pytest.mark.parametrize("D", [520, 4100, 4101, 12000])
@pytest.mark.parametrize("mean,dev", [(10000.0, 1e-2), (-3e5, 1.0), (1e3, 1e-3), (1.0, 1e-6), (0.0, 1.0)])
def test_layer_norm_rounds_the_mean_alone(cuda, mean, dev, D, first):
    """Rows far from 0 in fp32, with and without a first value far out.  The mean is off by two roundings
    of its own (a warp's, the row's) and by a row's length in roundings of the deviations; the
    differences from it by one of theirs."""
    z = randn(6, D, seed=D).double()
    z[::2, 0] += first
    x = (mean + dev * z).float().to(cuda)
    w = torch.ones(D, device=cuda, requires_grad=True)
    y = layer_norm(x, w, None, eps=1e-12)
    X = x.double().cpu()
    mu = X.mean(-1, keepdim=True)
    d = X - mu
    r = (d.square().mean(-1, keepdim=True) + 1e-12).rsqrt()
    dmu = 2 * U * mu.abs() + 64 * U * (d.abs().mean(-1, keepdim=True) + d.abs().amax(-1, keepdim=True))
    # r: half of what its sum of squares is off by - 22 roundings (of a lane's values, of the lanes) nine
    # times, as up to 8/9 of the sum are taken off again, and those over warps - and of dmu squared
    dn = r * dmu + (d * r).abs() * (128 * U + 0.5 * (r * dmu).square())
    near(y, d * r, dn)
    dy = randn(6, D, seed=10, device=cuda)
    (dw,) = torch.autograd.grad(y, w, dy)
    g = dy.double().cpu()
    # 2 more: of the mean that the backward is given, and of its use
    near(dw, (g * d * r).sum(0), (g.abs() * (dn + 2 * U * mu.abs() * r)).sum(0) + 10 * U * (g * d * r).abs().sum(0))


@pytest.mark.parametrize("residual,saved", [(False, "full"), (True, "full"), (False, "8bit")])
@pytest.mark.parametrize("D", [520, 1001, 4100, pytest.param(5120, marks=pytest.mark.gpu), pytest.param(16384, marks=pytest.mark.gpu)])
def test_layer_norm_of_rows_with_values_far_out(device, D, residual, saved):
    """single values thousands of times the others, first in a row or in a tile: the others keep their places"""
    x = randn(8, D, seed=D)
    for i, c in enumerate([0, 256, 1, D - 1]):
        x[i, c] = 1e4
    x[4, 0], x[4, D // 2] = 1e4, -1e4
    x[5, ::256] = 3e3
    x[6, :8] = -2e4
    norm_case(device, 8, D, torch.float32, x=x.to(device), residual=residual, saved=saved)


@pytest.mark.parametrize("D", [8, 300, 301, 4100, pytest.param(16384, marks=pytest.mark.gpu)])
def test_layer_norm_of_rows_with_infinities(device, D):
    """NaN throughout, wherever they are, and their gradients; the rows beside them are not touched"""
    for dtype in TYPES:
        x = randn(9, D, seed=D, dtype=dtype, device=device)
        for i, (c, v) in enumerate([(0, math.inf), (D // 2, -math.inf), (D - 1, math.inf), (0, math.nan), (D - 1, math.nan)]):
            x[i, c] = v
        x[5] = math.inf
        x.requires_grad_()
        y = layer_norm(x)
        (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
        assert y[:6].isnan().all() and dx[:6].isnan().all()
        assert torch.equal(y[6:], layer_norm(x[6:])) and torch.isfinite(dx[6:]).all()
    # squares beyond 32 bits: a deviation without end
    x = torch.full((2, D), 1e25, device=device)
    x[:, ::2] = -3e25
    assert (layer_norm(x) == 0).all()


@pytest.mark.parametrize("wtype", TYPES)
def test_layer_norm_with_a_bias_alone(device, wtype):
    for dtype in TYPES:
        for D in (72, 1001):
            norm_case(device, 40, D, dtype, wtype=wtype, weight=False)
            norm_case(device, 40, D, dtype, wtype=wtype, weight=False, residual=True, saved="8bit")


# ---------------------------------------------------------------------------
# embedding
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [256, 1001])
@pytest.mark.parametrize("scale", [-2.0, 0.0, 1e300, math.inf, -math.inf, math.nan])
def test_rows_of_absent_ids_are_0(device, scale, D, dtype):
    """whatever the scale, and without a sign"""
    ids = torch.tensor([3, -1, 8, 7, 1 << 40, -100], device=device)
    w = randn(8, D, seed=1, dtype=dtype, device=device).requires_grad_()
    y = embedding(ids, w, scale)
    absent = y.detach()[[1, 2, 4, 5]]
    assert (absent == 0).all() and not torch.signbit(absent).any()
    here = (w.detach().float() * scale).to(dtype)[[3, 7]]
    assert torch.equal(y.detach()[[0, 3]].nan_to_num(nan=5.0), here.nan_to_num(nan=5.0))
    (dw,) = torch.autograd.grad(y, w, torch.ones_like(y))
    rows = dw[[0, 1, 2, 4, 5, 6]]
    assert (rows == 0).all() and not torch.signbit(rows).any()
