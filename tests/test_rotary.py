"""rotary_embedding against its formula in 64 bits, on the CPU and on the GPU.

Tolerance: the output is rounded once (half a step of the type, relative to the value);
before that, cos and sin carry at most 2^-22 (2 ulp of 32-bit sincospi and the reduced
angle's rounding times 2 pi) and two products and a sum 2^-23 of |a| + |b| each, so
2^-20 (|a| + |b|) f bounds the rest."""

import math

import pytest
import torch

from zeroq_b200.ops import RopeScaling, apply_rope, rotary_embedding
from zeroq_b200.ops.rope import _rope_frequencies


def exact(x, positions, theta, R, interleaved, scaling, sign=1.0):
    """64-bit rotation as a product of complex numbers, and the sum of each pair's sizes."""
    freq, factor = _rope_frequencies(R, float(theta), scaling)
    ang = positions.double().cpu()[..., None, None] * torch.tensor(freq, dtype=torch.float64) * sign
    turn = torch.polar(torch.full_like(ang, factor), ang)
    y = x.double().cpu().clone()
    size = torch.zeros_like(y)
    a, b = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    both = y[..., a].abs() + y[..., b].abs()
    c = torch.complex(y[..., a].contiguous(), y[..., b].contiguous()) * turn
    y[..., a], y[..., b] = c.real, c.imag
    size[..., a] = size[..., b] = both * factor
    return y, size


def check(got, x, *args, sign=1.0):
    want, size = exact(x, *args, sign=sign)
    tol = torch.finfo(got.dtype).eps / 2 * want.abs() + 2.0 ** -20 * size
    if got.dtype == torch.float16:
        tol += 2.0 ** -25   # half a step below fp16's normal range
    off = (got.double().cpu() - want).abs()
    assert (off <= tol).all(), (off - tol).max()


SCALINGS = [None, RopeScaling("linear", 4.0), RopeScaling("ntk", 8.0), RopeScaling("yarn", 8.0, 4096),
            RopeScaling("yarn", 2.0, 2048, attention_factor=1.0)]


def case(device, tokens, hq, hk, D, R, dtype, interleaved, scaling, far=262144, fused=True, shape=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    if fused:   # column ranges of one q/k/v buffer
        qkv = torch.randn(tokens, (hq + 2 * hk) * D, generator=g).to(device=device, dtype=dtype)
        q = qkv[:, : hq * D].view(tokens, hq, D)
        k = qkv[:, hq * D: (hq + hk) * D].view(tokens, hk, D)
    else:
        q = torch.randn(tokens, hq, D, generator=g).to(device=device, dtype=dtype)
        k = torch.randn(tokens, hk, D, generator=g).to(device=device, dtype=dtype)
    pos = torch.randint(0, far, (tokens,), generator=g)
    pos = pos.to(torch.int32 if seed % 2 else torch.int64).to(device)
    q.requires_grad_(), k.requires_grad_()
    args = (pos, 10000.0, R, interleaved, scaling)
    yq, yk = rotary_embedding(q, k, *args)
    check(yq, q.detach(), *args)
    check(yk, k.detach(), *args)
    gq, gk = torch.randn(yq.shape, generator=g).to(yq), torch.randn(yk.shape, generator=g).to(yk)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
    check(dq, gq, *args, sign=-1.0)
    check(dk, gk, *args, sign=-1.0)


@pytest.mark.parametrize("scaling", SCALINGS)
@pytest.mark.parametrize("interleaved", [False, True])
def test_reference_matches_formula(scaling, interleaved):
    case("cpu", 33, 4, 2, 64, 32, torch.float32, interleaved, scaling)


def test_half_layout_equals_apply_rope():
    q, k = torch.randn(2, 16, 4, 64), torch.randn(2, 16, 2, 64)
    yq, yk = rotary_embedding(q, k, torch.arange(16), theta=500.0)
    rq, rk = apply_rope(q, k, 500.0)
    assert torch.allclose(yq, rq, atol=1e-5) and torch.allclose(yk, rk, atol=1e-5)


def test_gradient_against_differences():
    q = torch.randn(5, 2, 12, dtype=torch.float64, requires_grad=True)
    pos = torch.tensor([0, 7, 100, 3, 3])
    for inter in (False, True):
        assert torch.autograd.gradcheck(
            lambda x: rotary_embedding(x, None, pos, rotary_dim=8, interleaved=inter,
                                       scaling=RopeScaling("yarn", 4.0, 64))[0], (q,))


def test_scaling_limits():
    assert _rope_frequencies(64, 10000.0, RopeScaling("linear", 1.0)) == _rope_frequencies(64, 10000.0, None)
    f, _ = _rope_frequencies(64, 10000.0, None)
    n, _ = _rope_frequencies(64, 10000.0, RopeScaling("ntk", 8.0))
    assert n[0] == f[0] and math.isclose(n[-1], f[-1] / 8.0, rel_tol=1e-12)
    y, m = _rope_frequencies(64, 10000.0, RopeScaling("yarn", 8.0, 4096))
    assert y[0] == f[0] and math.isclose(y[-1], f[-1] / 8.0, rel_tol=1e-12) and m == 0.1 * math.log(8.0) + 1.0


def test_a_fake_call_leaves_nothing_to_the_real_ones():
    from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode

    from zeroq_b200.ops.rope import _rope_turns

    with FakeTensorMode():   # as a trace of a model makes it: the first call with these parameters
        _rope_turns(64, 4321.0, None)
        rotary_embedding(torch.empty(3, 1, 64), None, torch.arange(3), theta=4321.0)
    kept, factor = _rope_turns(64, 4321.0, None)
    assert not isinstance(kept, FakeTensor) and factor == 1.0
    turns = torch.frombuffer(bytearray(kept), dtype=torch.float64)
    freq, _ = _rope_frequencies(64, 4321.0, None)
    assert turns.tolist() == [f / (2 * math.pi) for f in freq]


@pytest.mark.parametrize("bad", [
    dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=66), dict(theta=0.5),
    dict(positions=torch.arange(5)), dict(positions=torch.arange(8.0)), dict(k=torch.randn(8, 2, 32)),
    dict(k=torch.randn(8, 2, 64).double()), dict(q=torch.zeros(8, 2, 64, dtype=torch.int32), k=None),
    dict(q=torch.randn(8, 64), k=None)])
def test_refusals(bad):
    args = dict(q=torch.randn(8, 4, 64), k=torch.randn(8, 2, 64), positions=torch.arange(8))
    args.update(bad)
    with pytest.raises((ValueError, TypeError)):
        rotary_embedding(**args)


@pytest.mark.parametrize("bad", [("dynamic", 2.0), ("linear", 0.5), ("yarn", float("nan"))])
def test_scaling_refusals(bad):
    with pytest.raises(ValueError):
        RopeScaling(*bad)


# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,hq,hk,D,R", [
    (1, 28, 4, 128, 128), (37, 4, 4, 64, 64), (1000, 6, 2, 80, 40), (257, 3, 1, 128, 64),
    (129, 2, 1, 20, 6),     # widths that are not whole vectors
    (5000, 8, 2, 96, 96), (64, 1, 1, 256, 256), (33, 2, 2, 130, 2)])
def test_kernel_matches_formula(cuda, dtype, interleaved, tokens, hq, hk, D, R):
    case(cuda, tokens, hq, hk, D, R, dtype, interleaved, SCALINGS[(tokens + D) % len(SCALINGS)], seed=tokens)


@pytest.mark.gpu
@pytest.mark.parametrize("scaling", SCALINGS)
def test_kernel_scalings(cuda, scaling):
    case(cuda, 301, 4, 1, 128, 128, torch.bfloat16, False, scaling, fused=False)


@pytest.mark.gpu
def test_kernel_strides_shapes_and_partial_gradients(cuda):
    pos = torch.arange(24, device=cuda, dtype=torch.int32) * 11 - 40     # negative positions turn back
    # [B, S, H, D] with positions of one row; heads outermost in memory; an odd storage offset
    base = torch.randn(2 * 4 * 24 * 64 + 1, device=cuda, dtype=torch.bfloat16)[1:]
    q = base.view(2, 4, 24, 64).transpose(1, 2).requires_grad_()
    k = torch.randn(2, 24, 64, 2, device=cuda, dtype=torch.bfloat16).transpose(2, 3)   # no unit stride
    args = (pos, 1e6, 64, False, None)
    yq, yk = rotary_embedding(q, k, *args)
    check(yq, q.detach(), *args)
    check(yk, k, *args)
    gq = torch.randn_like(yq)
    dq, = torch.autograd.grad(yq, q, gq, retain_graph=True)   # k's gradient is not asked for
    check(dq, gq, *args, sign=-1.0)
    only, none = rotary_embedding(q.detach(), None, *args)
    assert none is None and torch.equal(only, yq)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(yq, q, gq, create_graph=True)
    with pytest.raises(RuntimeError, match="rotary"):          # the entry's own checks
        from zeroq_b200.ops import _ext
        _ext.ext().rotary(q.detach()[0], None, pos[:5], torch.ones(32, dtype=torch.float64),
                          torch.empty(24, 4, 64, device=cuda, dtype=torch.bfloat16), None, False, 1.0, 1.0)


@pytest.mark.gpu
def test_kernel_empty_and_far_position(cuda):
    q = torch.randn(0, 4, 64, device=cuda, dtype=torch.bfloat16)
    yq, _ = rotary_embedding(q, None, torch.zeros(0, dtype=torch.int64, device=cuda))
    assert yq.shape == q.shape
    q = torch.randn(2, 1, 64, device=cuda)
    pos = torch.tensor([2 ** 31 + 12345, 0], device=cuda)     # past 32 bits
    yq, _ = rotary_embedding(q, None, pos)
    # 2^31 x 2^-53 of a turn: 64-bit angles are off by 2^-21 radians there at most
    want, size = exact(q, pos, 10000.0, 64, False, None)
    assert ((yq.double().cpu() - want).abs() <= 2.0 ** -19 * size + 2.0 ** -23 * want.abs()).all()
    assert torch.equal(yq[1], q[1])


@pytest.mark.gpu
def test_kernel_in_a_graph_and_on_another_stream(cuda):
    q = torch.randn(100, 4, 128, device=cuda, dtype=torch.bfloat16)
    pos = torch.arange(100, device=cuda)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side, _ = rotary_embedding(q, None, pos, theta=77.0)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):   # a base that no call had before: nothing is set up on the device
        y, _ = rotary_embedding(q, None, pos, theta=78.0)
    pos.add_(5)
    q.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, rotary_embedding(q, None, pos, theta=78.0)[0])
    assert torch.equal(side, rotary_embedding(q / 2, None, pos - 5, theta=77.0)[0])
