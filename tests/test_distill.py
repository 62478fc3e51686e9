"""distillation_loss against its formula in 64 bits.

Tolerances.  A row's loss is a sum of terms each formed in 32 bits from exp2 and log2 of
relative error 2^-22 and sums of V terms in partial sums: 2^-17 (tau^2 + |loss|) bounds it
(V <= 2^18 in at least 512 partial sums: at most 512 additions each, errors of both signs).
A gradient entry is g (a tau (q - p) + (1 - a)(r - 1)) with q, p, r of the same relative
error, at most 2^-17 g (a tau + 1 - a) in all, and one rounding of its type."""

import pytest
import torch

from zeroq_b200.ops import distillation_loss
from zeroq_b200.ops.distill import MAX_TEACHER_ENTRIES, distillation_reference


def make(M, V, K, dtype, device="cpu", wide=None, seed=0, short=True, teacher=torch.float32, ids=torch.int64):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(M, wide or V, generator=g) * 3).to(dtype).to(device)
    at = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(M)])
    if short:
        at[torch.rand(M, K, generator=g) < 0.1] = -1
    t = (torch.randn(M, K, generator=g) * 3).to(teacher).to(device)
    y = torch.randint(0, V, (M,), generator=g)
    y[torch.rand(M, generator=g) < 0.2] = -100
    return z, at.to(ids).to(device), t, y.to(device)


def exact(z, ids, t, y, T, a, V, g=None, mean=True):
    """(loss rows, gradient) in 64 bits from the definition, row by row over the vocabulary."""
    z64 = z.detach().double().cpu()[:, :V]
    ids, t = ids.cpu().long(), t.double().cpu()
    M = z64.shape[0]
    on = torch.ones(M, dtype=torch.bool) if y is None else (y.cpu() >= 0) & (y.cpu() < V)
    rows, grad = torch.zeros(M, dtype=torch.float64), torch.zeros(z.shape, dtype=torch.float64)
    for m in range(M):
        if not on[m]:
            continue
        p = torch.zeros(V, dtype=torch.float64)
        keep = (ids[m] >= 0) & (ids[m] < V) & (t[m] > -float("inf"))
        d = torch.zeros(V, dtype=torch.float64)
        if keep.any():
            w = torch.softmax(t[m][keep] / T, 0)
            lq = torch.log_softmax(z64[m] / T, 0)
            p.index_add_(0, ids[m][keep], w)
            rows[m] = a * T * T * (w * w.log() - w * lq[ids[m][keep]]).sum()
            d += a * T * (lq.exp() - p)
        if a < 1:
            lr = torch.log_softmax(z64[m], 0)
            rows[m] -= (1 - a) * lr[y[m].item()]
            d += (1 - a) * lr.exp()
            d[y[m].item()] -= 1 - a
        grad[m, :V] = d
    n = max(1, int(on.sum()))
    scale = torch.full((M,), 1.0 / n, dtype=torch.float64) if mean else g.double().cpu()
    return rows, grad * scale[:, None], n, scale


def check(z, ids, t, y, T, a, V, reduction="mean", upstream=1.0, exact_of=None):
    z = z.detach().requires_grad_()
    loss = distillation_loss(z, ids, t, y, temperature=T, alpha=a, vocab=V, reduction=reduction)
    if reduction == "mean":
        grad, = torch.autograd.grad(loss * upstream, z)
        rows, want, n, scale = exact(z, ids, t, y, T, a, V)
        want, scale = want * upstream, scale * abs(upstream)
        value = rows.sum() / n
        tol = 2.0 ** -17 * (T * T + rows.abs().sum() / n)
        assert loss.dtype == torch.float32 and abs(loss.item() - value.item()) <= tol
        # an upstream gradient that is no power of two rounds once more
        steps = 1 if upstream == 1.0 or z.dtype == torch.float16 else 2
    else:
        g = torch.rand(z.shape[0], device=z.device) + 0.5
        grad, = torch.autograd.grad(loss, z, g)
        rows, want, n, scale = exact(z, ids, t, y, T, a, V, g, mean=False)
        assert (loss.detach().double().cpu() - rows).abs().le(2.0 ** -17 * (T * T + rows.abs())).all()
        steps = 1
    tol = steps * torch.finfo(z.dtype).eps / 2 * want.abs() + 2.0 ** -17 * (a * T + 1 - a) * scale[:, None]
    if z.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    off = (grad.double().cpu() - want).abs()
    assert (off <= tol).all(), (off / tol).max()
    assert (grad[:, V:] == 0).all()
    if y is not None:
        assert (grad[((y < 0) | (y >= V))] == 0).all()


@pytest.mark.parametrize("T,a", [(1.0, 1.0), (2.0, 0.5), (1.5, 0.0), (3.0, 1.0)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_reference_matches_definition(T, a, reduction):
    check(*make(9, 50, 7, torch.float32), T, a, 50, reduction)


def test_ignore_index_within_the_vocabulary():
    z, ids, t, y = make(9, 50, 7, torch.float32)
    y[:] = torch.arange(9) % 4
    out = torch.where(y == 2, -100, y)
    for r in ("mean", "none"):
        assert torch.equal(distillation_loss(z, ids, t, y, alpha=0.5, ignore_index=2, reduction=r),
                           distillation_loss(z, ids, t, out, alpha=0.5, reduction=r))


def test_gradient_against_differences():
    z, ids, t, y = make(5, 11, 4, torch.float64)
    z.requires_grad_()
    assert torch.autograd.gradcheck(
        lambda x: distillation_loss(x, ids, t, y, temperature=2.0, alpha=0.6, reduction="none"), (z,))


@pytest.mark.parametrize("bad", [
    dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("inf")), dict(alpha=1.5), dict(alpha=-0.1),
    dict(alpha=0.5, targets=None), dict(vocab=0), dict(vocab=51), dict(reduction="sum"),
    dict(targets=torch.zeros(3, dtype=torch.int64)), dict(targets=torch.zeros(6)),
    dict(teacher_ids=torch.zeros(6, 4)), dict(teacher_ids=torch.zeros(5, 4, dtype=torch.int64)),
    dict(teacher_logits=torch.zeros(6, 3)), dict(logits=torch.zeros(6, 50, dtype=torch.int64)),
    dict(teacher_ids=torch.zeros(6, MAX_TEACHER_ENTRIES + 1, dtype=torch.int64),
         teacher_logits=torch.zeros(6, MAX_TEACHER_ENTRIES + 1))])
def test_refusals(bad):
    args = dict(logits=torch.zeros(6, 50), teacher_ids=torch.zeros(6, 4, dtype=torch.int64),
                teacher_logits=torch.zeros(6, 4), targets=torch.zeros(6, dtype=torch.int64))
    args.update(bad)
    with pytest.raises((ValueError, TypeError)):
        distillation_loss(**args)


# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,a", [(1.0, 1.0), (1.0, 0.3), (2.0, 0.5), (1.5, 1.0), (4.0, 0.0)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_kernel_matches_definition(cuda, dtype, T, a, reduction):
    check(*make(67, 1003, 9, dtype, cuda, wide=1024), T, a, 1003, reduction)


@pytest.mark.gpu
@pytest.mark.parametrize("M,V,wide,K", [
    (1, 1, 1, 1), (1, 7, 7, 3), (3, 33, 40, 33), (5, 50257, 50304, 64), (2, 152064, 152064, 1024),
    (40, 8191, 8191, 5),      # rows of an odd pitch: every alignment
    (150, 4099, 4104, 1), (700, 515, 515, 128), (1, 40000, 40000, 0)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_kernel_sizes(cuda, M, V, wide, K, dtype):
    z, ids, t, y = make(M, V, K, dtype, cuda, wide=wide, seed=M + V, ids=torch.int32 if M % 2 else torch.int64,
                        teacher=torch.bfloat16 if K == 64 else torch.float32)
    y[0] = V - 1
    check(z, ids, t, y, 2.0, 0.5, V)
    check(z, ids, t, y, 1.0, 0.5, V, reduction="none")


@pytest.mark.gpu
def test_kernel_repeated_ids_and_targets_among_them(cuda):
    z, ids, t, y = make(30, 600, 40, torch.float32, cuda, short=False)
    ids[:, 1] = ids[:, 0]
    ids[:, 7] = ids[:, 0]
    ids[::2, 20:] = ids[::2, 3:4]
    y[:] = ids[:, 0]
    y[::3] = ids[::3, 5]
    check(z, ids, t, y, 2.0, 0.5, 600)
    check(z, ids, t, y, 1.0, 0.9, 600, reduction="none")


@pytest.mark.gpu
def test_kernel_rows_that_count_nothing(cuda):
    z, ids, t, y = make(20, 300, 8, torch.bfloat16, cuda)
    ids[3] = -1                        # no entries: the hard term alone
    t[4] = float("-inf")
    ids[5] = 300 + torch.arange(8)     # outside the vocabulary
    y[3:6] = 7
    check(z, ids, t, y, 2.0, 0.5, 300)
    check(z, ids, t, None, 2.0, 1.0, 300)
    y[:] = -100
    y[1] = 300                         # outside as well
    y[2] = -5
    check(z, ids, t, y, 2.0, 0.5, 300)
    loss = distillation_loss(z, ids, t, y, alpha=0.5)
    assert loss.item() == 0.0


@pytest.mark.gpu
def test_kernel_infinite_logits(cuda):
    z, ids, t, y = make(12, 5000, 6, torch.float32, cuda, short=False)
    y[:] = 4000
    z[:, :2048] = float("-inf")        # banned tokens: whole vectors and whole threads of them
    ids = ids.clamp_min(2048)
    z[torch.arange(12), 4000] = 1.0
    for r in range(12):
        z[r, ids[r]] = 0.5
    t[0, 0] = float("-inf")
    check(z, ids, t, y, 1.0, 0.5, 5000)
    check(z, ids, t, y, 3.0, 0.5, 5000, reduction="none")
    z[2, ids[2, 1]] = float("-inf")    # the student rules out what the teacher wants
    z[5, 3000] = float("nan")
    t[7, 2] = float("nan")
    t[8, 3] = float("inf")
    rows = distillation_loss(z, ids, t, y, temperature=2.0, alpha=0.5, reduction="none")
    want = distillation_reference(z, ids, t, y, temperature=2.0, alpha=0.5, reduction="none")
    assert rows[2].item() == float("inf") and want[2].item() == float("inf")
    assert torch.equal(torch.isnan(rows), torch.isnan(want)) and torch.isnan(rows).sum() == 3


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("upstream", [0.25, 3.0])
def test_kernel_upstream_gradient(cuda, dtype, upstream):
    check(*make(33, 777, 5, dtype, cuda), 2.0, 0.5, 777, upstream=upstream)


@pytest.mark.gpu
def test_fp16_gradient_takes_the_loss_scale_before_rounding(cuda):
    """At 2^12 the scaled gradient is normal where the unscaled one is below fp16's range."""
    z, ids, t, y = make(2000, 900, 5, torch.float16, cuda)
    check(z, ids, t, y, 2.0, 0.5, 900, upstream=2.0 ** 12)


@pytest.mark.gpu
def test_kernel_strided_logits_second_backward_and_no_grad(cuda):
    z, ids, t, y = make(10, 256, 4, torch.bfloat16, cuda, wide=320)
    part = z[:, :256]                                            # rows apart
    check(part, ids, t, y, 1.0, 0.5, 256)
    check(z[1:9, 3:200], ids[1:9], t[1:9], y[1:9], 1.0, 0.5, 190)   # an odd start
    check(z.t().contiguous().t(), ids, t, y, 1.0, 0.5, 256)       # columns outermost
    check(z[:1].expand(10, 320), ids, t, y, 1.0, 0.5, 256)        # one row for all
    leaf = z.detach().requires_grad_()
    loss = distillation_loss(leaf, ids, t, y, alpha=0.5, vocab=256)
    loss.backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="handed over"):
        loss.backward()
    with torch.no_grad():
        again = distillation_loss(leaf, ids, t, y, alpha=0.5, vocab=256)
    assert abs(again.item() - loss.item()) <= 2.0 ** -20 * abs(loss.item())


@pytest.mark.gpu
def test_kernel_refuses_rows_that_do_not_fit_and_second_derivatives(cuda):
    z = torch.zeros(1, 500000, device=cuda)
    ids, t = torch.zeros(1, 2, dtype=torch.int64, device=cuda), torch.zeros(1, 2, device=cuda)
    with pytest.raises(RuntimeError, match="bytes"):
        distillation_loss(z, ids, t)
    z, ids, t, y = make(4, 50, 3, torch.float32, cuda)
    for r in ("mean", "none"):
        leaf = z.detach().requires_grad_()
        loss = distillation_loss(leaf, ids, t, y, alpha=0.5, reduction=r)
        with pytest.raises(RuntimeError, match="not differentiable"):
            torch.autograd.grad(loss.sum(), leaf, create_graph=True)
    y[1] = 7
    assert torch.equal(distillation_loss(z, ids, t, y, alpha=0.5, ignore_index=7),
                       distillation_loss(z, ids, t, torch.where(y == 7, -100, y), alpha=0.5))


@pytest.mark.gpu
def test_kernel_is_deterministic_and_replays_in_a_graph(cuda):
    z, ids, t, y = make(300, 2000, 16, torch.bfloat16, cuda)
    z.requires_grad_()

    def step():
        loss = distillation_loss(z, ids, t, y, temperature=2.0, alpha=0.5)
        # (a live eager graph of z would tie the captured one to another stream)
        return loss.detach(), torch.autograd.grad(loss, z)[0]

    first = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grad = step()
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, first[0]) and torch.equal(grad, first[1])
    with torch.no_grad():
        z.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    now = step()
    assert torch.equal(loss, now[0]) and torch.equal(grad, now[1]) and not torch.equal(now[1], first[1])
