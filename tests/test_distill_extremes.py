"""distillation_loss on rows at the ends of their type's range, against its formula in 64 bits.

Tolerances as for ordinary rows: every term of a loss row is formed in 32 bits from exp2 and
log2 of relative error 2^-22, so 2^-17 (tau^2 + |loss|) bounds a row, and 2^-17 g (a tau + 1 - a)
with one rounding of the type a gradient entry.  Differences from the row's largest value are
exact here or so large that their exponential is 0."""

import pytest
import torch

from zeroq_b200.ops import distillation_loss


def exact(z, ids, t, y, T, a, V, g):
    """(loss rows, gradient) of sum(g * rows) in 64 bits."""
    z64, ids, t64 = z.detach().double().cpu()[:, :V], ids.cpu().long(), t.double().cpu()
    on = (y.cpu() >= 0) & (y.cpu() < V)
    w = torch.softmax((t64 / T).masked_fill((ids < 0) | (ids >= V), -float("inf")), -1)
    p = torch.zeros_like(z64).scatter_add_(1, ids.clamp(0, V - 1), w)
    lq, lr = torch.log_softmax(z64 / T, -1), torch.log_softmax(z64, -1)
    label = y.cpu().clamp(0, V - 1)[:, None]
    cross = torch.where(p > 0, p * lq, torch.zeros_like(p)).sum(-1)
    rows = a * T * T * (torch.xlogy(w, w).sum(-1) - cross) - (1 - a) * lr.gather(1, label)[:, 0]
    d = a * T * (lq.exp() - p) + (1 - a) * lr.exp()
    d.scatter_add_(1, label, torch.full_like(label, a - 1, dtype=torch.float64))
    return torch.where(on, rows, 0.0), torch.where(on, g, 0.0)[:, None] * d


def check(z, ids, t, y, T, a, V):
    """Rows with a gradient each, and their mean."""
    u, sub = torch.finfo(z.dtype).eps / 2, 2.0 ** -25 if z.dtype == torch.float16 else 0.0
    n = int(((y >= 0) & (y < V)).sum())
    for reduction, g in (("none", torch.linspace(0.5, 1.5, len(y), dtype=torch.float64)),
                         ("mean", torch.full((len(y),), 1.0 / n, dtype=torch.float64))):
        leaf = z.detach().requires_grad_()
        loss = distillation_loss(leaf, ids, t, y, temperature=T, alpha=a, vocab=V, reduction=reduction)
        up = g.float().to(z.device) if reduction == "none" else torch.ones((), device=z.device)
        grad, = torch.autograd.grad(loss, leaf, up)
        rows, want = exact(z, ids, t, y, T, a, V, g)
        tol = 2.0 ** -17 * (T * T + rows.abs())
        if reduction == "mean":
            rows, tol = rows.sum() / n, tol.sum() / n
        assert ((loss.detach().double().cpu() - rows).abs() <= tol).all(), (loss, rows)
        tol = u * want.abs() + 2.0 ** -17 * (a * T + 1 - a) * g[:, None] + sub
        assert ((grad.double().cpu()[:, :V] - want).abs() <= tol).all()
        assert (grad[:, V:] == 0).all()


def make(M, V, K, dtype, teacher, device, wide=None):
    g = torch.Generator().manual_seed(M + V)
    z = (torch.randn(M, wide or V, generator=g) * 3).to(dtype).to(device)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(M)]).to(device)
    t = (torch.randn(M, K, generator=g) * 3).to(teacher).to(device)
    y = torch.randint(0, V, (M,), generator=g)
    y[::5] = -100
    return z, ids, t, y.to(device)


def lowest_teacher(dtype, teacher, device="cpu"):
    """Entries at and near the type's lowest value are entries, not none."""
    z, ids, t, y = make(12, 300, 6, dtype, teacher, device)
    low = torch.finfo(teacher).min
    t[1] = low                    # all alike: uniform
    t[2, :3] = low                # next to ordinary ones: nothing of the mass
    t[3, 1:] = low
    t[4] = low
    t[4, 4] = 0.75 * low          # all of the mass
    t[6] = -low
    ids[7, 2:], t[7] = -1, low    # two entries
    return z, ids, t, y


TEMPERATURES = [(1.0, 1.0), (1.0, 0.4), (2.0, 0.5), (0.5, 1.0), (1.5, 0.3), (4.0, 0.5), (3.0, 0.0)]


@pytest.mark.parametrize("T,a", TEMPERATURES)
def test_reference_teacher_at_the_lowest_value(T, a):
    check(*lowest_teacher(torch.float32, torch.float32), T, a, 300)


@pytest.mark.gpu
@pytest.mark.parametrize("teacher", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,a", TEMPERATURES)
def test_kernel_teacher_at_the_lowest_value(cuda, teacher, T, a):
    check(*lowest_teacher(torch.float32, teacher, cuda), T, a, 300)
    check(*lowest_teacher(torch.bfloat16, teacher, cuda), T, a, 300)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,offset", [
    (torch.float32, 30001.0), (torch.float32, -1e6), (torch.bfloat16, -999.0), (torch.float16, -6e4), (torch.float16, 3e4)])
@pytest.mark.parametrize("T,a", TEMPERATURES)
def test_kernel_logits_with_an_offset(cuda, dtype, offset, T, a):
    """A shift of a row's logits drops out, as far as their type holds their differences."""
    for V in (300, 5000):
        z, ids, t, y = make(12, V, 6, torch.float32, torch.float32, cuda)
        z = z.round() + offset
        z[1] = offset                      # all alike
        z[2, V // 2:] = offset + 5
        check(z.to(dtype), ids, t, y, T, a, V)


def masked_logits(V, dtype, device="cpu", wide=None):
    """Rows with a part of the vocabulary masked out: whole blocks of columns, all but the
    teacher's entries and the target, single columns."""
    z, ids, t, y = make(20, V, 6, dtype, torch.float32, device, wide)
    low = torch.finfo(dtype).min
    values = (low, -1e10, -1e9, -3e38, -1e30) if low < -1e5 else (low, -6e4, -3e4, -65504.0, -5e4)
    for r in range(20):
        value = values[r % 5]
        keep = torch.cat([ids[r], y[r: r + 1].clamp_min(0)])
        row = z[r].clone()
        if r < 5:
            z[r] = value                       # everything
        elif r < 10:
            z[r, : V // 2] = value             # the first half: whole threads, warps and blocks begin with it
        elif r < 15:
            z[r, V // 2:] = value
        else:
            z[r, ::3] = value
        z[r, keep] = row[keep]                 # but these
    y[y < 0] = 1
    y[3], y[8] = -100, V
    z[torch.arange(20, device=device), y.clamp(0, V - 1)] = 0.5
    return z, ids, t, y


@pytest.mark.parametrize("T,a", TEMPERATURES)
def test_reference_masked_vocabulary(T, a):
    check(*masked_logits(300, torch.float32), T, a, 300)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,a", TEMPERATURES)
@pytest.mark.parametrize("V,wide", [(7, 7), (300, 300), (1003, 1024), (50257, 50304), (152064, 152064)])
def test_kernel_masked_vocabulary(cuda, V, wide, T, a, dtype):
    check(*masked_logits(V, dtype, cuda, wide), T, a, V)


def far_logits(V, dtype, teacher=torch.float32, device="cpu", wide=None):
    """Rows whose largest logit lies far from 0: masks that left nothing, and others."""
    z, ids, t, y = make(20, V, 6, dtype, teacher, device, wide)
    g = torch.Generator().manual_seed(V)
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    rows = [r for r in range(20) if r % 5]      # (every fifth counts nothing)
    z[rows[0]] = low                            # a mask by the lowest value over everything
    for r, value in zip(rows[1:6], (-1e9, -1e10, -1e30, 3e9, 1e37) if high > 1e5 else (-6e4, -3e4, -65504.0, 6e4, 5e4)):
        z[r] = value
    z[rows[6]] = high
    r = rows[7]                                 # a mask over everything but the teacher's entries and the target
    keep = torch.cat([ids[r], y[r: r + 1]])
    z[r], z[r, keep] = low, z[r, keep].clone()
    r = rows[8]                                 # lowest values, and -inf behind them
    z[r] = low
    z[r, torch.randperm(V, generator=g)[: V // 2].to(device)] = -float("inf")
    z[r, ids[r]] = z[r, y[r]] = low
    for r, base in zip(rows[9:15], (-2.0 ** 26, -2.0 ** 25, -4.66e7, 4.66e7, 2.0 ** 24, -1.2e7)):
        steps = torch.randint(0, 9, z[r].shape, generator=g).to(device)   # next to where the kernel's forms meet
        z[r] = base + 4 * steps if high > 1e5 else steps.to(dtype)
    z[rows[15], : V // 2] = -1e9 if high > 1e5 else low       # ordinary rows with a part masked out
    ids[rows[15]] = V // 2 + torch.arange(6, device=device)
    y[rows[15]] = V - 1
    return z, ids, t, y


@pytest.mark.parametrize("T,a", TEMPERATURES)
def test_reference_logits_far_from_zero(T, a):
    check(*far_logits(300, torch.float32), T, a, 300)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,a", TEMPERATURES)
@pytest.mark.parametrize("V,wide", [(300, 300), (1003, 1024), (50257, 50304), (152064, 152064)])
def test_kernel_logits_far_from_zero(cuda, V, wide, T, a, dtype):
    check(*far_logits(V, dtype, device=cuda, wide=wide), T, a, V)


@pytest.mark.gpu
def test_kernel_low_temperatures(cuda):
    """Ordinary logits over a small temperature are far from 0 as well."""
    for dtype in (torch.float32, torch.float16):
        check(*far_logits(777, dtype, device=cuda), 0.01, 0.5, 777)
        check(*far_logits(777, dtype, device=cuda), 0.001, 1.0, 777)


@pytest.mark.gpu
def test_kernel_a_batch_of_rows_far_from_zero(cuda):
    """More of them than a block looks at together, repeated ids and a target among them."""
    z, ids, t, y = make(2500, 200, 40, torch.bfloat16, torch.float32, cuda)
    z[::2] = torch.finfo(z.dtype).min
    z[1] = 0.5
    ids[::4, 20:] = ids[::4, :1]
    y[::6] = ids[::6, 3]
    check(z, ids, t, y, 2.0, 0.5, 200)
    check(z, ids, t, y, 1.0, 0.5, 200)
