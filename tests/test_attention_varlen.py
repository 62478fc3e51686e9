"""flash_attention_varlen and PackedSequences against the formulas in 64 bits.

Tolerances, with u = half a step of the type and e = 2^-11 (the exponentials' 2^-13.6, as it
enters P and, through the row sums, again; and the scores' 32-bit products):
  O   (u + e) sum P|v| + u|O|
  dV  (u + e) sum P|dO| + u|dV|
  dS  (u + e)|dS| + P (sum |dO| tol(O)), since delta is formed from the rounded O
  dQ  scale sum tol(dS)|K| + u|dQ|, dK likewise.
fp16 P and dS below the normal range are off by up to 2^-25 each."""

import math

import pytest
import torch

from zeroq_b200.ops import PackedSequences, flash_attention_varlen
from zeroq_b200.ops.attention import attention_varlen_reference

E = 2.0 ** -11


def inputs(lengths, tail, hq, hk, D, dtype, device, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    T = sum(lengths) + tail
    qkv = (torch.randn(T, (hq + 2 * hk) * D, generator=g) * std).to(dtype).to(device)
    q = qkv[:, : hq * D].view(T, hq, D)
    k = qkv[:, hq * D: (hq + hk) * D].view(T, hk, D)
    v = qkv[:, (hq + hk) * D:].view(T, hk, D)
    do = torch.randn(T, hq, D, generator=g).to(dtype).to(device)
    cu = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).to(device)
    return q, k, v, do, cu


def exact(q, k, v, do, lengths, causal, scale):
    """Outputs, gradients and their tolerances (as factors above) in 64 bits, on the inputs' device."""
    u = torch.finfo(q.dtype).eps / 2
    sub = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    dev = q.device
    q, k, v, do = (t.detach().double() for t in (q, k, v, do))
    share = q.shape[1] // k.shape[1]
    zero = lambda t: torch.zeros_like(t)  # noqa: E731
    out = {n: (zero(t), zero(t)) for n, t in (("o", q), ("dq", q), ("dk", k), ("dv", v))}
    a = 0
    for n in lengths:
        r = slice(a, a + n)
        a += n
        hidden = torch.ones(n, n, dtype=torch.bool, device=dev).triu(1) if causal else None
        for h in range(q.shape[1]):
            hk = h // share
            Q, K, V, G = q[r, h], k[r, hk], v[r, hk], do[r, h]
            s = Q @ K.T * scale
            if causal:
                s = s.masked_fill(hidden, -math.inf)
            p = torch.softmax(s, -1) if n else s
            seen = (p > 0).double()
            o = p @ V
            to = (u + E) * (p @ V.abs()) + u * o.abs() + sub * (seen @ V.abs())
            ds = p * (G @ V.T - (G * o).sum(-1, keepdim=True))
            tds = (u + E) * ds.abs() + p * (G.abs() * to).sum(-1, keepdim=True) + sub * seen
            for name, at, value, tol in (
                    ("o", h, o, to),
                    ("dq", h, scale * ds @ K, scale * tds @ K.abs()),
                    ("dk", hk, scale * ds.T @ Q, scale * tds.T @ Q.abs()),
                    ("dv", hk, p.T @ G, (u + E) * (p.T @ G.abs()) + sub * (seen.T @ G.abs()))):
                out[name][0][r, at] += value
                out[name][1][r, at] += tol
    for name in ("dq", "dk", "dv"):
        out[name][1].add_(u * out[name][0].abs())
    if sub:
        for name in out:
            out[name][1].add_(sub)
    return out


def check(lengths, tail, hq, hk, D, dtype, device, causal=True, scale=None, seed=0, std=1.0, poison=False):
    q, k, v, do, cu = inputs(lengths, tail, hq, hk, D, dtype, device, seed, std)
    if poison:   # padding rows that hold anything
        for t in (q, k, v, do):
            t[sum(lengths):] = float("nan")
            t[sum(lengths)::2] = float("inf")
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = flash_attention_varlen(*leaves, cu, causal=causal, scale=scale)
    got = dict(zip(("o", "dq", "dk", "dv"), (o.detach(),) + torch.autograd.grad(o, leaves, do)))
    want = exact(q, k, v, do, lengths, causal, 1 / math.sqrt(D) if scale is None else scale)
    for name, (value, tol) in want.items():
        x = got[name]
        assert x.dtype == dtype and x.shape == value.shape
        assert (x[sum(lengths):] == 0).all(), name
        off = (x.double() - value).abs()
        assert (off <= tol).all(), (name, (off / tol.clamp_min(1e-300)).max().item(), off.max().item())


# ---------------------------------------------------------------------------
@pytest.mark.parametrize("causal", [True, False])
def test_reference_matches_formula(causal):
    check([3, 0, 17, 1, 40], 5, 4, 2, 24, torch.float32, "cpu", causal)


def test_reference_gradient_against_differences():
    q, k, v, do, cu = inputs([3, 4], 1, 2, 1, 4, torch.float64, "cpu")
    f = lambda *t: flash_attention_varlen(*t, cu)  # noqa: E731
    assert torch.autograd.gradcheck(f, tuple(t.clone().requires_grad_() for t in (q, k, v)))


def test_positions_and_bounds():
    s = PackedSequences(torch.tensor([0, 3, 3, 7]), 9)
    assert s.positions.tolist() == [0, 1, 2, 0, 1, 2, 3, 0, 0]
    assert s.bounds() == [(0, 3), (3, 3), (3, 7)]


@pytest.mark.parametrize("cu,total", [([0, 8], 8), (None, 8), (torch.tensor([0, 8]), 8.5), (torch.tensor([0, 8]), None)])
def test_packed_refuses_other_kinds_of_arguments(cu, total):
    with pytest.raises(TypeError, match="PackedSequences"):
        PackedSequences(cu, total)


@pytest.mark.parametrize("seqs", [[0, 8], None, 8])
def test_attention_refuses_other_kinds_of_divisions(seqs):
    q = torch.zeros(8, 2, 16)
    with pytest.raises(TypeError, match="flash_attention_varlen"):
        flash_attention_varlen(q, q, q, seqs)


def test_attention_refuses_heads_of_no_width():
    q = torch.zeros(8, 2, 0)
    with pytest.raises(ValueError, match="flash_attention_varlen"):
        flash_attention_varlen(q, q, q, torch.tensor([0, 8]))


def test_a_division_is_the_one_it_was_made_with():
    cu = torch.tensor([0, 3, 8], dtype=torch.int32)
    q = torch.randn(8, 2, 16)
    s = PackedSequences(cu, 8)
    want = flash_attention_varlen(q, q, q, s)
    cu[1] = 6                       # the caller's tensor goes on to the next batch
    assert s.bounds() == [(0, 3), (3, 8)] and s.positions.tolist() == [0, 1, 2, 0, 1, 2, 3, 4]
    assert torch.equal(flash_attention_varlen(q, q, q, s), want)


def test_a_device_by_another_spelling():
    """"cpu:0" for "cpu", as "cuda" for "cuda:0": the device is the one that the rows are on."""
    q = torch.randn(8, 2, 16)
    s = PackedSequences(torch.tensor([0, 3, 8]), 8, device="cpu:0")
    assert s.device == q.device == s.cu_seqlens.device
    assert torch.equal(flash_attention_varlen(q, q, q, s), flash_attention_varlen(q, q, q, torch.tensor([0, 3, 8])))


@pytest.mark.gpu
def test_a_device_without_an_index(cuda):
    q = torch.randn(8, 2, 64, device=cuda, dtype=torch.bfloat16)
    for cu in (torch.tensor([0, 3, 8]), torch.tensor([0, 3, 8], dtype=torch.int32, device=cuda)):
        s = PackedSequences(cu, 8, device="cuda")
        assert s.device == q.device == s.positions.device
        assert torch.equal(flash_attention_varlen(q, q, q, s), flash_attention_varlen(q, q, q, cu))


@pytest.mark.parametrize("cu,total", [
    (torch.tensor([1, 3]), 5), (torch.tensor([0, 4, 3]), 5), (torch.tensor([0, 6]), 5), (torch.tensor([[0, 3]]), 5),
    (torch.tensor([0.0, 3.0]), 5), (torch.tensor([], dtype=torch.int32), 5), (torch.tensor([0]), -1)])
def test_packed_refusals(cu, total):
    with pytest.raises((ValueError, TypeError)):
        PackedSequences(cu, total)


@pytest.mark.parametrize("bad", [
    dict(q=torch.zeros(8, 4)), dict(k=torch.zeros(7, 2, 16)), dict(v=torch.zeros(8, 1, 16)),
    dict(q=torch.zeros(8, 3, 16)), dict(k=torch.zeros(8, 2, 16).double()), dict(scale=0.0), dict(scale=-1.0),
    dict(scale=float("nan")), dict(seqs=PackedSequences(torch.tensor([0, 9]), 9)), dict(seqs=torch.tensor([0, 9]))])
def test_refusals(bad):
    args = dict(q=torch.zeros(8, 4, 16), k=torch.zeros(8, 2, 16), v=torch.zeros(8, 2, 16), seqs=torch.tensor([0, 8]))
    args.update(bad)
    with pytest.raises((ValueError, TypeError)):
        flash_attention_varlen(**args)


# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("lengths,tail", [
    ([], 5), ([0, 0], 0), ([1], 0), ([128, 256, 0, 1, 300, 129], 17), ([5000, 3, 0, 700], 1),
    ([i % 7 for i in range(3000)], 40), ([70000, 2000], 0)])
def test_plan_tables(cuda, lengths, tail):
    T = sum(lengths) + tail
    cu = torch.tensor([0] + lengths).cumsum(0)
    s = PackedSequences(cu.to(cuda), T)
    host = PackedSequences(cu, T)
    assert torch.equal(s.positions.cpu(), host.positions)
    n = len(lengths)
    words = s.plan.cpu()
    caps = [(T + 255) // 256 + n] + [(T + 127) // 128 + n] * 2
    tables, at = [], 0
    for c in caps:
        tables.append(words[at: at + 4 * c].view(c, 4))
        at += 4 * c
    meta = words[at: at + 5].tolist()
    assert meta[3:] == [0, sum(lengths)]
    for kind, rows in enumerate((256, 128, 128)):
        want, slot = set(), 0
        for a, b in host.bounds():
            for t in range(0, (b - a + rows - 1) // rows):
                want.add((a, b - a, t, slot))
                slot += 1
        got = [tuple(r) for r in tables[kind][: meta[kind]].tolist()]
        assert len(got) == len(set(got)) == meta[kind] and set(got) == want
        work = [(L - t * rows if kind == 2 else min(t * rows + rows, L)) for _, L, t, _ in got]
        unit = 64
        while (T + 63) // unit >= 1024:
            unit *= 2
        cls = [(w + 63) // 64 * 64 // unit for w in work]
        assert cls == sorted(cls, reverse=True)


@pytest.mark.gpu
@pytest.mark.parametrize("extra", [0, 2])
def test_plan_of_more_tiles_than_32_bits_count(cuda, extra):
    """2^18 sequences over all of 2^20 rows, which fall back to 0 in between: 2^31 tiles of
    128 rows.  The tables keep the sequences that fit, and nothing else."""
    T, pairs = 1 << 20, (1 << 18) + extra
    cu = torch.tensor([0, T], dtype=torch.int32, device=cuda).repeat(pairs)
    n = cu.numel() - 1
    s = PackedSequences(cu, T)
    words, at = s.plan.cpu(), 0
    caps = [T // 256 + n] + [T // 128 + n] * 2
    meta = words[4 * sum(caps):][:3].tolist()
    for cap, count, rows in zip(caps, meta, (256, 128, 128)):
        fit = cap // (T // rows)                         # whole sequences
        assert count == fit * (T // rows)
        start, length, tile, slot = words[at: at + 4 * count].view(count, 4).unbind(1)
        at += 4 * cap
        assert (start == 0).all() and (length == T).all()
        assert torch.equal(slot.sort().values, torch.arange(count, dtype=torch.int32))
        assert torch.equal(tile, slot % (T // rows))
    from zeroq_b200.ops import _ext
    assert _ext.ext().gemm_status(0)[0] == 324


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,tail,hq,hk,D", [
    ([1], 0, 1, 1, 128),
    ([128], 0, 2, 1, 128),
    ([1, 63, 64, 65, 127, 128, 129], 3, 4, 2, 128),
    ([255, 256, 257, 0, 383, 1], 0, 3, 1, 64),
    ([700, 2, 513], 100, 7, 1, 80),
    ([33, 300], 1, 2, 2, 8),
    ([200, 129, 77], 0, 4, 4, 72),
    ([1025], 0, 6, 3, 120)])
def test_kernels_match_formula(cuda, dtype, causal, lengths, tail, hq, hk, D):
    check(lengths, tail, hq, hk, D, dtype, cuda, causal, seed=sum(lengths) + D)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_kernels_long_and_many(cuda, D):
    check([4097, 100], 0, 2, 1, D, torch.bfloat16, cuda)
    check([(i * 37) % 90 for i in range(60)], 9, 2, 2, D, torch.bfloat16, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
def test_unset_padding_does_not_enter(cuda, causal):
    check([130, 1, 60, 255], 150, 4, 2, 128, torch.bfloat16, cuda, causal, poison=True)
    check([130, 1, 60, 255], 150, 4, 2, 64, torch.float16, cuda, causal, poison=True)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
def test_a_neighbour_does_not_enter(cuda, causal):
    """A document of NaN and infinities between two others changes neither."""
    lengths = [100, 77, 200]
    q, k, v, do, cu = inputs(lengths, 0, 4, 2, 128, torch.bfloat16, cuda)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    o = flash_attention_varlen(*leaves, cu, causal=causal)
    clean = (o.detach(),) + torch.autograd.grad(o, leaves, do)
    for t in (q, k, v, do):
        t[100:177] = float("nan")
        t[120:130] = float("inf")
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    o = flash_attention_varlen(*leaves, cu, causal=causal)
    dirty = (o.detach(),) + torch.autograd.grad(o, leaves, do)
    for a, b in zip(clean, dirty):
        assert torch.equal(a[:100], b[:100]) and torch.equal(a[177:], b[177:])


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_a_later_value_does_not_enter_however_large(cuda, D):
    """A masked key's weight is 0, not merely small: values near the type's largest behind
    the mask change no row before them."""
    q, k, v, do, cu = inputs([300, 60], 9, 4, 2, D, torch.bfloat16, cuda)
    v = v.contiguous()
    clean = flash_attention_varlen(q, k, v, cu)
    for first in (1, 64, 150, 257):
        large = v.clone()
        large[first:300] = 2.0 ** 127
        o = flash_attention_varlen(q, k, large, cu)
        assert torch.equal(o[:first], clean[:first]) and torch.equal(o[300:], clean[300:])


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_scores_that_overflow_downwards_weigh_nothing(cuda, D):
    """The first 150 keys, a whole key tile among them, score -2^140 scale: -inf in 32 bits."""
    q, k, v, do, cu = inputs([300], 0, 2, 1, D, torch.bfloat16, cuda)
    q, k = torch.zeros_like(q), k.clone()
    q[..., 0] = 2.0 ** 70
    k[..., 0] = 0
    k[:150, :, 0] = -2.0 ** 70
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = flash_attention_varlen(*leaves, cu)
    got = (o.detach(),) + torch.autograd.grad(o, leaves, do)
    want = exact(q, k, v, do, [300], True, 1 / math.sqrt(D))
    for x, (value, tol) in zip(got, want.values()):   # the rows before see nothing else
        assert ((x[150:].double() - value[150:]).abs() <= tol[150:]).all()
    assert torch.isnan(got[0][:150]).all()


@pytest.mark.gpu
def test_large_scores_move_the_running_maximum(cuda):
    check([600, 300], 0, 2, 1, 128, torch.bfloat16, cuda, seed=3, std=1.0, scale=1.0)
    check([600, 300], 0, 2, 1, 64, torch.bfloat16, cuda, causal=False, seed=4, scale=0.01)


@pytest.mark.gpu
def test_strides_shared_plan_and_partial_gradients(cuda):
    lengths = [150, 90]
    q, k, v, do, cu = inputs(lengths, 0, 4, 2, 64, torch.bfloat16, cuda)
    seqs = PackedSequences(cu.long().cpu(), 240, device=cuda)
    want = flash_attention_varlen(q.contiguous(), k.contiguous(), v.contiguous(), cu)
    heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert torch.equal(flash_attention_varlen(*heads_first, seqs), want)
    odd = [torch.empty(240 * t.shape[1] * 64 + 1, device=cuda, dtype=t.dtype)[1:].view(t.shape).copy_(t) for t in (q, k, v)]
    assert torch.equal(flash_attention_varlen(*odd, seqs), want)
    one = k[:, :1].expand(240, 2, 64)     # one kv head for both
    assert torch.equal(flash_attention_varlen(q, one, one, seqs),
                       flash_attention_varlen(q, one.contiguous(), one.contiguous(), seqs))
    leaf = q.detach().requires_grad_()
    flash_attention_varlen(leaf, k, v, seqs).sum().backward()     # an expanded gradient; k, v take none
    full = q.detach().requires_grad_()
    o = flash_attention_varlen(full, k, v, seqs)
    o.backward(torch.ones_like(o))
    assert torch.equal(leaf.grad, full.grad)


@pytest.mark.gpu
def test_no_sequence_one_head_and_one_row(cuda):
    q = torch.randn(70, 2, 64, device=cuda, dtype=torch.bfloat16, requires_grad=True)
    o = flash_attention_varlen(q, q, q, torch.zeros(1, dtype=torch.int32, device=cuda))
    dq, = torch.autograd.grad(o, q, torch.ones_like(o))
    assert (o == 0).all() and (dq == 0).all()
    # axes of one with strides that no tensor map could take
    base = torch.randn(40 * 64, device=cuda, dtype=torch.bfloat16)
    odd = base.as_strided((40, 1, 64), (64, 3, 1))
    cu = torch.tensor([0, 40], dtype=torch.int32, device=cuda)
    assert torch.equal(flash_attention_varlen(odd, odd, odd, cu), flash_attention_varlen(*[base.view(40, 1, 64)] * 3, cu))
    one = base.as_strided((1, 2, 64), (7, 64, 1))
    cu1 = torch.tensor([0, 1], dtype=torch.int32, device=cuda)
    assert torch.equal(flash_attention_varlen(one, one, one, cu1), one)


@pytest.mark.gpu
def test_sequences_out_of_order_stay_in_bounds(cuda):
    """The host cannot see such a division: it gives nothing useful, within the buffers."""
    q = torch.randn(300, 2, 64, device=cuda, dtype=torch.bfloat16, requires_grad=True)
    for cu in ([0, 300, 0, 300, 0, 300, 0, 300], [-50, 7000, 2 ** 31 - 1], [200, 100, -2 ** 31, 150], [300, 0]):
        o = flash_attention_varlen(q, q, q, torch.tensor(cu, device=cuda).to(torch.int32))
        torch.autograd.grad(o, q, torch.ones_like(o))
    torch.cuda.synchronize()
    from zeroq_b200.ops import _ext
    assert _ext.ext().gemm_status(0)[0] in (0, 324)   # 324: a division with more tiles than rows could give
    assert _ext.ext().gemm_status(0)[0] == 0


@pytest.mark.gpu
def test_second_derivatives_are_refused(cuda):
    q, k, v, do, cu = inputs([10], 0, 2, 2, 64, torch.bfloat16, cuda)
    leaf = q.detach().requires_grad_()
    o = flash_attention_varlen(leaf, k, v, cu)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(o, leaf, do, create_graph=True)


@pytest.mark.gpu
def test_kernel_refusals(cuda):
    q, k, v, do, cu = inputs([10], 0, 2, 2, 128, torch.bfloat16, cuda)
    with pytest.raises(TypeError):
        flash_attention_varlen(q.float(), k.float(), v.float(), cu)
    for D in (4, 12, 136):
        t = torch.zeros(10, 2, D, device=cuda, dtype=torch.bfloat16)
        with pytest.raises(ValueError):
            flash_attention_varlen(t, t, t, cu)
    with pytest.raises(ValueError):
        flash_attention_varlen(q, k, v, PackedSequences(torch.tensor([0, 10]), 10))   # on the CPU
    from zeroq_b200.ops import _ext
    s = PackedSequences(cu, 10)
    with pytest.raises(RuntimeError, match="plan"):
        _ext.ext().attn_varlen_fwd(q, k, v, s.plan, 2, torch.empty_like(q), torch.empty(2, 10, device=cuda), None, True, 0.1)


@pytest.mark.gpu
def test_repeatable_in_a_graph_with_changing_sequences(cuda):
    q, k, v, do, cu = inputs([200, 300, 12], 0, 4, 2, 128, torch.bfloat16, cuda)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]

    def step():
        o = flash_attention_varlen(*leaves, cu)
        return (o.detach(),) + torch.autograd.grad(o, leaves, do)

    first = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, side))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for lengths in ([200, 300, 12], [1, 500, 11], [512, 0, 0]):
        cu.copy_(torch.tensor([0] + lengths).cumsum(0).to(torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))
    from zeroq_b200.ops import _ext
    assert _ext.ext().gemm_status(0)[0] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128])
def test_blocks_that_take_over_items(cuda, dtype, causal, D):
    """Several dQ items (128 queries of a head) to each SM: documents of one to three key
    tiles between longer ones, so that items start on odd and even key tiles."""
    lengths = [60, 100, 190, 700, 30, 129, 400, 64, 65, 0, 1, 1000, 130, 20, 150, 63]
    sms = torch.cuda.get_device_properties(cuda).multi_processor_count
    per_head = sum((n + 127) // 128 for n in lengths)
    hk = 3 * sms // (2 * per_head) + 1
    hq = 2 * hk
    assert per_head * hq > 3 * sms
    check(lengths, 77, hq, hk, D, dtype, cuda, causal, seed=D)
    q, k, v, do, cu = inputs(lengths, 77, hq, hk, D, dtype, cuda, seed=D)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]

    def step():
        o = flash_attention_varlen(*leaves, cu, causal=causal)
        return (o.detach(),) + torch.autograd.grad(o, leaves, do)

    first = step()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, step()))
    from zeroq_b200.ops import _ext
    assert _ext.ext().gemm_status(0)[0] == 0


@pytest.mark.gpu
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two devices")
def test_tensors_on_another_device_than_the_current_one(cuda):
    other = torch.device("cuda", 1)
    with torch.cuda.device(0):   # (the first work of this device: its status words are set up there)
        check([130, 1, 60], 5, 4, 2, 128, torch.bfloat16, other)
        from zeroq_b200.ops import _ext
        assert _ext.ext().gemm_status(1)[0] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,lost", [(torch.bfloat16, 8), (torch.float16, 5)])
def test_the_forward_keeps_eight_more_bits_of_o(cuda, dtype, lost):
    """Equal scores: every weight is 1 and the sum of a row's is in its lse, so the 32-bit O
    is sum(v) exp(-lse).  With its byte O lacks the pattern's last `lost` bits, 2^(lost - 23)
    of it; lse's logarithm adds 2^-20, and sums of up to 40 values 40 steps of 2^-23 of their
    mean size.  A value of 32 bits lies at a tie that is rounded down (the kept bits even, those
    behind them 100..0) with probability 2^-(lost + 9); its byte reads the other way.  Rows of
    two and three keys must not do so more often.  Heads share their values in pairs here, so
    of N values at most N 2^-(lost + 9) and six deviations, of pairs, are such."""
    from zeroq_b200.ops import _ext

    lengths = list(range(1, 41))
    q, k, v, do, cu = inputs(lengths, 0, 4, 2, 64, dtype, cuda)
    q = torch.zeros_like(q)
    seqs = PackedSequences(cu, q.shape[0])
    o, low = torch.empty_like(q), torch.empty(q.shape, dtype=torch.int8, device=cuda)
    lse = torch.empty(4, q.shape[0], device=cuda)
    _ext.ext().attn_varlen_fwd(q, k, v, seqs.plan, seqs.n, o, lse, low, True, 0.125)
    got = (o.float().view(torch.int32) + (low.int() << lost)).view(torch.float32).double()
    got = torch.where(o == 0, 0.0, got)
    total, size, a = torch.zeros_like(got), torch.zeros_like(got), 0
    for n in lengths:
        r = slice(a, a + n)
        a += n
        both = v[r].double().repeat_interleave(2, 1)
        total[r], size[r] = both.cumsum(0), both.abs().cumsum(0)
    down = torch.exp(-lse.double()).T[:, :, None]
    want, size = total * down, size * down
    off = (got - want).abs()
    tol = (2.0 ** (lost - 23) + 2.0 ** -20) * want.abs() + 40 * 2.0 ** -23 * size
    if dtype == torch.float16:   # below the normal range the byte counts 2^-11 of the value
        tol = tol + torch.where(want.abs() < 2.0 ** -14, 2.0 ** -11 * want.abs() + 2.0 ** -25, 0.0)
    ties = off.numel() * 2.0 ** -(lost + 9)
    wrong = off > tol
    assert wrong.sum() <= ties + 6 * math.sqrt(2 * ties) and (low[wrong] == -128).all()
    assert ((o.double() - want).abs() > tol).float().mean() > 0.5    # (what the byte is for)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_delta_is_formed_from_them(cuda, dtype):
    """Two tokens with one key: dS of the second is +d and -d, whose sum is twice what delta
    is off by, so dQ = 0 unless the two round apart.  Off by 2^-16 of O, at steps of 2^-8 of
    d, a few rows in a hundred do; from the rounded O half of them would."""
    q, k, v, do, cu = inputs([2] * 400, 0, 4, 4, 64, dtype, cuda)
    k = k.clone()
    k[1::2] = k[::2]
    leaf = q.detach().requires_grad_()
    o = flash_attention_varlen(leaf, k, v, cu)
    dq, = torch.autograd.grad(o, leaf, do)
    assert (dq[1::2] != 0).any(-1).float().mean() < 0.1


@pytest.mark.gpu
def test_many_short_and_empty_sequences(cuda):
    check([1, 0, 2, 3, 0, 0, 65, 1, 5, 130] * 20, 3, 4, 2, 64, torch.bfloat16, cuda)
    check([1, 0, 2, 3, 0, 0, 65, 1, 5, 130] * 20, 0, 2, 2, 128, torch.float16, cuda, causal=False)


@pytest.mark.gpu
def test_the_backwards_workspace_goes_with_the_rows(cuda):
    """20000 sequences of one token, 8 heads: statistics of 128 rows each were 165 MB; inputs,
    outputs and gradients are 2.6 MB each."""
    T = 20000
    q, k, v, do = (torch.randn(T, 8, 8, device=cuda, dtype=torch.bfloat16) for _ in range(4))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    seqs = PackedSequences(torch.arange(T + 1, dtype=torch.int32, device=cuda), T)
    o = flash_attention_varlen(*leaves, seqs)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    dq, dk, dv = torch.autograd.grad(o, leaves, do)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < 40e6
    assert torch.equal(o, v) and torch.equal(dv, do)
    # one key: P = 1 and dS = 0, off by sum |dO| tol(O) as above
    u = 2.0 ** -8
    off = (do.double().abs() * (2 * u + E) * v.double().abs()).sum(-1, keepdim=True) * 8 ** -0.5 * (1 + u)
    assert (dq.double().abs() <= off * k.double().abs()).all() and (dk.double().abs() <= off * q.double().abs()).all()
