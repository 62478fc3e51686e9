"""Packed documents, a teacher and stretched contexts through the decoder and the trainer."""

import pytest
import torch

import zeroq_b200 as zq
from zeroq_b200.models import DecoderLM, get_config
from zeroq_b200.ops import PackedSequences, RopeScaling
from zeroq_b200.train import Trainer

LENGTHS = [5, 1, 19, 40]


def model(device="cpu", dtype=torch.float32, **kw):
    kw = {"n_layers": 2, "n_kv_heads": 2, "vocab_size": 200, "d_model": 128, "n_heads": 2, "ffn_dim": 192, **kw}
    return DecoderLM(get_config("tiny", **kw), device=device, dtype=dtype).init_dense_(std=0.1, seed=0)


def batch(device="cpu", lengths=LENGTHS, tail=3, k=6, seed=0, vocab=200):
    g = torch.Generator().manual_seed(seed)
    T = sum(lengths) + tail
    ids, y = torch.randint(0, vocab, (2, 1, T), generator=g)
    y[0, sum(lengths):] = -100
    y[0, ::7] = -100
    top = torch.stack([torch.randperm(vocab, generator=g)[:k] for _ in range(T)])[None]
    cu = torch.tensor([0] + lengths).cumsum(0)
    teacher = (top.to(device), torch.randn(1, T, k, generator=g).to(device))
    return ids.to(device), y.to(device), cu.to(device), teacher


@pytest.mark.parametrize("scaling", [None, RopeScaling("yarn", 4.0, 16)])
@pytest.mark.parametrize("checkpointing", [False, True])
def test_packed_logits_and_gradients_are_the_documents_own(scaling, checkpointing):
    """fp32 on the CPU: sums of at most 192 products in other orders, 2 layers deep, and a
    normalisation each: 1e-4 of the largest value is over a hundred roundings."""
    m = model(rope_scaling=scaling, activation_checkpointing=checkpointing, train_embeddings=True)
    ids, y, cu, _ = batch()
    loss = m(ids, y, cu_seqlens=cu)
    loss.backward()
    grad = m.embed_tokens.weight.grad.clone()
    m.zero_grad()
    logits = m(ids, cu_seqlens=cu)
    total, counted = 0.0, 0
    for a, b in zip(cu.tolist(), cu.tolist()[1:]):
        alone = m(ids[:, a:b])
        assert (alone - logits[:, a:b]).abs().max() <= 1e-4 * alone.abs().max()
        n = int((y[0, a:b] >= 0).sum())
        if n:
            total = total + m(ids[:, a:b], y[:, a:b]) * n
            counted += n
    total = total / counted
    total.backward()
    assert abs(total.item() - loss.item()) <= 1e-5 * abs(loss.item())
    assert (m.embed_tokens.weight.grad - grad).abs().max() <= 1e-4 * grad.abs().max()


def test_teacher_loss_and_its_limits():
    m = model()
    ids, y, cu, teacher = batch()
    hard = m(ids, y, cu_seqlens=cu)
    assert torch.allclose(m(ids, y, cu_seqlens=cu, teacher=teacher, alpha=0.0), hard, rtol=1e-5)
    soft = m(ids, y, cu_seqlens=cu, teacher=teacher, alpha=1.0, temperature=2.0)
    both = m(ids, y, cu_seqlens=cu, teacher=teacher, alpha=0.25, temperature=2.0)
    assert torch.allclose(both, 0.25 * soft + 0.75 * hard, rtol=1e-5)


def test_refusals():
    m = model()
    ids, y, cu, teacher = batch()
    with pytest.raises(ValueError):
        m(ids.view(2, -1), cu_seqlens=cu)
    with pytest.raises(ValueError):
        m(ids, y, cu_seqlens=PackedSequences(cu, ids.shape[1] + 1))
    with pytest.raises(ValueError):
        m(ids, teacher=teacher)
    m = model("cpu", n_layers=1)
    t = Trainer(m, torch.optim.SGD(m.parameters(), lr=0.0), torch.device("cpu"))
    t._graph_on = True
    with pytest.raises(ValueError):
        t.step_device(ids, y, cu_seqlens=cu)


def test_trainer_step_takes_the_batch():
    m = model(train_embeddings=True)
    ids, y, cu, teacher = batch()
    t = Trainer(m, torch.optim.SGD([p for p in m.parameters() if p.requires_grad], lr=0.1), torch.device("cpu"))
    before = m.embed_tokens.weight.detach().clone()
    loss = t.step_device(ids, y, cu_seqlens=cu, teacher=teacher, alpha=0.5)
    assert torch.isfinite(loss) and not torch.equal(before, m.embed_tokens.weight)


@pytest.mark.gpu
@pytest.mark.parametrize("head_dim", [64, 128])
def test_gpu_documents_do_not_touch_each_other(cuda, head_dim):
    """Rotary, attention and the mixed loss in one training step of a 4-bit model with
    LoRA: a document's logits, and the gradients of its loss, do not move by a bit when
    another document's tokens change."""
    cfg = dict(head_dim=head_dim, d_model=256, n_heads=4, n_kv_heads=2, ffn_dim=512, vocab_size=1000, lora_r=16)
    m = model(cuda, torch.bfloat16, **cfg)
    zq.initialize(m, zq.ZeroQConfig(compute_dtype=torch.bfloat16, compute_in_4bit=True, gather_once=True,
                                    exclude_modules=["lm_head", "embed_tokens"]), trainable_patterns=("lora_", "norm"))
    with torch.no_grad():
        for n, p in m.named_parameters():
            if "lora_B" in n:
                p.normal_(0, 0.02, generator=torch.Generator(device=cuda).manual_seed(1))
    lengths = [130, 77, 300]
    ids, y, cu, teacher = batch(cuda, lengths, tail=5, k=8, vocab=1000)
    y[0, 130:207] = -100                        # the second document trains nothing

    def step(ids):
        m.zero_grad()
        logits = m(ids, cu_seqlens=cu)
        loss = m(ids, y, cu_seqlens=cu, teacher=teacher, temperature=2.0, alpha=0.5)
        loss.backward()
        grads = {n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None}
        return logits.detach(), loss.detach(), grads

    first = step(ids)
    other = ids.clone()
    other[0, 130:207] = (other[0, 130:207] + 17) % 1000
    second = step(other)
    keep = [r for r in range(512) if not 130 <= r < 207]
    assert torch.isfinite(first[1]) and any("lora_A" in n for n in first[2])
    assert torch.equal(first[0][0, keep], second[0][0, keep])
    assert not torch.equal(first[0][0, 130:207], second[0][0, 130:207])
    assert torch.equal(first[1], second[1])
    assert all(torch.isfinite(g).all() for g in first[2].values())


@pytest.mark.gpu
def test_gpu_trainer_steps_on_changing_divisions(cuda):
    m = model(cuda, torch.bfloat16, head_dim=128, d_model=256, lora_r=16, rope_scaling=RopeScaling("linear", 2.0))
    zq.initialize(m, zq.ZeroQConfig(compute_dtype=torch.bfloat16, compute_in_4bit=True, gather_once=True,
                                    exclude_modules=["lm_head", "embed_tokens"]), trainable_patterns=("lora_", "norm"))
    opt = zq.ShardedAdamW(m.trainable_parameters(), lr=1e-3)
    t = Trainer(m, opt, cuda)
    for lengths in ([200, 56], [1, 1, 254], [256], [0, 13, 200]):
        ids, y, cu, teacher = batch(cuda, lengths, tail=256 - sum(lengths), k=4)
        assert torch.isfinite(t.step_device(ids, y, cu_seqlens=cu, teacher=teacher, temperature=2.0))
    ids, y, _, _ = batch(cuda, [256], tail=0)
    assert torch.isfinite(t.step_device(ids, y))   # unpacked, with the scaled positions
    from zeroq_b200.ops import _ext
    assert _ext.ext().gemm_status(0)[0] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [True, False])
def test_gpu_forward_mode_is_refused(cuda, grad):
    """A tangent is not dropped without a word, with the backward's graph or without."""
    from torch.autograd import forward_ad

    from zeroq_b200.ops import distillation_loss, flash_attention_varlen, rotary_embedding

    q = torch.randn(8, 2, 64, device=cuda, dtype=torch.bfloat16)
    z = torch.randn(8, 50, device=cuda)
    pos, cu = torch.arange(8, device=cuda), torch.tensor([0, 8], dtype=torch.int32, device=cuda)
    top = torch.zeros(8, 2, dtype=torch.int64, device=cuda), torch.zeros(8, 2, device=cuda)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        dual, dz = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (q, z))
        for call in (lambda: rotary_embedding(dual, None, pos), lambda: rotary_embedding(q, dual, pos),
                     lambda: flash_attention_varlen(q, q, dual, cu), lambda: flash_attention_varlen(dual, q, q, cu),
                     lambda: distillation_loss(dz, *top), lambda: distillation_loss(dz, *top, reduction="none")):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


@pytest.mark.gpu
@pytest.mark.parametrize("head_dim", [64, 128])
def test_gpu_gradients_of_rows_stay_within_their_document(cuda, head_dim):
    """The loss's gradient with respect to the tokens' embeddings: 0 for every row of a
    document without targets and of the padding, and for the other rows the same to the bit
    whatever tokens that document holds.  (The weights' gradients are sums over the rows by
    atomics, in any order.)"""
    cfg = dict(head_dim=head_dim, d_model=256, n_heads=4, n_kv_heads=2, ffn_dim=512, vocab_size=1000, lora_r=16)
    m = model(cuda, torch.bfloat16, **cfg)
    zq.initialize(m, zq.ZeroQConfig(compute_dtype=torch.bfloat16, compute_in_4bit=True, gather_once=True,
                                    exclude_modules=["lm_head", "embed_tokens"]), trainable_patterns=("lora_", "norm"))
    with torch.no_grad():
        for n, p in m.named_parameters():
            if "lora_B" in n:
                p.normal_(0, 0.02, generator=torch.Generator(device=cuda).manual_seed(1))
    ids, y, cu, teacher = batch(cuda, [130, 77, 300], tail=5, k=8, vocab=1000)
    y[0, 130:207] = -100
    leaves = []

    def leaf(module, args, out):
        leaves.append(out.detach().requires_grad_())
        return leaves[-1]

    m.embed_tokens.register_forward_hook(leaf)

    def gradient(ids):
        m.zero_grad()
        m(ids, y, cu_seqlens=cu, teacher=teacher, temperature=2.0, alpha=0.5).backward()
        return leaves[-1].grad[0]

    first = gradient(ids)
    other = ids.clone()
    other[0, 130:207] = (other[0, 130:207] + 17) % 1000
    second = gradient(other)
    for g in (first, second):
        assert torch.isfinite(g).all() and (g[:130] != 0).any(-1).float().mean() > 0.9
        assert (g[130:207] == 0).all() and (g[507:] == 0).all()
    assert torch.equal(first[:130], second[:130]) and torch.equal(first[207:], second[207:])


_FIRST_CALL = """
import sys, torch
sys.path.insert(0, {root!r})
from zeroq_b200.ops import _ext, distillation_loss, flash_attention_varlen, rotary_embedding
dev = torch.device("cuda", 0)
q = torch.randn(100, 2, 64, device=dev, dtype=torch.bfloat16)
cu = torch.tensor([0, 60, 100], dtype=torch.int32, device=dev)
z, pos = torch.randn(8, 50, device=dev), torch.arange(100, device=dev)
top = torch.zeros(8, 2, dtype=torch.int64, device=dev), torch.zeros(8, 2, device=dev)
calls = dict(attention=lambda: flash_attention_varlen(q, q, q, cu), rotary=lambda: rotary_embedding(q, None, pos)[0],
             distill=lambda: distillation_loss(z, *top))
call = calls[{name!r}]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = call()
graph.replay()
torch.cuda.synchronize()
assert torch.equal(y, call()) and _ext.ext().gemm_status(0)[0] == 0
"""


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["attention", "rotary", "distill"])
def test_gpu_first_call_of_a_process_may_be_captured(cuda, name):
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", _FIRST_CALL.format(root=root, name=name)], capture_output=True,
                          text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
