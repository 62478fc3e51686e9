"""embedding, layer norm, 8-bit activations and token log probabilities together in the decoder
and the trainer, in checkpoints, on other streams and in captured graphs."""

import copy

import pytest
import torch

import zeroq_b200 as zq
from zeroq_b200.models import DecoderLM, LayerNorm, get_config
from zeroq_b200.ops import (add_layer_norm, checkpoint_8bit, dequantize_activation, embedding, gelu, layer_norm,
                            quantize_activation, swiglu, token_logprobs)
from zeroq_b200.train import Trainer
from zeroq_b200.utils.checkpoint import enable_gradient_checkpointing

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.fixture(params=DEVICES)
def device(request):
    if request.param == "cuda":
        request.getfixturevalue("cuda")
    return request.param


def model(device="cpu", dtype=torch.float32, seed=0, **more):
    cfg = get_config("tiny", **{"d_model": 64, "n_layers": 2, "n_heads": 2, "n_kv_heads": 2, "head_dim": 32, "ffn_dim": 96,
                                "vocab_size": 200, "norm": "layernorm", "embed_scale": 8.0, "train_embeddings": True, **more})
    torch.manual_seed(seed)
    m = DecoderLM(cfg, device=device, dtype=dtype).init_dense_(seed=seed)
    return m


def batch(device="cpu", B=2, S=24, vocab=200):
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(0, vocab, (B, S), generator=g)
    y = torch.roll(ids, -1, 1)
    y[:, :5] = -100
    return ids.to(device), y.to(device)


def grads(m):
    return {n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None}


def test_logprobs_are_the_loss_and_a_teacher():
    m = model()
    ids, y = batch()
    out = m.logprobs(ids, y, top_k=6)
    assert out.logprobs.shape == (2, 24) and out.top_ids.shape == (2, 24, 6)
    loss = m(ids, y)
    assert torch.allclose(-out.logprobs.sum() / (y != -100).sum(), loss, rtol=1e-5)
    m.zero_grad()
    loss.backward()
    a = grads(m)
    m.zero_grad()
    (-out.logprobs.sum() / (y != -100).sum()).backward()
    b = grads(m)
    assert set(a) == set(b) and any("norm.bias" in n for n in a) and "embed_tokens.weight" in a
    for n in a:
        assert torch.allclose(a[n], b[n], rtol=1e-4, atol=1e-6), n
    # the top alternatives of the model itself as a teacher: no distance where they hold everything
    whole = m.logprobs(ids, y, top_k=200)
    teacher = (whole.top_ids, whole.top_logprobs.detach())
    assert abs(float(m(ids, y, teacher=teacher, alpha=1.0).detach())) < 1e-5
    assert m.logprobs(ids).logprobs is None


def test_embedding_scale_and_padding():
    m, plain = model(), model(embed_scale=None)
    plain.load_state_dict(m.state_dict())
    ids, _ = batch()
    assert torch.allclose(m.embed_tokens(ids), 8.0 * plain.embed_tokens(ids))
    assert (m.embed_tokens(torch.full((1, 3), -100)) == 0).all()
    assert isinstance(m.norm, LayerNorm)
    assert model(norm="rmsnorm", embed_scale=None)(ids).shape == (2, 24, 200)
    with pytest.raises(ValueError, match="norm is"):
        model(norm="batchnorm")
    with pytest.raises(ValueError, match="'full' or '8bit'"):
        model(saved_activations="4bit")


def test_num_params_counts_the_biases():
    for norm in ("rmsnorm", "layernorm"):
        m = model(norm=norm, embed_scale=None, vocab_size=256)
        assert m.cfg.num_params() == sum(p.numel() for p in m.parameters()), norm


# ---------------------------------------------------------------------------
# checkpoints in 8 bits
# ---------------------------------------------------------------------------
def test_checkpoint_gradients_are_those_at_the_kept_inputs(device):
    torch.manual_seed(0)
    lin = torch.nn.Linear(200, 200).to(device)
    x = torch.randn(6, 200, device=device)
    flag, w = torch.arange(6, device=device), torch.nn.Parameter(torch.randn(200, device=device))

    def fn(x, flag, w, none, scale=1.0):
        assert none is None and flag.dtype == torch.int64
        return torch.tanh(lin(x)) * w * scale + flag[:, None], x * 2

    y, z = checkpoint_8bit(fn, x.requires_grad_(), flag, w, None, scale=3.0)
    want, _ = fn(x, flag, w, None, 3.0)
    assert torch.equal(y, want)
    got = torch.autograd.grad(y.square().sum() + z.sum(), [x, w, *lin.parameters()])
    kept = dequantize_activation(quantize_activation(x)).requires_grad_()
    assert not torch.equal(kept, x)
    y2, z2 = fn(kept, flag, w, None, 3.0)
    expect = torch.autograd.grad([y2, z2], [kept, w, *lin.parameters()], [2 * want.detach(), torch.ones_like(z2)])
    for a, b in zip(got, expect):
        assert torch.equal(a, b)


def test_checkpoint_of_an_input_without_gradient(device):
    """parameters inside get their gradients all the same"""
    lin = torch.nn.Linear(64, 64).to(device)
    x = torch.randn(3, 64, device=device)
    checkpoint_8bit(lin, x).sum().backward()
    assert lin.weight.grad is not None
    with torch.no_grad():
        assert torch.equal(checkpoint_8bit(lin, x), lin(x))
    assert checkpoint_8bit(lambda: 3) == 3


def test_checkpoint_keeps_a_byte_an_element():
    """nothing that the function saves, and no exact input, is held until the backward"""
    import gc
    import weakref

    x = torch.randn(8, 1024, requires_grad=True)
    h = x * 1.0
    seen = []

    def fn(h):
        t = torch.sin(h)
        if torch.is_grad_enabled() and not seen:
            seen.append(weakref.ref(t))
        return torch.exp(t)

    y = checkpoint_8bit(fn, h)
    kept = weakref.ref(h)
    del h
    gc.collect()
    assert kept() is None and seen[0]() is None
    y.sum().backward()
    assert torch.isfinite(x.grad).all()


@pytest.mark.parametrize("checkpointing", [False, True])
def test_decoder_with_8_bits(device, checkpointing):
    """the loss does not move by a bit, the gradients by about the kept inputs' half step"""
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    more = dict(d_model=256, head_dim=64, n_heads=4, n_kv_heads=4, ffn_dim=512)
    for act in ("swiglu", "gelu"):
        full = model(device, dtype, ffn_act=act, **more)
        kept = model(device, dtype, ffn_act=act, saved_activations="8bit", activation_checkpointing=checkpointing, **more)
        kept.load_state_dict(full.state_dict())
        ids, y = batch(device, S=32)
        losses = []
        for m in (full, kept):
            loss = m(ids, y)
            loss.backward()
            losses.append(loss.detach())
        if device == "cpu" or checkpointing:
            assert torch.equal(*losses)
        a, b = grads(full), grads(kept)
        assert set(a) == set(b)
        for n in a:
            # a sanity bound: 1 / 254 of a group's largest in each input is a few per cent of a gradient
            assert (a[n] - b[n]).norm() <= 0.1 * a[n].norm() + 1e-6, n


def test_enable_gradient_checkpointing_in_8_bits():
    m = model()
    ids, y = batch()
    want = m(ids, y)
    enable_gradient_checkpointing(m, saved="8bit")
    loss = m(ids, y)
    assert torch.equal(loss, want)
    loss.backward()
    assert all(p.grad is not None for n, p in m.named_parameters() if p.requires_grad)
    with pytest.raises(ValueError, match="without reentrance"):
        enable_gradient_checkpointing(m, use_reentrant=True, saved="8bit")
    with pytest.raises(ValueError, match="'full' or '8bit'"):
        enable_gradient_checkpointing(m, saved="1bit")
    with pytest.raises(ValueError, match="found none"):
        enable_gradient_checkpointing(torch.nn.Linear(2, 2), saved="8bit")


# ---------------------------------------------------------------------------
# a policy's training step
# ---------------------------------------------------------------------------
def policy_loss(m, ids, y, old, advantage):
    out = m.logprobs(ids, y, temperature=0.9)
    counted = (y != -100).float()
    ratio = (out.logprobs - old).exp()
    return -((ratio * advantage).sum() + 0.01 * (out.entropy * counted).sum()) / counted.sum()


def test_policy_step_gradients_against_differences():
    m = model().double()
    ids, y = batch()
    with torch.no_grad():
        old = m.logprobs(ids, y, temperature=0.9).logprobs - 0.1
    advantage = torch.randn(2, 24, generator=torch.Generator().manual_seed(5), dtype=torch.float64)
    m.zero_grad()
    policy_loss(m, ids, y, old, advantage).backward()
    # Along the gradient the slope is its length.  Rotary positions, attention and the activation
    # round to 32 bits, so a loss of size 1 is off by some 2^-22, the quotient by 2^-22 / eps =
    # 2.4e-4; the third derivative's term is eps^2 |g|^3 at most.
    eps = 1e-3
    for name in ("embed_tokens.weight", "layers.1.mlp_norm.weight", "norm.bias"):
        p = m.get_parameter(name)
        length = float(p.grad.norm())
        d = p.grad / length
        with torch.no_grad():
            p += eps * d
            up = policy_loss(m, ids, y, old, advantage)
            p -= 2 * eps * d
            down = policy_loss(m, ids, y, old, advantage)
            p += eps * d
        assert abs(float((up - down) / (2 * eps)) - length) <= 5e-4 + 1e-3 * length, name


@pytest.mark.gpu
def test_gpu_policy_step_follows_the_cpu(cuda):
    """one step of the whole set in bf16 against the same model in fp32 on the CPU"""
    more = dict(d_model=256, head_dim=64, n_heads=4, n_kv_heads=4, ffn_dim=512, vocab_size=1000)
    ref = model("cpu", **more)
    m = model(cuda, torch.bfloat16, saved_activations="8bit", **more)
    m.load_state_dict(ref.state_dict())
    ids, y = batch(S=64, vocab=1000)
    with torch.no_grad():
        old = ref.logprobs(ids, y, temperature=0.9).logprobs
    advantage = torch.randn(2, 64, generator=torch.Generator().manual_seed(5))
    a = policy_loss(ref, ids, y, old, advantage)
    a.backward()
    b = policy_loss(m, ids.to(cuda), y.to(cuda), old.to(cuda), advantage.to(cuda))
    b.backward()
    assert abs(float(a) - float(b)) < 0.05
    x, z = grads(ref), grads(m)
    for n in x:
        u, v = x[n].flatten(), z[n].float().cpu().flatten()
        assert torch.nn.functional.cosine_similarity(u, v, 0) > 0.97, n


@pytest.mark.gpu
def test_gpu_graph_steps_are_eager_steps(cuda):
    """the trainer's captured step with layer norms, a scaled embedding and 8-bit activations"""
    more = dict(d_model=256, head_dim=64, n_heads=4, n_kv_heads=4, ffn_dim=512, vocab_size=1000, train_embeddings=False,
                lora_r=8, ffn_act="gelu")
    for kw in (dict(saved_activations="8bit"), dict(saved_activations="8bit", activation_checkpointing=True), {}):
        losses = []
        for graph in (False, True):
            m = model(cuda, torch.bfloat16, **more, **kw)
            zq.initialize(m, zq.ZeroQConfig(compute_dtype=torch.bfloat16, compute_in_4bit=True, gather_once=True,
                                            exclude_modules=["lm_head", "embed_tokens"]), trainable_patterns=("lora_", "norm"))
            t = Trainer(m, zq.ShardedAdamW(m.trainable_parameters(), lr=1e-3), cuda)
            if graph:
                t.enable_cuda_graph()
            ids, y = batch(S=64, vocab=1000)
            losses.append([t.step(torch.roll(ids, i, 1), torch.roll(y, i, 1)) for i in range(4)])
        assert torch.allclose(torch.tensor(losses[0]), torch.tensor(losses[1]), rtol=2e-3), losses


# ---------------------------------------------------------------------------
# streams and graphs
# ---------------------------------------------------------------------------
def calls(g, device):
    """name -> (leaves, function of the leaves, upstream gradients)"""
    r = lambda *s, dtype=torch.bfloat16: torch.randn(*s, generator=g).to(device=device, dtype=dtype)  # noqa: E731
    ids = torch.randint(0, 500, (300,), generator=g).to(device)
    many = torch.randint(0, 500, (9000,), generator=g).to(device)
    y = torch.randint(0, 70000, (5,), generator=g).to(device)
    return {
        "embedding": ([r(500, 264)], lambda w: [embedding(ids, w, 2.0)], [r(300, 264)]),
        "embedding_many": ([r(500, 40)], lambda w: [embedding(many, w)], [r(9000, 40)]),
        "norm": ([r(100, 640), r(100, 640), r(640, dtype=torch.float32), r(640, dtype=torch.float32)],
                 lambda x, d, w, b: list(add_layer_norm(x, d, w, b)), [r(100, 640), r(100, 640)]),
        "norm_8bit": ([r(100, 5000), r(5000, dtype=torch.float32)], lambda x, w: [layer_norm(x, w, saved="8bit")], [r(100, 5000)]),
        "gelu": ([r(100, 640)], lambda x: [gelu(x, saved="8bit")], [r(100, 640)]),
        "swiglu": ([r(100, 640), r(100, 640)], lambda x, u: [swiglu(x, u, saved="8bit")], [r(100, 640)]),
        "checkpoint": ([r(64, 640)], lambda x: [checkpoint_8bit(lambda v: gelu(v) * v, x)], [r(64, 640)]),
        "logprobs": ([r(5, 70016)], lambda z: list(token_logprobs(z, y, 7, vocab=70000)[:3]),
                     [r(5, dtype=torch.float32), r(5, dtype=torch.float32), r(5, 7, dtype=torch.float32)]),
    }


NAMES = ["embedding", "embedding_many", "norm", "norm_8bit", "gelu", "swiglu", "checkpoint", "logprobs"]


def run(leaves, fn, ups):
    outs = fn(*leaves)
    return [o.detach() for o in outs] + list(torch.autograd.grad(outs, leaves, ups))


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_gpu_other_streams_and_graphs(cuda, name):
    """the same bits on a side stream, in a captured forward and backward, and replayed on other inputs"""
    leaves, fn, ups = calls(torch.Generator().manual_seed(1), cuda)[name]
    other, _, other_ups = calls(torch.Generator().manual_seed(2), cuda)[name]
    for t in leaves + other:
        t.requires_grad_()
    want, want2 = run(leaves, fn, ups), run(other, fn, other_ups)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(leaves, fn, ups)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    static = [t.detach().clone().requires_grad_() for t in leaves]
    static_ups = [t.clone() for t in ups]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(static, fn, static_ups)
    for values, grads_, expect in ((leaves, ups, want), (other, other_ups, want2), (leaves, ups, want)):
        with torch.no_grad():
            for a, b in zip(static + static_ups, list(values) + list(grads_)):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, expect))


@pytest.mark.gpu
def test_gpu_two_calls_at_once(cuda):
    """two streams, each with its own tensors: nothing is shared"""
    sets = [calls(torch.Generator().manual_seed(s), cuda) for s in (1, 2)]
    for s in sets:
        for leaves, _, _ in s.values():
            for t in leaves:
                t.requires_grad_()
    want = [{n: run(*s[n]) for n in NAMES} for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        got = []
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append({n: run(*s[n]) for n in NAMES})
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for n in NAMES:
                assert all(torch.equal(x, z) for x, z in zip(a[n], b[n])), n


@pytest.mark.gpu
def test_gpu_forward_mode_is_refused(cuda):
    import torch.autograd.forward_ad as fwd

    with fwd.dual_level():
        x = fwd.make_dual(torch.randn(4, 64, device="cuda"), torch.ones(4, 64, device="cuda"))
        y = torch.zeros(4, dtype=torch.int64, device="cuda")
        for call in (lambda: layer_norm(x), lambda: token_logprobs(x, y), lambda: embedding(y, x)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


def test_a_copied_model_keeps_its_choices():
    m = copy.deepcopy(model(saved_activations="8bit"))
    assert m.embed_tokens.scale == 8.0 and m.norm.saved == "8bit" and m.layers[0].act_saved == "8bit"


def test_layer_norm_biases_go_through_checkpoint_files(tmp_path):
    from zeroq_b200.utils.loading import hf_to_decoder_name, save_hf_checkpoint, stream_load

    m = model(vocab_size=256)
    g = torch.Generator().manual_seed(4)
    for n, p in m.named_parameters():
        if "norm" in n:
            p.data += torch.randn(p.shape, generator=g)
    path = str(tmp_path / "model.safetensors")
    save_hf_checkpoint(m, path)
    again = model(seed=1, vocab_size=256)
    counts = stream_load(again, path)
    assert counts["skipped"] == 0 and counts["copied"] == len(list(m.parameters()))
    for (n, a), b in zip(m.named_parameters(), again.parameters()):
        assert torch.equal(a, b), n
    ids, _ = batch()
    assert torch.equal(m(ids), again(ids))
    assert hf_to_decoder_name("model.layers.1.input_layernorm.bias") == "layers.1.attn_norm.bias"
    assert hf_to_decoder_name("model.norm.bias") == "norm.bias"
    # into a decoder whose norms have none
    assert stream_load(model(seed=1, vocab_size=256, norm="rmsnorm"), path)["skipped"] == 5
