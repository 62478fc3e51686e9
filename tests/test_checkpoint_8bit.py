"""What an 8-bit checkpoint keeps in 8 bits and what it keeps as it is: gradients against those of
the same function at the kept activations and the exact rest, to the bit."""

import pytest
import torch

from zeroq_b200.ops import checkpoint_8bit, dequantize_activation, quantize_activation

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.fixture(params=DEVICES)
def device(request):
    if request.param == "cuda":
        request.getfixturevalue("cuda")
    return request.param


def attention(h, mask, bias=None):
    s = h @ h.transpose(-1, -2) / 8 + mask
    return torch.softmax(s if bias is None else s + bias, -1) @ h


def inputs(device, low, S=24):
    torch.manual_seed(1)
    h = torch.randn(2, S, 64).to(device).requires_grad_()
    mask = torch.full((S, S), low).triu(1).to(device)
    return h, mask, torch.randn(2, S, 64).to(device)


def at_kept(h):
    return dequantize_activation(quantize_activation(h)).requires_grad_()


@pytest.mark.parametrize("low", [float("-inf"), torch.finfo(torch.float32).min, -1e9])
def test_a_mask_is_kept_as_it_is(device, low):
    """a mask in one tensor with a position bias of ordinary size, which 8 bits would lose"""
    h, mask, dy = inputs(device, low)
    bias = torch.randn(24, 24).to(device)
    (got,) = torch.autograd.grad(checkpoint_8bit(attention, h, mask + bias), h, dy)
    k = at_kept(h)
    (want,) = torch.autograd.grad(attention(k, mask + bias), k, dy)
    assert torch.isfinite(got).all() and torch.equal(got, want)
    (exact,) = torch.autograd.grad(attention(h, mask + bias), h, dy)
    assert not torch.equal(got, exact)   # (h itself is kept in 8 bits)


def test_a_bias_with_a_gradient_is_kept_as_it_is(device):
    """learned position biases with the mask added in: not of the hidden states' shape"""
    h, mask, dy = inputs(device, float("-inf"))
    table = torch.randn(24, 24).to(device).requires_grad_()
    bias = table[None] + mask
    got = torch.autograd.grad(checkpoint_8bit(attention, h, torch.zeros_like(mask), bias), (h, table), dy, retain_graph=True)
    k = at_kept(h)
    want = torch.autograd.grad(attention(k, torch.zeros_like(mask), table[None] + mask), (k, table), dy)
    assert all(torch.isfinite(a).all() and torch.equal(a, b) for a, b in zip(got, want))


def test_every_input_of_the_first_activations_shape_is_kept_in_8_bits(device):
    """a residual stream and its addend"""
    h, _, dy = inputs(device, 0.0)
    delta = torch.randn(2, 24, 64).to(device).requires_grad_()
    cos = torch.randn(24, 64).to(device)
    fn = lambda h, cos, d: torch.tanh(h * cos + d)  # noqa: E731
    got = torch.autograd.grad(checkpoint_8bit(fn, h, cos, delta), (h, delta), dy)
    a, b = at_kept(h), at_kept(delta)
    want = torch.autograd.grad(fn(a, cos, b), (a, b), dy)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("args,names", [((), ("h", "d")), (("h",), ("d",))])
def test_inputs_by_name_are_kept_like_the_others(device, args, names):
    """called by name alone, too: recomputed, from 8 bits, and nothing exact is held"""
    import gc
    import weakref

    leaf = torch.randn(6, 200, device=device, requires_grad=True)
    calls = []

    def fn(h, d, scale=2.0):
        calls.append(1)
        return torch.sin(h) * torch.exp(d) * scale

    def inputs():
        return {"h": leaf * 1.0, "d": leaf * 0.5}

    now = inputs()
    held = [weakref.ref(t) for t in now.values()]
    y = checkpoint_8bit(fn, *(now[n] for n in args), **{n: now[n] for n in names}, scale=3.0)
    want = fn(**inputs(), scale=3.0)
    assert torch.equal(y, want)
    del now
    gc.collect()
    assert all(r() is None for r in held)
    calls.clear()
    (got,) = torch.autograd.grad(y.sum(), leaf)
    assert len(calls) == 1
    again = {n: at_kept(t.detach().requires_grad_()) for n, t in inputs().items()}
    a, b = torch.autograd.grad(fn(**again, scale=3.0).sum(), list(again.values()))
    assert torch.allclose(got, a + 0.5 * b, rtol=1e-6, atol=1e-6)


def test_a_mask_by_name_is_kept_as_it_is(device):
    h, mask, dy = inputs(device, float("-inf"))
    (got,) = torch.autograd.grad(checkpoint_8bit(attention, mask=mask, h=h), h, dy)
    k = at_kept(h)
    (want,) = torch.autograd.grad(attention(k, mask), k, dy)
    assert torch.equal(got, want)


class Block(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.lin = torch.nn.Linear(200, 200)
        self.calls = 0

    def forward(self, h, mask=None):
        self.calls += 1
        return torch.tanh(self.lin(h)) * (1.0 if mask is None else torch.exp(mask))


class Stack(torch.nn.Module):
    def __init__(self, by_name=False):
        super().__init__()
        self.layers = torch.nn.ModuleList([Block(), Block()])
        self.by_name = by_name

    def forward(self, h, mask=None):
        for layer in self.layers:
            h = layer(h=h, mask=mask) if self.by_name else layer(h, mask)
        return h


def stack_gradients(m, x, mask, read):
    """by hand, every layer recomputed from `read` of its input"""
    a = [x]
    with torch.no_grad():
        for layer in m.layers:
            a.append(layer.lin(a[-1]).tanh() * torch.exp(mask))
    g, out = torch.ones_like(x), {}
    for i in (1, 0):
        k = read(a[i]).requires_grad_()
        lin = m.layers[i].lin
        g, out[f"layers.{i}.lin.weight"], out[f"layers.{i}.lin.bias"] = torch.autograd.grad(
            torch.tanh(lin(k)) * torch.exp(mask), [k, lin.weight, lin.bias], g)
    return out


@pytest.mark.parametrize("by_name", [False, True])
@pytest.mark.parametrize("before", [None, "full", "8bit"])
@pytest.mark.parametrize("saved", ["full", "8bit"])
def test_enabled_checkpoints_are_what_was_asked_for_last(device, saved, before, by_name):
    from zeroq_b200.utils.checkpoint import enable_gradient_checkpointing

    torch.manual_seed(0)
    m = Stack(by_name).to(device)
    x = torch.randn(6, 200, device=device)
    mask = torch.zeros(200, device=device)
    mask[3] = float("-inf")
    if before:
        enable_gradient_checkpointing(m, saved=before)
    enable_gradient_checkpointing(m, saved=saved)
    m(x.requires_grad_(), mask).sum().backward()
    assert [layer.calls for layer in m.layers] == [2, 2]   # (once more each, not nested)
    full = stack_gradients(m, x.detach(), mask, lambda t: t.detach().clone())
    kept = stack_gradients(m, x.detach(), mask, lambda t: at_kept(t).detach())
    want, other = (kept, full) if saved == "8bit" else (full, kept)
    for n, p in m.named_parameters():
        assert torch.equal(p.grad, want[n]), n
        assert not torch.equal(p.grad, other[n]) or n == "layers.1.lin.bias", n
