"""How the attention calls behave in a program: derivatives that they do not have, and what they take for granted."""
import pytest
import torch

from gpt_neox_amd import _lib
from gpt_neox_amd.fused_attention import window_attention
from gpt_neox_amd.paged_cache import PagedKVCache, paged_attention

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["native", "ctypes"])
def path(request, monkeypatch):
    if request.param == "ctypes":
        monkeypatch.setattr(_lib, "calls", lambda *tensors: None)
    return request.param


def normal(shape, device, seed, dtype=torch.bfloat16):
    gen = torch.Generator(device=device).manual_seed(seed)
    return torch.randn(shape, generator=gen, device=device).to(dtype)


@pytest.mark.parametrize("of", [0, 1, 2])
def test_a_second_derivative_is_refused(device, path, of):
    qkv = [normal((40, 1, 2, 64), device, i) for i in range(3)]
    qkv[of].requires_grad_()
    out = window_attention(*qkv, window=9)
    (grad,) = torch.autograd.grad(out.float().square().sum(), qkv[of], create_graph=True)
    want = torch.autograd.grad(window_attention(*qkv, window=9).float().square().sum(), qkv[of])[0]
    assert torch.equal(grad, want) and grad.requires_grad
    # a penalty on the gradient beside a loss: the loss alone has a gradient, the penalty's may not be left out
    with pytest.raises(RuntimeError, match="no second derivative"):
        (out.float().sum() + grad.float().square().sum()).backward()


def test_a_second_derivative_with_a_constant_gradient_is_refused(device, path):
    q, k, v = (normal((40, 1, 2, 64), device, i).requires_grad_() for i in range(3))
    out = window_attention(q, k, v, window=9)
    grads = torch.autograd.grad(out, (q, k, v), torch.ones_like(out), create_graph=True)
    for g in grads:
        with pytest.raises(RuntimeError, match="no second derivative"):
            torch.autograd.grad(g.float().square().sum(), (q, k, v), allow_unused=True, retain_graph=True)
    # and where nothing goes back through them, gradients of a recorded backward pass are those of any other
    again = torch.autograd.grad(window_attention(q, k, v, window=9), (q, k, v), torch.ones_like(out))
    assert all(torch.equal(x, y) for x, y in zip(grads, again)) and not any(g.requires_grad for g in again)


@pytest.mark.parametrize("bounds", [{"max_query": 2**32 + 1}, {"max_query": -1}, {"max_query": 1, "max_context": -5}, {"max_query": 1, "max_context": 2**32 + 7},
                                    {"max_query": 1, "max_context": 0}, {"max_query": 2**62}, {"max_query": 1, "max_context": 2**30}])
def test_bounds_that_no_length_can_have_are_refused(device, path, bounds):
    # (in 32 bits 2^32 + 1 would be 1: all tokens behind the first would have been left out)
    cache = PagedKVCache.allocate(4, 16, 2, 64, torch.int8, device)
    table = torch.arange(4, device=device).view(1, 4).int()
    starts, lengths = (torch.tensor(x, dtype=torch.int32, device=device) for x in ([0, 3], [40]))
    with pytest.raises(RuntimeError, match="max_query|max_context"):
        paged_attention(normal((3, 4, 64), device, 5), cache, table, starts, lengths, **bounds)


@pytest.mark.parametrize("change", [
    lambda t: t[:-1] if t.dim() == 4 else t, lambda t: t.float() if t.dtype == torch.bfloat16 else t, lambda t: t[:-1] if t.dtype == torch.float32 else t,
    lambda t: t[..., :32] if t.dim() == 4 and t.shape[2] == 1 else t, lambda t: t[:1] if t.dtype == torch.int32 else t,
    lambda t: t.long() if t.dtype == torch.int32 else t, lambda t: t.cpu() if t.dtype == torch.float32 else t])
def test_saved_tensors_that_hooks_have_changed_are_refused(device, path, change):
    q = normal((40, 2, 2, 64), device, 0).requires_grad_()
    k, v = (normal((40, 2, 1, 64), device, i) for i in (1, 2))
    lengths = torch.tensor([40, 30], dtype=torch.int32, device=device)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
        out = window_attention(q, k, v, window=9, key_lengths=lengths)
    with pytest.raises(RuntimeError, match="shapes and dtypes|lengths have changed|device|GPU"):
        out.backward(torch.ones_like(out))


def test_saved_tensors_of_another_layout_are_those_of_before(device, path):
    q, k, v = (normal((40, 2, 2, 64), device, i).requires_grad_() for i in range(3))
    want = torch.autograd.grad(window_attention(q, k, v, window=9), (q, k, v), torch.ones_like(q))

    def spread(t):
        wide = t.new_empty((*t.shape[:-1], 2 * t.shape[-1]))
        wide[..., ::2] = t
        return wide[..., ::2]

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, spread):
        out = window_attention(q, k, v, window=9)
    assert all(torch.equal(x, y) for x, y in zip(want, torch.autograd.grad(out, (q, k, v), torch.ones_like(q))))
