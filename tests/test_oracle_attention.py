"""The 64-bit attention oracle against autograd, central differences and torch's own 8-bit floats (CPU)."""
import math

import pytest
import torch

from oracle import attention as A


def tensors(sq, sk, b, h, h_kv, d, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(*s, generator=g, dtype=torch.float64) for s in ((sq, b, h, d), (sk, b, h_kv, d), (sk, b, h_kv, d), (sq, b, h, d))]


def loss(q, k, v, g, **kw):
    return (A.window_attention(q, k, v, **kw)["out"] * g).sum()


@pytest.mark.parametrize("sq,sk,window,sinks,lengths", [
    (6, 6, None, 0, None), (6, 9, 2, 1, None), (9, 5, 3, 0, None), (7, 7, 1, 2, [7, 3]), (8, 8, 2, 0, [0, 2]), (1, 1, 0, 0, None)])
def test_gradients_are_those_of_differences(sq, sk, window, sinks, lengths):
    q, k, v, g = tensors(sq, sk, 2, 4, 2, 8)
    kw = dict(window=window, sinks=sinks, key_lengths=lengths, scale=0.7)
    res = A.window_attention(q, k, v, grad=g, **kw)
    gen = torch.Generator().manual_seed(1)
    for name, x in (("dq", q), ("dk", k), ("dv", v)):
        step = torch.randn(x.shape, generator=gen, dtype=torch.float64)
        eps = 1e-5
        args = {"dq": 0, "dk": 1, "dv": 2}[name]
        hi, lo = [q, k, v], [q, k, v]
        hi[args], lo[args] = x + eps * step, x - eps * step
        got = (loss(*hi, g, **kw) - loss(*lo, g, **kw)) / (2 * eps)
        # third derivatives are of order 10 here: eps^2 of them, and the cancellation of two sums of order 100
        assert abs(got - (res[name] * step).sum()) < 1e-6


def test_output_is_the_softmax_of_the_visible_scores():
    q, k, v, g = tensors(5, 8, 1, 2, 1, 4, seed=3)
    got = A.window_attention(q, k, v, window=2, sinks=1, scale=0.5)["out"]
    for i in range(5):
        p = i + 3
        keys = [j for j in range(8) if j <= p and (j >= p - 2 or j < 1)]
        for h in range(2):
            s = torch.stack([q[i, 0, h] @ k[j, 0, 0] for j in keys]) * 0.5
            want = torch.softmax(s, 0) @ torch.stack([v[j, 0, 0] for j in keys])
            assert torch.allclose(got[i, 0, h], want, atol=1e-12)


def test_a_query_that_sees_nothing_gives_zeros_and_no_gradient():
    q, k, v, g = tensors(6, 3, 1, 1, 1, 4)
    res = A.window_attention(q, k, v, grad=g)
    assert (res["out"][:3] == 0).all() and (res["dq"][:3] == 0).all() and (res["out"][3:] != 0).all()


def test_e4m3_rounding_is_torchs():
    x = torch.cat((torch.linspace(-448, 448, 40001), torch.randn(20000) * 0.01, torch.randn(20000) * 1e-3,
                   torch.arange(0, 256).to(torch.uint8).view(torch.float8_e4m3fn).float().nan_to_num(0)))
    ties = (x.to(torch.float8_e4m3fn).float() + 2.0**-4).clamp(-448, 448)
    for t in (x, ties):
        assert torch.equal(A.round_e4m3(t.double()).float(), t.to(torch.float8_e4m3fn).float())


def test_int8_codes_at_ties_and_zero_rows():
    x = torch.tensor([[127.0, 0.5, 1.5, -2.5], [0.0, 0.0, 0.0, 0.0], [254.0, 1.0, 3.0, -127.0]])
    y, scale = A.encode(x, torch.int8)
    assert y.tolist() == [[127, 0, 2, -2], [0, 0, 0, 0], [127, 0, 2, -64]]
    assert scale.tolist() == [1.0, 0.0, 2.0]


def test_visible_follows_the_window_rule():
    sees = A.visible(4, 6, window=1, sinks=1, length=5)
    assert sees.int().tolist() == [[1, 1, 1, 0, 0, 0], [1, 0, 1, 1, 0, 0], [1, 0, 0, 1, 1, 0], [1, 0, 0, 0, 1, 0]]
    assert math.prod(A.visible(3, 0).shape) == 0
