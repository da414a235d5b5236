"""Window attention with sinks against the 64-bit oracle, forward and backward.

Every comparison is elementwise against the bound that the oracle derives from the roundings the kernels make
(probabilities and score gradients rounded to the type, the output rounded once, 32-bit sums).
"""
import math

import pytest
import torch

from gpt_neox_amd import _lib
from gpt_neox_amd.fused_attention import window_attention
from oracle import attention as A

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


def normal(shape, dtype, device, seed, times=1.0):
    gen = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn(shape, generator=gen, device=device) * times).to(dtype)


def inputs(sq, sk, b, h, h_kv, d, dtype, device, seed=1, times=1.0):
    return (normal((sq, b, h, d), dtype, device, seed, times), normal((sk, b, h_kv, d), dtype, device, seed + 1),
            normal((sk, b, h_kv, d), dtype, device, seed + 2), normal((sq, b, h, d), dtype, device, seed + 3))


def check(got, want, bound, what):
    assert got.shape == want.shape, what
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all(), what
    assert (err <= bound).all(), (what, err.max().item(), (err / bound.clamp(min=1e-30)).max().item())


def run(q, k, v, g, **kw):
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    out = window_attention(q, k, v, **kw)
    return (out.detach(), *torch.autograd.grad(out, (q, k, v), g))


def compare(q, k, v, g, lengths=None, **kw):
    dtype = q.dtype
    want = A.window_attention(q, k, v, grad=g, dtype=dtype, key_lengths=lengths, **kw)
    on_gpu = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=q.device)
    got = run(q, k, v, g, key_lengths=on_gpu, **kw)
    for name, t in zip(("out", "dq", "dk", "dv"), got):
        check(t, want[name], want[name + "_bound"], name)
    # without a gradient: the same output, bit for bit
    with torch.no_grad():
        assert torch.equal(window_attention(q, k, v, key_lengths=on_gpu, **kw), got[0])
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sq,sk", [(1, 1), (1, 7), (2, 2), (7, 1), (31, 33), (32, 32), (64, 64), (65, 63), (100, 300), (300, 100), (129, 129), (257, 260)])
def test_lengths_from_one_on(device, dtype, sq, sk):
    compare(*inputs(sq, sk, 2, 4, 2, 64, dtype, device), window=40, sinks=3)
    compare(*inputs(sq, sk, 1, 2, 2, 128, dtype, device, seed=9))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [8, 16, 40, 64, 72, 80, 96, 104, 128, 136, 192, 256])
def test_head_dims(device, dtype, d):
    compare(*inputs(150, 150, 1, 4, 2, d, dtype, device), window=60, sinks=2)


@pytest.mark.parametrize("h,h_kv", [(1, 1), (3, 1), (4, 4), (5, 1), (6, 2), (12, 3), (16, 2), (40, 1), (9, 9)])
def test_groups_of_heads(device, h, h_kv):
    compare(*inputs(90, 90, 2, h, h_kv, 64, torch.bfloat16, device), window=30, sinks=1)


@pytest.mark.parametrize("window,sinks", [
    (None, 0), (0, 0), (0, 1), (1, 0), (31, 0), (32, 4), (63, 64), (64, 65), (100, 130), (200, 300), (1000, 0), (10, 1000), (None, 5),
    (2**31 - 1, 2**31 - 1)])
def test_windows_and_sinks(device, window, sinks):
    compare(*inputs(330, 330, 1, 4, 2, 64, torch.bfloat16, device), window=window, sinks=sinks)


@pytest.mark.parametrize("window,sinks,h,h_kv", [(64, 4, 4, 1), (300, 140, 2, 2), (128, 1, 6, 2)])
def test_rows_far_behind_the_window_reach_the_sinks(device, window, sinks, h, h_kv):
    # thousands of rows whose only part in the first key tiles is the sinks: summed in several pieces
    compare(*inputs(2600, 2600, 1, h, h_kv, 128, torch.float16, device), window=window, sinks=sinks)


@pytest.mark.parametrize("h,h_kv,sinks", [(32, 32, 1400), (24, 12, 1100), (40, 20, 2000)])
def test_many_sinks_over_many_heads(device, h, h_kv, sinks):
    # more key tiles hold sinks than the rows behind their window can be cut for
    compare(*inputs(2050, 2048, 1, h, h_kv, 16, torch.bfloat16, device), window=64, sinks=sinks)


@pytest.mark.parametrize("h,h_kv,lengths", [(4, 1, None), (6, 2, [1300, 40]), (3, 1, [0, 1301])])
def test_key_gradients_in_pieces_under_a_bare_causal_mask(device, h, h_kv, lengths):
    # few key tiles, whose first ones have many more rows than the last: pieces of one size, fewer of them for later tiles
    compare(*inputs(1301, 1301, 2, h, h_kv, 64, torch.bfloat16, device), lengths=lengths)
    compare(*inputs(700, 1301, 2, h, h_kv, 64, torch.bfloat16, device), lengths=lengths, window=1250, sinks=3)


@pytest.mark.parametrize("lengths", [[0, 0, 0], [1, 200, 199], [64, 128, 63], [200, 500, -3]])
@pytest.mark.parametrize("window,sinks", [(50, 0), (50, 4), (None, 0)])
def test_key_lengths_leave_rows_empty(device, lengths, window, sinks):
    q, k, v, g = inputs(200, 200, 3, 4, 4, 64, torch.float16, device)
    got = compare(q, k, v, g, lengths=[min(max(n, 0), 200) for n in lengths], window=window, sinks=sinks)
    as_given = torch.tensor(lengths, dtype=torch.int32, device=device)
    again = run(q, k, v, g, key_lengths=as_given, window=window, sinks=sinks)
    assert all(torch.equal(x, y) for x, y in zip(got, again))
    for i, n in enumerate(lengths):
        assert (got[2][max(n, 0):, i] == 0).all() and (got[3][max(n, 0):, i] == 0).all()


@pytest.mark.parametrize("d", [64, 80, 128, 256])
def test_what_lies_behind_a_length_may_be_anything(device, d):
    q, k, v, g = inputs(130, 130, 2, 2, 1, d, torch.bfloat16, device)
    lengths = torch.tensor([70, 33], dtype=torch.int32, device=device)
    clean = run(q, k, v, g, key_lengths=lengths, window=100, sinks=2)
    for poison in (math.nan, math.inf, -math.inf, torch.finfo(torch.bfloat16).min):
        for i, n in enumerate((70, 33)):
            k[n:, i] = poison
            v[n:, i] = poison
        assert all(torch.equal(x, y) for x, y in zip(run(q, k, v, g, key_lengths=lengths, window=100, sinks=2), clean))


def test_a_far_nan_stays_where_it_is_seen(device):
    q, k, v, g = inputs(700, 700, 1, 2, 2, 64, torch.float16, device)
    clean = window_attention(q, k, v, window=100)
    v[10] = math.nan
    k[10] = math.nan
    out = window_attention(q, k, v, window=100)
    # seen by rows 10 .. 110; its tile of 64 keys by the workgroups of rows up to 255
    assert torch.isnan(out[10:111]).all()
    assert torch.equal(out[256:], clean[256:])


@pytest.mark.parametrize("scale", [0.3, -0.3, 0.0, 1.0, 3.0])
def test_scales(device, scale):
    compare(*inputs(140, 140, 1, 2, 2, 64, torch.bfloat16, device), window=70, sinks=2, scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_scores(device, dtype):
    compare(*inputs(200, 200, 1, 2, 1, 128, dtype, device, times=30.0), window=90, sinks=4)


def test_scores_that_rise_and_fall_along_the_keys(device):
    # the running maximum has to follow, and what was summed before it to be scaled down
    q, k, v, g = inputs(512, 512, 1, 2, 2, 64, torch.bfloat16, device)
    ramp = torch.linspace(-6, 6, 512, device=device).view(-1, 1, 1, 1)
    for t in (ramp, -ramp, ramp.abs()):
        compare(q.abs(), (k.abs() * t).to(k.dtype), v, g, window=400, sinks=8)


# ---- layouts ----------------------------------------------------------------------------------------------------
def fused_view(sq, b, h, h_kv, d, dtype, device):
    mixed = normal((sq, b, h + 2 * h_kv, d), dtype, device, 4)
    return mixed[:, :, :h], mixed[:, :, h:h + h_kv], mixed[:, :, h + h_kv:]


def batch_first(sq, b, h, h_kv, d, dtype, device):
    return tuple(normal((b, n, sq, d), dtype, device, 5 + i).permute(2, 0, 1, 3) for i, n in enumerate((h, h_kv, h_kv)))


def dim_strided(sq, b, h, h_kv, d, dtype, device):
    return tuple(normal((sq, b, n, 2 * d), dtype, device, 8 + i)[..., ::2] for i, n in enumerate((h, h_kv, h_kv)))


def misaligned(sq, b, h, h_kv, d, dtype, device):
    def one(n, seed):
        flat = normal((sq * b * n * d + 3,), dtype, device, seed)
        return flat[3:].view(sq, b, n, d)

    return one(h, 11), one(h_kv, 12), one(h_kv, 13)


def odd_rows(sq, b, h, h_kv, d, dtype, device):
    return tuple(normal((sq, b, n, d + 1), dtype, device, 14 + i)[..., :d] for i, n in enumerate((h, h_kv, h_kv)))


def broadcast_keys(sq, b, h, h_kv, d, dtype, device):
    q = normal((sq, b, h, d), dtype, device, 17)
    k, v = (normal((sq, 1, 1, d), dtype, device, s).expand(sq, b, h_kv, d) for s in (18, 19))
    return q, k, v


@pytest.mark.parametrize("layout", [fused_view, batch_first, dim_strided, misaligned, odd_rows, broadcast_keys])
@pytest.mark.parametrize("b,d", [(2, 64), (1, 96)])
def test_layouts(device, layout, b, d):
    q, k, v = layout(120, b, 4, 2, d, torch.bfloat16, device)
    g = normal((4, b, 120, d), torch.bfloat16, device, 20).permute(2, 1, 0, 3)
    got = compare(q, k, v, g, window=50, sinks=2)
    dense = run(q.contiguous(), k.contiguous(), v.contiguous(), g.contiguous(), window=50, sinks=2)
    assert all(torch.equal(x, y) for x, y in zip(got, dense))


def test_gradients_of_broadcast_inputs_are_summed(device):
    q = normal((40, 2, 4, 64), torch.float16, device, 21)
    k, v = (normal((40, 1, 1, 64), torch.float16, device, s).requires_grad_() for s in (22, 23))
    g = normal((40, 2, 4, 64), torch.float16, device, 24)
    out = window_attention(q, k.expand(40, 2, 2, 64), v.expand(40, 2, 2, 64), window=9)
    dk, dv = torch.autograd.grad(out, (k, v), g)
    want = A.window_attention(q, k.detach().expand(40, 2, 2, 64), v.detach().expand(40, 2, 2, 64), window=9, grad=g, dtype=q.dtype)
    for name, t in (("dk", dk), ("dv", dv)):
        # (the four gradients, rounded each, are summed by torch in that type)
        bound = want[name + "_bound"].sum((1, 2)) + 4 * A.ROUND[q.dtype] * want[name].abs().sum((1, 2))
        assert ((t.double().view(40, 64) - want[name].sum((1, 2))).abs() <= bound).all()


def test_strides_beyond_32_bits(device):
    # keys and values whose tokens lie 2^26 elements apart: the last one starts at 2^32 elements
    big = torch.empty((66 << 26,), dtype=torch.float16, device=device)
    k = big.as_strided((66, 1, 2, 64), (1 << 26, 64, 64, 1))
    v = big.as_strided((66, 1, 2, 64), (1 << 26, 64, 64, 1), 1024)
    k.copy_(normal((66, 1, 2, 64), torch.float16, device, 30))
    v.copy_(normal((66, 1, 2, 64), torch.float16, device, 31))
    q, g = normal((66, 1, 4, 64), torch.float16, device, 32), normal((66, 1, 4, 64), torch.float16, device, 33)
    got = compare(q, k, v, g, window=20, sinks=2)
    assert all(torch.equal(x, y) for x, y in zip(got, run(q, k.contiguous(), v.contiguous(), g, window=20, sinks=2)))
    # and queries
    qq = big.as_strided((66, 1, 4, 64), (1 << 26, 256, 64, 1), 4096)
    qq.copy_(q)
    assert all(torch.equal(x, y) for x, y in zip(got, run(qq, k, v, g, window=20, sinks=2)))


# ---- how it is called ---------------------------------------------------------------------------------------------
def test_the_same_inputs_give_the_same_bits(device):
    args = inputs(600, 600, 2, 8, 2, 128, torch.bfloat16, device)
    first = run(*args, window=100, sinks=4)
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(first, run(*args, window=100, sinks=4)))


def test_on_another_stream(device):
    args = inputs(300, 300, 1, 4, 2, 64, torch.bfloat16, device)
    want = run(*args, window=100, sinks=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(*args, window=100, sinks=4)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_without_the_native_calls_the_same_bits(device, monkeypatch):
    args = inputs(300, 300, 2, 4, 2, 96, torch.float16, device)
    kw = dict(window=100, sinks=4, key_lengths=torch.tensor([300, 77], dtype=torch.int32, device=device))
    want = run(*args, **kw)
    monkeypatch.setattr(_lib, "calls", lambda *tensors: None)
    assert all(torch.equal(x, y) for x, y in zip(want, run(*args, **kw)))


def test_saved_tensor_hooks(device):
    args = inputs(130, 130, 1, 4, 2, 64, torch.bfloat16, device)
    want = run(*args, window=30, sinks=1)
    with torch.autograd.graph.save_on_cpu():
        q, k, v = (t.clone().requires_grad_() for t in args[:3])
        out = window_attention(q, k, v, window=30, sinks=1)
    got = torch.autograd.grad(out, (q, k, v), args[3])
    assert all(torch.equal(x, y) for x, y in zip(want[1:], got))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.float() if t.dtype == torch.bfloat16 else t):
        out = window_attention(q, k, v, window=30, sinks=1)
    with pytest.raises(RuntimeError, match="shapes and dtypes"):
        out.backward(args[3])


def test_gradients_are_only_those_asked_for(device):
    q, k, v, g = inputs(64, 64, 1, 2, 2, 64, torch.bfloat16, device)
    want = run(q, k, v, g, window=10)
    qq = q.clone().requires_grad_()
    (dq,) = torch.autograd.grad(window_attention(qq, k, v, window=10), qq, g)
    assert torch.equal(dq, want[1])
    vv = v.clone().requires_grad_()
    (dv,) = torch.autograd.grad(window_attention(q, k, vv, window=10), vv, g)
    assert torch.equal(dv, want[3])


def test_gradient_against_differences(device):
    q, k, v, g = inputs(80, 80, 1, 2, 1, 64, torch.float16, device)
    kw = dict(window=25, sinks=2)
    got = run(q, k, v, g, **kw)
    want = A.window_attention(q, k, v, grad=g, dtype=q.dtype, **kw)
    for n, name in enumerate(("dq", "dk", "dv")):
        step = normal((q, k, v)[n].shape, torch.float64, device, 40 + n)
        hi, lo = [t.double() for t in (q, k, v)], [t.double() for t in (q, k, v)]
        hi[n], lo[n] = hi[n] + 1e-4 * step, lo[n] - 1e-4 * step
        diff = sum(s * (A.window_attention(*t, **kw)["out"] * g.double()).sum() for s, t in ((1, hi), (-1, lo))) / 2e-4
        # the kernel's gradient may be off by its bound in every element, the difference by its third derivative's 1e-8
        bound = (want[name + "_bound"] * step.abs()).sum() + 1e-4
        assert abs((got[n + 1].double() * step).sum() - diff) <= bound, name


@pytest.mark.parametrize("sq,sk,b", [(0, 5, 1), (5, 0, 1), (5, 5, 0), (0, 0, 2)])
def test_empty_calls(device, sq, sk, b):
    q, k, v, g = inputs(sq, sk, b, 2, 1, 64, torch.bfloat16, device)
    out, dq, dk, dv = run(q, k, v, g)
    for x, y in ((out, q), (dq, q), (dk, k), (dv, v)):
        assert x.shape == y.shape and (x == 0).all()


def test_refusals(device):
    q, k, v, _ = inputs(8, 8, 1, 4, 2, 64, torch.bfloat16, device)
    cases = [
        ((q[0], k, v), {}, "4D"), ((q.float(), k.float(), v.float()), {}, "fp16 and bf16"), ((q, k.half(), v), {}, "same dtype"),
        ((q, k, v[:4]), {}, "same shape"), ((q, k[..., :32], v[..., :32]), {}, "head dim"), ((q[..., :20], k[..., :20], v[..., :20]), {}, "multiple of 8"),
        ((q[:, :, :3], k, v), {}, "multiple of 2 key heads"), ((q, k, v), {"window": -2}, "window"), ((q, k, v), {"window": 1.5}, "window"),
        ((q, k, v), {"sinks": -1}, "sinks"), ((q, k, v), {"key_lengths": torch.tensor([8], device=device)}, "int32"),
        ((q, k, v), {"key_lengths": torch.tensor([8], dtype=torch.int32)}, "GPU"), ((q.cpu(), k, v), {}, "GPU"),
        ((q, k, v), {"scale": math.nan}, "finite"),
    ]
    for args, kw, message in cases:
        with pytest.raises(RuntimeError, match=message):
            window_attention(*args, **kw)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q, q)
        with pytest.raises((RuntimeError, NotImplementedError)):
            window_attention(dual, k, v)
