"""Attention at the ends of the number range: running maxima, small and large values, against the 64-bit oracle."""
import pytest
import torch

from gpt_neox_amd.fused_attention import window_attention
from gpt_neox_amd.paged_cache import PagedKVCache, paged_attention, slots_of
from oracle import attention as A

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
I8, F8 = torch.int8, torch.float8_e4m3fn


def normal(shape, dtype, device, seed, times=1.0):
    gen = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn(shape, generator=gen, device=device) * times).to(dtype)


def within(got, want, bound):
    assert torch.isfinite(got).all()
    err = (got.double() - want).abs()
    assert (err <= bound).all(), (err.max().item(), (err / bound.clamp(min=1e-300)).max().item())


def one_sequence(k, v, codes, page=64):
    """``k``, ``v`` ``[n, h_kv, d]`` of one sequence in a cache, and its table."""
    n, h_kv, d = k.shape
    pages = -(-n // page)
    cache = PagedKVCache.allocate(pages + 1, page, h_kv, d, codes, k.device)
    table = torch.arange(pages, 0, -1, device=k.device).view(1, pages).int()
    cache.write(k, v, slots_of(table, torch.zeros(n, device=k.device), torch.arange(n, device=k.device), page))
    return cache, table


def attend_paged(q, cache, table, context, **kw):
    starts = torch.tensor([0, q.shape[0]], dtype=torch.int32, device=q.device)
    lengths = torch.tensor([context], dtype=torch.int32, device=q.device)
    return paged_attention(q, cache, table, starts, lengths, max_query=q.shape[0], max_context=context, **kw)


def held(cache, table, n):
    """The keys and values ``[n, h_kv, d]`` that a cache of codes holds, in 64 bits."""
    return [A.gather(table[0], cache.page_size, n, t.float()).double() * A.gather(table[0], cache.page_size, n, s).double()[..., None]
            for t, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]


# ---- the running maximum -------------------------------------------------------------------------------------------
def steps(d, dtype, device):
    """Queries and keys whose scores come from the last 16 dims alone, and rise from tile to tile by 20 to 70 powers of two:
    a maximum taken of anything but the whole sum is off by far more than the slack that it is kept with."""
    sk, sq = 1024, 40
    gen = torch.Generator(device=device).manual_seed(d)
    level = torch.randint(0, 3, (sk // 32,), generator=gen, device=device).repeat_interleave(32) * 24.0
    level = level + torch.arange(sk, device=device) // 256 * 20.0
    q = torch.zeros((sq, 1, 2, d), device=device)
    q[..., -16:] = 1.0
    q[..., : d - 16] = torch.randn((sq, 1, 2, d - 16), generator=gen, device=device) * 0.01
    k = torch.randn((sk, 1, 2, d), generator=gen, device=device) * 0.01
    k[..., -16:] += (level / 16)[:, None, None, None]
    return q.to(dtype), k.to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 96, 128, 256])
def test_the_maximum_is_that_of_the_whole_sums(device, dtype, d):
    q, k = steps(d, dtype, device)
    v = normal(k.shape, dtype, device, 3)
    want = A.window_attention(q, k, v, scale=0.69, dtype=dtype)
    with torch.no_grad():
        got = window_attention(q, k, v, scale=0.69)
    within(got, want["out"], want["out_bound"])
    cache, table = one_sequence(k[:, 0], v[:, 0], dtype)
    within(attend_paged(q[:, 0], cache, table, k.shape[0], scale=0.69), want["out"][:, 0], want["out_bound"][:, 0])


# ---- small and large values ----------------------------------------------------------------------------------------
def typical_error(q, k, v, sees, scale, dtype):
    """One head in 64 bits: the output, and the variance that rounding each weighted value and the output to the type may
    leave in it.  An error of one rounding is even over half a unit in the last place on both sides, so its variance is a third of
    (unit roundoff * value)^2 at most, or of half the type's smallest step squared; errors of different keys are independent."""
    out, p = A.one_head(q, k, v, sees, scale)
    u, tiny = A.ROUND[dtype], A.TINY[dtype]
    return out, (u * u * (p.square() @ v.square() + out.square()) + tiny * tiny) / 3


def typically_within(got, want, variance):
    # a quarter more than the roundings' own size: room for the 32-bit part, a tenth of it, and for what a mean over
    # thousands of elements may be off by
    assert torch.isfinite(got).all()
    err, most = (got.double() - want).square().mean().sqrt(), variance.mean().sqrt()
    assert err <= 1.25 * most, (err / most).item()


def sink_and_rest(n, h_kv, d, dtype, device, times, above, seed):
    """Keys and values ``[n, h_kv, d]``: values of the size ``times``; where ``above`` is given the first key's score is that much above
    the others' (queries carry 4 in their last dim, with a scale of 1), and its value a hundred times smaller."""
    k, v = normal((n, h_kv, d), dtype, device, seed, 0.02), normal((n, h_kv, d), dtype, device, seed + 1, times)
    k[..., -1] = 0
    if above:
        k[0, :, -1] = above / 4
        v[0] *= 0.01
    return k, v


@pytest.mark.parametrize("codes", [I8, F8])
@pytest.mark.parametrize("times,above", [(1.0, 0), (0.1, 0), (0.01, 0), (0.002, 0), (1.0, 6), (0.3, 8), (0.05, 10)])
@pytest.mark.parametrize("n,new", [(250, 1), (3000, 1), (250, 60), (3000, 60)])
def test_codes_keep_the_precision_of_half(device, codes, times, above, n, new):
    h, h_kv, d = 8, 4, 64
    k, v = sink_and_rest(n, h_kv, d, torch.float16, device, times, above, 5)
    q = normal((new, h, d), torch.float16, device, 7)
    q[..., -1] = 4
    cache, table = one_sequence(k, v, codes)
    got = attend_paged(q, cache, table, n, scale=1.0)
    hk, hv = held(cache, table, n)
    sees = A.visible(new, n, device=device)
    want, variance = torch.empty(got.shape, dtype=torch.float64, device=device), torch.empty(got.shape, dtype=torch.float64, device=device)
    for x in range(h):
        want[:, x], variance[:, x] = typical_error(q[:, x].double(), hk[:, x // 2], hv[:, x // 2], sees, 1.0, q.dtype)
    typically_within(got, want, variance)


@pytest.mark.parametrize("codes", [I8, F8, torch.float16])
@pytest.mark.parametrize("n,new", [(250, 1), (3000, 1), (250, 60), (3000, 60)])
def test_values_near_the_largest_of_half(device, codes, n, new):
    # scores that rise, behind every wave's first keys, by a little less than what the running maximum may lag behind
    h, d = 4, 64
    k = normal((n, h, d), torch.float16, device, 8, 0.02)
    k[..., -1] = torch.where(torch.arange(n, device=device) % 256 < 128, 0.0, 7.2 * 0.6931 / 4)[:, None]
    v = (normal((n, h, d), torch.float16, device, 9).sign() * 60000).to(torch.float16)
    q = normal((new, h, d), torch.float16, device, 10)
    q[..., -1] = 4
    cache, table = one_sequence(k, v, codes)
    got = attend_paged(q, cache, table, n, scale=1.0)
    quantised = codes in (I8, F8)
    want, bound = A.paged_attention(q, cache.k.float() if quantised else cache.k, cache.v.float() if quantised else cache.v, cache.k_scale,
                                    cache.v_scale, table, [0, new], [n], scale=1.0, dtype=q.dtype)
    within(got, want, bound)


@pytest.mark.parametrize("codes", [I8, F8])
@pytest.mark.parametrize("new", [1, 60])
def test_large_values_that_the_maximum_leaves_behind(device, codes, new):
    # the first keys' values are 2^13 times the others', and their scores 30 powers of two below: their products come first,
    # and are nothing in the end
    n, h, d = 2000, 4, 64
    k, v = normal((n, h, d), torch.float16, device, 11, 0.02), normal((n, h, d), torch.float16, device, 12)
    behind = torch.arange(n, device=device) % 256 < 128  # (so in every part of a split axis)
    k[..., -1] = torch.where(behind, 0.0, 30 * 0.6931 / 4)[:, None]
    v *= torch.where(behind, 2.0**13, 1.0)[:, None, None]
    q = normal((new, h, d), torch.float16, device, 13)
    q[..., -1] = 4
    cache, table = one_sequence(k, v, codes)
    got = attend_paged(q, cache, table, n, scale=1.0)
    hk, hv = held(cache, table, n)
    sees = A.visible(new, n, device=device)
    want, variance = torch.empty(got.shape, dtype=torch.float64, device=device), torch.empty(got.shape, dtype=torch.float64, device=device)
    for x in range(h):
        want[:, x], variance[:, x] = typical_error(q[:, x].double(), hk[:, x], hv[:, x], sees, 1.0, q.dtype)
    typically_within(got, want, variance)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("above", [0, 8, 11, 13])
@pytest.mark.parametrize("n,new", [(250, 1), (3000, 1), (250, 60), (3000, 60)])
def test_probabilities_far_below_a_sink_without_a_value(device, dtype, above, n, new):
    h, d = 4, 64
    k, v = sink_and_rest(n, h, d, dtype, device, 100.0, above, 14)
    if above:
        v[0] = 0
    q = normal((new, h, d), dtype, device, 16)
    q[..., -1] = 4
    cache, table = one_sequence(k, v, dtype)
    got = attend_paged(q, cache, table, n, scale=1.0)
    sees = A.visible(new, n, device=device)
    want, variance = torch.empty(got.shape, dtype=torch.float64, device=device), torch.empty(got.shape, dtype=torch.float64, device=device)
    for x in range(h):
        want[:, x], variance[:, x] = typical_error(q[:, x].double(), k[:, x].double(), v[:, x].double(), sees, 1.0, dtype)
    typically_within(got, want, variance)
    with torch.no_grad():
        typically_within(window_attention(q[:, None], k[:, None], v[:, None], scale=1.0)[:, 0], want, variance)


# ---- gradients -----------------------------------------------------------------------------------------------------
def gradients(q, k, v, g, sees, scale, dtype):
    """One head ``[n, d]`` in 64 bits: the three gradients, and as in ``typical_error`` the variance that rounding P, dS and
    the results to the type may leave in each."""
    q, k, v, g = (t.double() for t in (q, k, v, g))
    out, p = A.one_head(q, k, v, sees, scale)
    ds = p * (g @ v.T - (g * out).sum(1, keepdim=True)) * scale
    u, tiny = A.ROUND[dtype], A.TINY[dtype]
    want = (ds @ k, ds.T @ q, p.T @ g)
    terms = (ds.square() @ k.square(), ds.T.square() @ q.square(), p.T.square() @ g.square())
    return want, [(u * u * (t + w.square()) + tiny * tiny) / 3 for t, w in zip(terms, want)]


def check_gradients(q, k, v, g, heads, rows=None, sink=False, **kw):
    """Heads ``heads`` of a call without shared keys; ``rows``: the tokens whose ``dq`` is looked at, each list by itself.  With
    ``sink`` the first key's gradients, a few numbers far larger than the others, are held to four deviations each."""
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(window_attention(*leaves, scale=0.125, **kw), leaves, g)
    sees = A.visible(q.shape[0], k.shape[0], kw.get("window"), kw.get("sinks", 0), device=q.device)
    for x in heads:
        want, variance = gradients(q[:, 0, x], k[:, 0, x], v[:, 0, x], g[:, 0, x], sees, 0.125, q.dtype)
        for some in rows or [slice(None)]:
            typically_within(got[0][some, 0, x], want[0][some], variance[0][some])
        for i in (1, 2):
            typically_within(got[i][sink:, 0, x], want[i][sink:], variance[i][sink:])
            if sink:
                within(got[i][0, 0, x], want[i][0], 4 * variance[i][0].sqrt())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("times", [300.0, 1.0, 1e-2, 1e-3, 1e-4])
@pytest.mark.parametrize("n,h,d,kw", [
    (4096, 2, 64, {}), (4096, 32, 64, {}), (4096, 2, 128, {"window": 2000, "sinks": 4}), (2000, 2, 96, {}), (1500, 2, 256, {}), (300, 3, 64, {"window": 100})])
def test_gradients_of_small_and_large_sizes(device, dtype, times, n, h, d, kw):
    q, k, v = (normal((n, 1, h, d), dtype, device, 20 + i) for i in range(3))
    g = normal((n, 1, h, d), dtype, device, 23, times)
    check_gradients(q, k, v, g, (0, h - 1), **kw)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_different_sizes_in_one_tile(device, dtype):
    n = 2000
    q, k, v = (normal((n, 1, 2, 64), dtype, device, 30 + i) for i in range(3))
    small = torch.arange(n, device=device) % 3 == 0
    g = (normal((n, 1, 2, 64), torch.float32, device, 33) * torch.where(small, 1e-3, 10.0)[:, None, None, None]).to(dtype)
    check_gradients(q, k, v, g, (0, 1), rows=[small, ~small])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("above", [9, 12])
def test_gradients_of_values_far_below_a_sink(device, dtype, above):
    # probabilities of about 2^-13 and 2^-17 for all keys but the first
    k, v = sink_and_rest(2500, 2, 64, dtype, device, 1.0, above, 40)
    q = normal((2500, 1, 2, 64), dtype, device, 42)
    q[..., -1] = 32
    check_gradients(q, k[:, None], v[:, None], normal(q.shape, dtype, device, 43), (0, 1), sink=True)
