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
