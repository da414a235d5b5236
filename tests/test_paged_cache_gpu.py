"""The paged cache (codes and scales bit by bit) and attention over it against the 64-bit oracle."""
import math

import pytest
import torch

from gpt_neox_amd import _lib
from gpt_neox_amd.paged_cache import PagedKVCache, paged_attention, slots_of
from oracle import attention as A

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
I8, F8 = torch.int8, torch.float8_e4m3fn


def gen(device, seed):
    return torch.Generator(device=device).manual_seed(seed)


def normal(shape, dtype, device, seed, times=1.0):
    return (torch.randn(shape, generator=gen(device, seed), device=device) * times).to(dtype)


def flat(t):
    """[pages, page_size, ...] -> [slots, ...] (a view for what the cache allocates)"""
    return t.view(-1, *t.shape[2:])


def values(codes):
    return codes.float().double()


# ---- the cache ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("codes", [I8, F8])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,heads,d,page", [(1, 1, 16, 1), (5, 3, 64, 4), (37, 2, 80, 16), (100, 5, 96, 48), (300, 8, 128, 64), (33, 2, 256, 7)])
def test_codes_and_scales_bit_by_bit(device, dtype, codes, tokens, heads, d, page):
    pages = tokens // page + 3
    cache = PagedKVCache.allocate(pages, page, heads, d, codes, device)
    k, v = normal((tokens, heads, d), dtype, device, 1, 3.0), normal((tokens, heads, d), dtype, device, 2)
    slots = torch.randperm(pages * page, generator=gen(device, 3), device=device)[:tokens]
    cache.write(k, v, slots)
    for x, held, scales in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        want, scale = A.encode(x, codes)
        assert torch.equal(values(flat(held)[slots] if codes == I8 else flat(held.view(I8))[slots].view(F8)), want)
        assert torch.equal(flat(scales)[slots], scale)
    others = torch.ones(pages * page, dtype=torch.bool, device=device)
    others[slots] = False
    assert (flat(cache.k.view(I8))[others] == 0).all() and (flat(cache.v_scale)[others] == 0).all()
    # and back: the product in 32 bits, rounded once
    for out in DTYPES:
        rk, rv = cache.read(slots, out)
        for x, got in ((k, rk), (v, rv)):
            want, scale = A.encode(x, codes)
            assert torch.equal(got, (want.float() * scale[..., None]).to(out))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("codes", [I8, F8])
def test_ties_and_extremes(device, dtype, codes):
    top = A.LARGEST[codes]
    rows = [
        torch.arange(16) + 0.5,                       # with the largest code at the end: ties between whole numbers
        torch.arange(16) * 0.25 - 2,
        torch.zeros(16),
        torch.full((16,), torch.finfo(dtype).max),
        torch.full((16,), torch.finfo(dtype).tiny),
        torch.arange(16) * (2.0**-133 if dtype == torch.bfloat16 else 2.0**-24),  # subnormal
        torch.tensor([torch.finfo(dtype).max, torch.finfo(dtype).tiny] * 8),
        torch.cat((torch.tensor([3.0]), torch.arange(1, 16) * 1.5 / 127)),        # ties that no power of two scales
        torch.cat((torch.tensor([7.0]), (torch.arange(1, 16) * 2 + 17) * 7.0 / 448)),
        torch.cat((torch.tensor([-5.0]), torch.arange(1, 16) * 0.3125)),
    ]
    x = torch.stack(rows).to(dtype).to(device)
    for i in (0, 1):
        x[i, 15] = top / 2
    x = x[:, None, :].contiguous()
    cache = PagedKVCache.allocate(2, 8, 1, 16, codes, device)
    slots = torch.arange(x.shape[0], device=device)
    cache.write(x, -x, slots)
    want, scale = A.encode(x, codes)
    held = flat(cache.k.view(I8))[slots].view(codes)
    assert torch.equal(values(held), want)
    assert torch.equal(flat(cache.k_scale)[slots], scale)
    assert torch.equal(values(flat(cache.v.view(I8))[slots].view(codes)), -want)


@pytest.mark.parametrize("codes", [I8, F8])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_row_with_an_infinity_or_nan_reads_back_as_nan(device, codes, bad):
    cache = PagedKVCache.allocate(1, 8, 2, 64, codes, device)
    k, v = normal((8, 2, 64), torch.bfloat16, device, 4), normal((8, 2, 64), torch.bfloat16, device, 5)
    k[3, 1, 17] = bad
    cache.write(k, v, torch.arange(8, device=device))
    rk, rv = cache.read(torch.arange(8, device=device))
    assert torch.isnan(rk[3, 1]).all() and torch.isfinite(rv).all()
    rk[3, 1] = 0
    assert torch.isfinite(rk).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [8, 72, 128, 256])
def test_a_cache_in_16_bits_keeps_every_bit(device, dtype, d):
    cache = PagedKVCache.allocate(9, 5, 3, d, dtype, device)
    k, v = normal((40, 3, d), dtype, device, 6), normal((40, 3, d), dtype, device, 7)
    k[0, 0, 0], v[1, 0, 0] = math.nan, math.inf
    slots = torch.randperm(45, generator=gen(device, 8), device=device)[:40]
    cache.write(k, v, slots)
    rk, rv = cache.read(slots, dtype)
    assert torch.equal(rk.view(torch.int16), k.view(torch.int16)) and torch.equal(rv.view(torch.int16), v.view(torch.int16))


@pytest.mark.parametrize("codes", [I8, torch.bfloat16])
@pytest.mark.parametrize("slot_type", [torch.int32, torch.int64])
def test_slots_outside_the_cache(device, codes, slot_type):
    cache = PagedKVCache.allocate(4, 4, 2, 64, codes, device)
    slots = torch.tensor([3, -1, 16, 0, -(2**31), 2**31 - 1, 15], dtype=slot_type, device=device)
    k, v = normal((7, 2, 64), torch.bfloat16, device, 9), normal((7, 2, 64), torch.bfloat16, device, 10)
    cache.write(k, v, slots)
    inside = torch.tensor([0, 3, 6], device=device)
    rk, rv = cache.read(slots)
    for t in (rk, rv):
        outside = torch.ones(7, dtype=torch.bool, device=device)
        outside[inside] = False
        assert (t[outside] == 0).all() and (t[inside] != 0).any(-1).all()
    written = flat(cache.k.view(I8) if codes == I8 else cache.k).ne(0).any(-1).any(-1).nonzero().flatten().tolist()
    assert written == [0, 3, 15]


def test_strided_inputs_and_a_cache_for_all_layers(device):
    layers = 3
    k_all = torch.zeros((6, layers, 8, 2, 64), dtype=I8, device=device)
    v_all, ks, vs = torch.zeros_like(k_all), torch.zeros((6, layers, 8, 2), device=device), torch.zeros((6, layers, 8, 2), device=device)
    mixed = normal((20, 8, 64), torch.float16, device, 11)  # q, k and v of a projection: 4 + 2 + 2 heads
    slots = torch.randperm(48, generator=gen(device, 12), device=device)[:20]
    for layer in range(layers):
        cache = PagedKVCache(k_all[:, layer], v_all[:, layer], ks[:, layer], vs[:, layer])
        cache.write(mixed[:, 4:6], mixed[:, 6:], slots)
        rk, rv = cache.read(slots, torch.float16)
        for x, got in ((mixed[:, 4:6], rk), (mixed[:, 6:], rv)):
            want, scale = A.encode(x, I8)
            assert torch.equal(got, (want.float() * scale[..., None]).half())
    # an odd layout is copied first
    odd = normal((64, 2, 20), torch.float16, device, 13).permute(2, 1, 0)
    cache.write(odd, odd, slots)
    rk, _ = cache.read(slots, torch.float16)
    want, scale = A.encode(odd, I8)
    assert torch.equal(rk, (want.float() * scale[..., None]).half())


@pytest.mark.parametrize("codes", [F8, torch.float16])
def test_offsets_beyond_32_bits(device, codes):
    # pages 2^24 elements apart, 300 of them: slots behind 2^32 elements
    size = 300 << 24
    step = (1 << 24, 64, 64, 1)

    def one():
        if codes == F8:
            return torch.zeros(size, dtype=I8, device=device).as_strided((300, 16, 1, 64), step).view(F8)
        return torch.empty(size, dtype=codes, device=device).as_strided((300, 16, 1, 64), step)

    scales = [torch.zeros((300, 16, 1), device=device) for _ in "kv"] if codes == F8 else [None, None]
    cache = PagedKVCache(one(), one(), *scales)
    n = 2000
    k, v = normal((n, 1, 64), torch.float16, device, 14), normal((n, 1, 64), torch.float16, device, 15)
    table = torch.randperm(300, generator=gen(device, 16), device=device)[:126].view(1, 126).int()
    table[0, 125] = 299
    slots = slots_of(table, torch.zeros(n, device=device), torch.arange(n, device=device), 16)
    cache.write(k, v, slots)
    rk, rv = cache.read(slots, torch.float16)
    if codes != F8:
        assert torch.equal(rk, k) and torch.equal(rv, v)
    for new in (1, 40):
        q = normal((new, 4, 64), torch.float16, device, 17)
        starts = torch.tensor([0, new], dtype=torch.int32, device=device)
        lengths = torch.tensor([n], dtype=torch.int32, device=device)
        got = paged_attention(q, cache, table, starts, lengths, max_query=new)
        want, bound = A.paged_attention(q, rk.view(125, 16, 1, 64), rv.view(125, 16, 1, 64), None, None,
                                        torch.arange(125, device=device).view(1, 125), starts, lengths, dtype=torch.float16)
        if codes == F8:  # (rk and rv were rounded to 16 bits, the kernel multiplies by the scales in 32)
            bound = bound * 3
        assert ((got.double() - want).abs() <= bound).all()


# ---- attention ------------------------------------------------------------------------------------------------------
def sequences(device, dtype, codes, new, context, h, h_kv, d, page, seed=20):
    """A cache of garbage with the sequences' keys and values in pages of their own, in random order; its tables."""
    b = len(new)
    width = max(1, -(-max(context) // page)) + 1
    pages = b * width + 2
    order = torch.randperm(pages, generator=gen(device, seed), device=device)
    table = order[: b * width].view(b, width).int()
    cache = PagedKVCache.allocate(pages, page, h_kv, d, codes, device)
    # what no sequence has written is NaN, and table entries behind a sequence's end name no page
    if codes in (I8, F8):
        cache.k_scale.fill_(math.nan)
        cache.v_scale.fill_(math.nan)
        if codes == F8:
            cache.k.view(I8).fill_(0x7F)
            cache.v.view(I8).fill_(0x7F)
    else:
        cache.k.fill_(math.nan)
        cache.v.fill_(math.inf)
    for s in range(b):
        n = context[s]
        if n:
            k, v = normal((n, h_kv, d), dtype, device, seed + 2 * s + 1), normal((n, h_kv, d), dtype, device, seed + 2 * s + 2)
            at = torch.arange(n, device=device)
            cache.write(k, v, slots_of(table, torch.full((n,), s, device=device), at, page))
        used = -(-n // page)
        table[s, used:] = torch.tensor([-1, 2**31 - 1], dtype=torch.int32, device=device).repeat(width)[: width - used]
    starts = torch.tensor([sum(new[:s]) for s in range(b + 1)], dtype=torch.int32, device=device)
    lengths = torch.tensor(context, dtype=torch.int32, device=device)
    q = normal((sum(new), h, d), dtype, device, seed + 99, 1.5)
    return q, cache, table, starts, lengths


def check(q, cache, table, starts, lengths, max_query=None, max_context=None, **kw):
    max_query = max_query or max(1, int((starts[1:] - starts[:-1]).max()))
    got = paged_attention(q, cache, table, starts, lengths, max_query=max_query, max_context=max_context, **kw)
    quantised = cache.k_scale is not None
    want, bound = A.paged_attention(q, values(cache.k) if quantised else cache.k, values(cache.v) if quantised else cache.v,
                                    cache.k_scale, cache.v_scale, table.clamp(0, cache.pages - 1), starts, lengths, dtype=q.dtype, **kw)
    assert torch.isfinite(got).all()
    err = (got.double() - want).abs()
    assert (err <= bound).all(), (err.max().item(), (err / bound.clamp(min=1e-30)).max().item())
    return got


@pytest.mark.parametrize("codes", [I8, F8, None])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [16, 64, 80, 96, 128, 256])
def test_single_tokens(device, dtype, codes, d):
    check(*sequences(device, dtype, codes or dtype, [1, 1, 1, 1, 1], [1, 2, 33, 400, 64], 4, 2, d, 16))
    check(*sequences(device, dtype, codes or dtype, [1, 1], [700, 129], 8, 1, d, 48), window=100, sinks=3)


@pytest.mark.parametrize("codes", [I8, F8, None])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [16, 64, 80, 96, 128, 256])
def test_chunks(device, dtype, codes, d):
    check(*sequences(device, dtype, codes or dtype, [40, 1, 17], [40, 300, 90], 4, 2, d, 16))
    check(*sequences(device, dtype, codes or dtype, [70, 33], [500, 129], 8, 1, d, 48), window=100, sinks=3)


@pytest.mark.parametrize("d", [8, 40, 128, 136, 256])
@pytest.mark.parametrize("new,context", [([601, 500], [3001, 700]), ([1025], [1030]), ([300, 0, 301], [5000, 9, 301])])
def test_many_rows_in_a_few_parts(device, d, new, context):
    args = sequences(device, torch.bfloat16, torch.bfloat16, new, context, 8, 2, d, 64)
    got = check(*args)
    assert torch.equal(got, check(*args))
    check(*args, window=700, sinks=5)


@pytest.mark.parametrize("codes", [I8, F8, torch.float16])
def test_many_rows_in_a_few_parts_in_half(device, codes):
    check(*sequences(device, torch.float16, codes, [601, 500], [3001, 700], 8, 2, 96, 64))


@pytest.mark.parametrize("page", [1, 3, 16, 31, 32, 64, 100, 256])
@pytest.mark.parametrize("codes", [I8, torch.bfloat16])
def test_page_sizes(device, page, codes):
    for new in ([1, 1], [50, 20]):
        check(*sequences(device, torch.bfloat16, codes, new, [321, 64], 4, 2, 64, page))


@pytest.mark.parametrize("h,h_kv,new", [(1, 1, 1), (16, 1, 1), (17, 1, 1), (5, 1, 3), (6, 2, 5), (3, 1, 6), (64, 2, 1), (12, 12, 16), (12, 12, 17), (40, 1, 9)])
def test_rows_around_the_change_of_kernels(device, h, h_kv, new):
    check(*sequences(device, torch.float16, torch.float16, [new, max(1, new - 1)], [new, 777], h, h_kv, 64, 16))


@pytest.mark.parametrize("codes", [I8, torch.float16])
@pytest.mark.parametrize("new,context", [([1], [20001]), ([1, 1], [9000, 100]), ([30], [12345]), ([200, 3], [6000, 5000])])
def test_long_sequences_are_split(device, codes, new, context):
    args = sequences(device, torch.float16, codes, new, context, 4, 2, 64, 64)
    got = check(*args)
    assert torch.equal(got, check(*args))  # the same bits again
    check(*args, window=3000, sinks=5)


@pytest.mark.parametrize("window,sinks", [(0, 0), (0, 2), (15, 0), (16, 40), (500, 700), (None, 9), (2**31 - 1, 2**31 - 1)])
def test_windows_and_sinks(device, window, sinks):
    for new in ([1, 1, 1], [20, 45, 1]):
        check(*sequences(device, torch.bfloat16, torch.bfloat16, new, [600, 45, 31], 4, 2, 64, 16), window=window, sinks=sinks)


@pytest.mark.parametrize("codes", [I8, torch.bfloat16])
def test_sequences_without_tokens_or_keys(device, codes):
    got = check(*sequences(device, torch.bfloat16, codes, [1, 0, 1, 0], [5, 7, 0, 0], 4, 2, 64, 16))
    assert (got[1] == 0).all()
    got = check(*sequences(device, torch.bfloat16, codes, [30, 0, 20], [10, 7, 0], 4, 2, 64, 16))  # more tokens than keys
    assert (got[:20] == 0).all() and (got[20:30] != 0).any() and (got[30:] == 0).all()


@pytest.mark.parametrize("scale", [-0.4, 0.0, 2.0])
def test_scales(device, scale):
    for new in ([1, 1], [33, 10]):
        check(*sequences(device, torch.bfloat16, I8, new, [100, 333], 4, 2, 64, 16), scale=scale)


def test_bounds_larger_than_the_lengths(device):
    args = sequences(device, torch.bfloat16, I8, [3, 1], [300, 77], 4, 2, 64, 16)
    for max_query, max_context in ((3, 300), (3, 301), (4, 5000), (60, None)):  # other kernels and numbers of parts
        check(*args, max_query=max_query, max_context=max_context)


def test_layouts(device):
    q, cache, table, starts, lengths = sequences(device, torch.float16, torch.float16, [3, 40], [50, 222], 4, 2, 64, 16)
    want = check(q, cache, table, starts, lengths)
    wide = torch.zeros((43, 9, 64), dtype=torch.float16, device=device)
    wide[:, 1:5] = q
    assert torch.equal(check(wide[:, 1:5], cache, table, starts, lengths), want)
    assert torch.equal(check(q.transpose(0, 2).contiguous().transpose(0, 2), cache, table, starts, lengths), want)
    big = torch.full((table.shape[0], table.shape[1] * 2), -1, dtype=torch.int32, device=device)
    big[:, : table.shape[1]] = table
    assert torch.equal(check(q, cache, big[:, : table.shape[1]], starts, lengths), want)
    spread = torch.full((table.shape[0], table.shape[1] * 2), -1, dtype=torch.int32, device=device)
    spread[:, ::2] = table
    assert torch.equal(check(q, cache, spread[:, ::2], starts, lengths), want)


def test_tables_that_point_outside_are_kept_inside(device):
    q, cache, table, starts, lengths = sequences(device, torch.bfloat16, I8, [1, 30], [60, 90], 4, 2, 64, 16)
    for broken_starts, broken_lengths in ((starts, lengths + 100000), (starts, lengths * -1), (starts * 1000, lengths), (starts.flip(0), lengths)):
        for max_query in (1, 30):
            paged_attention(q, cache, table, broken_starts, broken_lengths, max_query=max_query)
    torch.cuda.synchronize()


def test_a_key_that_is_nan_is_not_seen_through_the_mask(device):
    # codes: a hidden key's NaN scale must not reach the row through its zero probability
    q, cache, table, starts, lengths = sequences(device, torch.bfloat16, I8, [1, 40], [100, 140], 4, 2, 64, 16)
    want = paged_attention(q, cache, table, starts, lengths, max_query=40, window=20)
    for s, j in ((0, 79 - 1), (1, 100 - 22)):  # just outside the window of the first row that looks there
        cache.k_scale[table[s, j // 16].long(), j % 16] = math.nan
        cache.v_scale[table[s, j // 16].long(), j % 16] = math.nan
    assert torch.equal(paged_attention(q, cache, table, starts, lengths, max_query=40, window=20), want)


def test_in_a_graph(device):
    q, cache, table, starts, lengths = sequences(device, torch.bfloat16, I8, [1, 1], [3000, 900], 8, 2, 128, 64)
    k, v = normal((2, 2, 128), torch.bfloat16, device, 50), normal((2, 2, 128), torch.bfloat16, device, 51)
    slots = torch.tensor([-1, -1], device=device)

    def step():
        cache.write(k, v, slots)
        return paged_attention(q, cache, table, starts, lengths, max_query=1, max_context=4096)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):  # the lengths and the query change between the replays
        lengths.copy_(torch.tensor([3000 - 500 * i, 900 - 200 * i], dtype=torch.int32))
        q.copy_(normal(q.shape, q.dtype, device, 60 + i))
        slots.copy_(slots_of(table, torch.arange(2, device=device), lengths - 1, 64))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step())


def test_on_another_stream(device):
    args = sequences(device, torch.bfloat16, I8, [1, 1], [3000, 900], 8, 2, 128, 64)
    want = paged_attention(*args, max_query=1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = paged_attention(*args, max_query=1)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@pytest.mark.parametrize("codes", [I8, torch.float16])
def test_without_the_native_calls_the_same_bits(device, codes, monkeypatch):
    def everything():
        q, cache, table, starts, lengths = sequences(device, torch.float16, codes, [1, 30], [3000, 900], 8, 2, 128, 64)
        return (paged_attention(q, cache, table, starts, lengths, max_query=30, window=700, sinks=2),
                paged_attention(q[:1], cache, table[:1], starts[:2], lengths[:1], max_query=1, max_context=3000),
                *cache.read(torch.arange(60, device=device), torch.float16))

    want = everything()
    monkeypatch.setattr(_lib, "calls", lambda *tensors: None)
    for x, y in zip(want, everything()):
        assert torch.equal(x.view(torch.int16), y.view(torch.int16))


def test_no_tokens_at_all(device):
    q, cache, table, starts, lengths = sequences(device, torch.bfloat16, I8, [1], [10], 4, 2, 64, 16)
    assert paged_attention(q[:0], cache, table, starts * 0, lengths, max_query=1).shape == (0, 4, 64)
    none = torch.empty((0, 2, 64), dtype=torch.bfloat16, device=device)
    cache.write(none, none, torch.empty(0, dtype=torch.int64, device=device))
    assert cache.read(torch.empty(0, dtype=torch.int64, device=device))[0].shape == (0, 2, 64)


# ---- refusals ---------------------------------------------------------------------------------------------------------
def test_refusals(device):
    k = torch.zeros((4, 16, 2, 64), dtype=I8, device=device)
    s = torch.zeros((4, 16, 2), device=device)
    for args, message in (
        ((k, k[:2], s, s), "same shape"), ((k.int(), k.int(), s, s), "a cache holds"), ((k, k), "needs k_scale"), ((k.half(), k.half(), s, s), "takes none"),
        ((k, k, s, s[:2]), "scales must be"), ((k, k, s.half(), s.half()), "scales must be"), ((k.cpu(), k.cpu(), s, s), "GPU"),
        ((k[..., :24], k[..., :24], s, s), "multiple of 16"), ((k[..., 1:33], k[..., 1:33], s, s), "16-byte boundary"),
        ((k[:0], k[:0], s[:0], s[:0]), "at least one page"), ((k[..., ::2], k[..., ::2], s, s), "dense"),
    ):
        with pytest.raises(RuntimeError, match=message):
            PagedKVCache(*args)
    cache = PagedKVCache(k, k.clone(), s, s.clone())
    half = PagedKVCache.allocate(4, 16, 2, 64, torch.float16, device)
    x = torch.zeros((3, 2, 64), dtype=torch.bfloat16, device=device)
    slots = torch.arange(3, device=device)
    for call, message in (
        (lambda: cache.write(x, x, slots.float()), "int32 or int64"), (lambda: cache.write(x, x, slots[:2]), "shape"),
        (lambda: cache.write(x.float(), x.float(), slots), "fp16 and bf16"), (lambda: cache.write(x, x.half(), slots), "one dtype"),
        (lambda: half.write(x, x, slots), "goes with"), (lambda: half.read(slots), "goes with"), (lambda: cache.read(slots, torch.float32), "fp16 and bf16"),
        (lambda: cache.write(x.cpu(), x.cpu(), slots), "GPU"), (lambda: cache.read(slots.cpu()), "GPU"),
    ):
        with pytest.raises(RuntimeError, match=message):
            call()
    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16, device=device)
    with pytest.raises(RuntimeError, match="no gradients"):
        paged_attention(q.clone().requires_grad_(), cache, None, None, None, max_query=1)
    table = torch.zeros((2, 3), dtype=torch.int32, device=device)
    starts, lengths = torch.tensor([0, 1, 2], dtype=torch.int32, device=device), torch.tensor([5, 6], dtype=torch.int32, device=device)
    for change, message in (
        ({"q": q[0]}, "3D"), ({"q": q.float()}, "fp16 and bf16"), ({"q": q[..., :32]}, "head dim"), ({"q": q[:, :3]}, "multiple of 2 key heads"),
        ({"query_starts": starts[:2]}, "query_starts"), ({"context_lengths": lengths.long()}, "context_lengths"), ({"page_table": table[:1]}, "page_table"),
        ({"page_table": table.cpu()}, "GPU"), ({"window": -1}, "window"), ({"sinks": -1}, "sinks"), ({"max_query": 0}, "max_query"),
        ({"max_context": 0}, "max_context"), ({"cache": half}, "goes with"),
    ):
        kw = {"q": q, "cache": cache, "page_table": table, "query_starts": starts, "context_lengths": lengths, "max_query": 1, **change}
        with pytest.raises(RuntimeError, match=message):
            paged_attention(**kw)
