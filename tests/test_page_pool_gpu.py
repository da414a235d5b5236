"""The page pool against the oracle's, which serves one sequence after the other; and a step as it is used."""
import random

import pytest
import torch

from gpt_neox_amd import PagedKVCache, PagePool, _lib, paged_attention
from oracle import attention as A
from oracle import pages as P

pytestmark = pytest.mark.gpu


def int32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def twin(pool):
    return P.Pool(pool.page_table.tolist(), pool.lengths.tolist(), pool.free.tolist(), pool.left.item(), pool.page_size)


def agree(pool, want):
    assert pool.lengths.tolist() == want.lengths and pool.left.item() == want.left
    assert pool.page_table.tolist() == want.table and pool.free.tolist() == want.free


def extend(pool, want, new, most=None):
    most = sum(max(n, 0) for n in new) if most is None else most
    step = pool.extend(int32(new, pool.device), max_tokens=most)
    starts, positions, slots, granted = want.extend(new, most)
    assert step.query_starts.tolist() == starts and step.granted.tolist() == granted
    assert step.positions.tolist() == positions and step.slots.tolist() == slots
    assert step.slots.dtype == torch.int64 and step.positions.dtype == step.query_starts.dtype == torch.int32
    agree(pool, want)
    return step


def truncate(pool, want, keep):
    pool.truncate(int32(keep, pool.device))
    want.truncate(keep)
    agree(pool, want)


# both forms of the call: places in the kernel that counts (up to 8192 tokens), and in one of their own
@pytest.mark.parametrize("sequences,most", [(1, 1), (1, 40000), (3, 200), (64, 1), (63, 300), (1000, 12), (1023, 2), (1024, 9), (1025, 9), (2500, 3), (2500, 20)])
@pytest.mark.parametrize("page_size", [1, 16, 48, 256])
def test_random_steps(device, sequences, most, page_size):
    rng = random.Random(sequences * 1000 + most + page_size)
    columns = -(-3 * most // page_size) + 1
    need = sequences * (-(-most * 2 // page_size) + 1)
    for pages in (need * 2, max(1, need // 3)):  # enough, and too few
        pool = PagePool.allocate(pages, page_size, sequences, columns, device)
        want = twin(pool)
        for turn in range(5):
            new = [rng.choice([0, 1, rng.randint(0, most), most, -3]) for _ in range(sequences)]
            extend(pool, want, new)
            keep = [rng.choice([n, 0, max(0, n - rng.randint(0, most)), n + 5, -1]) for n in want.lengths]
            truncate(pool, want, keep)


@pytest.mark.parametrize("most", [0, 1, 6, 7, 100, 8192, 8193, 20000])
def test_max_tokens(device, most):
    pool = PagePool.allocate(40, 4, 4, 20, device)
    extend(pool, twin(pool), [3, 4, 0, 2], most)


def test_a_draft_that_is_dropped_leaves_the_pool_as_it_was(device):
    pool = PagePool.allocate(300, 16, 40, 20, device)
    want = twin(pool)
    extend(pool, want, [i * 7 % 90 for i in range(40)])
    before = [t.clone() for t in (pool.page_table, pool.lengths, pool.free, pool.left)]
    extend(pool, want, [5] * 40)
    pool.truncate(before[1])
    for x, y in zip(before, (pool.page_table, pool.lengths, pool.free, pool.left)):
        assert torch.equal(x, y)


def test_what_the_tensors_say_beyond_themselves_is_kept_inside(device):
    # lengths behind the table, more free pages than there are, pages that are none: nothing is read or written outside
    for left, lengths, numbers in ((1000, [5, 4000, -7], 2**31 - 1), (-5, [2**31 - 1] * 3, -1), (10, [17, 16, 15], -(2**31))):
        pool = PagePool(torch.full((3, 2), numbers, dtype=torch.int32, device=device), int32(lengths, device), torch.full((10,), numbers, dtype=torch.int32, device=device),
                        int32([left], device), page_size=16)
        pool.extend(int32([2**31 - 1, 1, 20], device), max_tokens=50)
        pool.extend(int32([9, -(2**31), 2**31 - 1], device), max_tokens=9000)
        pool.truncate(int32([0, 3, -9], device))
        assert 0 <= pool.left.item() <= 10
    torch.cuda.synchronize()


def test_layouts(device):
    wide = torch.full((5, 12), -9, dtype=torch.int32, device=device)
    wide[:, :7] = -1
    pool = PagePool(wide[:, :7], int32([0] * 5, device), torch.arange(50, dtype=torch.int32, device=device), int32([50], device), page_size=8)
    want = twin(pool)
    new = torch.zeros(10, dtype=torch.int32, device=device)
    new[::2] = int32([9, 8, 0, 41, 56], device)
    step = pool.extend(new[::2], max_tokens=114)
    assert want.extend(new[::2].tolist(), 114)[2] == step.slots.tolist()
    truncate(pool, want, [1, 0, 0, 16, 17])
    assert (wide[:, 7:] == -9).all()


def test_more_than_a_workgroup_gives_back_at_once(device):
    pool = PagePool.allocate(9000, 2, 3, 5000, device)
    want = twin(pool)
    extend(pool, want, [9999, 1, 4000])
    truncate(pool, want, [3, 0, 4000])
    extend(pool, want, [0, 9000, 17])
    truncate(pool, want, [0, 0, 0])
    assert pool.left.item() == 9000 and (pool.page_table == -1).all()


@pytest.mark.parametrize("empty", [0, 1, 1023, 1024, 2500])
def test_many_sequences_without_tokens(device, empty):
    # between the sequences of a workgroup's tokens, and behind the last one
    new = []
    for n in (3, 1021, 1, 1024, 7000, 2, 900, 130):
        new += [n] + [0] * empty
    pool = PagePool.allocate(2600, 4, len(new), 1750, device)
    want = twin(pool)
    extend(pool, want, new)
    extend(pool, want, [1] * len(new), max(8200, len(new) + 5))
    truncate(pool, want, [3 * (i % 2) for i in range(len(new))])


def test_outputs_do_not_share(device):
    # writing into one output leaves the others and the pool
    pool = PagePool.allocate(50, 16, 7, 10, device)
    step = pool.extend(int32([5, 0, 17, 3, 1, 0, 9], device), max_tokens=41)
    kept = [t.clone() for t in step]
    for i, t in enumerate(step):
        assert t.is_contiguous() and t.shape == kept[i].shape
        t.fill_(1)
        for j in range(i + 1, 4):
            assert torch.equal(step[j], kept[j])
    assert [t.dtype for t in step] == [torch.int32, torch.int32, torch.int64, torch.bool]


def test_in_inference_mode(device):
    pool, cache = PagePool.allocate(20, 16, 3, 8, device), PagedKVCache.allocate(20, 16, 2, 64, torch.float4_e2m1fn_x2, device)
    new = int32([20, 0, 5], device)
    with torch.inference_mode():
        step = pool.extend(new, max_tokens=25)
        kv = torch.randn((25, 2, 64), device=device).bfloat16()
        cache.write(kv, kv, step.slots)
        out = paged_attention(kv, cache, pool.page_table, step.query_starts, pool.lengths, max_query=20)
        step.positions.add_(1)
        assert (step.slots + 0).tolist() == [*range(20), *range(32, 37)] and step.positions.tolist() == [*range(1, 21), *range(1, 6)]
    assert torch.isfinite(out).all() and step.granted.all()
    pool.truncate(int32([0, 0, 0], device))
    assert pool.left.item() == 20


def test_on_another_stream(device):
    pool = PagePool.allocate(100, 16, 5, 20, device)
    want = twin(pool)
    new = int32([100, 0, 33, 16, 1], device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step = pool.extend(new, max_tokens=150)
        pool.truncate(int32([90, 0, 0, 16, 1], device))
    torch.cuda.current_stream().wait_stream(side)
    assert step.slots.tolist() == want.extend(new.tolist(), 150)[2]
    want.truncate([90, 0, 0, 16, 1])
    assert pool.lengths.tolist() == want.lengths and pool.free.tolist()[: want.left] == want.free[: want.left]


@pytest.mark.parametrize("codes", ["fp4", "int8"])
def test_the_example_serves_with_a_pool(device, codes):
    import os
    import sys

    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import windowed_layer

    assert 0 < windowed_layer.main(["--codes", codes]) < 1


def test_refusals(device):
    pool = PagePool.allocate(9, 16, 4, 3, device)
    new = int32([1] * 4, device)
    for call, message in (
        (lambda: pool.extend(new[:3], max_tokens=4), r"new_tokens must be int32 \[4\]"), (lambda: pool.extend(new.long(), max_tokens=4), "int32"),
        (lambda: pool.extend(new, max_tokens=-1), "max_tokens"), (lambda: pool.extend(new, max_tokens=2**30), "max_tokens"), (lambda: pool.extend(new.cpu(), max_tokens=4), "GPU"),
        (lambda: pool.extend(new, max_tokens=2.5), "max_tokens"), (lambda: pool.truncate(new[None]), r"lengths must be int32 \[4\]"), (lambda: pool.truncate(new.cpu()), "GPU"),
    ):
        with pytest.raises(RuntimeError, match=message):
            call()
    assert pool.lengths.tolist() == [0] * 4 and pool.left.item() == 9
    with pytest.raises(AttributeError, match="cannot be replaced"):
        pool.lengths = new


def test_without_the_native_calls_the_same(device, monkeypatch):
    monkeypatch.setattr(_lib, "calls", lambda *tensors: None)
    pool = PagePool.allocate(200, 16, 30, 20, device)
    want = twin(pool)
    extend(pool, want, [i * 7 % 90 for i in range(30)])
    extend(pool, want, [1] * 30, 9000)
    truncate(pool, want, [i * 3 for i in range(30)])


def test_in_a_graph(device):
    # a step with the pool, the cache and the attention, replayed while new sequences come and others end
    b, h, h_kv, d, page = 3, 4, 2, 64, 16
    pool, other = (PagePool.allocate(60, page, b, 20, device) for _ in range(2))
    caches = [PagedKVCache.allocate(60, page, h_kv, d, torch.float4_e2m1fn_x2, device) for _ in range(2)]
    new, keep = int32([100, 37, 60], device), int32([0] * 3, device)
    q, k, v = (torch.zeros((200, n, d), dtype=torch.bfloat16, device=device) for n in (h, h_kv, h_kv))

    def step(pool, cache):
        pool.truncate(keep)
        s = pool.extend(new, max_tokens=200)
        cache.write(k, v, s.slots)
        return paged_attention(q, cache, pool.page_table, s.query_starts, pool.lengths, max_query=200, max_context=320), s

    for p, c in ((pool, caches[0]), (other, caches[1])):
        step(p, c)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, places = step(pool, caches[0])
    for turn, (kept, count) in enumerate([([100, 0, 60], [1, 130, 1]), ([101, 130, 61], [5, 5, 5]), ([103, 131, 61], [1, 1, 1]), ([104, 0, 0], [90, 50, 60])]):
        keep.copy_(int32(kept, device))
        new.copy_(int32(count, device))
        for t in (q, k, v):
            t.normal_(generator=torch.Generator(device=device).manual_seed(turn))
        graph.replay()
        torch.cuda.synchronize()
        eager, where = step(other, caches[1])
        n = sum(count)
        assert torch.equal(out[:n], eager[:n]) and all(torch.equal(x, y) for x, y in zip(places, where))
        assert torch.equal(pool.page_table, other.page_table) and torch.equal(pool.lengths, other.lengths) and torch.equal(pool.free, other.free)


@pytest.mark.parametrize("codes", [torch.float4_e2m1fn_x2, torch.int8, torch.bfloat16])
def test_generation_as_it_is_used(device, codes):
    # prompts, drafts of which some tokens are dropped, a sequence that ends and another in its place: after every step the
    # attention is that over each sequence's own keys, in the order in which they came
    b, h, h_kv, d, page = 4, 4, 2, 64, 16
    pool = PagePool.allocate(50, page, b, 16, device)
    cache = PagedKVCache.allocate(50, page, h_kv, d, codes, device)
    g = torch.Generator(device=device).manual_seed(7)
    held = [torch.zeros((0, 2, h_kv, d), dtype=torch.bfloat16, device=device) for _ in range(b)]
    steps = [([70, 33, 0, 128], None), ([1, 1, 1, 1], None), ([5, 5, 5, 5], [72, 35, 6, 131]), ([1, 0, 1, 90], [73, 0, 7, 221]), ([3, 61, 1, 1], None)]
    for new, keep in steps:
        n = sum(new)
        q = torch.randn((n, h, d), generator=g, device=device).bfloat16()
        kv = torch.randn((n, 2, h_kv, d), generator=g, device=device).bfloat16()
        step = pool.extend(int32(new, device), max_tokens=n)
        assert step.granted.all()
        cache.write(kv[:, 0], kv[:, 1], step.slots)
        longest = int(pool.lengths.max())
        got = paged_attention(q, cache, pool.page_table, step.query_starts, pool.lengths, max_query=max(new), max_context=longest)
        # what the cache holds of them: its own reading, in 32 bits for int8
        rk, rv = cache.read(step.slots, torch.bfloat16)
        if codes == torch.bfloat16:
            assert torch.equal(rk, kv[:, 0]) and torch.equal(rv, kv[:, 1])
        at = step.query_starts.tolist()
        for s in range(b):
            held[s] = torch.cat((held[s], torch.stack((rk, rv), 1)[at[s] : at[s + 1]]))
            if at[s] == at[s + 1]:
                continue
            m = held[s].shape[0]
            assert pool.lengths[s].item() == m
            whole = held[s].view(1, m, 2, h_kv, d)
            want, bound = A.paged_attention(q[at[s] : at[s + 1]], whole[:, :, 0], whole[:, :, 1], None, None, torch.zeros((1, 1), dtype=torch.int32, device=device),
                                            int32([0, at[s + 1] - at[s]], device), int32([m], device), dtype=torch.bfloat16)
            if codes == torch.int8:
                # the kernel multiplies by the scales in 32 bits, the reading was rounded to 16 once more: half a unit of a
                # value, and of a key's part of a score (2^-9 of the sum of |q k| / 8, which is below 24 here)
                bound = bound + 2.0**-9 * (1 + 2 * 24) * whole[0, :, 1].abs().amax()
            assert ((got[at[s] : at[s + 1]].double() - want).abs() <= bound).all()
        if keep is not None:
            pool.truncate(int32(keep, device))
            held = [t[:n] for t, n in zip(held, keep)]
