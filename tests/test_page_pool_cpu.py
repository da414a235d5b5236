"""The page pool and 4-bit caches without a GPU: refusals, and what cannot be replaced."""
import ctypes

import pytest
import torch

from gpt_neox_amd import _lib
from gpt_neox_amd.page_pool import PagePool
from gpt_neox_amd.paged_cache import PagedKVCache

F4 = torch.float4_e2m1fn_x2


@pytest.fixture(scope="module")
def p():
    """An aligned address that is never read."""
    buf = ctypes.create_string_buffer(4096)
    yield (ctypes.addressof(buf) + 255) & ~255
    del buf


def st(*values):
    return (ctypes.c_int64 * len(values))(*values)


def refused(status, code, message):
    assert status == code
    assert message.encode() in _lib.lib().neox_fused_last_error()


def test_extend(p):
    def call(**change):
        a = dict(starts=p, positions=p, slots=p, granted=p, ws=p, table=p, lengths=p, free=p, left=p, new=p, sequences=4, columns=3, stride=3, pages=9,
                 page=16, most=7, stream=None)
        a.update(change)
        return _lib.lib().neox_pages_extend(*a.values())

    for change, code, message in (
        ({"table": None}, -1, "page_table is null"), ({"lengths": p + 2}, -5, "lengths"), ({"free": None}, -1, "free_pages"), ({"left": p + 1}, -5, "left"),
        ({"new": None}, -1, "numbers"), ({"sequences": 0}, -3, "sequences=0"), ({"columns": -1}, -3, "columns=-1"), ({"pages": 1 << 30}, -3, "pages"),
        ({"page": 0}, -3, "page_size=0"), ({"stride": 2}, -4, "table stride 2"), ({"most": -1}, -3, "max_tokens=-1"), ({"most": 1 << 30}, -3, "max_tokens"),
        ({"starts": None}, -1, "output"), ({"slots": None}, -1, "output"), ({"ws": None}, -1, "workspace"), ({"slots": p + 4}, -5, "misaligned"),
        ({"positions": p + 2}, -5, "misaligned"),
    ):
        refused(call(**change), code, message)


def test_truncate(p):
    def call(**change):
        a = dict(table=p, lengths=p, free=p, left=p, keep=p, sequences=4, columns=3, stride=3, pages=9, page=16, stream=None)
        a.update(change)
        return _lib.lib().neox_pages_truncate(*a.values())

    for change, code, message in (({"keep": None}, -1, "numbers"), ({"free": p + 2}, -5, "free_pages"), ({"pages": 0}, -3, "pages=0"), ({"stride": 0}, -4, "stride")):
        refused(call(**change), code, message)


def test_a_pool_looks_at_its_tensors():
    def t(*shape):
        return torch.zeros(shape, dtype=torch.int32)

    for args, message in (
        ((t(4), t(4), t(9), t(1)), "page_table must be a 2D"), ((t(4, 3).long(), t(4), t(9), t(1)), "int32"), ((t(4, 3), t(5), t(9), t(1)), r"lengths must be int32 \[4\]"),
        ((t(4, 3), t(4), t(9), t(2)), r"left int32 \[1\]"), ((t(4, 0), t(4), t(9), t(1)), "not be empty"), ((t(4, 6)[:, ::2], t(4), t(9), t(1)), "dense"),
        ((t(1, 3).expand(4, 3), t(4), t(9), t(1)), "overlap"), ((t(4, 3), t(4), t(0), t(1)), "not be empty"),
    ):
        with pytest.raises(RuntimeError, match=message):
            PagePool(*args, page_size=16)
    for size in (0, -1, 2.0, True, 2**30):
        with pytest.raises(RuntimeError, match="page_size"):
            PagePool(t(4, 3), t(4), t(9), t(1), page_size=size)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        PagePool(t(4, 3), t(4), t(9), t(1), page_size=16)


@pytest.mark.parametrize("name", ["page_table", "lengths", "free", "left", "page_size", "sequences", "columns", "pages", "device"])
def test_what_was_checked_cannot_be_replaced(name):
    pool = object.__new__(PagePool)
    setattr(pool, name, 1)
    with pytest.raises(AttributeError, match="cannot be replaced"):
        setattr(pool, name, 2)
    pool.label = "all layers"
    pool.label = "layer 4"


def paged(p, **change):
    a = dict(out=p, ws=None, size=0, q=p, kc=p, vc=p, ks=p, vs=p, table=p, starts=p, lengths=p, b=2, tokens=2, max_query=1, max_context=100, h=4, h_kv=2,
             d=64, pages=8, page=16, columns=7, stride=7, os=st(256, 64), qs=st(256, 64), kcs=st(1024, 64, 32), vcs=st(1024, 64, 32), kss=st(64, 4, 2),
             vss=st(64, 4, 2), scale=0.1, window=-1, sinks=0, dtype=_lib.NEOX_BF16, cache=_lib.NEOX_F4, stream=None)
    a.update(change)
    return _lib.lib().neox_paged_attention(*a.values())


def test_attention_over_4_bits(p):
    wide = dict(os=st(384, 96), qs=st(384, 96))
    for change, code, message in (
        ({"d": 48}, -3, "multiple of 32"), ({"d": 16}, -3, "multiple of 32"), ({"ks": None}, -1, "k_scales"), ({"vs": None}, -1, "v_scales"),
        ({"kc": p + 8}, -5, "k_cache"), ({"kcs": st(1024, 64, 16)}, -4, "k_cache head stride"), ({"vcs": st(1024, 72, 32)}, -4, "multiple of 16"),
        ({"kss": st(64, 4, 1)}, -4, "k_scales head stride"), ({"d": 96, "vss": st(64, 6, 3), "kcs": st(1536, 96, 48), "vcs": st(1536, 96, 48), **wide}, -4, "k_scales"),
        ({"vss": st(-64, 4, 2)}, -4, "negative"), ({"kss": st(1 << 31, 4, 2)}, -4, "below 2^31"), ({"cache": 6}, -2, "the cache must hold"),
        ({"max_context": 100000}, -1, "workspace is null"),
    ):
        refused(paged(p, **change), code, message)


def test_more_blocks_than_a_launch_has(p):
    strides = dict(h=48, h_kv=1, os=st(64 * 64, 64), qs=st(64 * 64, 64), kcs=st(512, 32, 32), vcs=st(512, 32, 32), kss=st(32, 2, 2), vss=st(32, 2, 2))
    refused(paged(p, b=1 << 29, max_query=1, max_context=16, **strides), -3, "too large for one call")


def test_writing_4_bits(p):
    def write(**change):
        a = dict(kc=p, vc=p, ks=p, vs=p + 1, k=p, v=p, slots=p, wide=1, tokens=3, h=2, d=64, pages=4, page=16, kcs=st(1024, 64, 32), vcs=st(1024, 64, 32),
                 kss=st(64, 4, 2), vss=st(64, 4, 2), k2=st(128, 64), v2=st(128, 64), dtype=_lib.NEOX_F16, cache=_lib.NEOX_F4, stream=None)
        a.update(change)
        return _lib.lib().neox_cache_write(*a.values())

    for change, code, message in (({"d": 48}, -3, "multiple of 32"), ({"vs": None}, -1, "v_scales"), ({"k2": st(128, 32)}, -4, "k head stride"), ({"dtype": _lib.NEOX_F4}, -2, "fp16 and bf16")):
        refused(write(**change), code, message)


def test_a_cache_in_4_bits_looks_at_its_tensors():
    def codes(*shape):
        return torch.zeros(shape, dtype=torch.uint8).view(F4)

    def scales(*shape):
        return torch.zeros(shape, dtype=torch.uint8).view(torch.float8_e8m0fnu)

    k, s = codes(4, 16, 2, 32), scales(4, 16, 2, 2)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        PagedKVCache(k, k, s, s)
    with pytest.raises(RuntimeError, match="a cache holds"):
        PagedKVCache(k.view(torch.uint8), k.view(torch.uint8), s, s)
    with pytest.raises(RuntimeError, match="multiple of 32"):
        PagedKVCache.allocate(4, 16, 2, 48, F4, "cpu")


HUGE = 1 << 24  # blocks of 256 threads: a launch has less than 2^32 in one direction


@pytest.mark.parametrize("cache", [_lib.NEOX_F4, _lib.NEOX_I8, _lib.NEOX_BF16])
@pytest.mark.parametrize("change", [
    dict(b=HUGE, max_context=16, h=1, h_kv=1), dict(b=HUGE - 3, max_context=16, h=1, h_kv=1), dict(b=HUGE // 3 + 1, max_context=16, h=6, h_kv=3),
    dict(b=HUGE // 2, max_query=100, max_context=100, h=4, h_kv=2),
    dict(b=1, tokens=HUGE // 32, max_query=1, max_context=100000, h=32, h_kv=2, ws=True, size=1 << 62),  # (the parts' join: a block for each row)
])
def test_launches_that_do_not_fit(p, cache, change):
    codes = 2 if cache == _lib.NEOX_F4 else 1
    wide = {n: st(4096, 256, 64 // codes) for n in ("kcs", "vcs")}
    change = {**change, **({"ws": p} if "ws" in change else {})}
    refused(paged(p, cache=cache, os=st(2048, 64), qs=st(2048, 64), **wide, **change), -3, "too large for one call")


def test_blocks_of_rows_that_do_not_fit(p):
    strides = dict(h=48, h_kv=1, os=st(64 * 64, 64), qs=st(64 * 64, 64))  # three blocks of 16 rows
    refused(paged(p, b=HUGE // 3 + 1, max_query=1, max_context=16, **strides), -3, "too large for one call")


@pytest.mark.parametrize("cache,d,into,back", [(_lib.NEOX_F4, 32, None, 2**30 - 1), (_lib.NEOX_F4, 256, 2**28, 2**27), (_lib.NEOX_F4, 160, 2**28 - 1, 2**27),
                                               (_lib.NEOX_I8, 128, 2**29, 2**28), (_lib.NEOX_F16, 256, 2**27, 2**27)])
def test_caches_whose_launches_do_not_fit(p, cache, d, into, back):
    # tokens of one head, from 2 to 32 threads each
    row = d // 2 if cache == _lib.NEOX_F4 else d
    outside, held, scales = st(d, d), st(64 * row, row, row), st(64, 8, 8)
    lib, types = _lib.lib(), (_lib.NEOX_F16, cache, None)
    refused(lib.neox_cache_read(p, p, p, p, p, p, p, 1, back, 1, d, 4, 16, outside, outside, held, held, scales, scales, *types), -3, "too large for one call")
    if into:
        refused(lib.neox_cache_write(p, p, p, p, p, p, p, 1, into, 1, d, 4, 16, held, held, scales, scales, outside, outside, *types), -3, "too large for one call")
