"""Argument errors of the attention and cache entry points: reported before any HIP call, so on a machine without a GPU."""
import ctypes

import pytest
import torch

from gpt_neox_amd import _lib
from gpt_neox_amd.fused_attention import window_attention
from gpt_neox_amd.paged_cache import PagedKVCache, paged_attention, slots_of

F16, BF16, F32, I8, F8 = _lib.NEOX_F16, _lib.NEOX_BF16, _lib.NEOX_F32, _lib.NEOX_I8, _lib.NEOX_F8


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


def window_fwd(p, **change):
    a = dict(out=p, low=p, lse=p, q=p, k=p, v=p, lengths=None, b=2, sq=8, sk=8, h=4, h_kv=2, d=64, qs=st(512, 256, 64), ks=st(256, 128, 64),
             vs=st(256, 128, 64), os=st(512, 256, 64), scale=0.1, window=4, sinks=1, dtype=BF16, stream=None)
    a.update(change)
    return _lib.lib().neox_window_attention_fwd(*a.values())


def test_window_attention_forward(p):
    for change, code, message in (
        ({"dtype": F32}, -2, "fp16 and bf16"), ({"q": None}, -1, "q is null"), ({"out": None}, -1, "out is null"), ({"v": p + 8}, -5, "16-byte"),
        ({"lse": p + 2}, -5, "misaligned"), ({"lengths": p + 1}, -5, "misaligned"), ({"b": 0}, -3, "b=0"), ({"sq": 0}, -3, "sq=0"), ({"sk": -1}, -3, "sk=-1"),
        ({"h": 5}, -3, "multiple of h_kv"), ({"h_kv": 0}, -3, "multiple of h_kv"), ({"d": 60}, -3, "head dim 60"), ({"d": 264}, -3, "head dim 264"),
        ({"qs": None}, -1, "q strides"), ({"qs": st(-512, 256, 64)}, -4, "negative"), ({"ks": st(256, 128, 60)}, -4, "multiple of 8"),
        ({"vs": st(256, 128, 32)}, -4, "smaller than d"), ({"os": st(1 << 31, 256, 64)}, -4, "below 2^31"), ({"scale": float("nan")}, -3, "finite"),
        ({"scale": float("inf")}, -3, "finite"), ({"sinks": -1}, -3, "sinks"), ({"b": 1 << 20, "sq": 1 << 20}, -3, "too large"),
    ):
        refused(window_fwd(p, **change), code, message)


def test_window_attention_backward(p):
    lib, need = _lib.lib(), ctypes.c_int64()
    sizes = (2, 8, 8, 4, 2, 64)
    assert lib.neox_window_attention_bwd_workspace(need, *sizes, 4, 1) == 0 and need.value == 4 * 2 * 4 * 8
    assert lib.neox_window_attention_bwd_workspace(need, 1, 4096, 4096, 32, 8, 128, 1024, 4) == 0 and need.value > 4 * 32 * 4096
    refused(lib.neox_window_attention_bwd_workspace(None, *sizes, 4, 1), -1, "bytes is null")
    refused(lib.neox_window_attention_bwd_workspace(need, 2, 8, 8, 4, 3, 64, 4, 1), -3, "multiple of h_kv")
    q3, k3 = st(512, 256, 64), st(256, 128, 64)

    def bwd(**change):
        a = dict(dq=p, dk=p, dv=p, ws=p, size=256, dout=p, out=p, low=p, lse=p, q=p, k=p, v=p, lengths=None, b=2, sq=8, sk=8, h=4, h_kv=2, d=64, s0=q3, s1=k3,
                 s2=k3, s3=q3, s4=q3, s5=q3, s6=k3, s7=k3, scale=0.1, window=4, sinks=1, dtype=F16, stream=None)
        a.update(change)
        return lib.neox_window_attention_bwd(*a.values())

    for change, code, message in (
        ({"dtype": I8}, -2, "fp16 and bf16"), ({"dq": None}, -1, "dq is null"), ({"lse": None}, -1, "lse is null"), ({"ws": None}, -1, "workspace is null"),
        ({"size": 255}, -3, "needs 256"), ({"dout": p + 4}, -5, "dout"), ({"s1": st(256, 128, 8)}, -4, "dk head stride"), ({"s4": st(4, 256, 64)}, -4, "out stride"),
    ):
        refused(bwd(**change), code, message)


def paged(p, **change):
    a = dict(out=p, ws=None, size=0, q=p, kc=p, vc=p, ks=p, vs=p, table=p, starts=p, lengths=p, b=2, tokens=2, max_query=1, max_context=100, h=4, h_kv=2,
             d=64, pages=8, page=16, columns=7, stride=7, os=st(256, 64), qs=st(256, 64), kcs=st(2048, 128, 64), vcs=st(2048, 128, 64), kss=st(32, 2, 1),
             vss=st(32, 2, 1), scale=0.1, window=-1, sinks=0, dtype=BF16, cache=I8, stream=None)
    a.update(change)
    return _lib.lib().neox_paged_attention(*a.values())


def test_paged_attention(p):
    for change, code, message in (
        ({"dtype": F8}, -2, "fp16 and bf16"), ({"cache": F16}, -2, "the cache must hold"), ({"cache": F32}, -2, "the cache must hold"), ({"table": None}, -1, "page_table"),
        ({"starts": p + 2}, -5, "query_starts"), ({"lengths": None}, -1, "context_lengths"), ({"ks": None}, -1, "k_scales"), ({"kc": p + 8}, -5, "k_cache"),
        ({"b": 0}, -3, "b=0"), ({"tokens": 0}, -3, "tokens=0"), ({"max_query": 0}, -3, "max_query=0"), ({"max_context": 1 << 30}, -3, "max_context"),
        ({"h": 3}, -3, "multiple of h_kv"), ({"d": 40}, -3, "multiple of 16"), ({"pages": 0}, -3, "pages=0"), ({"page": 0}, -3, "page_size=0"),
        ({"columns": 0}, -3, "column"), ({"stride": -1}, -3, "column"), ({"kcs": st(2048, 128, 72)}, -4, "multiple of 16"), ({"vss": st(32, 2, 0)}, -4, "v_scales"),
        ({"qs": st(256, 32)}, -4, "q head stride"), ({"max_context": 100000}, -1, "workspace is null"),
        ({"max_context": 100000, "ws": p, "size": 64}, -3, "needs"), ({"sinks": -2}, -3, "sinks"),
    ):
        refused(paged(p, **change), code, message)
    need = ctypes.c_int64(-1)
    size = _lib.lib().neox_paged_attention_workspace
    assert size(need, 2, 2, 1, 100, 4, 2, 64, -1, 0) == 0 and need.value == 0
    assert size(need, 1, 1, 1, 1000, 4, 2, 64, -1, 0) == 0 and need.value == 4 * 4 * 65 * 4
    assert size(need, 1, 1, 1, 1000, 4, 2, 64, 100, 4) == 0 and need.value == 0  # what the window shows needs no splitting
    refused(size(None, 2, 2, 1, 100, 4, 2, 64, -1, 0), -1, "bytes is null")
    refused(size(need, 2, 2, 1, 100, 4, 2, 64, -1, -1), -3, "sinks")


def test_cache_calls(p):
    lib = _lib.lib()

    def write(**change):
        a = dict(kc=p, vc=p, ks=p, vs=p, k=p, v=p, slots=p, wide=1, tokens=3, h=2, d=64, pages=4, page=16, kcs=st(2048, 128, 64), vcs=st(2048, 128, 64),
                 kss=st(32, 2, 1), vss=st(32, 2, 1), k2=st(128, 64), v2=st(128, 64), dtype=BF16, cache=F8, stream=None)
        a.update(change)
        return lib.neox_cache_write(*a.values())

    for change, code, message in (
        ({"dtype": F32}, -2, "fp16 and bf16"), ({"cache": F16}, -2, "the cache must hold"), ({"k": None}, -1, "k is null"), ({"v": p + 4}, -5, "v must be"),
        ({"slots": p + 4}, -5, "slots"), ({"slots": None}, -1, "slots"), ({"tokens": 0}, -3, "0 tokens"), ({"tokens": 1 << 30}, -3, "2^30"), ({"h": 0}, -3, "h_kv=0"),
        ({"d": 24}, -3, "multiple of 16"), ({"k2": st(128, 60)}, -4, "k stride"), ({"v2": None}, -1, "v strides"), ({"kcs": st(2048, 120, 64)}, -4, "k_cache"),
        ({"vs": None}, -1, "v_scales"), ({"pages": 1 << 30}, -3, "pages"),
    ):
        refused(write(**change), code, message)
    refused(lib.neox_cache_read(None, p, p, p, p, p, p, 0, 3, 2, 64, 4, 16, st(128, 64), st(128, 64), st(2048, 128, 64), st(2048, 128, 64), st(32, 2, 1),
                                st(32, 2, 1), BF16, I8, None), -1, "neox_cache_read: k is null")


def test_there_is_no_cpu_fallback():
    q = torch.zeros(4, 1, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        window_attention(q, q, q)
    k = torch.zeros(2, 16, 2, 64, dtype=torch.int8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        PagedKVCache(k, k, torch.zeros(2, 16, 2), torch.zeros(2, 16, 2))


def test_slots_of():
    table = torch.tensor([[5, 2, 7], [1, 0, 3]], dtype=torch.int32)
    sample, position = torch.tensor([0, 0, 1, 1]), torch.tensor([0, 9, 4, 11])
    assert slots_of(table, sample, position, 4).tolist() == [20, 29, 0, 15]
    assert callable(paged_attention)
