"""A paged key/value cache in 16, 8 or 4 bits, and the attention of new tokens over it.

:class:`PagedKVCache` holds the keys and values of many sequences in pages of a fixed number of tokens; which pages
belong to a sequence is the caller's page table (or a :class:`~gpt_neox_amd.page_pool.PagePool`'s).  New keys and values
are quantised as they are written (:meth:`PagedKVCache.write`) to int8 or 8-bit floats with an fp32 scale for each token
and head, to 4-bit floats with a power of two for every 32 values, or kept in 16 bits;
:func:`paged_attention` reads them where they lie, for one new token of each sequence (generation) or many (prompts in
chunks), with or without a window and sinks as in :func:`~gpt_neox_amd.fused_attention.window_attention`.  Nothing
here looks at the page table, the lengths or the slots on the host, so a step can be recorded into a HIP graph.
"""
import ctypes
import math
import operator

import torch

from . import _lib
from .fused_attention import check_window

_HALF = (torch.float16, torch.bfloat16)
_CODES = {torch.int8: _lib.NEOX_I8, torch.float8_e4m3fn: _lib.NEOX_F8, torch.float4_e2m1fn_x2: _lib.NEOX_F4}
_F4_GROUP = 32  # values of a 4-bit cache that share a scale


class PagedKVCache:
    """Keys and values ``[pages, page_size, heads, dim]`` in fp16, bf16, int8 or float8_e4m3fn, the last two with scales
    ``[pages, page_size, heads]`` in fp32, or in float4_e2m1fn_x2, two values to an element (``dim / 2`` of them, the first value
    in the low half), with scales ``[pages, page_size, heads, dim / 32]`` in float8_e8m0fnu, one for each 32 neighbouring values.
    Slot ``page * page_size + i`` is token ``i`` of a page.

    Values in 4 bits are 0, 0.5, 1, 1.5, 2, 3, 4 or 6 times a power of two, with a sign.  ``write`` takes the least power of
    which seven times is no less than the 32 values' largest magnitude, from 2^-125 up to 2^125 (bf16) or 2^13 (fp16), and rounds to
    the nearest of these, to the even code at ties; what is above six times the power becomes six times.  A token's
    head that holds an infinity or a NaN gets NaN scales and reads back as NaN, as in 8 bits.  (In a cache filled otherwise, scales above
    2^125 count as NaN, and values whose scale is below 2^-125 may count as zero.)

    The tensors may be views (of one buffer for all layers, say) as long as every head's values are dense and start on
    16-byte boundaries.  They are looked at once, here, and stay: other tensors are another cache.
    """

    _FIXED = frozenset(("k", "v", "k_scale", "v_scale", "pages", "page_size", "heads", "dim", "dtype", "device", "quantised", "_strides"))

    def __setattr__(self, name, value):
        if name in self._FIXED and name in self.__dict__:
            raise AttributeError(f"{name} of a cache cannot be replaced: make a PagedKVCache of the new tensors")
        super().__setattr__(name, value)

    def __init__(self, k, v, k_scale=None, v_scale=None):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype:
            raise RuntimeError("k and v must have the same shape [pages, page_size, heads, dim] and dtype")
        if k.dtype not in _HALF and k.dtype not in _CODES:
            raise RuntimeError(f"a cache holds fp16, bf16, int8, float8_e4m3fn or float4_e2m1fn_x2, not {k.dtype}")
        _lib.require_gpu(k, v, k_scale, v_scale)
        self.quantised = k.dtype in _CODES
        per_piece, packed = 16 // k.element_size(), 2 if k.dtype == torch.float4_e2m1fn_x2 else 1
        dim = k.shape[3] * packed
        if k.shape[3] % per_piece or not 8 <= dim <= 256:
            raise RuntimeError(f"head dim {dim} must be a multiple of {per_piece * packed} up to 256 for a cache in {k.dtype}")
        if k.numel() == 0:
            raise RuntimeError("a cache needs at least one page, one token per page and one head")
        for t in (k, v):
            if t.stride(3) != 1 or t.data_ptr() % 16 or any(s % per_piece for n, s in zip(t.shape[:3], t.stride()) if n > 1):
                raise RuntimeError("every head's values must be dense and start on a 16-byte boundary")
        if self.quantised != (k_scale is not None) or self.quantised != (v_scale is not None):
            raise RuntimeError("a cache in 8 or 4 bits needs k_scale and v_scale, one in 16 bits takes none")
        if packed == 2:
            shape = (*k.shape[:3], dim // _F4_GROUP)
            for t in (k_scale, v_scale):
                if t.shape != shape or t.dtype != torch.float8_e8m0fnu:
                    raise RuntimeError(f"scales must be float8_e8m0fnu {list(shape)}")
                if t.stride(3) != 1 and t.shape[3] > 1:
                    raise RuntimeError("the scales of a token's head must be dense")
        elif self.quantised:
            for t in (k_scale, v_scale):
                if t.shape != k.shape[:3] or t.dtype != torch.float32:
                    raise RuntimeError(f"scales must be float32 {list(k.shape[:3])}")
        for t in (v, k_scale, v_scale):
            if t is not None and t.device != k.device:
                raise RuntimeError("all tensors must be on the same device")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.pages, self.page_size, self.heads, self.dim = *k.shape[:3], dim
        self.dtype, self.device = k.dtype, k.device
        # the scales of 8 bits have no dense axis of their own: [..., None] gives row_strides one to leave out
        scales = [_lib.row_strides(t[..., None] if t.dim() == 3 else t) if t is not None else None for t in (k_scale, v_scale)]
        self._strides = (_lib.row_strides(k), _lib.row_strides(v), *scales)

    @classmethod
    def allocate(cls, pages, page_size, heads, dim, dtype=torch.int8, device="cuda"):
        """A cache of zeros."""
        if dtype == torch.float4_e2m1fn_x2:
            if dim % _F4_GROUP:
                raise RuntimeError(f"head dim {dim} must be a multiple of {_F4_GROUP} up to 256 for a cache in {dtype}")
            k, v, k_scale, v_scale = (torch.zeros((pages, page_size, heads, dim // n), dtype=torch.uint8, device=device) for n in (2, 2, _F4_GROUP, _F4_GROUP))
            return cls(k.view(dtype), v.view(dtype), k_scale.view(torch.float8_e8m0fnu), v_scale.view(torch.float8_e8m0fnu))
        k, v = (torch.zeros((pages, page_size, heads, dim), dtype=torch.int8, device=device).view(dtype) if dtype in _CODES
                else torch.zeros((pages, page_size, heads, dim), dtype=dtype, device=device) for _ in "kv")
        if dtype not in _CODES:
            return cls(k, v)
        return cls(k, v, *(torch.zeros((pages, page_size, heads), dtype=torch.float32, device=device) for _ in "kv"))

    def _code(self, dtype):
        """The library's name for the cache's type next to tensors of ``dtype``."""
        if dtype not in _HALF:
            raise RuntimeError("Only fp16 and bf16 are supported")
        if not self.quantised and dtype != self.dtype:
            raise RuntimeError(f"a cache in {self.dtype} goes with tensors of that dtype, not {dtype}")
        return _CODES[self.dtype] if self.quantised else _lib.dtype_code(dtype)

    def _pointers(self):
        return _lib.ptr(self.k), _lib.ptr(self.v), _lib.ptr(self.k_scale), _lib.ptr(self.v_scale)

    def _check_slots(self, slots):
        if slots.dim() != 1 or slots.dtype not in (torch.int32, torch.int64):
            raise RuntimeError("slots must be a 1D tensor of int32 or int64")
        _lib.require_gpu(slots)
        if slots.device != self.device:
            raise RuntimeError("all tensors must be on the same device")
        return slots.contiguous()

    def write(self, k, v, slots):
        """Quantises (or copies) ``k``, ``v`` ``[tokens, heads, dim]`` into ``slots`` ``[tokens]``.  A negative slot, or one
        behind the end, is skipped; no slot may be named twice."""
        calls = _lib.calls(k, v, slots)
        if calls is not None and calls.cache_write(self.k, self.v, self.k_scale, self.v_scale, k, v, slots):
            return
        slots = self._check_slots(slots)
        shape = (slots.shape[0], self.heads, self.dim)
        if k.shape != shape or v.shape != shape or k.dtype != v.dtype:
            raise RuntimeError(f"k and v must have the shape {list(shape)} and one dtype")
        code = self._code(k.dtype)
        _lib.require_gpu(k, v)
        if k.device != self.device or v.device != self.device:
            raise RuntimeError("all tensors must be on the same device")
        if k.numel() == 0:
            return
        k, v = _lib.in_pieces(k.detach()), _lib.in_pieces(v.detach())
        with _lib.device_guard(k):
            _lib.check(_lib.lib().neox_cache_write(
                *self._pointers(), k.data_ptr(), v.data_ptr(), slots.data_ptr(), slots.dtype == torch.int64, shape[0], self.heads,
                self.dim, self.pages, self.page_size, *self._strides, _lib.row_strides(k), _lib.row_strides(v),
                _lib.dtype_code(k.dtype), code, _lib.current_stream(k)))

    def read(self, slots, dtype=torch.bfloat16):
        """The keys and values of ``slots`` ``[tokens]``, each ``[tokens, heads, dim]`` in ``dtype`` (fp16 or bf16; of a cache
        in 16 bits: its own); zeros for a slot outside the cache."""
        calls = _lib.calls(slots)
        if calls is not None:
            out = calls.cache_read(self.k, self.v, self.k_scale, self.v_scale, slots, dtype)
            if out is not None:
                return out
        slots = self._check_slots(slots)
        code = self._code(dtype)
        k, v = (torch.empty((slots.shape[0], self.heads, self.dim), dtype=dtype, device=self.device) for _ in "kv")
        if k.numel() == 0:
            return k, v
        with _lib.device_guard(k):
            _lib.check(_lib.lib().neox_cache_read(
                k.data_ptr(), v.data_ptr(), *self._pointers(), slots.data_ptr(), slots.dtype == torch.int64, slots.shape[0],
                self.heads, self.dim, self.pages, self.page_size, _lib.row_strides(k), _lib.row_strides(v), *self._strides,
                _lib.dtype_code(dtype), code, _lib.current_stream(k)))
        return k, v


def slots_of(page_table, sample, position, page_size):
    """The slots of tokens: ``page_table`` ``[b, columns]``, ``sample`` and ``position`` ``[tokens]`` (which sequence a token
    belongs to, and where it stands there) -> int64 ``[tokens]``."""
    sample, position = sample.long(), position.long()
    return page_table[sample, position // page_size].long() * page_size + position % page_size


def paged_attention(q, cache, page_table, query_starts, context_lengths, *, max_query, max_context=None, scale=None, window=None,
                    sinks=0):
    """Causal attention of the newest tokens of ``b`` sequences over their pages -> ``[tokens, h, d]``.

    ``q`` ``[tokens, h, d]`` holds the sequences one behind the other: sequence ``s`` the rows ``query_starts[s]`` to
    ``query_starts[s + 1]`` (int32 ``[b + 1]``).  Its keys, those of its new tokens among them, are already in ``cache``:
    ``context_lengths[s]`` of them (int32 ``[b]``), key ``j`` in page ``page_table[s, j // page_size]`` (int32
    ``[b, columns]``).  The last token stands at the last key; ``window`` and ``sinks`` as in ``window_attention``.  A token that
    sees no key gets zeros; a row of ``q`` that no sequence covers is left unspecified.  There is no backward pass.

    ``max_query`` and ``max_context`` (default: what ``page_table`` has room for) are known to the host and must not be
    smaller than the longest entries of the tensors, which only the kernels look at: they choose the kernel and the number
    of parts that the keys are split into.  What a table says beyond them is not computed.
    """
    if torch.is_grad_enabled() and q.requires_grad or _lib.in_dual_level() and _lib.carries_tangent(q):
        raise RuntimeError("paged_attention computes no gradients: call it under torch.no_grad() or on q.detach()")
    window, sinks = check_window(window, sinks)
    calls = _lib.calls(q, page_table, query_starts, context_lengths)
    if calls is not None:
        out = calls.paged_attention(q, cache.k, cache.v, cache.k_scale, cache.v_scale, page_table, query_starts, context_lengths, max_query,
                                    max_context, 1.0 / math.sqrt(cache.dim) if scale is None else scale,
                                    window, sinks)
        if out is not None:
            return out
    if q.dim() != 3:
        raise RuntimeError(f"expected 3D tensor, got q with {q.dim()} dims")
    code = cache._code(q.dtype)
    (tokens, h, d), b = q.shape, context_lengths.shape[0] if context_lengths.dim() == 1 else -1
    if d != cache.dim:
        raise RuntimeError(f"q has head dim {d}, the cache {cache.dim}")
    if h == 0 or h % cache.heads:
        raise RuntimeError(f"{h} query heads must be a multiple of {cache.heads} key heads")
    if context_lengths.dtype != torch.int32 or b < 1:
        raise RuntimeError("context_lengths must be int32 [sequences]")
    if query_starts.dtype != torch.int32 or query_starts.shape != (b + 1,):
        raise RuntimeError(f"query_starts must be int32 [{b + 1}]")
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != b or page_table.shape[1] < 1:
        raise RuntimeError(f"page_table must be int32 [{b}, columns]")
    _lib.require_gpu(q, page_table, query_starts, context_lengths)
    for t in (q, page_table, query_starts, context_lengths):
        if t.device != cache.device:
            raise RuntimeError("all tensors must be on the same device")
    if max_context is None:
        max_context = page_table.shape[1] * cache.page_size
    for name, n in (("max_query", max_query), ("max_context", max_context)):
        if not 1 <= operator.index(n) < 2**30:  # (a C integer would take what is left of a larger one in 32 bits)
            raise RuntimeError(f"{name}={n} must be at least 1 and below 2^30")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    out = torch.empty((tokens, h, d), dtype=q.dtype, device=q.device)
    if tokens == 0:
        return out
    q = _lib.in_pieces(q.detach())
    if page_table.stride(1) != 1:
        page_table = page_table.contiguous()
    query_starts, context_lengths = query_starts.contiguous(), context_lengths.contiguous()
    lib = _lib.lib()
    need = ctypes.c_int64()
    _lib.check(lib.neox_paged_attention_workspace(need, b, tokens, max_query, max_context, h, cache.heads, d, window, sinks))
    workspace = torch.empty(need.value, dtype=torch.uint8, device=q.device) if need.value else None
    with _lib.device_guard(q):
        _lib.check(lib.neox_paged_attention(
            out.data_ptr(), _lib.ptr(workspace), need.value, q.data_ptr(), *cache._pointers(), page_table.data_ptr(),
            query_starts.data_ptr(), context_lengths.data_ptr(), b, tokens, max_query, max_context, h, cache.heads, d, cache.pages,
            cache.page_size, page_table.shape[1], page_table.stride(0), _lib.row_strides(out), _lib.row_strides(q), *cache._strides,
            scale, window, sinks, _lib.dtype_code(q.dtype), code, _lib.current_stream(q)))
    return out
