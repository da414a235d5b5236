"""Which pages of a :class:`~gpt_neox_amd.paged_cache.PagedKVCache` belong to which sequence, kept on the GPU.

:class:`PagePool` holds the page tables and lengths of many sequences and the list of pages that nobody has.
:meth:`PagePool.extend` gives the new tokens of every sequence their places, and new pages where they begin one, from
their numbers alone; :meth:`PagePool.truncate` takes pages back from sequences that end or drop tokens.  What they
return goes into ``cache.write`` and ``paged_attention`` as it is, and nothing looks at it on the host, so that a step
can be recorded into a HIP graph.  One pool serves the caches of all layers.
"""
from typing import NamedTuple

import torch

from . import _lib


class PoolStep(NamedTuple):
    """Where the new tokens of a step stand, the sequences one behind the other.

    ``query_starts`` int32 ``[sequences + 1]``: the first token of every sequence, and the end; ``positions`` int32
    ``[max_tokens]``: where a token stands in its sequence (0 behind the last one); ``slots`` int64 ``[max_tokens]``: its slot
    of the cache (-1 behind the last one, and for a sequence that was not granted); ``granted`` bool ``[sequences]``.
    """

    query_starts: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor
    granted: torch.Tensor


class PagePool:
    """``page_table`` ``[sequences, columns]`` (the pages of every sequence in order, -1 behind them), ``lengths``
    ``[sequences]`` (the tokens each has), ``free`` ``[pages]`` and ``left`` ``[1]``: the pages ``free[:left]`` belong to nobody, and
    the last of them is the next to be given.  All int32 on one GPU; the calls change them in place, on the current
    stream.  They are looked at once, here, and stay.
    """

    _FIXED = frozenset(("page_table", "lengths", "free", "left", "page_size", "sequences", "columns", "pages", "device"))

    def __setattr__(self, name, value):
        if name in self._FIXED and name in self.__dict__:
            raise AttributeError(f"{name} of a pool cannot be replaced: make a PagePool of the new tensors")
        super().__setattr__(name, value)

    def __init__(self, page_table, lengths, free, left, *, page_size):
        for name, t, dims in (("page_table", page_table, 2), ("lengths", lengths, 1), ("free", free, 1), ("left", left, 1)):
            if t.dim() != dims or t.dtype != torch.int32:
                raise RuntimeError(f"{name} must be a {dims}D tensor of int32")
            if t.numel() == 0 or t.stride(-1) != 1 and t.shape[-1] > 1:
                raise RuntimeError(f"{name} must not be empty, and its last axis dense")
        if lengths.shape[0] != page_table.shape[0] or left.shape[0] != 1:
            raise RuntimeError(f"lengths must be int32 [{page_table.shape[0]}], left int32 [1]")
        if page_table.shape[0] > 1 and page_table.stride(0) < page_table.shape[1]:
            raise RuntimeError("the rows of page_table must not overlap")
        if isinstance(page_size, bool) or not isinstance(page_size, int) or not 1 <= page_size < 2**30:
            raise RuntimeError(f"page_size must be a positive integer below 2^30, got {page_size!r}")
        _lib.require_gpu(page_table, lengths, free, left)
        if any(t.device != page_table.device for t in (lengths, free, left)):
            raise RuntimeError("all tensors must be on the same device")
        self.page_table, self.lengths, self.free, self.left, self.page_size = page_table, lengths, free, left, page_size
        (self.sequences, self.columns), self.pages, self.device = page_table.shape, free.shape[0], page_table.device

    @classmethod
    def allocate(cls, pages, page_size, sequences, columns, device="cuda"):
        """A pool of ``pages`` free pages, page 0 the first to be given, and ``sequences`` empty sequences."""
        table = torch.full((sequences, columns), -1, dtype=torch.int32, device=device)
        free = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=device)
        return cls(table, torch.zeros(sequences, dtype=torch.int32, device=device), free,
                   torch.full((1,), pages, dtype=torch.int32, device=device), page_size=page_size)

    def _stride(self):
        return self.page_table.stride(0) if self.sequences > 1 else 0

    def _state(self):
        return tuple(t.data_ptr() for t in (self.page_table, self.lengths, self.free, self.left))

    def _check(self, name, t):
        if t.dtype != torch.int32 or t.shape != (self.sequences,):
            raise RuntimeError(f"{name} must be int32 [{self.sequences}]")
        _lib.require_gpu(t)
        if t.device != self.device:
            raise RuntimeError("all tensors must be on the same device")
        return t.contiguous()

    def extend(self, new_tokens, *, max_tokens):
        """Places for ``new_tokens`` ``[sequences]`` (int32; below zero counts as none) more tokens of every sequence -> a
        :class:`PoolStep`, with ``lengths`` and ``page_table`` grown by them.

        Sequences are served in order, each wholly or not at all: one whose table row would be too short, whose
        tokens go beyond ``max_tokens``, or that needs pages when it and those before it need more than are left keeps what it has,
        and ``granted`` says so; its tokens have no slots (and attention over them means nothing).  ``max_tokens``
        is the host's number of rows: at least the sum of ``new_tokens``.
        """
        if type(max_tokens) is not int or not 0 <= max_tokens < 2**30:
            raise RuntimeError(f"max_tokens must be an integer from 0 to below 2^30, got {max_tokens!r}")
        calls = _lib.calls(new_tokens)
        if calls is not None:
            step = calls.pages_extend(self.page_table, self.lengths, self.free, self.left, new_tokens, self.page_size, max_tokens)
            if step is not None:
                return PoolStep(*step)
        new_tokens = self._check("new_tokens", new_tokens)
        starts, workspace = (torch.empty(self.sequences + 1, dtype=torch.int32, device=self.device) for _ in range(2))
        positions = torch.empty(max_tokens, dtype=torch.int32, device=self.device)
        slots = torch.empty(max_tokens, dtype=torch.int64, device=self.device)
        granted = torch.empty(self.sequences, dtype=torch.bool, device=self.device)
        with _lib.device_guard(new_tokens):
            _lib.check(_lib.lib().neox_pages_extend(
                starts.data_ptr(), positions.data_ptr(), slots.data_ptr(), granted.data_ptr(), workspace.data_ptr(), *self._state(),
                new_tokens.data_ptr(), self.sequences, self.columns, self._stride(), self.pages, self.page_size, max_tokens,
                _lib.current_stream(new_tokens)))
        return PoolStep(starts, positions, slots, granted)

    def truncate(self, lengths):
        """Cuts every sequence to ``lengths`` ``[sequences]`` (int32; 0 ends it, its own length or more leaves it).  The pages behind go
        back onto the list, the last one first: dropping what the last ``extend`` brought makes the pool what it was."""
        calls = _lib.calls(lengths)
        if calls is not None and calls.pages_truncate(self.page_table, self.lengths, self.free, self.left, lengths, self.page_size):
            return
        lengths = self._check("lengths", lengths)
        with _lib.device_guard(lengths):
            _lib.check(_lib.lib().neox_pages_truncate(*self._state(), lengths.data_ptr(), self.sequences, self.columns, self._stride(), self.pages,
                                                      self.page_size, _lib.current_stream(lengths)))
