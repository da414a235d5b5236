"""Attention over a window of keys and a few first ones, without stored scores.

:func:`window_attention` computes what the softmax module of ``fused_softmax`` and the two products around it compute
for a causal mask with a sliding window (``sliding_window_width``), in one kernel that never writes the scores; its
backward pass recomputes them.  Two things come on top: the first ``sinks`` keys stay visible to every query, and
query heads may share key heads.  The kernels are those of ``csrc/attention_kernels.hpp``, through
``neox_window_attention_fwd`` and ``neox_window_attention_bwd``; there is no CPU fallback.
"""
import ctypes
import math

import torch

from . import _lib

_HALF = (torch.float16, torch.bfloat16)


def check_window(window, sinks):
    """``window`` as the kernels take it: -1 for none."""
    if window is None:
        window = -1
    elif isinstance(window, bool) or not isinstance(window, int) or window < 0:
        raise RuntimeError(f"window must be a non-negative integer or None, got {window!r}")
    if isinstance(sinks, bool) or not isinstance(sinks, int) or sinks < 0:
        raise RuntimeError(f"sinks must be a non-negative integer, got {sinks!r}")
    return min(window, 2**31 - 1), min(sinks, 2**31 - 1)


def _forward(q, k, v, scale, window, sinks, key_lengths, for_backward):
    (sq, b, h, d), (sk, _, h_kv, _) = q.shape, k.shape
    out = torch.empty((sq, b, h, d), dtype=q.dtype, device=q.device)
    lse = torch.empty(b * h * sq, dtype=torch.float32, device=q.device) if for_backward else None
    low = torch.empty_like(out) if for_backward else None
    if out.numel() == 0 or sk == 0:
        return out.zero_(), low, lse
    q, k, v = _lib.in_pieces(q), _lib.in_pieces(k), _lib.in_pieces(v)
    with _lib.device_guard(q):
        _lib.check(_lib.lib().neox_window_attention_fwd(
            out.data_ptr(), _lib.ptr(low), _lib.ptr(lse), q.data_ptr(), k.data_ptr(), v.data_ptr(),
            _lib.ptr(key_lengths), b, sq, sk, h, h_kv, d,
            _lib.row_strides(q), _lib.row_strides(k), _lib.row_strides(v), _lib.row_strides(out), scale, window, sinks,
            _lib.dtype_code(q.dtype), _lib.current_stream(q)))
    return out, low, lse


def _check_saved(q, k, v, out, low, lse, key_lengths):
    """A saved-tensor hook may have given back other tensors than were left with it: the kernels take for granted what was
    looked at in the forward pass."""
    _lib.require_gpu(q, k, v, out, low, lse, key_lengths)
    if any(t is not None and t.device != q.device for t in (k, v, out, low, lse, key_lengths)):
        raise RuntimeError("the saved tensors must be on one device")
    if (q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or k.shape[1] != q.shape[1] or k.shape[3] != q.shape[3]
            or any(t.shape != q.shape for t in (out, low)) or any(t.dtype != q.dtype for t in (k, v, out, low))
            or q.dtype not in _HALF or lse.dtype != torch.float32 or lse.numel() != out.numel() // max(1, q.shape[3])):
        raise RuntimeError("the saved tensors must have the shapes and dtypes of the forward pass")
    if key_lengths is not None and (key_lengths.dtype != torch.int32 or key_lengths.shape != q.shape[1:2] or not key_lengths.is_contiguous()):
        raise RuntimeError("the saved key lengths have changed")


class _OnlyOnce(torch.autograd.Function):
    """Hands on the gradients ``dq, dk, dv`` of a backward pass that is itself recorded (``create_graph=True``), as
    results of the tensors they were computed from: the kernels have no second derivative, and asking for one has to fail
    and not to leave a term out."""

    @staticmethod
    def forward(ctx, dq, dk, dv, *sources):
        return dq, dk, dv

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("window_attention has no second derivative")


class WindowAttention(torch.autograd.Function):
    """``apply(q, k, v, scale, window, sinks, key_lengths)``; see :func:`window_attention`, which checks the arguments."""

    @staticmethod
    def forward(ctx, q, k, v, scale, window, sinks, key_lengths):
        out, low, lse = _forward(q, k, v, scale, window, sinks, key_lengths, True)
        ctx.save_for_backward(q, k, v, out, low, lse, key_lengths)
        ctx.call = (scale, window, sinks)
        return out

    @staticmethod
    def backward(ctx, grad):
        sources = (*ctx.saved_tensors[:3], grad)
        with torch.no_grad():
            grads = WindowAttention._gradients(ctx, grad)
        if torch.is_grad_enabled() and any(t.requires_grad for t in sources):
            grads = _OnlyOnce.apply(*grads, *sources)
        return (*grads, None, None, None, None)

    @staticmethod
    def _gradients(ctx, grad):
        q, k, v, out, low, lse, key_lengths = ctx.saved_tensors
        _check_saved(q, k, v, out, low, lse, key_lengths)
        (sq, b, h, d), (sk, _, h_kv, _) = q.shape, k.shape
        dq = torch.empty((sq, b, h, d), dtype=q.dtype, device=q.device)
        dk, dv = (torch.empty((sk, b, h_kv, d), dtype=q.dtype, device=q.device) for _ in "kv")
        if out.numel() == 0 or sk == 0:
            return dq.zero_(), dk.zero_(), dv.zero_()
        if grad.shape != out.shape or grad.dtype != out.dtype or grad.device != out.device:
            raise RuntimeError("the gradient must have the shape, dtype and device of the attention's output")
        q, k, v, grad = (_lib.in_pieces(t) for t in (q, k, v, grad))
        out, low, lse = out.contiguous(), low.contiguous(), lse.contiguous()  # (a saved-tensor hook may have changed their layout)
        need = ctypes.c_int64()
        _lib.check(_lib.lib().neox_window_attention_bwd_workspace(need, b, sq, sk, h, h_kv, d, *ctx.call[1:]))
        workspace = torch.empty(need.value, dtype=torch.uint8, device=q.device)
        strides = [_lib.row_strides(t) for t in (dq, dk, dv, grad, out, q, k, v)]
        with _lib.device_guard(q):
            _lib.check(_lib.lib().neox_window_attention_bwd(
                dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), workspace.data_ptr(), need.value, grad.data_ptr(), out.data_ptr(),
                low.data_ptr(), lse.data_ptr(),
                q.data_ptr(), k.data_ptr(), v.data_ptr(), _lib.ptr(key_lengths),
                b, sq, sk, h, h_kv, d, *strides, *ctx.call, _lib.dtype_code(q.dtype), _lib.current_stream(q)))
        return dq, dk, dv


def window_attention(q, k, v, *, window=None, sinks=0, scale=None, key_lengths=None):
    """Causal attention of ``q`` ``[sq, b, h, d]`` over ``k``, ``v`` ``[sk, b, h_kv, d]`` -> ``[sq, b, h, d]``.

    Query ``i`` stands at position ``p = i + sk - sq`` and sees key ``j`` if ``j <= p`` and ``j >= p - window`` (the rule
    of GPT-NeoX's ``sliding_window_width``; ``window=None``: all of them) or ``j < sinks``.  ``key_lengths`` (int32
    ``[b]`` on the GPU) hides the keys from a sample's length on.  A query that sees no key gets zeros, and no gradient
    flows from it.  ``scale`` defaults to ``1 / sqrt(d)``.

    fp16 or bf16; ``h`` a multiple of ``h_kv``; ``d`` a multiple of 8, at most 256.  Any strides: tensors whose rows
    are dense and start on 16-byte boundaries (views into a fused QKV projection among them) are read as they lie,
    others are copied first.  Sums and the softmax are in fp32.  Gradients flow to ``q``, ``k`` and ``v``; those of shared
    key heads are summed in a fixed order, so the same inputs give the same bits.  There is no second derivative: going
    back through gradients taken with ``create_graph=True`` raises.
    """
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 4:
            raise RuntimeError(f"expected 4D tensor, got {name} with {t.dim()} dims")
    w, n = check_window(window, sinks)
    calls = _lib.calls(q, k, v) if key_lengths is None or type(key_lengths) is torch.Tensor else None
    if calls is not None:
        out = calls.window_attention(q, k, v, (1.0 / math.sqrt(max(1, q.shape[3]))) if scale is None else scale, w, n, key_lengths)
        if out is not None:
            return out
    if q.dtype not in _HALF:
        raise RuntimeError("Only fp16 and bf16 are supported")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise RuntimeError("q, k and v must have the same dtype")
    if k.shape != v.shape:
        raise RuntimeError(f"k and v must have the same shape, got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.shape[1] != q.shape[1] or k.shape[3] != q.shape[3]:
        raise RuntimeError(f"q {tuple(q.shape)} and k {tuple(k.shape)} must agree in samples and head dim")
    d = q.shape[3]
    if d % 8 or not 8 <= d <= 256:
        raise RuntimeError(f"head dim {d} must be a multiple of 8 from 8 to 256")
    if k.shape[2] == 0 or q.shape[2] % k.shape[2]:
        raise RuntimeError(f"{q.shape[2]} query heads must be a multiple of {k.shape[2]} key heads")
    _lib.require_gpu(q, k, v, key_lengths)
    if key_lengths is not None:
        if key_lengths.dtype != torch.int32 or key_lengths.shape != (q.shape[1],):
            raise RuntimeError(f"key_lengths must be int32 [{q.shape[1]}]")
        key_lengths = key_lengths.contiguous()
    for t in (k, v, key_lengths):
        if t is not None and t.device != q.device:
            raise RuntimeError("all tensors must be on the same device")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad) or (
            _lib.in_dual_level() and _lib.carries_tangent(q, k, v)):
        return WindowAttention.apply(q, k, v, scale, w, n, key_lengths)
    return _forward(q, k, v, scale, w, n, key_lengths, False)[0]
