"""Window attention, the paged cache and its codes in 64 bits, with error bounds (runs on any device).

Plain restatements of the definitions in ``include/neox_fused.h``, written without the product's code, and what a
kernel may differ from them by.  Test infrastructure: never imported by the product.
"""
import math

import torch

# half a unit in the last place, relative: what one rounding to the type costs (8 and 11 bits of significand)
ROUND = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16)}
# the smallest step of the type near zero, halved
TINY = {torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25}


def visible(sq, sk, window=None, sinks=0, length=None, device="cpu"):
    """``[sq, sk]``: which keys a query sees; the last query stands at the last key."""
    p = torch.arange(sq, device=device)[:, None] + (sk - sq)
    j = torch.arange(sk, device=device)[None, :]
    sees = j <= p
    if window is not None:
        sees = sees & ((j >= p - window) | (j < sinks))
    if length is not None:
        sees = sees & (j < length)
    return sees


def one_head(q, k, v, sees, scale):
    """``q [m, d]``, ``k``, ``v`` ``[n, d]``, ``sees [m, n]`` in float64 -> output, probabilities."""
    s = (q @ k.T) * scale
    s = torch.where(sees, s, -math.inf)
    top = s.amax(1, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    # (a hidden key has no part in the sum, whatever its value is)
    return p @ torch.where(sees.any(0)[:, None], v, 0.0), p


def one_head_bound(q, k, v, sees, scale, p, out, dtype, value_size=None):
    """What a 16-bit output may be off by: the probabilities are rounded to the type before they meet the values,
    the output after; scores, exponentials and sums are in 32 bits, whose part grows with the size of the scores."""
    u = ROUND[dtype]
    size = p @ (v.abs() if value_size is None else value_size)
    scores = abs(scale) * (q.abs() @ k.abs().T)
    scores = torch.where(sees, scores, 0.0).amax(1, keepdim=True)
    small = 2.0**-20 * (4 + scores)
    seen = sees.sum(1, keepdim=True).double()
    return (1.05 * u + small) * size + 1.05 * u * out.abs() + 2 * TINY[dtype] * (seen * v.abs().amax().clamp(min=1) + 1)


def window_attention(q, k, v, *, window=None, sinks=0, scale=None, key_lengths=None, grad=None, dtype=None):
    """``q [sq, b, h, d]``, ``k``, ``v`` ``[sk, b, h_kv, d]`` (any dtype) -> dict of float64 results: ``out``, and with ``grad``
    ``dq``, ``dk``, ``dv``; with ``dtype`` also ``<name>_bound``, the most a kernel in that type may differ by."""
    (sq, b, h, d), (sk, _, h_kv, _) = q.shape, k.shape
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    q, k, v = q.double(), k.double(), v.double()
    res = {"out": torch.zeros_like(q, memory_format=torch.contiguous_format)}
    names = ["out"]
    if grad is not None:
        grad = grad.double()
        res.update(dq=torch.zeros_like(res["out"]), dk=torch.zeros((sk, b, h_kv, d), dtype=torch.float64, device=q.device))
        res["dv"] = torch.zeros_like(res["dk"])
        names += ["dq", "dk", "dv"]
    if dtype is not None:
        for n in names:
            res[n + "_bound"] = torch.zeros_like(res[n])
        u = ROUND[dtype]
    for i in range(b):
        sees = visible(sq, sk, window, sinks, None if key_lengths is None else int(key_lengths[i]), q.device)
        used = sees.any(0)[:, None]
        for x in range(h):
            y = x // (h // h_kv)
            qh, kh, vh = q[:, i, x], torch.where(used, k[:, i, y], 0.0), torch.where(used, v[:, i, y], 0.0)
            out, p = one_head(qh, kh, vh, sees, scale)
            res["out"][:, i, x] = out
            if dtype is not None:
                bound = one_head_bound(qh, kh, vh, sees, scale, p, out, dtype)
                res["out_bound"][:, i, x] = bound
            if grad is None:
                continue
            g = grad[:, i, x]
            dp = g @ vh.T
            delta = (g * out).sum(1, keepdim=True)
            ds = p * (dp - delta)
            res["dq"][:, i, x] = scale * (ds @ kh)
            res["dk"][:, i, y] += scale * (ds.T @ qh)
            res["dv"][:, i, y] += p.T @ g
            if dtype is not None:
                # p comes again from the scores and the row's 32-bit sum; delta from the output as it was stored
                scores = torch.where(sees, abs(scale) * (qh.abs() @ kh.abs().T), 0.0).amax(1, keepdim=True)
                small = 2.0**-19 * (4 + scores)
                off_delta = (g.abs() * bound).sum(1, keepdim=True) + 2.0**-18 * (g.abs() @ vh.abs().T)
                off = p * (off_delta + small * (dp.abs() + delta.abs())) + 1.05 * u * ds.abs() + TINY[dtype]
                off = torch.where(sees, off, 0.0)
                res["dq_bound"][:, i, x] = abs(scale) * (off @ kh.abs())
                res["dk_bound"][:, i, y] += abs(scale) * (off.T @ qh.abs())
                res["dv_bound"][:, i, y] += ((1.05 * u + small) * p + torch.where(sees, TINY[dtype], 0.0)).T @ g.abs()
    if dtype is not None:
        for n in names[1:]:
            res[n + "_bound"] += 1.05 * u * res[n].abs() + 4 * TINY[dtype]
    return res


# ---- the cache -----------------------------------------------------------------------------------------------
LARGEST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def round_e4m3(y):
    """float64 values of magnitude <= 448 to the nearest value of the 8-bit float, ties to even: 4 bits of significand,
    exponents from -6, below that steps of 2^-9."""
    exponent = torch.floor(torch.log2(y.abs().clamp(min=2.0**-6)))
    # (log2 of a number just below a power of two may round up to it)
    exponent = torch.where(torch.exp2(exponent) > y.abs().clamp(min=2.0**-6), exponent - 1, exponent)
    step = torch.exp2(exponent - 3)
    return torch.round(y / step) * step


def encode(x, codes):
    """Rows ``[..., d]`` -> the codes' values (float64) and the scales (float32), as the cache holds them."""
    x = x.double()
    largest = x.abs().amax(-1, keepdim=True)
    y = x * LARGEST[codes] / torch.where(largest == 0, 1.0, largest)
    y = torch.round(y) if codes == torch.int8 else round_e4m3(y)
    return y, (largest.squeeze(-1) / LARGEST[codes]).float()


def gather(table_row, page_size, count, tensor):
    """Tokens 0 .. count of a sequence from ``tensor [pages, page_size, ...]``."""
    j = torch.arange(count, device=tensor.device)
    return tensor[table_row.long()[j // page_size], j % page_size]


def paged_attention(q, k, v, k_scale, v_scale, table, starts, lengths, *, window=None, sinks=0, scale=None, dtype=None):
    """``k``, ``v`` ``[pages, page_size, h_kv, d]`` as numbers (codes or values); scales ``[pages, page_size, h_kv]`` or None.
    Returns the output in float64 and its bound."""
    tokens, h, d = q.shape
    h_kv, page = k.shape[2], k.shape[1]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    out = torch.zeros((tokens, h, d), dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for s in range(len(lengths)):
        a, z, n = int(starts[s]), int(starts[s + 1]), int(lengths[s])
        if a == z or n == 0:
            continue
        sees = visible(z - a, n, window, sinks, None, q.device)
        for y in range(h_kv):
            kh, vh = (gather(table[s], page, n, t[:, :, y]).double() for t in (k, v))
            if k_scale is not None:
                kh = kh * gather(table[s], page, n, k_scale[:, :, y]).double()[:, None]
                vh = vh * gather(table[s], page, n, v_scale[:, :, y]).double()[:, None]
            for x in range(y * (h // h_kv), (y + 1) * (h // h_kv)):
                qh = q[a:z, x].double()
                o, p = one_head(qh, kh, vh, sees, scale)
                out[a:z, x] = o
                if dtype is not None:
                    bound[a:z, x] = one_head_bound(qh, kh, vh, sees, scale, p, o, dtype)
    return out, bound
