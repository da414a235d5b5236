"""Attention over windows and over a paged cache, as cases that a timing program can run.

A case is a dict of plain values; ``listed()`` names twelve of them, ``draw(rng)`` makes more of the same
ranges.  Three operators:

* ``window`` -- attention of queries ``[s, b, heads, d]`` over keys and values with fewer or as many heads, where a
  query sees the ``w`` keys before it, itself and the first few keys (sinks), and no key behind its sample's length;
  forward only, or forward and backward;
* ``cache`` -- new keys and values written into a paged cache of 8-bit codes with a scale for each token and head,
  and read back from there;
* ``paged`` -- attention of the newest tokens of each sequence over its pages of such a cache, or of one in 16 bits:
  single tokens (generation) or chunks of a prompt, with or without a window and sinks.

``run`` computes them in plain torch where ``own`` is false, and through the package's entry points where it is true.
"""
import math

import torch

own = False

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "int8": torch.int8, "fp8": torch.float8_e4m3fn}
_TOP = {"int8": 127.0, "fp8": 448.0}  # the largest magnitude a code of the cache holds


def _window(name, b, s, heads, kv, d, dtype, w, sinks, train=True, padded=False, fused=False):
    return {"name": name, "kind": "window", "b": b, "s": s, "heads": heads, "kv": kv, "d": d, "dtype": dtype, "w": w,
            "sinks": sinks, "train": train, "padded": padded, "fused": fused}


def _cache(name, tokens, kv, d, dtype, codes, page, pages):
    return {"name": name, "kind": "cache", "tokens": tokens, "kv": kv, "d": d, "dtype": dtype, "codes": codes,
            "page": page, "pages": pages}


def _paged(name, b, new, context, heads, kv, d, dtype, codes, page, w=-1, sinks=0, ragged=True):
    return {"name": name, "kind": "paged", "b": b, "new": new, "context": context, "heads": heads, "kv": kv, "d": d,
            "dtype": dtype, "codes": codes, "page": page, "w": w, "sinks": sinks, "ragged": ragged}


def listed():
    return [
        # a training step of a small model on short sequences: the host's own time counts
        _window("window_train_small", 2, 256, 8, 8, 64, "bf16", 100, 4),
        # a padded batch at an odd length: keys behind a sample's end are hidden, and rows far behind it see nothing
        _window("window_train_padded", 8, 1001, 16, 16, 64, "fp16", 256, 0, padded=True),
        # one layer at the 7B shape with grouped heads, a quarter of the context visible, on the fused QKV projection
        _window("window_train_grouped", 1, 4096, 32, 8, 128, "bf16", 1024, 4, fused=True),
        # long context, half of it visible: the largest
        _window("window_train_long", 1, 8192, 32, 32, 128, "bf16", 4096, 4),
        # evaluation of two documents at the 20B shape, no gradient
        _window("window_eval_20b", 2, 2048, 64, 64, 96, "fp16", 512, 4, train=False),
        # one generated token of each of 16 sequences into the cache of one layer, and back
        _cache("cache_tokens", 16, 8, 128, "bf16", "int8", 16, 512),
        # a prompt at the 20B shape, of an odd length, into pages that hold other sequences too
        _cache("cache_prompt", 2047, 64, 96, "fp16", "fp8", 64, 64),
        # the prompts of a large batch
        _cache("cache_prompts", 65536, 32, 128, "bf16", "int8", 64, 1536),
        # generation, the smallest: one token of four sequences of a 125M model, a cache in 16 bits
        _paged("paged_token_small", 4, 1, 517, 12, 12, 64, "fp16", "fp16", 16),
        # generation for many users: sequences of 2k to 8k tokens, codes in 8 bits, grouped heads
        _paged("paged_token_batch", 64, 1, 8192, 32, 8, 128, "bf16", "int8", 64),
        # one very long sequence, whose work has to be split over its keys
        _paged("paged_token_long", 1, 1, 131001, 32, 8, 128, "bf16", "bf16", 128),
        # chunks of four prompts, each over what its sequence has in the cache already
        _paged("paged_chunk", 4, 512, 16384, 32, 8, 128, "bf16", "fp8", 64, w=4096, sinks=4),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: any kind, its sizes spread over the logarithm of their range, odd ones among them."""
    kind = rng.choice(["window", "window", "window", "cache", "cache", "paged", "paged", "paged"])
    dtype = rng.choice(["fp16", "bf16"])
    d = rng.choice([64, 80, 96, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8, 12, 16])
    heads = kv * rng.choice([1, 1, 2, 4, 8])
    sinks = rng.choice([0, 1, 4, 16])
    if kind == "window":
        s = _log_int(rng, 48, 8192)
        if rng.random() < 0.5:  # training lengths are mostly multiples of 64, evaluation is any length
            s = max(64, s // 64 * 64)
        c = _window("", rng.choice([1, 2, 4, 8]), s, heads, kv, d, dtype, _log_int(rng, 16, 4096), sinks,
                    train=rng.random() < 0.7, padded=rng.random() < 0.3, fused=rng.random() < 0.5)
        # (the plain form holds the scores of every pair)
        while c["b"] * c["heads"] * c["s"] ** 2 * max(c["d"], 128) > 32 * 8192**2 * 128:
            c["s"] = c["s"] // 2 + 1
        return c
    codes = rng.choice(["int8", "fp8"])
    page = rng.choice([16, 32, 48, 64, 128, 256])
    if kind == "cache":
        tokens = _log_int(rng, 1, 65536)
        while tokens * kv * d > 65536 * 32 * 128:
            tokens = tokens // 2 + 1
        return _cache("", tokens, kv, d, dtype, codes, page, tokens // page * 3 // 2 + 4)
    if rng.random() < 0.4:
        codes = dtype
    if rng.random() < 0.6:  # generation: one token, or a few that are checked together
        b, new, context = rng.choice([1, 2, 4, 16, 64]), rng.choice([1, 1, 1, 2, 5]), _log_int(rng, 32, 131072)
    else:
        b, new, context = rng.choice([1, 2, 4]), _log_int(rng, 16, 1024), _log_int(rng, 1024, 32768)
    w = rng.choice([-1, -1, 128, 1024, 4096])
    c = _paged("", b, new, context, heads, kv, d, dtype, codes, page, w, sinks if w >= 0 else 0, rng.random() < 0.7)
    while c["b"] * c["context"] * c["kv"] * c["d"] > 64 * 8192 * 8 * 128 or \
            c["b"] * c["new"] * c["context"] * c["heads"] * c["d"] > 4 * 512 * 16384 * 32 * 128:
        c["context"] = c["context"] // 2 + 1
        c["new"] = min(c["new"], c["context"])
    return c


# ---- what a case's lengths are: part of the case, not of the seed -------------------------------------
def _key_lengths(c):
    """The samples' lengths of a padded batch: from all of s down to a quarter of it."""
    return [c["s"] - i * (c["s"] * 3 // 4) // max(1, c["b"] - 1) for i in range(c["b"])]


def _paged_lengths(c):
    """New tokens and tokens in the cache (the new ones among them) of every sequence."""
    new, context = [], []
    for i in range(c["b"]):
        part = i / max(1, c["b"] - 1) if c["ragged"] else 0.0
        n = max(1, c["new"] - int(part * c["new"] / 2))
        new.append(n)
        context.append(max(n, c["context"] - int(part * 0.75 * c["context"])))
    return new, context


def _visible(first, count, w, sinks, length):
    """Pairs that the queries at the positions first .. first + count - 1 see."""
    total = 0
    for p in range(first, first + count):
        end = min(p + 1, length)
        start = 0 if w < 0 else max(0, p - w)
        total += max(0, end - start) + (max(0, min(sinks, start, end)))
    return total


def work(case):
    """What a pass cannot do without: every input read once, every output written once, and the products over the
    visible pairs -- two forward, five backward (the scores again, and the gradients of the probabilities, the
    queries, the keys and the values)."""
    c = case
    if c["kind"] == "window":
        lengths = _key_lengths(c) if c["padded"] else [c["s"]] * c["b"]
        pairs = sum(_visible(0, c["s"], c["w"], c["sinks"], n) for n in lengths) * c["heads"]
        q, kv = c["b"] * c["s"] * c["heads"] * c["d"] * 2, c["b"] * c["s"] * c["kv"] * c["d"] * 2
        if c["train"]:  # q, k, v, the output's gradient; the output and the three gradients
            return {"bytes": 4 * q + 4 * kv, "flops": 14 * pairs * c["d"]}
        return {"bytes": 2 * q + 2 * kv, "flops": 4 * pairs * c["d"]}
    if c["kind"] == "cache":
        n = c["tokens"] * c["kv"]
        # k and v in, codes and scales out and in again, k and v out; a quotient and a product for each value
        return {"bytes": 2 * n * (4 * c["d"] + 2 * (c["d"] + 4)) + 8 * c["tokens"], "flops": 4 * n * c["d"]}
    new, context = _paged_lengths(c)
    pairs = touched = 0
    for n, t in zip(new, context):
        pairs += _visible(t - n, n, c["w"], c["sinks"], t) * c["heads"]
        start = 0 if c["w"] < 0 else max(0, t - n - c["w"])
        touched += t - start + min(c["sinks"], start)
    row = 2 * c["d"] if c["codes"] in ("fp16", "bf16") else c["d"] + 4
    return {"bytes": 2 * touched * c["kv"] * row + 4 * sum(new) * c["heads"] * c["d"], "flops": 4 * pairs * c["d"]}


# ---- inputs ---------------------------------------------------------------------------------------------
def _normal(shape, dtype, gen, times=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * times).to(dtype)


def _encode(x, codes):
    """Rows of the last dim as 8-bit codes with a scale each: largest magnitude / largest code."""
    top = _TOP[codes]
    x = x.float()
    largest = x.abs().amax(-1, keepdim=True)
    scaled = torch.where(largest > 0, x * top / largest, 0.0)
    values = torch.round(scaled) if codes == "int8" else scaled
    return values.to(_TYPES[codes]), (largest / top).squeeze(-1)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[c["dtype"]]
    state = {"case": c, "scale": 1.0 / math.sqrt(c["d"])}
    if c["kind"] == "window":
        b, s, heads, kv, d = c["b"], c["s"], c["heads"], c["kv"], c["d"]
        if c["fused"]:  # q, k and v as views into one projection
            mixed = _normal((s, b, heads + 2 * kv, d), dtype, gen)
            q, k, v = mixed[:, :, :heads], mixed[:, :, heads : heads + kv], mixed[:, :, heads + kv :]
        else:
            q, k, v = (_normal((s, b, n, d), dtype, gen) for n in (heads, kv, kv))
        state.update(q=q, k=k, v=v, lengths=None)
        if c["padded"]:
            state["lengths"] = torch.tensor(_key_lengths(c), dtype=torch.int32, device="cuda")
        if c["train"]:
            state["grad"] = _normal((s, b, heads, d), dtype, gen)
            for name in ("q", "k", "v"):
                state[name] = state[name].detach().requires_grad_()
        return state
    kv, d, page = c["kv"], c["d"], c["page"]
    if c["kind"] == "cache":
        pages = c["pages"]
        # keys have a few large channels, as they do behind a projection with outliers
        loud = torch.where(torch.rand(d, generator=gen, device="cuda") < 0.05, 8.0, 1.0)
        state["k"] = (_normal((c["tokens"], kv, d), torch.float32, gen) * loud).to(dtype)
        state["v"] = _normal((c["tokens"], kv, d), dtype, gen)
        state["slots"] = torch.randperm(pages * page, generator=gen, device="cuda")[: c["tokens"]]
        codes = [torch.zeros((pages, page, kv, d), dtype=torch.int8, device="cuda").view(_TYPES[c["codes"]]) for _ in "kv"]
        scales = [torch.zeros((pages, page, kv), dtype=torch.float32, device="cuda") for _ in "kv"]
    else:
        new, context = _paged_lengths(c)
        width = -(-max(context) // page)
        pages = c["b"] * width + 3
        table = torch.randperm(pages, generator=gen, device="cuda")[: c["b"] * width].view(c["b"], width).int()
        codes, scales = [], []
        for _ in "kv":
            x = _normal((pages, page, kv, d), dtype, gen)
            if c["codes"] in _TOP:
                x, scale = _encode(x, c["codes"])
                scales.append(scale)
            codes.append(x)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        state.update(q=_normal((starts[-1], c["heads"], d), dtype, gen, 1.5), table=table, max_new=max(new), longest=max(context),
                     starts=torch.tensor(starts, dtype=torch.int32, device="cuda"),
                     lengths=torch.tensor(context, dtype=torch.int32, device="cuda"))
        scales = scales or [None, None]
    state["codes"], state["scales"] = codes, scales
    if own:
        from gpt_neox_amd.paged_cache import PagedKVCache

        state["cache"] = PagedKVCache(codes[0], codes[1], scales[0], scales[1])
    return state


# ---- one pass ---------------------------------------------------------------------------------------------
def run(state):
    c = state["case"]
    return (_run_own if own else _run_plain)[c["kind"]](state, c)


def _own_window(state, c):
    from gpt_neox_amd.fused_attention import window_attention

    q, k, v = state["q"], state["k"], state["v"]
    out = window_attention(q, k, v, window=c["w"], sinks=c["sinks"], scale=state["scale"], key_lengths=state["lengths"])
    if not c["train"]:
        return out
    return (out.detach(), *torch.autograd.grad(out, (q, k, v), state["grad"]))


def _own_cache(state, c):
    cache = state["cache"]
    cache.write(state["k"], state["v"], state["slots"])
    return cache.read(state["slots"], dtype=state["k"].dtype)


def _own_paged(state, c):
    from gpt_neox_amd.paged_cache import paged_attention

    return paged_attention(state["q"], state["cache"], state["table"], state["starts"], state["lengths"],
                           max_query=state["max_new"], max_context=state["longest"], scale=state["scale"],
                           window=c["w"] if c["w"] >= 0 else None, sinks=c["sinks"])


_run_own = {"window": _own_window, "cache": _own_cache, "paged": _own_paged}


def _softmax(scores, hidden):
    """Probabilities over the last dim; a row without a visible key is zero everywhere."""
    scores = scores.masked_fill(hidden, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, 1.0, total)


def _plain_window(state, c):
    b, s, kv, d, group = c["b"], c["s"], c["kv"], c["d"], c["heads"] // c["kv"]
    dtype, scale = state["q"].dtype, state["scale"]

    def rows(x):  # [s, b, heads, d] -> [b, kv, heads / kv * s, d]
        return x.detach().float().permute(1, 2, 0, 3).reshape(b, kv, -1, d).contiguous()

    def back(x):
        return x.reshape(b, -1, s, d).permute(2, 0, 1, 3).to(dtype).contiguous()

    q, k, v = rows(state["q"]), rows(state["k"]), rows(state["v"])
    i = torch.arange(s, device="cuda")[:, None]
    j = torch.arange(s, device="cuda")[None, :]
    hidden = ((j > i) | ((j < i - c["w"]) & (j >= c["sinks"]))).expand(b, 1, 1, s, s)
    if state["lengths"] is not None:
        hidden = hidden | (j >= state["lengths"].view(b, 1, 1, 1, 1))
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(scale)
    p = _softmax(scores.view(b, kv, group, s, s), hidden).view(b, kv, group * s, s)
    out = torch.matmul(p, v)
    if not c["train"]:
        return back(out)
    g = rows(state["grad"])
    dv = torch.matmul(p.transpose(2, 3).contiguous(), g)
    dp = torch.matmul(g, v.transpose(2, 3).contiguous())
    ds = p * (dp - (g * out).sum(-1, keepdim=True)) * scale
    return back(out), back(torch.matmul(ds, k)), back(_keys_gradient(ds, q)), back(dv)


def _keys_gradient(ds, q):
    """The keys' gradient: the scores' gradients, transposed, times the queries."""
    return torch.matmul(ds.transpose(2, 3).contiguous(), q)


def _plain_cache(state, c):
    slots, dtype = state["slots"], state["k"].dtype

    def one(x, codes, scales):
        values, scale = _encode(x, c["codes"])
        codes.view(torch.int8).view(-1, c["kv"], c["d"])[slots] = values.view(torch.int8)
        scales.view(-1, c["kv"])[slots] = scale
        held = codes.view(torch.int8).view(-1, c["kv"], c["d"])[slots].view(codes.dtype)
        return (held.float() * scales.view(-1, c["kv"])[slots][..., None]).to(dtype)

    return (one(state["k"], state["codes"][0], state["scales"][0]), one(state["v"], state["codes"][1], state["scales"][1]))


def _plain_paged(state, c):
    b, kv, d, page, group = c["b"], c["kv"], c["d"], c["page"], c["heads"] // c["kv"]
    q, starts, lengths, new, longest = state["q"], state["starts"].long(), state["lengths"].long(), state["max_new"], state["longest"]
    j = torch.arange(longest, device="cuda")
    at = state["table"].long()[:, j // page] * page + j % page  # [b, longest]

    def held(codes, scales):
        x = codes.view(-1, kv, d)
        x = x.view(torch.int8)[at].view(codes.dtype).float() if scales is not None else x[at].float()
        if scales is not None:
            x = x * scales.view(-1, kv)[at][..., None]
        return x.transpose(1, 2).contiguous()  # [b, kv, longest, d]

    k, v = held(state["codes"][0], state["scales"][0]), held(state["codes"][1], state["scales"][1])
    count = starts[1:] - starts[:-1]
    t = torch.arange(new, device="cuda")
    rows = (starts[:-1, None] + t).clamp(max=q.shape[0] - 1)
    x = q[rows].float().view(b, new, kv, group, d).permute(0, 2, 3, 1, 4).reshape(b, kv, group * new, d)
    position = (lengths - count)[:, None, None] + t[None, :, None]  # [b, new, 1]
    hidden = (j > position) | (j >= lengths[:, None, None])
    if c["w"] >= 0:
        hidden = hidden | ((j < position - c["w"]) & (j >= c["sinks"]))
    scores = torch.matmul(x, k.transpose(2, 3).contiguous()).mul_(state["scale"])
    p = _softmax(scores.view(b, kv, group, new, longest), hidden[:, None, None])
    out = torch.matmul(p.view(b, kv, group * new, longest), v).view(b, c["heads"], new, d).transpose(1, 2)
    token = torch.arange(q.shape[0], device="cuda")
    sample = torch.searchsorted(starts, token, right=True) - 1
    return out[sample, token - starts[sample]].to(q.dtype)


_run_plain = {"window": _plain_window, "cache": _plain_cache, "paged": _plain_paged}


# ---- the definition in 64 bits ------------------------------------------------------------------------------
def _attend64(q, k, v, scale, sees, grad=None):
    """One head: q [m, d], k, v [n, d], sees [m, n]; the output, and the three gradients where grad is given."""
    s = (q @ k.T) * scale
    s[~sees] = -math.inf
    m = s.max(1, keepdim=True).values
    m[m == -math.inf] = 0
    e = torch.exp(s - m)
    z = e.sum(1, keepdim=True)
    z[z == 0] = 1
    p = e / z
    o = p @ v
    if grad is None:
        return o
    dp = grad @ v.T
    ds = p * (dp - (p * dp).sum(1, keepdim=True)) * scale
    return o, ds @ k, ds.T @ q, p.T @ grad


def _exact_window(state, c):
    s, group = c["s"], c["heads"] // c["kv"]
    q, k, v = (state[n].detach().double() for n in ("q", "k", "v"))
    o, dq, dk, dv = (torch.zeros_like(x, memory_format=torch.contiguous_format) for x in (q, q, k, v))
    pos = torch.arange(s, device="cuda")
    near = (pos[None, :] <= pos[:, None]) & ((pos[:, None] - pos[None, :] <= c["w"]) | (pos[None, :] < c["sinks"]))
    lengths = _key_lengths(c) if c["padded"] else [s] * c["b"]
    for n in range(c["b"]):
        sees = near & (pos[None, :] < lengths[n])
        for h in range(c["heads"]):
            one = (q[:, n, h], k[:, n, h // group], v[:, n, h // group], state["scale"], sees)
            if not c["train"]:
                o[:, n, h] = _attend64(*one)
                continue
            got = _attend64(*one, state["grad"][:, n, h].double())
            o[:, n, h], dq[:, n, h] = got[0], got[1]
            dk[:, n, h // group] += got[2]
            dv[:, n, h // group] += got[3]
    return (o, dq, dk, dv) if c["train"] else o


def _exact_cache(state, c):
    def one(x):
        x = x.double()
        largest = x.abs().max(-1, keepdim=True).values
        largest[largest == 0] = 1
        y = x * _TOP[c["codes"]] / largest
        if c["codes"] == "int8":
            y = torch.round(y)  # to even at ties
        else:  # 4 bits of significand, exponents from -6: the spacing of the codes around y
            step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0**-6))) - 3)
            y = torch.round(y / step) * step
        return y * largest / _TOP[c["codes"]]

    return one(state["k"]), one(state["v"])


def _exact_paged(state, c):
    page, group = c["page"], c["heads"] // c["kv"]
    new, context = _paged_lengths(c)
    q = state["q"].double()
    out = torch.zeros_like(q)
    first = 0
    for n, (m, t) in enumerate(zip(new, context)):
        places = torch.arange(t, device="cuda")
        pages, inside = state["table"][n].long()[places // page], places % page
        at = torch.arange(t - m, t, device="cuda")[:, None]
        sees = places[None, :] <= at
        if c["w"] >= 0:
            sees &= (at - places[None, :] <= c["w"]) | (places[None, :] < c["sinks"])

        def held(codes, scales, head):
            x = codes[:, :, head].float()[pages, inside].double()
            return x if scales is None else x * scales[:, :, head][pages, inside].double()[:, None]

        for g in range(c["kv"]):
            k = held(state["codes"][0], state["scales"][0], g)
            v = held(state["codes"][1], state["scales"][1], g)
            for h in range(g * group, (g + 1) * group):
                out[first : first + m, h] = _attend64(q[first : first + m, h], k, v, state["scale"], sees)
        first += m
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return {"window": _exact_window, "cache": _exact_cache, "paged": _exact_paged}[case["kind"]](state, case)
