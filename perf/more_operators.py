"""A paged cache of keys and values in 4 bits, the attention that reads it, and the pages' bookkeeping on the GPU, as
cases that a timing program can run.

A case is a dict of plain values; ``listed()`` names eleven of them, ``draw(rng)`` makes more of the same ranges.
Three operators, those of one step of a server that generates for many sequences:

* ``pool`` -- which pages and slots the new tokens of every sequence get, from their numbers alone, and the pages' way
  back when they are dropped: page tables, starts, positions and slots;
* ``cache`` -- new keys and values written into a paged cache of 4-bit floats (e2m1), 32 of which share a power of two,
  and read back from there;
* ``paged`` -- attention of the newest tokens of each sequence over its pages of such a cache: single tokens
  (generation), a few that are checked together, or chunks of a prompt, with or without a window and sinks.

``run`` computes them in plain torch where ``own`` is false, and through the package's entry points where it is true.
"""
import math

import torch

own = False

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_GROUP = 32  # values that share a scale
_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # what the codes 0 to 7 stand for; 8 to 15 are the same below zero
_LEAST, _MOST = -125, {"fp16": 13, "bf16": 125}  # exponents of scales: 6 * 2^most is a number of the type that was written
_NAN = 255  # as a scale; any other byte s stands for 2^(s - 127)


def _pool(name, b, new, context, page, columns, short=False):
    return {"name": name, "kind": "pool", "b": b, "new": new, "context": context, "page": page, "columns": columns, "short": short}


def _cache(name, tokens, kv, d, dtype, page, pages):
    return {"name": name, "kind": "cache", "tokens": tokens, "kv": kv, "d": d, "dtype": dtype, "page": page, "pages": pages}


def _paged(name, b, new, context, heads, kv, d, dtype, page, w=-1, sinks=0, ragged=True):
    return {"name": name, "kind": "paged", "b": b, "new": new, "context": context, "heads": heads, "kv": kv, "d": d,
            "dtype": dtype, "page": page, "w": w, "sinks": sinks, "ragged": ragged}


def listed():
    return [
        # generation, the smallest step: a token for each of 64 sequences, a few of which begin a page
        _pool("pool_tokens", 64, 1, 8192, 16, 513),
        # five tokens of a draft for each of 1000 short sequences, and all of them dropped again
        _pool("pool_drafts", 1000, 5, 700, 16, 48),
        # the prompts of a large batch, into an empty pool, and the batch's end; the pool is too small for the last ones
        _pool("pool_prompts", 256, 2048, 0, 64, 64, short=True),
        # one generated token of each of 16 sequences into the cache of one layer, and back
        _cache("cache_tokens", 16, 8, 128, "bf16", 16, 512),
        # a prompt at the 20B shape, of an odd length, into pages that hold other sequences too
        _cache("cache_prompt", 2047, 64, 96, "fp16", 64, 64),
        # the prompts of a large batch
        _cache("cache_prompts", 65536, 32, 128, "bf16", 64, 1536),
        # generation, the smallest: one token of four sequences of a 125M model
        _paged("paged_token_small", 4, 1, 517, 12, 12, 64, "fp16", 16),
        # generation for many users: sequences of 2k to 8k tokens, grouped heads
        _paged("paged_token_batch", 64, 1, 8192, 32, 8, 128, "bf16", 64),
        # one very long sequence, whose work has to be split over its keys
        _paged("paged_token_long", 1, 1, 131001, 32, 8, 128, "bf16", 128),
        # five tokens of a draft for each of 16 sequences, wide heads, pages that end inside every tile
        _paged("paged_draft", 16, 5, 4099, 16, 8, 256, "fp16", 48, w=1024, sinks=4),
        # chunks of four prompts, each over what its sequence has in the cache already
        _paged("paged_chunk", 4, 512, 16384, 32, 8, 128, "bf16", 64, w=4096, sinks=4),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: any kind, its sizes spread over the logarithm of their range, odd ones among them."""
    kind = rng.choice(["pool", "cache", "cache", "paged", "paged", "paged", "paged"])
    page = rng.choice([16, 32, 48, 64, 128, 256])
    if kind == "pool":
        b = _log_int(rng, 1, 4096)
        if rng.random() < 0.5:  # tokens of sequences in the middle
            new, context = rng.choice([1, 1, 2, 5]), _log_int(rng, 16, 16384)
        else:  # prompts, whole or in chunks
            new, context = _log_int(rng, 16, 131072), rng.choice([0, 0, _log_int(rng, 16, 16384)])
        while b * new > 524288:
            new = new // 2 + 1
        while b * (context // page) > 1 << 20:
            context //= 2
        return _pool("", b, new, context, page, -(-(new + context) // page) + rng.choice([0, 0, 1, 7]), rng.random() < 0.3)
    dtype = rng.choice(["fp16", "bf16"])
    d = rng.choice([32, 64, 96, 128, 128, 160, 256])
    kv = rng.choice([1, 2, 4, 8, 12, 16])
    if kind == "cache":
        tokens = _log_int(rng, 1, 65536)
        while tokens * kv * d > 65536 * 32 * 128:
            tokens = tokens // 2 + 1
        return _cache("", tokens, kv, d, dtype, page, tokens // page * 3 // 2 + 4)
    heads = kv * rng.choice([1, 1, 2, 4, 8])
    sinks = rng.choice([0, 1, 4, 16])
    if rng.random() < 0.65:  # generation: one token, or a few that are checked together
        b, new, context = rng.choice([1, 2, 4, 16, 64]), rng.choice([1, 1, 1, 2, 5]), _log_int(rng, 32, 131072)
    else:
        b, new, context = rng.choice([1, 2, 4]), _log_int(rng, 16, 1024), _log_int(rng, 1024, 32768)
    w = rng.choice([-1, -1, 128, 1024, 4096])
    c = _paged("", b, new, context, heads, kv, d, dtype, page, w, sinks if w >= 0 else 0, rng.random() < 0.7)
    while c["b"] * c["context"] * c["kv"] * c["d"] > 64 * 8192 * 8 * 128 or \
            c["b"] * c["new"] * c["context"] * c["heads"] * c["d"] > 4 * 512 * 16384 * 32 * 128:
        c["context"] = c["context"] // 2 + 1
        c["new"] = min(c["new"], c["context"])
    return c


# ---- what a case's lengths are: part of the case, not of the seed -------------------------------------
def _pool_lengths(c):
    """Tokens that every sequence has, and how many come: both from all of the case's number down to a quarter of it."""
    old, new = [], []
    for i in range(c["b"]):
        j = i * 7 % c["b"] if c["b"] % 7 else i  # the long ones are not all at the front
        old.append(c["context"] - j * (c["context"] * 3 // 4) // max(1, c["b"] - 1))
        new.append(max(1, c["new"] - i * (c["new"] * 3 // 4) // max(1, c["b"] - 1)))
    return old, new


def _pool_pages(c):
    """Pages of the pool: those that the sequences have, and room for what comes -- or for most of it."""
    old, new = _pool_lengths(c)
    have = sum(-(-n // c["page"]) for n in old)
    need = sum(-(-(n + m) // c["page"]) for n, m in zip(old, new)) - have
    return have, need, have + (need * 15 // 16 if c["short"] else need + 3)


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
    visible pairs."""
    c = case
    if c["kind"] == "pool":
        _, new = _pool_lengths(c)
        tokens, pages = sum(new), _pool_pages(c)[1]
        # numbers in and out of both calls; a slot and a position for each token; each page out of the list into its
        # table, and back
        return {"bytes": 33 * c["b"] + 12 * tokens + 20 * pages, "flops": 4 * tokens}
    row = c["d"] // 2 + c["d"] // _GROUP
    if c["kind"] == "cache":
        n = c["tokens"] * c["kv"]
        # k and v in, codes and scales out and in again, k and v out; a product each way for each value
        return {"bytes": 2 * n * (4 * c["d"] + 2 * row) + 8 * c["tokens"], "flops": 4 * n * c["d"]}
    new, context = _paged_lengths(c)
    pairs = touched = 0
    for n, t in zip(new, context):
        pairs += _visible(t - n, n, c["w"], c["sinks"], t) * c["heads"]
        start = 0 if c["w"] < 0 else max(0, t - n - c["w"])
        touched += t - start + min(c["sinks"], start)
    return {"bytes": 2 * touched * c["kv"] * row + 4 * sum(new) * c["heads"] * c["d"], "flops": 4 * pairs * c["d"]}


# ---- inputs ---------------------------------------------------------------------------------------------
def _normal(shape, dtype, gen, times=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * times).to(dtype)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _loud(x, gen):
    """Keys have a few large channels, as they do behind a projection with outliers."""
    return x.mul_(torch.where(torch.rand(x.shape[-1], generator=gen, device="cuda") < 0.05, 8.0, 1.0))


def _encode(x, dtype):
    """Rows of the last dim as 4-bit codes, two to a byte, and a byte for the scale of every 32 values: the least power
    of two of which seven times is no less than the largest of them.  A row that is not all finite gets no scale."""
    x = x.float()
    groups = x.unflatten(-1, (-1, _GROUP))
    largest = groups.abs().amax(-1)
    part, exponent = torch.frexp(largest)  # part * 2^exponent, part in [0.5, 1)
    exponent = exponent - 3 + (part > 0.875).int()
    exponent = torch.where(largest > 0, exponent, _LEAST).clamp(_LEAST, _MOST[dtype])
    y = torch.ldexp(groups, -exponent[..., None])
    size = y.abs()
    code = (size > 0.25).byte()
    for border, even in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (size >= border) if even else (size > border)
    code = (code + 8 * (y < 0).byte()).flatten(-2)
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    code = code.masked_fill(bad, 0)
    scale = (exponent + 127).masked_fill(bad, _NAN).byte()
    return code[..., 0::2] | code[..., 1::2] << 4, scale


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": c}
    if c["kind"] == "pool":
        old, new = _pool_lengths(c)
        have, _, pages = _pool_pages(c)
        order = torch.randperm(pages, generator=gen, device="cuda").int()
        table = torch.full((c["b"], c["columns"]), -1, dtype=torch.int32, device="cuda")
        count = (torch.tensor(old, device="cuda") + c["page"] - 1) // c["page"]
        held = torch.arange(c["columns"], device="cuda") < count[:, None]
        table[held] = order[:have]
        free = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
        free[: pages - have] = order[have:]
        state.update(table=table, lengths=_int32(old), free=free, left=_int32([pages - have]), new=_int32(new), keep=_int32(old),
                     tokens=sum(new))
        if own:
            from gpt_neox_amd.page_pool import PagePool

            state["pool"] = PagePool(table, state["lengths"], free, state["left"], page_size=c["page"])
        return state
    dtype, kv, d, page = _TYPES[c["dtype"]], c["kv"], c["d"], c["page"]
    if c["kind"] == "cache":
        pages = c["pages"]
        state["k"] = _loud(_normal((c["tokens"], kv, d), torch.float32, gen), gen).to(dtype)
        state["v"] = _normal((c["tokens"], kv, d), dtype, gen)
        state["slots"] = torch.randperm(pages * page, generator=gen, device="cuda")[: c["tokens"]]
        codes = [torch.zeros((pages, page, kv, d // 2), dtype=torch.uint8, device="cuda") for _ in "kv"]
        scales = [torch.zeros((pages, page, kv, d // _GROUP), dtype=torch.uint8, device="cuda") for _ in "kv"]
    else:
        new, context = _paged_lengths(c)
        width = -(-max(context) // page)
        pages = c["b"] * width + 3
        table = torch.randperm(pages, generator=gen, device="cuda")[: c["b"] * width].view(c["b"], width).int()
        codes, scales = [], []
        for which in "kv":
            # (a few heads at a time: the codes' intermediate forms are many times their size)
            x = [torch.empty((pages, page, kv, n), dtype=torch.uint8, device="cuda") for n in (d // 2, d // _GROUP)]
            for first in range(0, kv, 2):
                part = _normal((pages, page, min(2, kv - first), d), torch.float32, gen)
                part = (_loud(part, gen) if which == "k" else part).to(dtype)
                x[0][:, :, first : first + 2], x[1][:, :, first : first + 2] = _encode(part, c["dtype"])
            codes.append(x[0])
            scales.append(x[1])
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        state.update(q=_normal((starts[-1], c["heads"], d), dtype, gen), table=table, max_new=max(new), longest=max(context),
                     starts=_int32(starts), lengths=_int32(context), scale=1.0 / math.sqrt(d))
    state["codes"], state["scales"] = codes, scales
    if own:
        from gpt_neox_amd.paged_cache import PagedKVCache

        state["cache"] = PagedKVCache(*(x.view(torch.float4_e2m1fn_x2) for x in codes), *(x.view(torch.float8_e8m0fnu) for x in scales))
    return state


# ---- one pass ---------------------------------------------------------------------------------------------
def run(state):
    c = state["case"]
    return (_run_own if own else _run_plain)[c["kind"]](state, c)


def _own_pool(state, c):
    pool = state["pool"]
    step = pool.extend(state["new"], max_tokens=state["tokens"])
    pool.truncate(state["keep"])
    return step.query_starts, step.positions, step.slots, step.granted, pool.page_table, pool.lengths, pool.free, pool.left


def _own_cache(state, c):
    cache = state["cache"]
    cache.write(state["k"], state["v"], state["slots"])
    return cache.read(state["slots"], dtype=state["k"].dtype)


def _own_paged(state, c):
    from gpt_neox_amd.paged_cache import paged_attention

    return paged_attention(state["q"], state["cache"], state["table"], state["starts"], state["lengths"],
                           max_query=state["max_new"], max_context=state["longest"], scale=state["scale"],
                           window=c["w"] if c["w"] >= 0 else None, sinks=c["sinks"])


_run_own = {"pool": _own_pool, "cache": _own_cache, "paged": _own_paged}


def _plain_pool(state, c):
    page, tokens = c["page"], state["tokens"]
    table, lengths, free, left = state["table"], state["lengths"], state["free"], state["left"]
    # the new tokens' pages, those on top of the list of free ones first; who does not fit gets none
    new, old, room = state["new"].long().clamp(min=0), lengths.long(), left.long()
    ends = torch.cumsum(new, 0)
    have = (old + page - 1) // page
    fits = (old + new <= c["columns"] * page) & (ends <= tokens)
    need = torch.where(fits, (old + new + page - 1) // page - have, 0)
    upto = torch.cumsum(need, 0)
    granted = fits & ((need == 0) | (upto <= room))
    starts = torch.cat((torch.zeros_like(ends[:1]), ends))
    token = torch.arange(tokens, device="cuda")
    sample = torch.searchsorted(ends, token, right=True)
    inside = token - starts[sample]
    position = old[sample] + inside
    column = position // page
    first = upto - need  # new pages of the sequences before
    at = column - have[sample]  # below zero: the page is there already
    source = (room - 1 - first[sample] - at).clamp(0, free.shape[0] - 1)
    number = torch.where(at < 0, table[sample, column.clamp(max=c["columns"] - 1)], free[source]).long()
    slots = torch.where(granted[sample], number * page + position % page, -1)
    begins = granted[sample] & (at >= 0) & ((position % page == 0) | (inside == 0))
    table[sample[begins], column[begins]] = number[begins].int()
    lengths.copy_(torch.where(granted, old + new, old))
    left.copy_(room - torch.where(granted & (need > 0), upto, 0).amax())
    # ... and back onto the list, the last one first
    old, room = lengths.long(), left.long()
    keep = torch.minimum(state["keep"].long().clamp(min=0), old)
    place = torch.arange(c["columns"], device="cuda")
    given = (place >= ((keep + page - 1) // page)[:, None]) & (place < ((old + page - 1) // page)[:, None])
    numbers = table[given].flip(0)
    free[room + torch.arange(numbers.shape[0], device="cuda")] = numbers
    table.masked_fill_(given, -1)
    lengths.copy_(keep)
    left.add_(numbers.shape[0])
    return starts.clamp(max=tokens).int(), position.int(), slots, granted, table, lengths, free, left


def _softmax(scores, hidden):
    """Probabilities over the last dim; a row without a visible key is zero everywhere."""
    scores = scores.masked_fill(hidden, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, 1.0, total)


def _decode(codes, scales):
    """Codes [..., d / 2] and scales [..., d / 32] as fp32 values [..., d]."""
    values = torch.tensor(_VALUES + tuple(-x for x in _VALUES), device="cuda")
    x = torch.stack((values[(codes & 15).int()], values[(codes >> 4).int()]), -1).flatten(-2)
    scale = torch.where(scales == _NAN, math.nan, torch.ldexp(torch.ones((), device="cuda"), scales.int() - 127))
    return (x.unflatten(-1, (-1, _GROUP)) * scale[..., None]).flatten(-2)


def _plain_cache(state, c):
    slots, dtype = state["slots"], state["k"].dtype

    def one(x, codes, scales):
        codes, scales = codes.view(-1, *codes.shape[2:]), scales.view(-1, *scales.shape[2:])
        codes[slots], scales[slots] = _encode(x, c["dtype"])
        return _decode(codes[slots], scales[slots]).to(dtype)

    return (one(state["k"], state["codes"][0], state["scales"][0]), one(state["v"], state["codes"][1], state["scales"][1]))


def _plain_paged(state, c):
    b, kv, d, page, group = c["b"], c["kv"], c["d"], c["page"], c["heads"] // c["kv"]
    q, starts, lengths, new, longest = state["q"], state["starts"].long(), state["lengths"].long(), state["max_new"], state["longest"]
    j = torch.arange(longest, device="cuda")
    at = state["table"].long()[:, j // page] * page + j % page  # [b, longest]

    def held(codes, scales):
        x = _decode(codes.view(-1, *codes.shape[2:])[at], scales.view(-1, *scales.shape[2:])[at])
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


_run_plain = {"pool": _plain_pool, "cache": _plain_cache, "paged": _plain_paged}


# ---- the definition in 64 bits ------------------------------------------------------------------------------
def _exact_pool(state, c):
    """One sequence after the other, on the host."""
    page, tokens = c["page"], state["tokens"]
    table, lengths, free = (state[n].cpu().long() for n in ("table", "lengths", "free"))
    left, new, keep = state["left"].item(), state["new"].tolist(), state["keep"].tolist()
    starts, granted, slots, positions = [0], [], torch.full((tokens,), -1), torch.zeros(tokens, dtype=torch.long)
    denied = False  # once the pool has had too few pages for one, none that needs a page gets any
    for s, n in enumerate(new):
        have, total = -(-lengths[s].item() // page), lengths[s].item() + n
        need = -(-total // page) - have
        yes = total <= c["columns"] * page and starts[-1] + n <= tokens
        if yes and need > 0:
            denied = denied or need > left
            yes = not denied
        at = torch.arange(lengths[s].item(), total)
        positions[starts[-1] : starts[-1] + n] = at
        if yes:
            for i in range(need):
                left -= 1
                table[s, have + i] = free[left]
            slots[starts[-1] : starts[-1] + n] = table[s, at // page] * page + at % page
            lengths[s] = total
        starts.append(starts[-1] + n)
        granted.append(yes)
    for s in reversed(range(c["b"])):
        n = min(keep[s], lengths[s].item())
        for column in reversed(range(-(-n // page), -(-lengths[s].item() // page))):
            free[left], table[s, column] = table[s, column], -1
            left += 1
        lengths[s] = n
    int32 = [torch.as_tensor(x).int() for x in (starts, positions, table, lengths, free, [left])]
    return int32[0], int32[1], slots, torch.tensor(granted), *int32[2:]


def _attend64(q, k, v, scale, sees):
    """One head: q [m, d], k, v [n, d], sees [m, n]."""
    s = (q @ k.T) * scale
    s[~sees] = -math.inf
    m = s.max(1, keepdim=True).values
    m[m == -math.inf] = 0
    e = torch.exp(s - m)
    z = e.sum(1, keepdim=True)
    z[z == 0] = 1
    return (e / z) @ v


def _exact_cache(state, c):
    def one(x):
        x = x.double().unflatten(-1, (-1, _GROUP))
        largest = x.abs().max(-1, keepdim=True).values
        e = torch.ceil(torch.log2(largest / 7)).clamp(_LEAST, _MOST[c["dtype"]])
        e = torch.where(largest > 7 * torch.exp2(e), e + 1, torch.where(largest <= 7 * torch.exp2(e - 1), e - 1, e))  # (log2 is not exact)
        e = e.clamp(_LEAST, _MOST[c["dtype"]])
        y = (x / torch.exp2(e)).clamp(-6, 6)
        # 2 bits of significand, exponents from 0: the spacing of the codes around y
        step = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0))
        return (torch.round(y / step) * step * torch.exp2(e)).flatten(-2)  # to even at ties

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
            x = codes[pages, inside, head].int()
            x = torch.stack((x % 16, x // 16), -1).flatten(-2).double()
            size, sign = x % 8, torch.where(x >= 8, -1.0, 1.0)
            # a code's lowest bit is its significand's, the two above are its exponent; none: a multiple of a half
            power = torch.exp2(torch.floor(size / 2) - 1)
            value = sign * torch.where(size < 2, size / 2, power * (1 + (size % 2) / 2))
            scale = torch.exp2(scales[pages, inside, head].double() - 127)
            return value * scale.repeat_interleave(_GROUP, -1)

        for g in range(c["kv"]):
            k = held(state["codes"][0], state["scales"][0], g)
            v = held(state["codes"][1], state["scales"][1], g)
            for h in range(g * group, (g + 1) * group):
                out[first : first + m, h] = _attend64(q[first : first + m, h], k, v, state["scale"], sees)
        first += m
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return {"pool": _exact_pool, "cache": _exact_cache, "paged": _exact_paged}[case["kind"]](state, case)
