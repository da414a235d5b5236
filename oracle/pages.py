"""The 4-bit codes of a paged cache in 64 bits, and the pages' bookkeeping one sequence after the other (any device).

Plain restatements of the definitions in ``include/neox_fused.h``, written without the product's code.  Test
infrastructure: never imported by the product.
"""
import torch

GROUP = 32
NAN = 255
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
LEAST, MOST = -125, {torch.float16: 13, torch.bfloat16: 125}


def exponents(x):
    """``x [..., d]`` in fp16 or bf16 -> int64 ``[..., d / 32]``: the least e with 7 * 2^e >= the largest of 32, within limits."""
    largest = x.double().abs().unflatten(-1, (-1, GROUP)).amax(-1)
    e = torch.full(largest.shape, LEAST, dtype=torch.int64, device=x.device)
    for power in range(MOST[x.dtype] - 1, LEAST - 1, -1):  # (a sequence of comparisons, with no logarithm to be rounded)
        e = torch.where((e == LEAST) & (largest > 7.0 * 2.0**power), power + 1, e)
    return e


def encode(x):
    """Rows ``[..., d]`` -> their values as the cache holds them (float64 ``[..., d]``; NaN where a row is not finite) and the scales'
    bytes (uint8 ``[..., d / 32]``).  Every value is compared with the sixteen that there are; the nearest is taken, at ties the one
    with an even code."""
    e = exponents(x)
    y = x.double().unflatten(-1, (-1, GROUP)) / torch.exp2(e.double())[..., None]
    best, far = torch.zeros_like(y), torch.full_like(y, float("inf"))
    order = [0, 2, 4, 6, 1, 3, 5, 7]  # even codes first: only a nearer odd one takes their place
    for code in order:
        for sign in (1.0, -1.0):
            value = sign * VALUES[code]
            nearer = (y - value).abs() < far
            best, far = torch.where(nearer, value, best), torch.where(nearer, (y - value).abs(), far)
    out = (best * torch.exp2(e.double())[..., None]).flatten(-2)
    bad = ~torch.isfinite(x.double()).all(-1, keepdim=True)
    return out.masked_fill(bad, float("nan")), (e + 127).masked_fill(bad, NAN).byte()


def decode(codes, scales):
    """Bytes ``[..., d / 2]`` and ``[..., d / 32]`` -> float64 ``[..., d]``; a row with a NaN scale is NaN,
    and so is one with a scale above the largest that is ever written."""
    scales = torch.where(scales > 127 + MOST[torch.bfloat16], NAN, scales)
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), dtype=torch.float64, device=codes.device)
    x = table[torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()]
    f = torch.exp2(scales.double() - 127).masked_fill(scales == NAN, float("nan")).repeat_interleave(GROUP, -1)
    return (x * f).masked_fill((scales == NAN).any(-1, keepdim=True), float("nan"))


class Pool:
    """The state and the calls of a page pool, in lists."""

    def __init__(self, table, lengths, free, left, page_size):
        self.table, self.lengths, self.free, self.left, self.page = [list(r) for r in table], list(lengths), list(free), left, page_size

    def extend(self, new, max_tokens):
        starts, positions, slots, granted, missing = [0], [], [], [], False
        total = 0
        for s, n in enumerate(new):
            n = max(n, 0)
            old, row = self.lengths[s], self.table[s]
            total += n
            need = -(-(old + n) // self.page) - -(-old // self.page)
            yes = old + n <= len(row) * self.page and total <= max_tokens
            if yes and need:
                # (what those before it asked for counts, whether they got it or not)
                missing = missing or need > self.left
                yes = not missing
            if yes:
                for i in range(need):
                    self.left -= 1
                    row[-(-old // self.page) + i] = self.free[self.left]
                self.lengths[s] = old + n
            for position in range(old, old + n):
                if len(positions) < max_tokens:
                    positions.append(position)
                    slots.append(row[position // self.page] * self.page + position % self.page if yes else -1)
            starts.append(min(total, max_tokens))
            granted.append(yes)
        rest = max_tokens - len(positions)
        return starts, positions + [0] * rest, slots + [-1] * rest, granted

    def truncate(self, lengths):
        for s in reversed(range(len(self.lengths))):
            keep = min(self.lengths[s], max(lengths[s], 0))
            for column in reversed(range(-(-keep // self.page), -(-self.lengths[s] // self.page))):
                self.free[self.left] = self.table[s][column]
                self.table[s][column] = -1
                self.left += 1
            self.lengths[s] = keep
