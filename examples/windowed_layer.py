"""One attention layer with a sliding window and sinks: a training step, a prompt in chunks, and generation.

    python examples/windowed_layer.py [--codes int8|fp8|16bit] [--window 256] [--sinks 4]

The layer rotates q and k (``apply_rotary_pos_emb``), and attends with ``window_attention`` in training.  For serving
it writes k and v into a ``PagedKVCache`` and attends with ``paged_attention``: the prompts of two sequences of
different lengths in chunks, then one token of both at a time.  What generation gives is compared with the training
path over the whole sequences; the difference is what the cache's 8-bit codes cost.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from gpt_neox_amd import PagedKVCache, RotaryEmbedding, apply_rotary_pos_emb, paged_attention, slots_of, window_attention  # noqa: E402

CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn, "16bit": torch.bfloat16}


class Layer(torch.nn.Module):
    """Projection to q, k and v (grouped heads), rotary, attention, projection back; hidden states ``[s, b, hidden]``."""

    def __init__(self, hidden, heads, kv_heads, window, sinks, max_positions, dtype=torch.bfloat16):
        super().__init__()
        self.heads, self.kv, self.dim = heads, kv_heads, hidden // heads
        self.window, self.sinks = window, sinks
        self.qkv = torch.nn.Linear(hidden, (heads + 2 * kv_heads) * self.dim, bias=False, dtype=dtype, device="cuda")
        self.dense = torch.nn.Linear(hidden, hidden, bias=False, dtype=dtype, device="cuda")
        self.rotary = RotaryEmbedding(self.dim, max_positions, precision=torch.float)

    def project(self, x, offset=0):
        mixed = self.qkv(x).view(*x.shape[:2], self.heads + 2 * self.kv, self.dim)
        q, k, v = mixed.split((self.heads, self.kv, self.kv), dim=2)
        cos, sin = self.rotary(x, seq_len=offset + x.shape[0])
        return (*apply_rotary_pos_emb(q, k, cos, sin, offset), v)

    def forward(self, x, key_lengths=None):
        q, k, v = self.project(x)
        out = window_attention(q, k, v, window=self.window, sinks=self.sinks, key_lengths=key_lengths)
        return self.dense(out.reshape(*x.shape))

    @torch.no_grad()
    def step(self, x, positions, cache, table, lengths):
        """New tokens of every sequence: ``x`` a list of ``[n, hidden]``, which stand at ``positions`` onwards; ``lengths``
        (int32 ``[b]``) counts them too.  Returns a list like ``x``."""
        parts = [self.project(t[:, None], p) for t, p in zip(x, positions)]
        q, k, v = (torch.cat([part[i][:, 0] for part in parts]) for i in range(3))
        count = [t.shape[0] for t in x]
        sample = torch.cat([torch.full((n,), s, device="cuda") for s, n in enumerate(count)])
        position = torch.cat([torch.arange(p, p + n, device="cuda") for p, n in zip(positions, count)])
        cache.write(k, v, slots_of(table, sample, position, cache.page_size))
        starts = torch.tensor([sum(count[:s]) for s in range(len(count) + 1)], dtype=torch.int32, device="cuda")
        out = paged_attention(q, cache, table, starts, lengths, max_query=max(count), max_context=max(p + n for p, n in zip(positions, count)),
                              window=self.window, sinks=self.sinks)
        return list(self.dense(out.view(out.shape[0], -1)).split(count))


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--codes", choices=sorted(CODES), default="int8")
    ap.add_argument("--window", type=int, default=256)
    ap.add_argument("--sinks", type=int, default=4)
    args = ap.parse_args(argv)
    torch.manual_seed(0)
    hidden, heads, kv, page = 1024, 16, 4, 64
    lengths = [700, 450]  # of the two sequences, once everything is generated
    prompts = [n - 40 for n in lengths]
    layer = Layer(hidden, heads, kv, args.window, args.sinks, 1024)

    # a training step on the padded batch
    x = torch.randn(max(lengths), 2, hidden, device="cuda").bfloat16()
    ends = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    y = layer(x, ends)
    valid = torch.arange(max(lengths), device="cuda")[:, None] < ends
    loss = (y.float().square().sum(-1) * valid).sum() / valid.sum()
    loss.backward()
    assert all(torch.isfinite(p.grad).all() for p in layer.parameters())
    print(f"training step: loss {loss.item():.4f}, |grad| {sum(p.grad.float().square().sum() for p in layer.parameters()).sqrt().item():.4f}")

    # serving: the prompts in chunks of 200 tokens, then a token at a time
    pages = sum(-(-n // page) for n in lengths) + 1
    cache = PagedKVCache.allocate(pages, page, kv, hidden // heads, CODES[args.codes])
    order = torch.randperm(pages - 1, device="cuda").int() + 1
    table = torch.zeros((2, -(-max(lengths) // page)), dtype=torch.int32, device="cuda")
    used = 0
    for s, n in enumerate(lengths):
        table[s, : -(-n // page)] = order[used : used + -(-n // page)]
        used += -(-n // page)
    got = [[], []]
    at = [0, 0]
    while at != lengths:
        count = [min(200, prompts[s] - at[s]) if at[s] < prompts[s] else min(1, lengths[s] - at[s]) for s in range(2)]
        new = [x[at[s] : at[s] + count[s], s] for s in range(2)]
        total = torch.tensor([a + n for a, n in zip(at, count)], dtype=torch.int32, device="cuda")
        for s, out in enumerate(layer.step(new, at, cache, table, total)):
            got[s].append(out)
        at = [a + n for a, n in zip(at, count)]
    worst = 0.0
    for s, n in enumerate(lengths):
        want = y[:n, s].detach().float()
        worst = max(worst, ((torch.cat(got[s]).float() - want).norm() / want.norm()).item())
    print(f"chunks and generation over the cache in {args.codes}: {worst:.4f} of the training path's norm away from it")
    return worst


if __name__ == "__main__":
    main()
