#!/usr/bin/env python3
"""A decoder layer served with this package's operators: what a program does with them, prompt and token by token.

    q, k, v = projection(norm(x));  q, k = rotate, append k, v to the paged cache;  x += projection(attention(q))
    x += mlp(norm(x))

The projections are `swiglu_down_*` (a row-major product with a [out, in] weight), the MLP is `fused_swiglu_mlp_*`; the norm is
elementary torch. Random weights. `python decoder_layer.py` runs a batch of prompts, then decodes some tokens of each, and
compares the decoded tokens' outputs with those of the whole sequences taken as prompts.
"""
import argparse
import math
import sys

import torch

import fsw_weights


class PagedCache:
    """Keys and values of one layer in pages of `page` tokens, and which pages each sequence has. Pages are handed out as
    tokens arrive; the table and the lengths are kept on the device, where the kernels read them."""

    def __init__(self, seqs, longest, kv_heads, channels, page, dtype, device):
        per_seq = -(-longest // page)
        self.page, self.longest, self.device = page, longest, device
        self.k = torch.empty(seqs * per_seq, kv_heads, page, channels, dtype=dtype, device=device)
        self.v = torch.empty_like(self.k)
        self.free = list(range(seqs * per_seq))
        self.pages = [[] for _ in range(seqs)]
        self.lengths = [0] * seqs
        self.per_seq = per_seq

    def grow(self, counts):
        """Room for counts[b] more tokens of sequence b -> positions and slots of the new tokens, packed, on the device."""
        for b, n in enumerate(counts):
            if self.lengths[b] + n > self.longest:
                raise ValueError("sequence %d would have %d tokens, the cache was made for %d" % (b, self.lengths[b] + n, self.longest))
        positions, slots = [], []
        for b, n in enumerate(counts):
            for t in range(self.lengths[b], self.lengths[b] + n):
                if t // self.page == len(self.pages[b]):
                    self.pages[b].append(self.free.pop())
                positions.append(t)
                slots.append(self.pages[b][t // self.page] * self.page + t % self.page)
            self.lengths[b] += n
        return self._int32(positions), self._int32(slots)

    def table(self):
        """(block table, lengths, longest) for attn_decode."""
        return (self._int32([p + [0] * (self.per_seq - len(p)) for p in self.pages]), self._int32(self.lengths), max(self.lengths))

    def _int32(self, values):
        return torch.tensor(values, dtype=torch.int32).to(self.device)


class DecoderLayer:
    def __init__(self, d, ff, heads, kv_heads, longest, dtype=torch.bfloat16, device="cuda:0", seed=0):
        import fused_mlp_module as m
        name = "bf16" if dtype == torch.bfloat16 else "fp16"
        self.append, self.decode, self.prompt, self.project, self.mlp = (
            getattr(m, op + name) for op in ("kv_append_", "attn_decode_", "attn_prompt_", "swiglu_down_", "fused_swiglu_mlp_"))
        self.heads, self.kv_heads, self.channels = heads, kv_heads, d // heads
        w = fsw_weights.make_inputs(1, d, ff, dtype, seed)
        self.w13, self.w2 = w["W13"].to(device), w["W2"].to(device)
        gen = torch.Generator().manual_seed(seed + 1)

        def weight(rows, cols):
            return (torch.randn(rows, cols, generator=gen) / math.sqrt(cols)).to(dtype).to(device)

        self.w_qkv = weight((heads + 2 * kv_heads) * self.channels, d)
        self.w_out = weight(d, heads * self.channels)
        rate = 10000.0 ** (-torch.arange(0, self.channels, 2, dtype=torch.float64) / self.channels)
        angle = torch.outer(torch.arange(longest, dtype=torch.float64), rate)
        self.cos_sin = torch.cat([angle.cos(), angle.sin()], 1).float().to(device)

    @staticmethod
    def norm(x):
        y = x.float()
        return (y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-5)).to(x.dtype)

    def _qkv(self, x):
        rows = self.project(self.norm(x), self.w_qkv).view(x.shape[0], -1, self.channels)
        return rows.split([self.heads, self.kv_heads, self.kv_heads], 1)

    def _finish(self, x, attended):
        x = x + self.project(attended.reshape(x.shape[0], -1), self.w_out)
        return x + self.mlp(self.norm(x), self.w13, self.w2)

    def prefill(self, x, lengths, cache):
        """x: the packed rows of new sequences' prompts."""
        for b, n in enumerate(lengths):
            if n and cache.lengths[b]:
                raise ValueError("sequence %d has tokens in the cache already" % b)
        q, k, v = self._qkv(x)
        positions, slots = cache.grow(lengths)
        q, k = self.append(q, k, v, self.cos_sin, positions, slots, cache.k, cache.v)
        starts = [0]
        for n in lengths:
            starts.append(starts[-1] + n)
        starts = torch.tensor(starts, dtype=torch.int32).to(x.device)
        return self._finish(x, self.prompt(q, k, v, starts, starts, self.channels ** -0.5))

    def step(self, x, cache):
        """x: one row per sequence, its next token."""
        q, k, v = self._qkv(x)
        positions, slots = cache.grow([1] * x.shape[0])
        q, _ = self.append(q, k, v, self.cos_sin, positions, slots, cache.k, cache.v)
        table, lengths, longest = cache.table()
        return self._finish(x, self.decode(q, cache.k, cache.v, table, lengths, longest, self.channels ** -0.5))


def run(d=1024, ff=2816, heads=16, kv_heads=4, prompts=(37, 5, 130), steps=9, page=16, dtype=torch.bfloat16, seed=0):
    """Largest difference, over the root mean square of the outputs, between tokens decoded one by one and the same tokens
    inside their whole sequences."""
    longest = max(prompts) + steps
    layer = DecoderLayer(d, ff, heads, kv_heads, longest, dtype, seed=seed)
    gen = torch.Generator().manual_seed(seed + 2)
    whole = [torch.randn(n + steps, d, generator=gen).to(dtype).to("cuda:0") for n in prompts]

    def new_cache():
        return PagedCache(len(prompts), longest, kv_heads, d // heads, page, dtype, "cuda:0")

    cache = new_cache()
    layer.prefill(torch.cat([x[:n] for x, n in zip(whole, prompts)]), list(prompts), cache)
    decoded = [layer.step(torch.stack([x[n + i] for x, n in zip(whole, prompts)]), cache) for i in range(steps)]
    want = layer.prefill(torch.cat(whole), [n + steps for n in prompts], new_cache()).split([n + steps for n in prompts])
    worst = 0.0
    for b, n in enumerate(prompts):
        got, ref = torch.stack([y[b] for y in decoded]).float(), want[b][n:].float()
        worst = max(worst, ((got - ref).abs().max() / ref.square().mean().sqrt()).item())
    return worst


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--d", type=int, default=1024)
    ap.add_argument("--ff", type=int, default=2816)
    ap.add_argument("--heads", type=int, default=16)
    ap.add_argument("--kv-heads", type=int, default=4)
    ap.add_argument("--prompts", type=int, nargs="+", default=[37, 5, 130])
    ap.add_argument("--steps", type=int, default=9)
    ap.add_argument("--page", type=int, default=16)
    args = ap.parse_args(argv)
    if not torch.cuda.is_available():
        sys.exit("decoder_layer.py needs the GPU: the extension has no CPU path")
    worst = run(args.d, args.ff, args.heads, args.kv_heads, tuple(args.prompts), args.steps, args.page)
    print("%d prompts, %d steps each: decoded tokens differ from whole sequences by %.1e of the outputs' size" %
          (len(args.prompts), args.steps, worst))


if __name__ == "__main__":
    main()
