#!/usr/bin/env python3
"""A decoder layer served with this package's operators: what a program does with them, prompt and token by token.

    q, k, v = projection(norm(x));  q, k = rotate, append k, v to the paged cache;  x += projection(attention(q))
    x += mlp(norm(x))

The projections are `swiglu_down_*` (a row-major product with a [out, in] weight), the MLP is `fused_swiglu_mlp_*`; the norm is
elementary torch. Random weights. `python decoder_layer.py` runs a batch of prompts, then decodes some tokens of each, and
compares the decoded tokens' outputs with those of the whole sequences taken as prompts.

`--eight`: the cache holds e4m3 elements (`kv_append8_*`, `attn_decode8_*`). `--prefix N`: all sequences begin with the same N tokens, which are
taken once and attended to together (`attn_shared_*`). `--turns N`: prompts come in N parts, each of which attends to what the cache holds of
the ones before (`kv_read_*`). `--sandwich`: norms with weights before and after both blocks, gates and a residual scale (`add_norm_*`).
"""
import argparse
import contextlib
import math
import sys

import torch

import fsw_weights

MOST_ROWS = 1 << 20  # of a call


class PagedCache:
    """Keys and values of one layer in pages of `page` tokens, and which pages each sequence has. Pages are handed out as
    tokens arrive; the table and the lengths are kept on the device, where the kernels read them."""

    def __init__(self, seqs, longest, kv_heads, channels, page, dtype, device, eight=False, prefix=0):
        """eight: e4m3 elements and their rows' scales. prefix: tokens that all sequences begin with, whole pages; longest, lengths and pages are of a
        sequence's own tokens behind them."""
        if prefix % page:
            raise ValueError("a shared prefix of %d tokens does not fill pages of %d" % (prefix, page))
        per_seq, shared = -(-longest // page), prefix // page
        self.page, self.longest, self.device, self.eight, self.prefix = page, longest, device, eight, prefix
        cells = (seqs * per_seq + shared, kv_heads, page)
        self.k = torch.empty(*cells, channels, dtype=torch.float8_e4m3fn if eight else dtype, device=device)
        self.v = torch.empty_like(self.k)
        self.arrays = [self.k, self.v]
        if eight:
            self.arrays += [torch.empty(cells, dtype=torch.float8_e8m0fnu, device=device) for _ in range(2)]
        self.free = list(range(seqs * per_seq + shared))
        self.prefix_pages = [self.free.pop() for _ in range(shared)]
        self.pages = [[] for _ in range(seqs)]
        self.lengths = [0] * seqs
        self.per_seq = per_seq

    def prefix_slots(self):
        """Positions and slots of the shared tokens."""
        slots = [p * self.page + t for p in self.prefix_pages for t in range(self.page)]
        return self._int32(range(self.prefix)), self._int32(slots)

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
                positions.append(self.prefix + t)
                slots.append(self.pages[b][t // self.page] * self.page + t % self.page)
            self.lengths[b] += n
        return self._int32(positions), self._int32(slots)

    @contextlib.contextmanager
    def growing(self, counts):
        """grow() for the length of a block: what is raised inside, a refused call say, gives the tokens' places back, so that the cache still has the
        tokens that it had."""
        lengths, pages = list(self.lengths), [len(p) for p in self.pages]
        try:
            yield self.grow(counts)
        except BaseException:
            self.lengths = lengths
            for own, n in zip(self.pages, pages):
                while len(own) > n:
                    self.free.append(own.pop())
            raise

    def table(self):
        """(block table, lengths, longest) for attn_decode."""
        return (self._int32([p + [0] * (self.per_seq - len(p)) for p in self.pages]), self._int32(self.lengths), max(self.lengths))

    def whole_table(self):
        """Pages of every sequence from its first token on, those of the prefix among them, for kv_read."""
        return self._int32([self.prefix_pages + p + [0] * (self.per_seq - len(p)) for p in self.pages])

    def _int32(self, values):
        return torch.tensor(list(values), dtype=torch.int32).to(self.device)


class DecoderLayer:
    def __init__(self, d, ff, heads, kv_heads, longest, dtype=torch.bfloat16, device="cuda:0", seed=0, sandwich=False):
        import fused_mlp_module as m
        name = "bf16" if dtype == torch.bfloat16 else "fp16"
        self.append, self.decode, self.prompt, self.project, self.mlp = (
            getattr(m, op + name) for op in ("kv_append_", "attn_decode_", "attn_prompt_", "swiglu_down_", "fused_swiglu_mlp_"))
        self.append8, self.decode8, self.shared, self.shared8, self.read, self.read8, self.add_norm, self.rms_norm = (
            getattr(m, op + name) for op in ("kv_append8_", "attn_decode8_", "attn_shared_", "attn_shared8_", "kv_read_", "kv_read8_", "add_norm_",
                                             "rms_norm_"))
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
        self.sandwich = sandwich
        if sandwich:  # weights of the norms before and after attention and MLP, and both gates
            vectors = (1 + 0.1 * torch.randn(6, d, generator=gen)).to(dtype).to(device)
            self.before_attn, self.after_attn, self.before_mlp, self.after_mlp, self.attn_gate, self.mlp_gate = vectors
            self.residual_scale = 0.5

    @staticmethod
    def norm(x):
        y = x.float()
        return (y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-5)).to(x.dtype)

    def _qkv(self, x):
        h = self.rms_norm(x, self.before_attn) if self.sandwich else self.norm(x)
        rows = self.project(h, self.w_qkv).view(x.shape[0], self.heads + 2 * self.kv_heads, self.channels)
        return rows.split([self.heads, self.kv_heads, self.kv_heads], 1)

    def _finish(self, x, attended):
        y = self.project(attended.flatten(1), self.w_out)
        if self.sandwich:
            x, h = self.add_norm(x, y, self.attn_gate, self.after_attn, self.before_mlp, self.residual_scale)
            return self.add_norm(x, self.mlp(h, self.w13, self.w2), self.mlp_gate, self.after_mlp, None, self.residual_scale)[0]
        x = x + y
        return x + self.mlp(self.norm(x), self.w13, self.w2)

    def _append(self, q, k, v, positions, slots, cache):
        """Rotated queries, and keys and values as later tokens will see them. Own tokens' positions go on behind the prefix's: a cache for as many tokens as
        the layer has angles, and a prefix beside them, would come to positions that have none, and keys that are NaN."""
        reach = cache.prefix + max(cache.lengths)
        if reach > self.cos_sin.shape[0]:
            raise ValueError("%d tokens in a row, the layer was made for %d" % (reach, self.cos_sin.shape[0]))
        if cache.eight:
            return self.append8(q, k, v, self.cos_sin, positions, slots, *cache.arrays)
        return (*self.append(q, k, v, self.cos_sin, positions, slots, cache.k, cache.v), v)

    def _prompts(self, x, lengths, positions, slots, cache):
        q, k, v = self._append(*self._qkv(x), positions, slots, cache)
        starts = self._starts(lengths, x.device)
        return self._finish(x, self.prompt(q, k, v, starts, starts, self.channels ** -0.5))

    @staticmethod
    def _starts(lengths, device):
        starts = [0]
        for n in lengths:
            starts.append(starts[-1] + n)
        return torch.tensor(starts, dtype=torch.int32).to(device)

    def prefill(self, x, lengths, cache):
        """x: the packed rows of new sequences' prompts."""
        for b, n in enumerate(lengths):
            if n and cache.lengths[b]:
                raise ValueError("sequence %d has tokens in the cache already" % b)
        if cache.prefix:
            raise ValueError("prompts behind a shared prefix extend what the cache holds: extend()")
        with cache.growing(lengths) as (positions, slots):
            return self._prompts(x, lengths, positions, slots, cache)

    def prefill_shared(self, x, cache):
        """x: the rows of the prefix that all of the cache's sequences begin with."""
        return self._prompts(x, [cache.prefix], *cache.prefix_slots(), cache)

    def extend(self, x, lengths, cache):
        """x: the packed rows of prompts that continue what the cache holds of their sequences. Every sequence's tokens are packed, those of the prefix
        once for each, so all sequences together have at most MOST_ROWS of them."""
        with cache.growing(lengths) as (positions, slots):
            held = [cache.prefix + n for n in cache.lengths]
            if sum(held) > MOST_ROWS:
                raise ValueError("%d cached tokens of all sequences together, kv_read takes %d" % (sum(held), MOST_ROWS))
            q = self._append(*self._qkv(x), positions, slots, cache)[0]
            starts = self._starts(held, x.device)
            k, v = (self.read8 if cache.eight else self.read)(*cache.arrays, cache.whole_table(), starts, sum(held))
            return self._finish(x, self.prompt(q, k, v, self._starts(lengths, x.device), starts, self.channels ** -0.5))

    def step(self, x, cache):
        """x: one row per sequence, its next token."""
        with cache.growing([1] * x.shape[0]) as (positions, slots):
            q = self._append(*self._qkv(x), positions, slots, cache)[0]
            table, lengths, longest = cache.table()
            own = (table, lengths, longest, self.channels ** -0.5)
            if cache.prefix:
                pages = cache._int32(cache.prefix_pages)
                return self._finish(x, (self.shared8 if cache.eight else self.shared)(q, *cache.arrays, pages, cache.prefix, *own))
            return self._finish(x, (self.decode8 if cache.eight else self.decode)(q, *cache.arrays, *own))


def run(d=1024, ff=2816, heads=16, kv_heads=4, prompts=(37, 5, 130), steps=9, page=16, dtype=torch.bfloat16, seed=0, eight=False, prefix=0, turns=1,
        sandwich=False):
    """Largest difference, over the root mean square of the outputs, between tokens decoded one by one and the same tokens
    inside their whole sequences."""
    if turns < 1:
        raise ValueError("prompts come in one part at least, not in %d" % turns)
    longest = prefix + max(prompts) + steps
    layer = DecoderLayer(d, ff, heads, kv_heads, longest, dtype, seed=seed, sandwich=sandwich)
    gen = torch.Generator().manual_seed(seed + 2)
    whole = [torch.randn(n + steps, d, generator=gen).to(dtype).to("cuda:0") for n in prompts]
    first = torch.randn(prefix, d, generator=gen).to(dtype).to("cuda:0")

    def new_cache(shared):
        return PagedCache(len(prompts), longest, kv_heads, d // heads, page, dtype, "cuda:0", eight, shared)

    cache = new_cache(prefix)
    if prefix:
        layer.prefill_shared(first, cache)
    for turn in range(turns):  # the prompts' parts of about the same length
        parts = [x[n * turn // turns:n * (turn + 1) // turns] for x, n in zip(whole, prompts)]
        take = layer.prefill if turn == 0 and not prefix else layer.extend
        take(torch.cat(parts), [p.shape[0] for p in parts], cache)
    decoded = [layer.step(torch.stack([x[n + i] for x, n in zip(whole, prompts)]), cache) for i in range(steps)]
    lengths = [prefix + n + steps for n in prompts]
    want = layer.prefill(torch.cat([torch.cat([first, x]) for x in whole]), lengths, new_cache(0)).split(lengths)
    worst = 0.0
    for b, n in enumerate(prompts):
        got, ref = torch.stack([y[b] for y in decoded]).float(), want[b][prefix + n:].float()
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
    ap.add_argument("--eight", action="store_true", help="a cache of 8 bits")
    ap.add_argument("--prefix", type=int, default=0, help="tokens that all sequences begin with, whole pages")
    ap.add_argument("--turns", type=int, default=1, help="parts that prompts come in")
    ap.add_argument("--sandwich", action="store_true", help="norms before and after both blocks, with gates")
    args = ap.parse_args(argv)
    if not torch.cuda.is_available():
        sys.exit("decoder_layer.py needs the GPU: the extension has no CPU path")
    worst = run(args.d, args.ff, args.heads, args.kv_heads, tuple(args.prompts), args.steps, args.page, eight=args.eight, prefix=args.prefix,
                turns=args.turns, sandwich=args.sandwich)
    print("%d prompts, %d steps each: decoded tokens differ from whole sequences by %.1e of the outputs' size" %
          (len(args.prompts), args.steps, worst))


if __name__ == "__main__":
    main()
