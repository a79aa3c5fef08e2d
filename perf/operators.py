"""Performance cases of the attention operators beside the SwiGLU forward: the other half of a decoder layer being served.

  op "append"   rotates the queries and keys of T new tokens by their positions and appends keys and values to a paged cache
  op "decode"   attention of one new token per sequence over the paged cache
  op "prompt"   causal attention of whole prompts, packed one behind the other

Hq query heads share Hkv key-value heads of D channels. Elements are bf16 or fp16; tables of cosines and sines are float32,
positions, slots, lengths, offsets and page numbers are int32. The cache is [pages, Hkv, page, D] for keys and for values.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _append(name, dtype, T, Hq, Hkv, D, rot, interleaved, page):
    return {"name": name, "op": "append", "dtype": dtype, "T": T, "Hq": Hq, "Hkv": Hkv, "D": D, "rot": rot,
            "interleaved": interleaved, "page": page}


def _attend(name, op, dtype, B, shortest, longest, Hq, Hkv, D, mix, page=0):
    case = {"name": name, "op": op, "dtype": dtype, "B": B, "shortest": shortest, "longest": longest, "Hq": Hq, "Hkv": Hkv,
            "D": D, "mix": mix}
    if op == "decode":
        case["page"] = page
    return case


def listed():
    return [
        # one new token of one sequence, a layer of width 4096: launches and latency count
        _append("append_1", "bf16", 1, 32, 8, 128, 128, False, 16),
        # a few short prompts, heads of 96 channels of which half are rotated, pairs side by side, odd pages
        _append("append_333_fp16", "fp16", 333, 20, 4, 96, 48, True, 24),
        # a full prefill batch, a layer of width 8192
        _append("append_8192", "bf16", 8192, 64, 8, 128, 128, False, 64),
        # one sequence, a few hundred tokens in: the shortest attention of a decode step
        _attend("decode_1", "decode", "bf16", 1, 300, 300, 32, 8, 128, 1, 16),
        # one sequence at the end of a very long context: its length has to be spread over the card
        _attend("decode_1_long", "decode", "bf16", 1, 131071, 131071, 64, 8, 128, 2, 64),
        # a small layer's decode batch, heads of 64 channels
        _attend("decode_16_d64", "decode", "bf16", 16, 1, 1500, 16, 4, 64, 3, 32),
        # a decode batch in the midst of serving, every length, as many key-value heads as query heads
        _attend("decode_40_mixed_fp16", "decode", "fp16", 40, 1, 4096, 40, 40, 128, 4, 16),
        # a large decode batch of sequences of about the same length, a layer of width 8192
        _attend("decode_128", "decode", "bf16", 128, 1700, 2300, 64, 8, 128, 5, 64),
        # one very short prompt through a small layer
        _attend("prompt_24", "prompt", "bf16", 1, 24, 24, 16, 4, 64, 6),
        # a packed batch of prompts of every length, one token among them, as many key-value heads as query heads
        _attend("prompt_13_ragged_fp16", "prompt", "fp16", 13, 1, 777, 40, 40, 128, 7),
        # an ordinary prompt through a layer of width 4096
        _attend("prompt_2000", "prompt", "bf16", 1, 2000, 2000, 32, 8, 128, 8),
        # a long prompt through a layer of width 8192
        _attend("prompt_8192", "prompt", "bf16", 1, 8192, 8192, 64, 8, 128, 9),
    ]


def lengths(case):
    """Tokens of each sequence: the shortest and the longest are among them, the others spread over the logarithm between."""
    B, lo, hi = case["B"], case["shortest"], case["longest"]
    rng = random.Random(case["mix"])
    out = [min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))) for _ in range(B)]
    out[0] = hi
    if B > 1:
        out[-1] = lo
    rng.shuffle(out)
    return out


MOST_PAIRS = 64 * 8192 * 8192 * 128     # score entries times channels of the largest prompt
MOST_CACHE = 40 * 4096 * 40 * 128       # keys times channels of the largest decode batch, padded to its longest sequence
MOST_APPEND = 8192 * 80 * 128           # elements of q, k and v of the largest append


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "prompt", "prompt"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    D = rng.choice([64, 80, 112, 128, 128, 128, 256])
    Hkv = rng.choice([1, 2, 4, 5, 8, 8, 16, 32])
    Hq = Hkv * rng.choice([1, 2, 4, 4, 7, 8] if Hkv <= 8 else [1, 2])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128, 256])
    mix = rng.randrange(1, 1 << 20)
    if op == "append":
        T = _log(rng, 1, min(16384, MOST_APPEND // ((Hq + 2 * Hkv) * D)))
        rot = rng.choice([D, D, D // 2])
        return {k: v for k, v in _append("", dtype, T, Hq, Hkv, D, rot, rng.random() < 0.3, page).items() if k != "name"}
    if op == "decode":
        B = _log(rng, 1, 128)
        longest = _log(rng, 1, min(131072, MOST_CACHE // (B * Hkv * D)))
        shortest = longest if B == 1 else _log(rng, 1, longest)
    else:
        B = _log(rng, 1, 24)
        longest = _log(rng, 1, min(8192, math.isqrt(MOST_PAIRS // (B * Hq * D))))
        shortest = longest if B == 1 else _log(rng, 1, longest)
    return {k: v for k, v in _attend("", op, dtype, B, shortest, longest, Hq, Hkv, D, mix, page).items() if k != "name"}


def _seeded(seed):
    """A generator of normal values on the GPU and one of whole numbers on the host, both from the seed."""
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, dtype, scale=1.0):
        return torch.empty(shape, dtype=dtype, device=dev).normal_(0.0, scale, generator=g)

    return dev, normal, random.Random(seed)


def _int32(values, dev):
    return torch.tensor(values, dtype=torch.int32).to(dev)


def prepare(case, seed):
    """What a layer has in hand before the call. Queries, keys and values lie in one row per token as a fused projection
    leaves them (what the rotation has written lies by itself); pages are handed out in no order, some are free."""
    dev, normal, rng = _seeded(seed)
    dtype, Hq, Hkv, D = DTYPES[case["dtype"]], case["Hq"], case["Hkv"], case["D"]
    st = {"op": case["op"], "dtype": case["dtype"], "scale": 1.0 / math.sqrt(D)}
    if case["op"] == "append":
        T, page, rot = case["T"], case["page"], case["rot"]
        qkv = normal(T, (Hq + 2 * Hkv) * D, dtype=dtype).view(T, Hq + 2 * Hkv, D)
        st["q"], st["k"], st["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
        rows = T + 4096
        pages = -(-T // page) + 8
        st["k_cache"] = normal(pages, Hkv, page, D, dtype=dtype)
        st["v_cache"] = normal(pages, Hkv, page, D, dtype=dtype)
        angle = torch.outer(torch.arange(rows, dtype=torch.float64),
                            10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot))
        st["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).float().to(dev)
        first = rng.randrange(4096)
        order = rng.sample(range(pages), pages)
        st["positions"] = _int32([first + t for t in range(T)], dev)
        st["slots"] = _int32([order[t // page] * page + t % page for t in range(T)], dev)
        st["interleaved"] = case["interleaved"]
        return st
    lens = lengths(case)
    if case["op"] == "decode":
        page = case["page"]
        used = [-(-n // page) for n in lens]
        pages = sum(used) + 8
        st["k_cache"] = normal(pages, Hkv, page, D, dtype=dtype)
        st["v_cache"] = normal(pages, Hkv, page, D, dtype=dtype)
        order = iter(rng.sample(range(pages), pages))
        width = max(used)
        st["block_table"] = _int32([[next(order) if i < n else 0 for i in range(width)] for n in used], dev)
        st["lengths"], st["max_len"] = _int32(lens, dev), max(lens)
        qkv = normal(len(lens), (Hq + 2 * Hkv) * D, dtype=dtype, scale=2.0).view(len(lens), Hq + 2 * Hkv, D)
        st["q"] = qkv[:, :Hq]
        return st
    T = sum(lens)
    qkv = normal(T, (Hq + 2 * Hkv) * D, dtype=dtype).view(T, Hq + 2 * Hkv, D)
    st["q"], st["k"], st["v"] = normal(T, Hq, D, dtype=dtype, scale=2.0), normal(T, Hkv, D, dtype=dtype), qkv[:, Hq + Hkv:]
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    st["starts"], st["max_len"] = _int32(starts, dev), max(lens)
    return st


def _rotate(x, cos, sin, interleaved):
    """x [T, H, D] in 32 bits; cos, sin [T, 1, R / 2]: the first R channels are turned in pairs, the others stay."""
    half = cos.shape[-1]
    pairs, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = pairs[..., 0::2], pairs[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = pairs[..., :half], pairs[..., half:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, rest], -1)


def _weights(scores, seen):
    """softmax over the last axis of the entries that are seen; a row that sees none weighs nothing."""
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    return p.div_(total.masked_fill(total == 0.0, 1.0))


def _plain_append(st):
    half = st["cos_sin"].shape[1] // 2
    cs = st["cos_sin"][st["positions"].long()].unsqueeze(1)
    cos, sin = cs[..., :half], cs[..., half:]
    dtype, page = st["q"].dtype, st["k_cache"].shape[2]
    q = _rotate(st["q"].float(), cos, sin, st["interleaved"]).to(dtype)
    k = _rotate(st["k"].float(), cos, sin, st["interleaved"]).to(dtype)
    slot = st["slots"].long()
    st["k_cache"][slot // page, :, slot % page] = k
    st["v_cache"][slot // page, :, slot % page] = st["v"]
    return {"q": q, "k": k, "k_cache": st["k_cache"], "v_cache": st["v_cache"]}


def _plain_decode(st):
    q, table, n = st["q"], st["block_table"].long(), st["max_len"]
    (B, Hq, D), Hkv = q.shape, st["k_cache"].shape[1]

    def rows(cache):  # [B, Hkv, longest, D]
        return cache[table].permute(0, 2, 1, 3, 4).reshape(B, Hkv, -1, D)[:, :, :n].float()

    scores = torch.matmul(q.float().view(B, Hkv, Hq // Hkv, D), rows(st["k_cache"]).transpose(2, 3)) * st["scale"]
    seen = torch.arange(n, device=q.device) < st["lengths"].view(B, 1, 1, 1)
    return torch.matmul(_weights(scores, seen), rows(st["v_cache"])).view(B, Hq, D).to(q.dtype)


def _plain_prompt(st):
    q, k, v, starts, n = st["q"], st["k"], st["v"], st["starts"].long(), st["max_len"]
    (T, Hq, D), Hkv, B = q.shape, k.shape[1], starts.numel() - 1
    at = torch.arange(n, device=q.device)
    lens = starts[1:] - starts[:-1]
    index = (starts[:-1, None] + at).clamp(max=T - 1)  # [B, longest]: a token's row, some other row behind the end

    def heads(x):  # [B, heads, longest, D]
        return x[index].permute(0, 2, 1, 3).float()

    qs = heads(q).reshape(B, Hkv, (Hq // Hkv) * n, D)
    scores = torch.matmul(qs, heads(k).transpose(2, 3)).mul_(st["scale"]).view(B, Hkv, Hq // Hkv, n, n)
    seen = (at <= at[:, None]) & (at < lens[:, None, None])  # [B, query, key]
    p = _weights(scores, seen[:, None, None]).view(B, Hkv, -1, n)
    o = torch.matmul(p, heads(v)).view(B, Hq, n, D).permute(0, 2, 1, 3).to(q.dtype)
    seq = torch.searchsorted(starts[1:], torch.arange(T, device=q.device), right=True)
    return o[seq, torch.arange(T, device=q.device) - starts[seq]]


def _module():
    path = os.path.abspath("fused-swiglu_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import fused_mlp_module
    return fused_mlp_module


def run(state):
    st = state
    if not own:
        return {"append": _plain_append, "decode": _plain_decode, "prompt": _plain_prompt}[st["op"]](st)
    m, bf16 = _module(), st["dtype"] == "bf16"
    if st["op"] == "append":
        f = m.kv_append_bf16 if bf16 else m.kv_append_fp16
        q, k = f(st["q"], st["k"], st["v"], st["cos_sin"], st["positions"], st["slots"], st["k_cache"], st["v_cache"],
                 st["interleaved"])
        return {"q": q, "k": k, "k_cache": st["k_cache"], "v_cache": st["v_cache"]}
    if st["op"] == "decode":
        f = m.attn_decode_bf16 if bf16 else m.attn_decode_fp16
        return f(st["q"], st["k_cache"], st["v_cache"], st["block_table"], st["lengths"], st["max_len"], st["scale"])
    f = m.attn_prompt_bf16 if bf16 else m.attn_prompt_fp16
    return f(st["q"], st["k"], st["v"], st["starts"], st["starts"], st["scale"])


def work(case):
    """Inputs once, outputs once. Multiplications and additions of the two products over the keys that each query sees."""
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    if case["op"] == "append":
        T = case["T"]
        return {"bytes": T * (2 * D * (2 * Hq + 5 * Hkv) + 4 * case["rot"] + 8), "flops": 3 * T * (Hq + Hkv) * case["rot"]}
    lens = lengths(case)
    if case["op"] == "decode":
        pages = sum(-(-n // case["page"]) for n in lens)
        return {"bytes": 4 * D * Hkv * sum(lens) + 4 * D * Hq * len(lens) + 4 * (pages + len(lens)),
                "flops": 4 * D * Hq * sum(lens)}
    return {"bytes": 4 * D * (Hq + Hkv) * sum(lens), "flops": 4 * D * Hq * sum(n * (n + 1) // 2 for n in lens)}


def exact(case, seed):
    """The definitions in float64, sequence by sequence. Pages that no token was appended to keep what they held."""
    st = prepare(case, seed)
    if case["op"] == "append":
        page, pos, slot = case["page"], st["positions"].long(), st["slots"].long()
        angles = st["cos_sin"].double()[pos]
        half = angles.shape[1] // 2
        turn = torch.complex(angles[:, :half], angles[:, half:])[:, None]

        def turned(x):
            x = x.double().clone()
            re, im = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["interleaved"] else (slice(0, half), slice(half, 2 * half))
            z = torch.complex(x[..., re], x[..., im]) * turn
            x[..., re], x[..., im] = z.real, z.imag
            return x

        out = {"q": turned(st["q"]), "k": turned(st["k"]), "k_cache": st["k_cache"].double(), "v_cache": st["v_cache"].double()}
        for name, rows in (("k_cache", out["k"]), ("v_cache", st["v"].double())):
            flat = out[name].transpose(1, 2).reshape(-1, case["Hkv"], case["D"])
            flat[slot] = rows
            out[name] = flat.view(-1, page, case["Hkv"], case["D"]).transpose(1, 2).contiguous()
        return out
    group, parts = case["Hq"] // case["Hkv"], []
    for b, n in enumerate(lengths(case)):
        if case["op"] == "decode":
            pages = st["block_table"][b, :-(-n // case["page"])].long()
            k, v = (c[pages].transpose(0, 1).reshape(case["Hkv"], -1, case["D"])[:, :n] for c in (st["k_cache"], st["v_cache"]))
            q, future = st["q"][b:b + 1], None
        else:
            rows = slice(int(st["starts"][b]), int(st["starts"][b]) + n)
            q, k, v = st["q"][rows], st["k"][rows].transpose(0, 1), st["v"][rows].transpose(0, 1)
            future = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1)
        o = torch.empty(q.shape, dtype=torch.float64, device=q.device)
        for h in range(case["Hq"]):
            s = (q[:, h].double() @ k[h // group].double().t()) * st["scale"]
            if future is not None:
                s = s.masked_fill(future, -math.inf)
            o[:, h] = torch.softmax(s, -1) @ v[h // group].double()
        parts.append(o)
    return torch.cat(parts)
