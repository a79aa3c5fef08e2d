"""Performance cases of a served decoder layer's other operators: an 8-bit cache, a prefix that a batch shares, norms around a block.

  op "append8"  rotates the queries and keys of T new tokens and appends keys and values to a paged cache of 8-bit elements
  op "read"     the keys and values of some sequences out of their pages, packed one behind the other (8- or 16-bit cache)
  op "decode8"  attention of one new token per sequence over the 8-bit cache
  op "shared"   attention of one new token per sequence whose keys are a prefix that all share and their own (8- or 16-bit cache)
  op "norm"     x' = x + scale * gate * norm(y), h = norm(x'): around a block of the layer

Hq query heads share Hkv key-value heads of D channels. Rows are bf16 or fp16. The 8-bit cache holds float8_e4m3fn elements
[pages, Hkv, page, D] and one power of two per row, float8_e8m0fnu [pages, Hkv, page]: a row stands for element * scale, with the
least scale under which the row's largest element is at most 448.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _append(name, dtype, T, Hq, Hkv, D, rot, interleaved, page):
    return {"name": name, "op": "append8", "dtype": dtype, "T": T, "Hq": Hq, "Hkv": Hkv, "D": D, "rot": rot,
            "interleaved": interleaved, "page": page}


def _cached(name, op, dtype, bits, B, shortest, longest, Hq, Hkv, D, page, mix, prefix=0):
    case = {"name": name, "op": op, "dtype": dtype, "bits": bits, "B": B, "shortest": shortest, "longest": longest, "Hkv": Hkv,
            "D": D, "page": page, "mix": mix}
    if op != "read":
        case["Hq"] = Hq
    if op == "shared":
        case["prefix"] = prefix
    return case


def _norm(name, dtype, T, d, post, gate):
    return {"name": name, "op": "norm", "dtype": dtype, "T": T, "d": d, "post": post, "gate": gate}


def listed():
    return [
        # one new token of one sequence, a layer of width 4096: launches and latency count
        _append("append8_1", "bf16", 1, 32, 8, 128, 128, False, 16),
        # a full prefill batch, a layer of width 8192
        _append("append8_8192", "bf16", 8192, 64, 8, 128, 128, False, 64),
        # earlier tokens of three short conversations whose next prompts are to see them, odd pages, a 16-bit cache
        _cached("read_3_fp16", "read", "fp16", 16, 3, 1, 700, 0, 4, 96, 24, 1),
        # the same for a batch of long ones out of the 8-bit cache
        _cached("read8_24", "read", "bf16", 8, 24, 100, 8192, 0, 8, 128, 64, 2),
        # the first tokens of a small batch: the shortest attention of a decode step
        _cached("decode8_3_fp16", "decode8", "fp16", 8, 3, 24, 700, 20, 4, 96, 24, 3),
        # one sequence at the end of a very long context: its length has to be spread over the card
        _cached("decode8_1_long", "decode8", "bf16", 8, 1, 131071, 131071, 64, 8, 128, 64, 4),
        # a large decode batch of sequences of about the same length, a layer of width 8192
        _cached("decode8_128", "decode8", "bf16", 8, 128, 1700, 2300, 64, 8, 128, 64, 5),
        # a few sequences behind a short instruction, as many key-value heads as query heads
        _cached("shared_6_fp16", "shared", "fp16", 16, 6, 1, 40, 40, 40, 128, 16, 6, 333),
        # a decode batch behind a long document, a layer of width 4096
        _cached("shared_64", "shared", "bf16", 16, 64, 1, 900, 32, 8, 128, 64, 7, 16384),
        # a large decode batch behind long instructions in the 8-bit cache, a layer of width 8192
        _cached("shared8_200", "shared", "bf16", 8, 200, 1, 1500, 64, 8, 128, 16, 8, 8000),
        # one token between two blocks of a layer of width 4096: launches and latency count
        _norm("norm_1", "bf16", 1, 4096, True, "channel"),
        # a full prefill batch, a layer of width 8192, with a gate of its own for every token
        _norm("norm_8192", "bf16", 8192, 8192, True, "token"),
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


MOST_APPEND = 8192 * 80 * 128                # elements of q, k and v of the largest append
MOST_READ = 24 * 4096 * 8 * 128              # keys times channels of the largest read
MOST_CACHE = 128 * 2300 * 8 * 128            # of the largest decode batch, padded to its longest sequence
MOST_PAIRS = 64 * 200 * (8000 + 1500) * 128  # score entries times channels of the largest shared attention
MOST_NORM = 8192 * 8192


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi)))))))


def draw(rng):
    op = rng.choice(["append8", "read", "decode8", "decode8", "shared", "shared", "norm"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    D = rng.choice([64, 80, 96, 112, 128, 128, 128, 256])
    Hkv = rng.choice([1, 2, 4, 5, 8, 8, 16, 32])
    Hq = Hkv * rng.choice([1, 2, 4, 4, 7, 8] if Hkv <= 8 else [1, 2])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128, 256])
    bits = 8 if op == "decode8" else rng.choice([8, 16])
    mix, prefix = rng.randrange(1, 1 << 20), 0
    if op == "append8":
        T = _log(rng, 1, min(16384, MOST_APPEND // ((Hq + 2 * Hkv) * D)))
        case = _append("", dtype, T, Hq, Hkv, D, rng.choice([D, D, D // 2]), rng.random() < 0.3, page)
    elif op == "norm":
        d = 8 * _log(rng, 16, 2048)
        case = _norm("", dtype, _log(rng, 1, min(16384, MOST_NORM // d)), d, rng.random() < 0.6,
                     rng.choice(["none", "channel", "token"]))
    else:
        B = _log(rng, 1, 32 if op == "read" else 256 if op == "shared" else 128)
        most = MOST_READ if op == "read" else MOST_CACHE
        longest = _log(rng, 1, min(4096 if op == "shared" else 131072, most // (B * Hkv * D)))
        shortest = longest if B == 1 else _log(rng, 1, longest)
        if op == "shared":
            prefix = _log(rng, 1, min(65536, most // (Hkv * D), max(1, MOST_PAIRS // (Hq * B * D) - longest)))
        case = _cached("", op, dtype, bits, B, shortest, longest, Hq, Hkv, D, page, mix, prefix)
    return {k: v for k, v in case.items() if k != "name"}


def _seeded(seed):
    """A generator of normal values on the GPU and one of whole numbers on the host, both from the seed."""
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, dtype, scale=1.0):
        return torch.empty(shape, dtype=dtype, device=dev).normal_(0.0, scale, generator=g)

    return dev, normal, random.Random(seed)


def _int32(values, dev):
    return torch.tensor(values, dtype=torch.int32).to(dev)


def _scales(x):
    """Exponents of a row's scale: the least e with max |x| <= 448 * 2^e, 448 = 0.875 * 2^9."""
    m, ex = torch.frexp(x.abs().amax(-1))
    return torch.where(m == 0, torch.zeros_like(ex), (ex - 9 + (m > 0.875)).clamp(min=-126))


def _power(e):
    """2^e in 32 bits, from its bits: a library's power is not always exact."""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _quantised(x):
    """Elements and scales of rows x in 32 or 64 bits. Elements have four significant bits and steps of 2^-9 at least."""
    e = _scales(x)
    y = x * _power(-e)[..., None]
    step = _power(torch.frexp(y)[1].clamp(min=-5) - 4)
    codes = (torch.round(y / step) * step).float().to(torch.float8_e4m3fn)
    return codes, (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _cache(case, pages, normal):
    """Keys and values of a cache, and the scales of both where it has 8 bits."""
    shape = (pages, case["Hkv"], case["page"], case["D"])
    if case.get("bits", 8) == 16:
        return [normal(*shape, dtype=DTYPES[case["dtype"]]) for _ in range(2)] + [None, None]
    (k, ks), (v, vs) = (_quantised(normal(*shape, dtype=torch.float32)) for _ in range(2))
    return [k, v, ks, vs]


def prepare(case, seed):
    """What a layer has in hand before the call. Queries, keys and values lie in one row per token as a fused projection
    leaves them; pages are handed out in no order, some are free."""
    dev, normal, rng = _seeded(seed)
    dtype = DTYPES[case["dtype"]]
    st = {"op": case["op"], "dtype": case["dtype"]}
    if case["op"] == "norm":
        T, d = case["T"], case["d"]
        st["x"], st["y"] = normal(T, d, dtype=dtype, scale=2.0), normal(T, d, dtype=dtype)
        st["gate"] = {"none": lambda: None, "channel": lambda: normal(d, dtype=dtype), "token": lambda: normal(T, d, dtype=dtype)}[case["gate"]]()
        st["post"] = normal(d, dtype=dtype, scale=0.1).add_(1.0) if case["post"] else None
        st["pre"] = normal(d, dtype=dtype, scale=0.1).add_(1.0)
        st["scale"], st["eps"] = 0.5, 1e-5
        return st
    Hkv, D, page = case["Hkv"], case["D"], case["page"]
    st["scale"], st["bits"] = 1.0 / math.sqrt(D), case.get("bits", 8)
    if case["op"] == "append8":
        T, Hq, rot = case["T"], case["Hq"], case["rot"]
        qkv = normal(T, (Hq + 2 * Hkv) * D, dtype=dtype).view(T, Hq + 2 * Hkv, D)
        st["q"], st["k"], st["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
        pages = -(-T // page) + 8
        st["cache"] = _cache(case, pages, normal)
        angle = torch.outer(torch.arange(T + 4096, dtype=torch.float64),
                            10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot))
        st["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).float().to(dev)
        first = rng.randrange(4096)
        order = rng.sample(range(pages), pages)
        st["positions"] = _int32([first + t for t in range(T)], dev)
        st["slots"] = _int32([order[t // page] * page + t % page for t in range(T)], dev)
        st["interleaved"] = case["interleaved"]
        return st
    lens = lengths(case)
    used, shared = [-(-n // page) for n in lens], -(-case.get("prefix", 0) // page)
    pages = sum(used) + shared + 8
    st["cache"] = _cache(case, pages, normal)
    order = iter(rng.sample(range(pages), pages))
    st["block_table"] = _int32([[next(order) if i < n else 0 for i in range(max(used))] for n in used], dev)
    if case["op"] == "read":
        starts = [0]
        for n in lens:
            starts.append(starts[-1] + n)
        st["starts"], st["tokens"] = _int32(starts, dev), starts[-1]
        return st
    st["lengths"], st["max_len"], Hq = _int32(lens, dev), max(lens), case["Hq"]
    if case["op"] == "shared":
        st["prefix"], st["prefix_len"] = _int32([next(order) for _ in range(shared)], dev), case["prefix"]
    qkv = normal(len(lens), (Hq + 2 * Hkv) * D, dtype=dtype, scale=2.0).view(len(lens), Hq + 2 * Hkv, D)
    st["q"] = qkv[:, :Hq]
    return st


def _rotate(x, cos, sin, interleaved):
    """x [T, H, D]; cos, sin [T, 1, R / 2]: the first R channels are turned in pairs, the others stay."""
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
    """softmax over the last axis of the entries that are seen."""
    scores = scores.masked_fill_(~seen, -math.inf)
    p = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    return p.div_(p.sum(-1, keepdim=True))


def _values(codes, scales):
    return codes.float() if scales is None else codes.float() * scales.float()[..., None]


def _plain_append(st):
    half = st["cos_sin"].shape[1] // 2
    cs = st["cos_sin"][st["positions"].long()].unsqueeze(1)
    dtype, page = st["q"].dtype, st["cache"][0].shape[2]
    q = _rotate(st["q"].float(), cs[..., :half], cs[..., half:], st["interleaved"]).to(dtype)
    cs = cs.double()  # keys in 64 bits: a value next to the border of two elements falls on its own side
    k = _quantised(_rotate(st["k"].double(), cs[..., :half], cs[..., half:], st["interleaved"]))
    v = _quantised(st["v"].float())
    slot = st["slots"].long()
    for cache, rows in zip(st["cache"], (k[0], v[0], k[1], v[1])):
        cache[slot // page, :, slot % page] = rows
    return _appended(q, _values(*k).to(dtype), _values(*v).to(dtype), st)


def _appended(q, k, v, st):
    return {"q": q, "k": k, "v": v, "k_cache": st["cache"][0], "v_cache": st["cache"][1], "k_scale": st["cache"][2], "v_scale": st["cache"][3]}


def _plain_read(st):
    starts, page = st["starts"].long(), st["cache"][0].shape[2]
    t = torch.arange(st["tokens"], device=starts.device)
    seq = torch.searchsorted(starts[1:], t, right=True)
    at = t - starts[seq]
    pages = st["block_table"].long()[seq, at // page]
    k, v, ks, vs = (None if c is None else c[pages, :, at % page] for c in st["cache"])
    dtype = DTYPES[st["dtype"]]
    return {"k": _values(k, ks).to(dtype), "v": _values(v, vs).to(dtype)}


def _rows(pages, n, codes, scales):
    """[..., Hkv, n, D] in 32 bits of the pages [..., count]."""
    x = _values(codes[pages], None if scales is None else scales[pages]).transpose(-4, -3)
    return x.reshape(*x.shape[:-3], -1, x.shape[-1])[..., :n, :]


def _plain_decode(st):
    q, table, n = st["q"], st["block_table"].long(), st["max_len"]
    (B, Hq, D), (k, v, ks, vs) = q.shape, st["cache"]
    Hkv = k.shape[1]
    scores = torch.matmul(q.float().view(B, Hkv, Hq // Hkv, D), _rows(table, n, k, ks).transpose(2, 3)) * st["scale"]
    seen = torch.arange(n, device=q.device) < st["lengths"].view(B, 1, 1, 1)
    return torch.matmul(_weights(scores, seen), _rows(table, n, v, vs)).view(B, Hq, D).to(q.dtype)


def _plain_shared(st):
    q, table, n, P = st["q"], st["block_table"].long(), st["max_len"], st["prefix_len"]
    (B, Hq, D), (k, v, ks, vs) = q.shape, st["cache"]
    Hkv, prefix = k.shape[1], st["prefix"].long()
    group = Hq // Hkv
    qs = q.float().view(B, Hkv, group, D)
    first = torch.matmul(qs.transpose(0, 1).reshape(Hkv, B * group, D), _rows(prefix, P, k, ks).transpose(1, 2))
    first = first.view(Hkv, B, group, P).transpose(0, 1)
    scores = torch.cat([first, torch.matmul(qs, _rows(table, n, k, ks).transpose(2, 3))], -1).mul_(st["scale"])
    at = torch.arange(P + n, device=q.device) - P
    w = _weights(scores, at < st["lengths"].view(B, 1, 1, 1))
    o = torch.matmul(w[..., :P].transpose(0, 1).reshape(Hkv, B * group, P), _rows(prefix, P, v, vs))
    o = o.view(Hkv, B, group, D).transpose(0, 1) + torch.matmul(w[..., P:], _rows(table, n, v, vs))
    return o.reshape(B, Hq, D).to(q.dtype)


def _normed(x, eps):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)


def _plain_norm(st):
    dtype, b = st["x"].dtype, st["y"].float()
    if st["post"] is not None:
        b = _normed(b, st["eps"]) * st["post"].float()
    if st["gate"] is not None:
        b = b * st["gate"].float()
    x = st["x"].float() + st["scale"] * b
    return {"x": x.to(dtype), "h": (_normed(x, st["eps"]) * st["pre"].float()).to(dtype)}


def _module():
    path = os.path.abspath("fused-swiglu_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import fused_mlp_module
    return fused_mlp_module


def run(state):
    st = state
    if not own:
        return {"append8": _plain_append, "read": _plain_read, "decode8": _plain_decode, "shared": _plain_shared,
                "norm": _plain_norm}[st["op"]](st)
    m, name = _module(), st["dtype"]
    if st["op"] == "norm":
        x, h = getattr(m, "add_norm_" + name)(st["x"], st["y"], st["gate"], st["post"], st["pre"], st["scale"], st["eps"])
        return {"x": x, "h": h}
    eight, cache = st["bits"] == 8, [c for c in st["cache"] if c is not None]
    if st["op"] == "append8":
        return _appended(*getattr(m, "kv_append8_" + name)(st["q"], st["k"], st["v"], st["cos_sin"], st["positions"], st["slots"], *cache,
                                                           st["interleaved"]), st)
    if st["op"] == "read":
        f = getattr(m, ("kv_read8_" if eight else "kv_read_") + name)
        k, v = f(*cache, st["block_table"], st["starts"], st["tokens"])
        return {"k": k, "v": v}
    if st["op"] == "decode8":
        return getattr(m, "attn_decode8_" + name)(st["q"], *cache, st["block_table"], st["lengths"], st["max_len"], st["scale"])
    f = getattr(m, ("attn_shared8_" if eight else "attn_shared_") + name)
    return f(st["q"], *cache, st["prefix"], st["prefix_len"], st["block_table"], st["lengths"], st["max_len"], st["scale"])


def work(case):
    """Inputs once, outputs once; a prefix once for all. Multiplications and additions of the products over the keys that each query sees."""
    if case["op"] == "norm":
        n, d = case["T"] * case["d"], case["d"]
        gate = {"none": 0, "channel": d, "token": n}[case["gate"]]
        return {"bytes": 2 * (4 * n + gate + d * (2 if case["post"] else 1)), "flops": n * (12 if case["post"] else 8)}
    Hkv, D = case["Hkv"], case["D"]
    row = 2 * Hkv * (D + 1 if case.get("bits", 8) == 8 else 2 * D)  # a token's keys and values in the cache
    if case["op"] == "append8":
        T, Hq = case["T"], case["Hq"]
        return {"bytes": T * (4 * D * (Hq + 2 * Hkv) + row + 4 * case["rot"] + 8), "flops": T * (3 * (Hq + Hkv) * case["rot"] + 6 * Hkv * D)}
    lens = lengths(case)
    pages = sum(-(-n // case["page"]) for n in lens)
    if case["op"] == "read":
        return {"bytes": sum(lens) * (row + 4 * Hkv * D) + 4 * (pages + len(lens) + 1), "flops": sum(lens) * 2 * Hkv * D}
    Hq, P = case["Hq"], case.get("prefix", 0)
    return {"bytes": (sum(lens) + P) * row + 4 * D * Hq * len(lens) + 4 * (pages + len(lens) + -(-P // case["page"])),
            "flops": 4 * D * Hq * (sum(lens) + P * len(lens))}


def _exact_row_elements(x):
    """Element values and scales (float64) of rows x, straight from the definition."""
    top = x.abs().amax(-1)
    e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -300) / 448.0))
    e = torch.where(top > 448.0 * _two_to(e), e + 1, e)
    e = torch.where(top <= 448.0 * _two_to(e - 1), e - 1, e)
    scale = _two_to(torch.where(top == 0, torch.zeros_like(e), e.clamp(min=-126)))
    y = x / scale[..., None]
    octave = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    octave = torch.where(y.abs() < _two_to(octave), octave - 1, octave).clamp(min=-6)
    ulp = _two_to(octave - 3)
    return torch.round(y / ulp) * ulp, scale


def _two_to(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def exact(case, seed):
    """The definitions in float64, sequence by sequence. Pages that no token was appended to keep what they held."""
    st = prepare(case, seed)
    if case["op"] == "norm":
        b = st["y"].double()
        if st["post"] is not None:
            b = b / torch.sqrt((b * b).sum(1, keepdim=True) / case["d"] + st["eps"]) * st["post"].double()
        x = st["x"].double() + st["scale"] * (1.0 if st["gate"] is None else st["gate"].double()) * b
        return {"x": x, "h": x / torch.sqrt((x * x).sum(1, keepdim=True) / case["d"] + st["eps"]) * st["pre"].double()}
    page, Hkv, D = case["page"], case["Hkv"], case["D"]
    cache = [None if c is None else c.double() for c in st["cache"]]
    if case["op"] == "append8":
        slot, angles = st["slots"].long(), st["cos_sin"].double()[st["positions"].long()]
        half = angles.shape[1] // 2
        turn = torch.complex(angles[:, :half], angles[:, half:])[:, None]

        def turned(x):
            x = x.double().clone()
            re, im = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["interleaved"] else (slice(0, half), slice(half, 2 * half))
            z = torch.complex(x[..., re], x[..., im]) * turn
            x[..., re], x[..., im] = z.real, z.imag
            return x

        out = {"q": turned(st["q"])}
        for i, (name, rows) in enumerate((("k", turned(st["k"])), ("v", st["v"].double()))):
            codes, scale = _exact_row_elements(rows)
            out[name] = codes * scale[..., None]
            for what, held, new in (("_cache", cache[i], codes), ("_scale", cache[i + 2][..., None], scale[..., None])):
                flat = held.transpose(1, 2).reshape(page * held.shape[0], Hkv, -1)
                flat[slot] = new
                out[name + what] = flat.view(-1, page, Hkv, held.shape[-1]).transpose(1, 2).reshape(held.shape if what == "_cache" else held.shape[:-1])
        return out

    def kept(pages, n):  # keys and values [Hkv, n, D] of a list of pages
        pages = pages.long()
        both = [c[pages] if s is None else c[pages] * s[pages][..., None] for c, s in zip(cache[:2], cache[2:])]
        return [x.transpose(0, 1).reshape(Hkv, -1, D)[:, :n] for x in both]

    rows, parts = [kept(st["block_table"][b, :-(-n // page)], n) for b, n in enumerate(lengths(case))], []
    if case["op"] == "read":
        return {"k": torch.cat([k.transpose(0, 1) for k, _ in rows]), "v": torch.cat([v.transpose(0, 1) for _, v in rows])}
    first = kept(st["prefix"], case["prefix"]) if case["op"] == "shared" else [torch.zeros(Hkv, 0, D, dtype=torch.float64, device=st["q"].device)] * 2
    for b, (k, v) in enumerate(rows):
        q = st["q"][b].double().view(Hkv, -1, D)
        s = torch.cat([q @ f.transpose(1, 2).contiguous() for f in (first[0], k)], 2)
        w = torch.softmax(s * st["scale"], -1)
        P = first[0].shape[1]
        parts.append(((w[..., :P] @ first[1]) + (w[..., P:] @ v)).reshape(-1, D))
    return torch.stack(parts)
