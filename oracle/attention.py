"""Plain float64 restatement, on the CPU, of the attention operators (test infrastructure only): one sequence and one head
at a time, straight from the definitions. Beside each output it returns the weighted sum of magnitudes that its error is
bounded by."""
import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # unit roundoff


def rotate(x, cos_sin, positions, interleaved):
    """x [T, H, D] -> float64 [T, H, D] with the first rot channels turned by the angles of positions."""
    x = x.cpu().double()
    out = x.clone()
    rot = cos_sin.shape[1]
    for i in range(rot // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        cos = cos_sin.cpu().double()[positions.cpu().long(), i].view(-1, 1)
        sin = cos_sin.cpu().double()[positions.cpu().long(), i + rot // 2].view(-1, 1)
        out[..., a] = x[..., a] * cos - x[..., b] * sin
        out[..., b] = x[..., b] * cos + x[..., a] * sin
    return out


def rotate_tolerance(x, ref, dtype):
    """One rounding of a sum of two fp32 products of values no larger than the largest input pair (sines and cosines <= 1)."""
    return U[dtype] * ref.abs() + 2.0 ** -22 * x.cpu().double().abs().amax() + 2.0 ** -25


def attend(q, k, v, scale, visible):
    """q [nq, D], k and v [nk, D], visible [nq]: row i sees the first visible[i] keys -> (o, sum w |v|), float64 [nq, D]."""
    q, k, v = q.cpu().double(), k.cpu().double(), v.cpu().double()
    o, mag = torch.zeros_like(q), torch.zeros_like(q)
    for i in range(q.shape[0]):
        n = int(visible[i])
        if n <= 0:
            continue
        s = (k[:n] @ q[i]) * scale
        w = torch.exp(s - s.max())
        w = w / w.sum()
        o[i], mag[i] = w @ v[:n], w @ v[:n].abs()
    return o, mag


def gather(cache, table_row, length):
    """Keys or values [length, Hkv, D] of one sequence from a [pages, Hkv, page_size, D] cache."""
    page = cache.shape[2]
    rows = [cache[int(table_row[j // page]), :, j % page] for j in range(length)]
    return torch.stack(rows) if rows else cache.new_zeros((0, cache.shape[1], cache.shape[3]))


def decode(q, k_cache, v_cache, table, lengths, scale):
    q, k_cache, v_cache = q.cpu(), k_cache.cpu(), v_cache.cpu()
    o = torch.zeros(q.shape, dtype=torch.float64)
    mag = torch.zeros_like(o)
    group = q.shape[1] // k_cache.shape[1]
    for b, n in enumerate(lengths):
        k, v = gather(k_cache, table[b], n), gather(v_cache, table[b], n)
        for h in range(q.shape[1]):
            o[b, h:h + 1], mag[b, h:h + 1] = attend(q[b, h:h + 1], k[:, h // group], v[:, h // group], scale, [n])
    return o, mag


def prompt(q, k, v, cu_q, cu_k, scale):
    q, k, v = q.cpu(), k.cpu(), v.cpu()
    o = torch.zeros(q.shape, dtype=torch.float64)
    mag = torch.zeros_like(o)
    group = q.shape[1] // k.shape[1]
    for b in range(len(cu_q) - 1):
        rq, rk = slice(cu_q[b], cu_q[b + 1]), slice(cu_k[b], cu_k[b + 1])
        nq, nk = cu_q[b + 1] - cu_q[b], cu_k[b + 1] - cu_k[b]
        visible = [min(nk, max(0, i + nk - nq + 1)) for i in range(nq)]
        for h in range(q.shape[1]):
            o[rq, h], mag[rq, h] = attend(q[rq, h], k[rk, h // group], v[rk, h // group], scale, visible)
    return o, mag


def tolerance(ref, mag, dtype, weights_rounded, keys):
    """Bound of |out - ref|. Output: one rounding, u |ref|. Weights: a relative error e of every weight moves a weighted mean by
    at most 2 e sum w |v|; e is u where the weights are rounded for a matrix product, plus what fp32 scores carry: products of 256 channels
    summed in any order are off by at most 256 2^-24 scale sum |q k| <= 2^-16 * 16 for the inputs of these tests. fp16 weights below 2^-14 are off by
    up to 2^-25 each, of a sum that is at least 1."""
    u = U[dtype]
    e = 2.0 ** -12 + (u if weights_rounded else 0.0)
    small = keys * 2.0 ** -25 * 4.0 if dtype == torch.float16 and weights_rounded else 0.0
    return u * ref.abs() + 2 * e * mag + small + 2.0 ** -24
