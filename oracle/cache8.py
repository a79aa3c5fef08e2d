"""Plain restatement, on the CPU in float64, of the cache in 8 bits (test infrastructure only): the elements by a search among all values
that an e4m3 number has, the exponent by trying them in turn."""
import torch

# e4m3: sign, 4 bits of exponent (bias 7), 3 of mantissa; code 127 is no number
VALUES = torch.tensor([(m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127],
                      dtype=torch.float64)


def power(e):
    """2^e in float64 of whole numbers from -1022 on."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def quantise(x, dtype):
    """x [..., D] float64, finite or not -> (codes uint8 [..., D], exponents + 127 uint8 [...]) for rows of `dtype`."""
    x = x.double()
    size = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))
    top = size.amax(-1)
    e = torch.full(top.shape, -126)
    for step in (128, 64, 32, 16, 8, 4, 2, 1):         # the largest e that is still too small, plus one
        e = torch.where(top > 448 * power(e + step - 1), e + step, e)
    e = torch.where(top == 0, torch.zeros_like(e), e)
    y = size / power(e)[..., None]
    most = VALUES[VALUES <= 448].expand(*top.shape, 127)
    limit = torch.where(most * power(e)[..., None] <= torch.finfo(dtype).max, most, torch.zeros_like(most)).amax(-1)
    y = torch.minimum(y, limit[..., None])
    above = torch.searchsorted(VALUES, y.contiguous()).clamp(max=126)
    below = (above - 1).clamp(min=0)
    up, down = VALUES[above] - y, y - VALUES[below]
    code = torch.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
    code = torch.where(torch.isfinite(x), code, torch.full_like(code, 127))
    return (code + 128 * torch.signbit(x).long()).to(torch.uint8), (e + 127).to(torch.uint8)


def held(codes, scales):
    """What codes uint8 [..., D] with scales uint8 [...] stand for, float64."""
    codes, scales = codes.cpu().long(), scales.cpu().long()
    x = torch.cat([VALUES, torch.tensor([float("nan")], dtype=torch.float64)])[codes % 128]
    x = torch.where(codes >= 128, -x, x) * power(scales - 127)[..., None]
    return torch.where(scales[..., None] == 255, torch.full_like(x, float("nan")), x)
