"""8-bit rows in 64 bits, from their definition: blocks of 32 values, the smallest power of two from
2^-127 on that brings the largest magnitude to at most 448, values rounded to the nearest e4m3
value, ties to the even code."""
import torch


def pow2(e):
    """2^e in fp64 for whole numbers e, exactly (the device's own powers are not)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def grid(device):
    """The finite magnitudes by code, 0 to 126."""
    c = torch.arange(127, dtype=torch.float64, device=device)
    f, m = torch.floor(c / 8), c % 8
    return torch.where(f == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * pow2(f - 7))


def rows8(v):
    """(codes uint8 [T, n], scale bytes uint8 [T, n/32], values fp64) of v [T, n] fp64, finite."""
    g = grid(v.device)
    mids = (g[1:] + g[:-1]) / 2
    b = v.unflatten(1, (-1, 32))
    top = b.abs().amax(2)
    e = torch.frexp(top).exponent - 10  # the search starts at least one below
    e = torch.where(top > 0, e, -127).clamp(min=-127)  # frexp calls 0 a half
    for _ in range(3):
        e = torch.where(top > 448 * pow2(e), e + 1, e)
    a = b * pow2(-e).unsqueeze(2)
    code = torch.searchsorted(mids, a.abs().contiguous())
    tie = (code < 126) & (a.abs() == mids[code.clamp(max=125)]) & (code % 2 == 1)
    code = code + tie.long()
    values = (g[code] * torch.sign(a) * pow2(e).unsqueeze(2)).flatten(1)
    return (code + 128 * torch.signbit(b).long()).flatten(1).to(torch.uint8), (e + 127).to(torch.uint8), values


def values8(rows):
    """fp64 values of MxRows (NaN for a scale byte of 255 and for the codes 127 and 255)."""
    c = rows.codes.view(torch.uint8).long()
    m = c & 127
    v = grid(c.device)[m.clamp(max=126)]
    v = torch.where(m == 127, float("nan"), torch.where(c >= 128, -v, v))
    s = rows.scales.int()
    s = torch.where(s == 255, float("nan"), pow2(s - 127))
    return (v.unflatten(1, (-1, 32)) * s.unsqueeze(2)).flatten(1)
