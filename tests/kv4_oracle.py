"""Plain forms of the 4-bit cache and of rotary positions for the tests: the group
quantiser (codes and powers must match it exactly), angles and turns in 64 bits."""
import math

import numpy as np
import torch

LEVELS = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
GROUP = 32


def quantise(x):
    """(values of the codes, scales' bytes) of rows of x (CPU) by the definition: groups of
    32, the least power of two 2^e with max <= 7 2^e (e from -100 to 125), nearest code, ties
    to the one of even number; max < 2^-100: byte 0 and zeros; not finite: byte 255, zeros."""
    g = x.double().unflatten(-1, (-1, GROUP))
    top = torch.where(torch.isnan(g).any(-1), torch.tensor(float("nan"), dtype=torch.float64), g.abs().amax(-1))
    fin = torch.isfinite(top)
    big = fin & (top >= 2.0 ** -100)
    safe = torch.where(big, top, torch.ones((), dtype=torch.float64))
    e = torch.ceil(torch.log2(safe / 7)).to(torch.int64)
    e = torch.where(safe > 7 * torch.exp2(e.double()), e + 1, e)            # log2 is off by a rounding next to a power
    e = torch.where(safe <= 7 * torch.exp2((e - 1).double()), e - 1, e).clamp(-100, 125)
    v = torch.where(big[..., None], g / torch.exp2(e.double())[..., None], torch.zeros((), dtype=torch.float64))
    near = (v.abs()[..., None] - LEVELS).abs()                                # [..., 8]
    best = near.amin(-1, keepdim=True)
    n = torch.where(near == best, torch.arange(8) % 2 * 8 + torch.arange(8), torch.full((), 99)).argmin(-1)  # an even number first
    codes = LEVELS[n] * torch.where(torch.signbit(v), -1.0, 1.0)
    byte = torch.where(big, e + 127, torch.where(fin, torch.zeros_like(e), torch.full_like(e, 255)))
    return codes.flatten(-2), byte.to(torch.uint8)


def unpack(codes):
    """Values of codes, uint8 [..., n / 2] -> float64 [..., n]."""
    n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    return LEVELS[n & 7] * torch.where(n > 7, -1.0, 1.0)


def values(codes, bytes_):
    """What a cache holds, float64: codes uint8 [..., slots, n / 2], bytes uint8 [..., groups, slots]."""
    p = torch.where(bytes_ == 255, torch.tensor(float("nan"), dtype=torch.float64), torch.exp2(bytes_.double() - 127))
    return unpack(codes) * p.transpose(-1, -2).repeat_interleave(GROUP, -1)


def angles(positions, frequencies):
    """(cos, sin) in 64 bits of the angles position * frequency, which are made and taken into one turn
    with 64 significant bits (with 53 they would be off by 2^-23 at positions of 2^30)."""
    a = positions.numpy().astype(np.longdouble)[..., None] * np.array(frequencies, dtype=np.longdouble)
    two_pi = np.longdouble("6.283185307179586476925286766559")
    a = torch.from_numpy((a - np.floor(a / two_pi) * two_pi).astype(np.float64))
    return a.cos(), a.sin()


def turned(x, positions, rotary_dim, interleaved, frequencies, magnitude=1.0, inverse=False):
    """x [..., tokens, heads, dim] in 64 bits, and how large the terms of each value are (for bounds)."""
    c, s = angles(positions, frequencies)
    c, s = c[..., None, :] * magnitude, (-s if inverse else s)[..., None, :] * magnitude
    h, y, size = rotary_dim // 2, x.double().clone(), x.double().abs().clone()
    first, second = (slice(0, rotary_dim, 2), slice(1, rotary_dim, 2)) if interleaved else (slice(0, h), slice(h, rotary_dim))
    a, b = x.double()[..., first], x.double()[..., second]
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    size[..., first], size[..., second] = ((a.abs() * c.abs() + b.abs() * s.abs()), (b.abs() * c.abs() + a.abs() * s.abs()))
    return y, size


def frequencies(rotary_dim, base=10000.0):
    return [base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]


def yarn(rotary_dim, base, factor, length, fast=32.0, slow=1.0):
    """Frequencies and magnitude of a context stretched by a ramp, written from the formulas pair by pair."""
    out = []
    at = lambda turns: rotary_dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    lo, hi = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), rotary_dim - 1)
    for i, f in enumerate(frequencies(rotary_dim, base)):
        r = min(max((i - lo) / max(hi - lo, 1e-3), 0), 1)
        out.append(f / factor * r + f * (1 - r))
    return out, 0.1 * math.log(factor) + 1


def bands(rotary_dim, base, factor, length, low=1.0, high=4.0):
    out = []
    for f in frequencies(rotary_dim, base):
        wave = 2 * math.pi / f
        if wave < length / high:
            out.append(f)
        elif wave > length / low:
            out.append(f / factor)
        else:
            w = (length / wave - low) / (high - low)
            out.append((1 - w) * f / factor + w * f)
    return out


def as_numpy(t):
    return np.nan_to_num(t.numpy(), nan=0.0)
