"""The quantised KV cache in 64 bits, from its definition.

TEST INFRASTRUCTURE ONLY (see oracle/__init__.py). Written apart from the
library: elements are found by searching the type's list of values.
"""
from __future__ import annotations

import math

import torch

E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
E4M3 = [m * 2.0 ** -9 for m in range(8)] + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)][:119]
TOP = {4: 7.0, 8: 464.0}
LARGEST_E = {4: 125, 8: 119}


def grid(bits):
    return torch.tensor(E2M1 if bits == 4 else E4M3, dtype=torch.float64)


def quantise(x, bits):
    """Vectors ``[..., 64]`` -> codes ``[..., 64]`` (one code per element, int64)
    and scale bytes ``[..., 2]``; the byte of a block of zeros is 1."""
    b = x.double().reshape(-1, 32)
    g = grid(bits)
    codes, scale = torch.zeros(b.shape, dtype=torch.int64), torch.zeros(b.shape[0], dtype=torch.int64)
    for i, block in enumerate(b.tolist()):
        if not all(math.isfinite(y) for y in block):
            scale[i] = 255
            continue
        most = max(abs(y) for y in block)
        e = -126
        if most:
            e = max(e, math.frexp(most / TOP[bits])[1] - 2)
            while most > math.ldexp(TOP[bits], e):
                e += 1
        e = min(e, LARGEST_E[bits])
        scale[i] = e + 127
        a = b[i].abs() * 2.0 ** -e
        upper = torch.searchsorted(g, a).clamp(1, len(g) - 1)
        lower = upper - 1
        to_up, to_low = g[upper] - a, a - g[lower]
        code = torch.where((to_up < to_low) | ((to_up == to_low) & (upper % 2 == 0)), upper, lower)
        codes[i] = code + (1 << (bits - 1)) * torch.signbit(b[i])
    return codes.reshape(x.shape), scale.reshape(*x.shape[:-1], 2)


def values(codes, scales, bits):
    """What element codes ``[..., 64]`` and scale bytes ``[..., 2]`` stand for, in 64 bits."""
    g = grid(bits)
    half = 1 << (bits - 1)
    v = torch.where(codes >= half, -1.0, 1.0).double() * g[codes % half]
    s = torch.where(scales == 0, torch.zeros((), dtype=torch.float64), 2.0 ** (scales.double() - 127))
    s = torch.where(scales == 255, torch.full((), math.nan, dtype=torch.float64), s)
    return v * s.repeat_interleave(32, -1)


def pack(codes, bits):
    """Element codes ``[..., 64]`` as the cache's bytes ``[..., 8 * bits]``, uint8."""
    c = codes.to(torch.uint8)
    return c if bits == 8 else c[..., 0::2] | (c[..., 1::2] << 4)


def unpack(codes, bits):
    """The cache's bytes as element codes, int64."""
    c = codes.long()
    return c if bits == 8 else torch.stack((c % 16, c // 16), -1).flatten(-2)


def decode_attention(q, k, v, used, scale):
    """``q [B, Hq, 64]`` over ``k, v [B, Hkv, C, 64]`` in 64 bits: zeros for a row with nothing used."""
    b, hq, d = q.shape
    hkv, c = k.shape[1:3]
    out = torch.zeros(b, hq, d, dtype=torch.float64)
    for i in range(b):
        n = max(0, min(int(used[i]), c))
        if n:
            qi = q[i].double().view(hkv, hq // hkv, d)
            s = qi @ k[i, :, :n].double().transpose(1, 2) * scale
            out[i] = (torch.softmax(s, -1) @ v[i, :, :n].double()).reshape(hq, d)
    return out
