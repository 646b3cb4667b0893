"""Plain 64-bit statements of the batch entries (include/dflash_batch.h), with the tolerances
that the kernels' roundings allow.  Everything here is torch on whatever device the inputs
are on; nothing calls the library."""
from __future__ import annotations

import math

import torch

BF16, FP16, FP32 = (torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32))


def values(part, bits, group):
    """float64 values of a cache tensor (data, scales, biases)."""
    data, s, b = part
    if bits == 16:
        return data.double()
    w = data.long() & 0xFFFFFFFF
    codes = torch.stack([(w >> k) & (2 ** bits - 1) for k in range(0, 32, bits)], -1).flatten(-2).double()
    wide = lambda t: t.double().repeat_interleave(group, -1)  # noqa: E731
    return codes * wide(s) + wide(b)


def quantise(x, bits, group):
    """(data, scales, biases) of rows x (float64 [..., d]) under the affine rule."""
    if bits == 16:
        return x.to(torch.bfloat16), None, None
    top = 2 ** bits - 1
    x = x.double().unflatten(-1, (-1, group))
    lo, hi = x.amin(-1), x.amax(-1)
    low = lo.abs() > hi.abs()
    edge, sign, span = torch.where(low, lo, hi), torch.where(low, 1.0, -1.0).double(), hi - lo
    tiny = span / top < 1e-7
    z = sign * torch.round(torch.where(tiny, edge / 1e-7, edge * top / span))
    s = torch.where(z != 0, edge / z, sign * (span / top).clamp(min=1e-7)).to(torch.bfloat16)
    b = torch.where(z != 0, edge, torch.zeros_like(edge)).to(torch.bfloat16)
    c = torch.round((x - b.double()[..., None]) / s.double()[..., None]).clamp(0, top).long().flatten(-2)
    c = c.unflatten(-1, (-1, 32 // bits))
    w = (c << torch.arange(0, 32, bits, device=x.device)).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32), s, b


def norm_rope(x, w, pos, rot, eps, theta):
    """float64 RMSNorm and rotate-half rotary embedding of heads x [rows, heads, d] at pos [rows]."""
    x = x.double()
    x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    if rot:
        freq = float(theta) ** (-torch.arange(0, rot, 2, device=x.device, dtype=torch.float64) / rot)
        a = (pos.double()[:, None] * freq)[:, None]
        p, q = x[..., :rot // 2], x[..., rot // 2:rot]
        x = torch.cat([p * a.cos() - q * a.sin(), q * a.cos() + p * a.sin(), x[..., rot:]], -1)
    return x


# The normalised element is off by at most 2^-16 relative in 32 bits (a sum of d <= 256 squares:
# 2^-16 of the sum, half of that in its root, and a few roundings), and a rotation adds cos and
# sin off by 2^-22 and 2^-24 for each of its operations; |rotated| <= sqrt(2) |row|max.
NORM = 2.0 ** -15


def depths(parents, T):
    """Row depths and visibility [T, T] of one tree given as a parent list (None: a chain)."""
    seen = torch.zeros(T, T, dtype=torch.bool)
    if parents is None:
        return list(range(T)), torch.tril(torch.ones(T, T, dtype=torch.bool))
    depth = []
    for t in range(T):
        r, d = t, 0
        while r >= 0:
            seen[t, r] = True
            p = parents[r] if r > 0 else -1
            r, d = (p, d + 1) if 0 <= p < r else (-1, d)
        depth.append(d)
    return depth, seen


def attention(q, k, v, seen, scale, eps_kv, eps_p):
    """softmax(scale q k^T) v in float64 for q [rows, d], k and v [keys, d] under seen
    [rows, keys], and how far a kernel may be off that rounds k and v to eps_kv and the
    probabilities to eps_p (relative) and adds in 32 bits: a score is off by
    delta = (eps_kv + d 2^-24) scale sum |q| |k|, a weight p / sum p then by a factor within
    e^(+-2 delta); the exponential in 32 bits adds 2^-21 + |score - max| 2^-23."""
    q, k, v = q.double(), k.double(), v.double()
    k, v = k.masked_fill(~seen.any(0)[:, None], 0.0), v.masked_fill(~seen.any(0)[:, None], 0.0)
    s = (q @ k.T * scale).masked_fill(~seen, -math.inf)
    p = torch.softmax(s, -1)
    size = ((q.abs() @ k.abs().T) * abs(scale)).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
    delta = (eps_kv + q.shape[1] * FP32) * size + 2.0 ** -21 + 2 * size * 2.0 ** -23
    spread = torch.expm1(2 * delta) + eps_kv + 2 * eps_p + k.shape[0] * FP32
    return p @ v, spread * (p @ v.abs())
