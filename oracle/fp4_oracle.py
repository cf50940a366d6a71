"""The 4-bit key/value cache in numpy, in 64 bits: the format and attention over it.

Test infrastructure: what include/nvk.h says of the format, restated from the definition (nearest
code by distance) rather than from the kernels' arithmetic.
"""
import numpy as np

GROUP = 32
MAGNITUDES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)


def quantise(x):
    """(codes uint8 [..., D], scale float16 [..., D / 32]) of rows x [..., D] (exact floats)."""
    x = np.asarray(x, dtype=np.float64)
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    top = np.abs(g).max(-1)
    finite = np.isfinite(top)
    with np.errstate(over="ignore"):
        scale = np.minimum(np.where(finite, top, 0) / 6, 65504.0).astype(np.float16)
    s = scale.astype(np.float64)[..., None]
    safe = np.where(finite[..., None], g, 0.0)
    # (beyond 6: 6; a distance to a far larger number would be the same for all codes in 64 bits)
    dist = np.abs(np.minimum(np.abs(safe), 6 * s)[..., None] - MAGNITUDES * s[..., None])
    # the nearest code; of two at the same distance the even one
    best = dist.min(-1, keepdims=True)
    near = dist == best
    order = np.array([0, 2, 4, 6, 1, 3, 5, 7])
    code = order[np.argmax(near[..., order], axis=-1)].astype(np.uint8)
    code = np.where(s > 0, code, 0).astype(np.uint8)
    code |= ((safe < 0).astype(np.uint8) << 3)
    scale = np.where(finite, scale, np.float16(np.nan)).astype(np.float16)
    return code.reshape(x.shape), scale


def places(d, keys):
    """places[i] = where dimension i of a row lies among its codes."""
    i = np.arange(d)
    if not keys:
        return i
    s, g, e = i // 32, i % 32 // 8, i % 8
    return ((d // 32) * g + s) * 8 + e


def pack(codes, keys):
    """Bytes [..., D / 2] of codes [..., D]."""
    row = np.zeros_like(codes)
    row[..., places(codes.shape[-1], keys)] = codes
    return row[..., 0::2] | (row[..., 1::2] << 4)


def unpack(data, keys):
    row = np.stack([data & 15, data >> 4], axis=-1).reshape(*data.shape[:-1], -1)
    return row[..., places(row.shape[-1], keys)]


def values(data, scale, keys):
    """Float64 [NB, P, H, D] that a cache's data [NB, H, P, D / 2] and scale [NB, H, D / 32, P]
    stand for."""
    c = unpack(data, keys)
    v = MAGNITUDES[c & 7] * np.where(c & 8, -1.0, 1.0)
    s = np.swapaxes(scale.astype(np.float64), -1, -2).repeat(GROUP, axis=-1)
    return np.swapaxes(v * s, 1, 2)


def store(rows, data, scale, slots, keys):
    """Scatters rows [N, H, D] into (data, scale) in place."""
    p = data.shape[2]
    codes, s = quantise(rows)
    packed = pack(codes, keys)
    for t, slot in enumerate(slots):
        if 0 <= slot < data.shape[0] * p:
            data[slot // p, :, slot % p] = packed[t]
            scale[slot // p, :, :, slot % p] = s[t]


def through_pages(n, g, d, groups, keys):
    """Whether n queries of g heads per kv head run over f16 pages of the keys and values, in a call
    of `groups` (sequence, kv head) pairs of at most `keys` keys."""
    chunks = -(-n * g // 16) * -(-keys // 64) * groups
    return n * g > 192 and d == 128 and g in (1, 2, 4, 8) and chunks >= 16384


def attention(q, k, v, n_keys, scale, pages=False):
    """One sequence: q [n, Hq, D], k / v [>= n_keys, Hkv, D]; query i sees keys j <= i + n_keys - n.
    Returns (out, size) [n, Hq, D]: the attention, and what its rounding errors are relative to:
    `size` bounds |kernel - out| without the rounding of the output itself.

    The kernel's probabilities are off by a relative 2 (D + 8) 2^-24 sum |q_i k_i| scale (the f32 sum of
    the score, in e^x, against the maximum) and, times the value's scale, by half a step of f16
    (2^-11 relative, 2^-25 at least); n_keys f32 additions and the exponential add 2 (n + 64) 2^-24.
    pages: keys, values and probabilities are off by half a step of f16 each, keys and values by 2^-22
    at least (f16 holds an eighth of them): in a score, that is 2^-11 sum |q_i k_i| scale
    + 2^-22 sum |q_i| scale, twice (against the maximum)."""
    n, hq, d = q.shape
    g = hq // k.shape[1]
    out, size = np.zeros((n, hq, d)), np.zeros((n, hq, d))
    for h in range(hq):
        kk, vv = k[:n_keys, h // g], v[:n_keys, h // g]
        for i in range(n):
            m = min(n_keys, i + n_keys - n + 1)
            if m <= 0:
                continue
            s = kk[:m] @ q[i, h] * scale
            off = (np.abs(kk[:m]) @ np.abs(q[i, h])).max() * scale
            e = np.exp(s - s.max())
            l = e.sum()
            out[i, h] = e @ vv[:m] / l
            rel = 2 * (d + 8) * 2.0 ** -24 * off + 2.0 ** -11 + 2 * (m + 64) * 2.0 ** -24
            if pages:
                rel += 2.0 ** -11 * (1 + 2 * off) + 2.0 ** -21 * np.abs(q[i, h]).sum() * scale
            size[i, h] = rel * (e @ np.abs(vv[:m]) / l) + 2.0 ** -25 * 6 * m / l
            size[i, h] += 2.0 ** -22 if pages else 0.0
    return out, size
