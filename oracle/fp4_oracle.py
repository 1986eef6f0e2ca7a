"""CPU restatement of the 4-bit paged cache and of attention over it, in
numpy and 64 bits: the definition the kernels are held to."""

from __future__ import annotations

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
NAN_SCALE = 255
D = 128


def encode(y):
    """e2m1 codes of y: the nearest value, ties to the even code, 6 beyond 6."""
    y = np.asarray(y, np.float64)
    a = np.minimum(np.abs(y), 6.0)
    hi = np.clip(np.searchsorted(GRID, a), 1, 7)
    to_hi, to_lo = GRID[hi] - a, a - GRID[hi - 1]
    code = np.where((to_hi < to_lo) | ((to_hi == to_lo) & (hi % 2 == 0)), hi, hi - 1)
    return (code | (np.signbit(y).astype(np.int64) << 3)).astype(np.uint8)


def decode(codes):
    v = GRID[codes & 7]
    return np.where(codes & 8, -v, v)


def quantize_k(x):
    """rows [..., 128] -> codes [..., 128] and scale bytes [..., 4]."""
    x = np.asarray(x, np.float64)
    b = x.reshape(x.shape[:-1] + (4, 32))
    amax = np.abs(b).max(-1)
    bad = ~np.isfinite(amax)
    m, p = np.frexp(np.where(bad, 1.0, amax))  # amax = m 2^p, m in [0.5, 1)
    e = np.where(amax == 0, -126, np.clip(p - 3 + (m >= 0.875), -126, 127))
    with np.errstate(invalid="ignore"):
        codes = encode(np.where(bad[..., None], 0.0, b / np.exp2(e.astype(np.float64))[..., None]))
    return codes.reshape(x.shape), np.where(bad, NAN_SCALE, e + 127).astype(np.uint8)


def quantize_v(x):
    """rows [..., 128] (float32 values) -> codes [..., 128] and fp32 scales."""
    x = np.asarray(x, np.float32)
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        amax = np.maximum(np.abs(x).max(-1), np.float32(1e-8)).astype(np.float32)
        bad = ~np.isfinite(amax)
        top = np.where(bad, np.float32(1), amax)
        y = (np.float32(0.75) * np.where(bad[..., None], np.float32(0), x)) / (
            np.float32(0.125) * top)[..., None]
        assert y.dtype == np.float32
        scale = np.where(bad, np.float32(np.nan), top / np.float32(6.0)).astype(np.float32)
    return encode(y), scale


def pack(codes):
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).astype(np.uint8)


def unpack(packed):
    return np.stack((packed & 15, packed >> 4), -1).reshape(packed.shape[:-1] + (-1,))


def store(key, value, caches, slots):
    """Writes the rows one token at a time into the numpy caches."""
    kc, vc, ks, vs = caches
    nb, _, bs = vc.shape[:3]
    kq, ke = quantize_k(key)
    vq, ve = quantize_v(value)
    for i, slot in enumerate(np.asarray(slots)):
        if not 0 <= slot < nb * bs:
            continue
        page, t = divmod(int(slot), bs)
        for h in range(key.shape[1]):
            kc[page, h, t // 16, :, t % 16] = pack(kq[i, h].reshape(4, 32))
            ks[page, h, t // 64, :, t % 16, t // 16 % 4] = ke[i, h]
            vc[page, h, t] = pack(vq[i, h])
            vs[page, h, t] = ve[i, h]


def rows(caches, pages, n):
    """K and V [H, n, 128] in 64 bits of the first n tokens of `pages`; a page
    outside the pool gives NaN rows."""
    kc, vc, ks, vs = caches
    nb, heads, bs = vc.shape[:3]
    k = np.full((heads, n, D), np.nan)
    v = np.full((heads, n, D), np.nan)
    for i, page in enumerate(pages[:-(-n // bs)]):
        if not 0 <= page < nb:
            continue
        m = min(bs, n - i * bs)
        kk = decode(unpack(kc[page]))  # [H, BS/16, 4, 16, 32]
        e = ks[page].transpose(0, 1, 4, 2, 3).reshape(heads, bs // 16, 4, 16)
        scale = np.where(e == NAN_SCALE, np.nan, np.exp2(e.astype(np.float64) - 127))
        kk = (kk * scale[..., None]).transpose(0, 1, 3, 2, 4).reshape(heads, bs, D)
        vv = decode(unpack(vc[page])) * vs[page].astype(np.float64)[..., None]
        k[:, i * bs:i * bs + m] = kk[:, :m]
        v[:, i * bs:i * bs + m] = vv[:, :m]
    return k, v


def attend(q, k, v, scale, seen):
    """q [n, Hq, 128] over k, v [H, keys, 128]; seen [n, keys].  Returns the
    output, and for error bounds: sum p |v| and the largest |scale| |q| |k|."""
    n, hq, _ = q.shape
    heads = k.shape[0]
    group = hq // heads
    out = np.zeros((n, hq, D))
    weight = np.zeros((n, hq, D))
    reach = np.zeros((n, hq))
    for h in range(hq):
        kh, vh = k[h // group], v[h // group]
        for i in range(n):
            at = np.flatnonzero(seen[i])
            if not len(at):
                continue
            s = kh[at] @ q[i, h].astype(np.float64) * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, h] = p @ vh[at]
            weight[i, h] = p @ np.abs(vh[at])
            reach[i, h] = abs(scale) * np.abs(q[i, h]).max() * np.abs(kh[at]).sum(-1).max()
    return out, weight, reach
