"""Shared by the GPU tests of attention weights, eviction and shared prefixes:
filled FP8 pools and the error bounds, derived from the kernels' roundings."""

from __future__ import annotations

import numpy as np
import torch

from oracle import fp8_oracle as O

DEV = "cuda"
D = 128


def pool(gen, num_blocks, heads, block, k_gain=1.0):
    """(numpy caches, the same on the GPU) of random K/V, an outlier channel in K."""
    arrays = []
    for gain in (k_gain, 1.0):
        x = torch.randn(num_blocks * block, heads, D, generator=gen) * gain
        if gain is k_gain:
            x[:, :, 7] *= 6
        q, s = O.quantize_rows(x.numpy())
        arrays.append((q.reshape(num_blocks, block, heads, D),
                       s.reshape(num_blocks, block, heads).astype(np.float32)))
    (kc, ks), (vc, vs) = arrays
    return [kc, vc, ks, vs], to_gpu([kc, vc, ks, vs])


def to_gpu(caches):
    kc, vc, ks, vs = (torch.from_numpy(np.ascontiguousarray(c)).to(DEV) for c in caches)
    return kc.view(torch.float8_e4m3fn), vc.view(torch.float8_e4m3fn), ks, vs


def to_cpu(caches):
    return [c.view(torch.uint8).cpu().numpy() if c.element_size() == 1 else c.cpu().numpy()
            for c in caches]


def tables_of(gen, lens, block, pool_size, width=0):
    """-1 padded tables of distinct pages."""
    pages = [-(-n // block) for n in lens]
    assert sum(pages) <= pool_size
    perm = torch.randperm(pool_size, generator=gen).tolist()
    t = np.full((len(lens), max(1, width, *pages)), -1, np.int32)
    for i, p in enumerate(pages):
        t[i, :p] = [perm.pop() for _ in range(p)]
    return t


def gpu(x, dtype=torch.int32):
    return torch.as_tensor(np.asarray(x), dtype=dtype).to(DEV)


def reach_of(q, k, scale):
    """The largest |scale| sum |q k| of any (query head, key), bounded by norms."""
    if k.shape[0] == 0 or q.shape[0] == 0:
        return 0.0
    return float(abs(scale) * np.sqrt((np.asarray(q, np.float64) ** 2).sum(-1).max()
                                      * (k ** 2).sum(-1).max()))


def weight_bound(reach, keys):
    """A probability's relative error: the score's 128 products are exact and
    summed in fp32 (2^-23 a term of reach), its scales add three roundings of
    2^-24; both move the weight and the denominator; exp2 and log2 1 ulp each
    at exponents of at most 2 reach (2^-23 of it); the denominator's sum over
    the keys 2^-24 each."""
    return 2 * reach * (128 * 2.0 ** -23 + 3 * 2.0 ** -24 + 2.0 ** -23) + keys * 2.0 ** -24 + 2.0 ** -20


def check_weights(got, want, old, reach, keys, rows):
    """Entries whose sums (want - old) are of `rows` probabilities each; sums and
    the addition to the old entry round by 2^-24 a step."""
    got, want, old = (np.asarray(x, np.float64) for x in (got, want, old))
    tol = np.abs(want - old) * (weight_bound(reach, keys) + rows * 2.0 ** -24)
    tol = tol + np.abs(want) * 2.0 ** -24 + 1e-37
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (
        f"{bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(got - want) / tol):.2f} of the "
        f"bound, first {np.argwhere(bad)[0]}")


def check_out(got, want, weight, reach, dtype, keys, vmax, weights):
    """Attention outputs, weight = sum p |v| of the row: the output's half step;
    `weights` roundings of each softmax weight to fp16, 2^-11 of sum p |v|, and
    below fp16's normal range 2^-25 of a unit in which the largest v_scale is at
    least 64, times a code of at most 448: 448 vmax 2^-24 / 64 a key, vmax the
    largest v_scale; the scores' errors as in weight_bound."""
    rel = weights * 2.0 ** -11 + weight_bound(reach, keys)
    tol = rel * weight + keys * 448 * vmax * 2.0 ** -30
    tol = tol + torch.finfo(dtype).eps / 2 * (np.abs(want) + tol) + 1e-30
    err = np.abs(got.double().cpu().numpy() - want)
    bad = ~(err <= tol)
    assert not bad.any(), (
        f"{bad.sum()} of {bad.size} off, worst {np.nanmax(err / tol):.2f} of the bound, "
        f"first {np.argwhere(bad)[0]}")
