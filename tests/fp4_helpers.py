"""Shared by the GPU tests of the 4-bit cache: numpy caches beside the GPU's,
and the error bounds, derived from the kernels' roundings."""

from __future__ import annotations

import numpy as np
import torch

import microserve_amd as M
from oracle import fp4_oracle as O

DEV = "cuda"
D = 128


def filled(gen, num_blocks, heads, block, k_gain=1.0, v_gain=1.0):
    """A pool of random K/V, every slot stored by the oracle's own quantizer:
    (numpy caches, the same on the GPU)."""
    n = num_blocks * block
    k = torch.randn(n, heads, D, generator=gen).numpy() * k_gain
    v = (torch.randn(n, heads, D, generator=gen) * v_gain).numpy()
    k[:, :, 7] *= 6  # an outlier channel
    caches = empty(num_blocks, heads, block)
    kc, vc, ks, vs = caches
    kq, ke = O.quantize_k(k)
    vq, ve = O.quantize_v(v)
    nb, bs = num_blocks, block
    kc[:] = O.pack(kq).reshape(nb, bs // 16, 16, heads, 4, 16).transpose(0, 3, 1, 4, 2, 5)
    ks[:] = ke.reshape(nb, bs // 64, 4, 16, heads, 4).transpose(0, 4, 1, 5, 3, 2)
    vc[:] = O.pack(vq).reshape(nb, bs, heads, 64).transpose(0, 2, 1, 3)
    vs[:] = ve.reshape(nb, bs, heads).transpose(0, 2, 1)
    return caches, to_gpu(caches)


def empty(num_blocks, heads, block):
    return [np.zeros(s, np.float32 if i == 3 else np.uint8)
            for i, s in enumerate(M.fp4_cache_shapes(num_blocks, block, heads))]


def to_gpu(caches):
    return tuple(torch.from_numpy(c).to(DEV) for c in caches)


def tables_of(gen, lens, block, pool, width=0):
    """-1 padded tables of distinct pages."""
    pages = [-(-n // block) for n in lens]
    assert sum(pages) <= pool
    perm = torch.randperm(pool, generator=gen).tolist()
    t = np.full((len(lens), max(1, width, *pages)), -1, np.int32)
    for i, p in enumerate(pages):
        t[i, :p] = [perm.pop() for _ in range(p)]
    return t


def check(got, want, weight, reach, dtype, keys, vmax, weights):
    """|got - want| elementwise, from the roundings of the kernels, with
    weight = sum p |v| and reach = |scale| max|q| max sum|k| of the row:

    * the output: half a step, eps / 2 of its magnitude;
    * the softmax weights: `weights` roundings to fp16, 2^-11 of sum p |v| each
      (decode: p * v_scale * f, one; prefill: p, v_scale * f, their product
      and the denominator's p, four);
    * weights below fp16's normal range, 2^-25 each of 1 = the row's largest p
      (prefill, twice: the sum and the denominator) or of a unit in which the
      largest v_scale is at least 64 (decode), times a code of at most 6: no
      more than 6 vmax 2^-24 a key;
    * the scores: the query's parts leave at most 2^-10 of a unit in which its
      largest element is at least 224, 2^-17.8 of it a dimension (decode,
      e4m3), or 2^-13 of one in which its block's largest is at least 3.75,
      2^-14.9 (prefill, e2m3); the product's fp32 sum of 128 x 3 terms at most
      384 x 2^-24: together 2^-14 of reach; the scale and the maximum's
      subtraction 2^-22 of reach.  Each moves a weight, and the denominator,
      by that much relatively;
    * exp2, the sums over the keys and the merge of the splits: 2^-18."""
    rel = weights * 2.0 ** -11 + 2 * reach * (2.0 ** -14 + 2.0 ** -22) + 2.0 ** -18
    tol = rel[..., None] * weight + keys * 6 * vmax * 2.0 ** -24
    tol = tol + torch.finfo(dtype).eps / 2 * (np.abs(want) + tol) + 1e-30
    err = np.abs(got.double().cpu().numpy() - want)
    bad = ~(err <= tol)
    assert not bad.any(), (
        f"{bad.sum()} of {bad.size} off, worst {np.nanmax(err / tol):.2f} of the bound, "
        f"first {np.argwhere(bad)[0]}")
