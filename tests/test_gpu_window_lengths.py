"""Windows whose sequences are longer than the tables or than the given bound: what
lies past the end is not counted, and a query sees all that lies before it."""

import numpy as np
import pytest
import torch

import microserve_amd as M
from oracle import weights_oracle as W
from tests import weights_helpers as H

pytestmark = pytest.mark.gpu
D = 128


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new,lens,pages,bound", [
    ([8], [600], 2, None),            # a table of 512 tokens
    ([8], [600], 3, 256), ([8, 5], [600, 90], 3, 300),  # a bound below the length
    ([40, 3, 70], [700, 513, 5000], 2, None),
    ([300], [400], 1, None),          # query i sees 101 + i of 256
    ([8], [2 ** 31 - 1], 2, None)])
def test_limits_follow_the_whole_length(new, lens, pages, bound, dtype, accumulate):
    gen = torch.Generator().manual_seed(sum(new))
    hq, hk, block, scale = 8, 2, 256, D ** -0.5
    total = pages * len(lens)
    host, dev = H.pool(gen, total, hk, block)
    tables = torch.randperm(total, generator=gen).reshape(len(lens), pages).numpy().astype(np.int32)
    old = torch.rand(total, hk, block, generator=gen)
    q = torch.randn(sum(new), hq, D, generator=gen).to(dtype)
    cu_q, cu_k = np.cumsum([0, *new]), np.cumsum([0, *lens])
    weights = old.to(H.DEV)
    M.fp8_window_attention_weights(
        q.to(H.DEV), dev[0], dev[2], H.gpu(tables), H.gpu(cu_q), H.gpu(cu_k), max(new), scale,
        weights, accumulate=accumulate, max_seqlen_k=bound)
    torch.cuda.synchronize()
    want, touched = old.double().numpy(), np.zeros(old.shape, bool)
    before = want.copy() if accumulate else np.zeros_like(want)
    reach = 0.0
    for b, (n, lq) in enumerate(zip(lens, new)):
        keys = min(n, pages * block, bound or n)
        k, ok = W.rows_of(host[0], host[2], tables[b], keys, block)
        rows = q[cu_q[b]:cu_q[b + 1]].double().numpy()
        p = W.probabilities(rows, k, ok, scale, n - lq + 1 + np.arange(lq))
        sums = W.by_kv_head(p, hk)
        W.record(want, sums, ok, tables[b], 0, lambda t: accumulate)
        W.record(touched, np.ones(sums.shape, bool), ok, tables[b], 0, lambda t: False)
        reach = max(reach, H.reach_of(rows, k, scale))
    got = weights.cpu().numpy()
    assert np.array_equal(got[~touched], old.numpy()[~touched]), "an entry beside the tokens"
    H.check_weights(got, want, np.where(touched, before, want), reach, pages * block,
                    hq // hk * max(new))


def test_a_range_of_more_tokens_than_an_int():
    """One query, a bound of 261632 and 67 million tokens in pages that repeat: by the
    bound a workgroup's range would hold 2^31 tokens and more."""
    heads, block, copies, scale = 8, 256, 262700, 0.05
    bound = 2044 * 128
    gen = torch.Generator().manual_seed(0)
    host, dev = H.pool(gen, 4, heads, block)
    table = torch.zeros(1, copies, dtype=torch.int32)
    table[0] = torch.arange(copies) % 3  # pages 0 to 2 in turn, then page 3
    table[0, -1] = 3
    lk = copies * block
    assert -(-copies * heads * 2044 // 512) * 256 > 2 ** 31
    q = torch.zeros(bound, heads, D, device=H.DEV).half()  # (the others are padding)
    q[0] = torch.randn(heads, D, generator=gen).half()
    weights = torch.full((4, heads, block), 7.0, device=H.DEV)
    M.fp8_window_attention_weights(q, dev[0], dev[2], table.to(H.DEV), H.gpu([0, 1]),
                                   H.gpu([0, lk]), bound, scale, weights, start=lk - block)
    got = weights.cpu().double().numpy()
    assert (got[:3] == 7).all()
    k, _ = W.rows_of(host[0], host[2], range(4), 4 * block, block)
    s = np.exp(np.einsum("hd,khd->hk", q[0].cpu().double().numpy(), k) * scale)
    times = np.repeat(np.bincount(table[0].numpy(), minlength=4), block)
    want = (s / (s * times).sum(-1, keepdims=True))[:, 3 * block:]
    # a lane adds the sum of 16 probabilities a tile to its running one: a rounding of
    # 2^-24 a tile, besides weight_bound's (the sum over keys there is this one)
    tol = H.weight_bound(H.reach_of(q[:1].cpu().double().numpy(), k, scale), copies + 32)
    assert (np.abs(got[3] - want) <= tol * want).all()
