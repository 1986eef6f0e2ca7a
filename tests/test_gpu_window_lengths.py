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
