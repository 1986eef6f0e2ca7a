"""The 4-bit attention where its arithmetic could give way: keys and queries
near the ends of their types, scores of any size, and queries whose parts
split unevenly."""

import numpy as np
import pytest
import torch

import microserve_amd as M
from microserve_amd import _lib
from oracle import fp4_oracle as O
from tests import fp4_helpers as H

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
HQ, HK, BLOCK = 16, 2, 128


def _i32(x):
    return torch.as_tensor(x, dtype=torch.int32, device=H.DEV)


def _want(q, host, tables, lens, scale):
    outs = []
    for i, n in enumerate(lens):
        k, v = O.rows(host, tables[i], n)
        outs.append(O.attend(q[i:i + 1].double().numpy(), k, v, scale, np.ones((1, n), bool)))
    return [np.concatenate(x) for x in zip(*outs)]


def _both(q, dev, tables, lens, scale):
    """(kernel, roundings of its weights, output): the decode under a table of a
    few pages and under a wide one, and the prefill of the one row."""
    args = (q.to(H.DEV), *dev, _i32(lens))
    wide = np.full((len(lens), 60), -1, np.int32)
    wide[:, :tables.shape[1]] = tables
    yield "joined", 1, M.fp4_decode_attention(*args, _i32(tables), scale)
    yield "split", 1, M.fp4_decode_attention(*args, _i32(wide), scale)
    cu = torch.arange(len(lens) + 1, dtype=torch.int32, device=H.DEV)
    yield "prefill", 4, M.fp4_varlen_prefill_attention(
        q.to(H.DEV), *dev, _i32(tables), cu, _i32(np.concatenate(([0], np.cumsum(lens)))), 1, scale)


@pytest.mark.parametrize("dtype,k_gain,q_gain", [
    (BF16, 1e35, 1e-34), (BF16, 1e33, 1e-32), (BF16, 1e-34, 1e33), (BF16, 1e30, 1e-30),
    (BF16, 1e20, 1e-33), (FP16, 1e6, 1e-6), (FP16, 1e7, 1e-7), (FP16, 1e-4, 1e4)])
def test_keys_and_queries_near_the_ends_of_their_types(dtype, k_gain, q_gain):
    """Scores of ordinary size from factors of any: the keys' block scales and
    the query's own cancel before anything overflows or is lost."""
    gen = torch.Generator().manual_seed(61)
    lens = [200, 70, 3]
    host, dev = H.filled(gen, 5, HK, BLOCK, k_gain=k_gain)
    tables = H.tables_of(gen, lens, BLOCK, 5)
    q = (torch.randn(3, HQ, 128, generator=gen) * q_gain).to(dtype)
    scale = 128 ** -0.5 / (k_gain * q_gain)
    want = _want(q, host, tables, lens, scale)
    for form, weights, got in _both(q, dev, tables, lens, scale):
        assert got.isfinite().all(), form
        H.check(got, *want, dtype, max(lens), host[3].max(), weights)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_scores_of_any_size_keep_the_largest_key(dtype):
    """Scores far beyond exp2's range: the row is its best key's value."""
    gen = torch.Generator().manual_seed(62)
    k_gain = 1e34 if dtype == BF16 else 1e30
    lens = [200, 70, 3]
    host, dev = H.filled(gen, 5, HK, BLOCK, k_gain=k_gain)
    tables = H.tables_of(gen, lens, BLOCK, 5)
    q = torch.randn(3, HQ, 128, generator=gen).to(dtype)
    for form, _, got in _both(q, dev, tables, lens, 1.0):
        got = got.double().cpu().numpy()
        assert np.isfinite(got).all(), form
        for i, n in enumerate(lens):
            k, v = O.rows(host, tables[i], n)
            for h in range(HQ):
                kh = k[h * HK // HQ]
                s = kh @ q[i, h].double().numpy()
                order = np.argsort(s)
                # (2^-14 of the reach is what a score may be off by)
                reach = q[i, h].abs().max().item() * np.abs(kh).sum(-1).max()
                if s[order[-1]] - s[order[-2]] < 2.0 ** -12 * reach:
                    continue
                best = v[h * HK // HQ, order[-1]]
                # the value's fp16 product, the weight and the output's type round once each
                tol = (2.0 ** -10 + torch.finfo(dtype).eps / 2) * np.abs(best) + 1e-6
                assert (np.abs(got[i, h] - best) <= tol).all(), (form, i, h)


@pytest.mark.parametrize("sign", [1, -1, 0])
@pytest.mark.parametrize("splits", [False, True])
def test_prefill_scores_that_leave_the_exponents_range_on_the_way(sign, splits):
    """Keys of growing size, from ordinary scores to 10^14, above zero (+1) or of
    either sign (0), or of shrinking size and all scores below zero (-1).  Rows
    whose best key is clear are its value; the others stay finite."""
    gen = torch.Generator().manual_seed(66)
    lq, lc = (20, 2400) if splits else (150, 420)
    lk = lq + lc
    pool = -(-lk // BLOCK)
    base = torch.randn(HK, 128, generator=gen)
    k = base * (1 + 0.3 * torch.randn(lk, HK, 128, generator=gen)) if sign else torch.randn(
        lk, HK, 128, generator=gen)
    k = k * 10 ** (torch.linspace(0, 12, lk) if sign >= 0 else torch.linspace(12, 4, lk))[
        :, None, None]
    v = torch.randn(lk, HK, 128, generator=gen)
    host = H.empty(pool, HK, BLOCK)
    O.store(k.numpy(), v.numpy(), host, np.arange(lk))
    dev, table = H.to_gpu(host), np.arange(pool)
    q = torch.randn(lq, HQ, 128, generator=gen)
    if sign:
        q = sign * base.repeat_interleave(HQ // HK, 0) + 0.1 * q
    q = q.to(BF16)
    need = _lib.load().mskv_fp8_prefill_bounded_workspace_bytes(1, lq, lq, lk, HQ, HK, 128, BLOCK,
                                                                pool)
    assert (need > 0) == splits
    got = M.fp4_chunk_prefill_attention(q.to(H.DEV), *dev, _i32(table), lc, 1.0)
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all()
    kk, vv = O.rows(host, table, lk)
    clear = 0
    for h in range(HQ):
        kh, vh = kk[h * HK // HQ], vv[h * HK // HQ]
        s = q[:, h].double().numpy() @ kh.T
        off = 2.0 ** -13 * q[:, h].abs().amax(-1).double().numpy()[:, None] * np.abs(kh).sum(-1)
        for i in range(lq):
            n = lc + i + 1
            best = s[i, :n].argmax()
            rest = np.delete(np.arange(n), best)
            # (each score is off by its own key's bound, and 60 units leave nothing of the others)
            if s[i, best] - off[i, best] < (s[i, rest] + off[i, rest]).max() + 60:
                continue
            clear += 1
            tol = (2.0 ** -9 + torch.finfo(BF16).eps / 2) * np.abs(vh[best]) + 1e-6
            assert (np.abs(got[i, h] - vh[best]) <= tol).all(), (h, i)
    assert clear > lq * HQ // 8


def _queries(kind, rows, dtype, gen):
    x = torch.randn(rows, HQ, 128, generator=gen)
    if kind == "borders":  # a block's largest at, just below and just above 1.875 * 2^k
        x = x.clamp(-1.5, 1.5)
        tops = torch.tensor([1.875, 1.8671875, 1.8828125, 1.9921875, 1.0, -1.875, 1.125, -2.0])
        at = torch.randint(0, 32, (rows, HQ, 4), generator=gen) + 32 * torch.arange(4)
        pick = tops[torch.randint(0, 8, (rows, HQ, 4), generator=gen)]
        x.scatter_(2, at, pick * 2.0 ** torch.randint(0, 3, (rows, HQ, 4), generator=gen))
    elif kind == "spread":  # elements 2^-16 to 1 of the row's largest
        x = torch.sign(x) * torch.exp2(-16 * torch.rand(x.shape, generator=gen))
    elif kind == "outlier":
        x[..., 5] *= 1000
        x[..., 40] *= 60
    elif kind == "empty blocks":
        x[:, ::2, 32:64] = 0
        x[:, 1, :] = 0
        x[:, 2, 1:] = 0
    elif kind == "largest":  # (q . k stays in fp32's range)
        x *= (65504 if dtype == FP16 else 1e35) / x.abs().max()
    elif kind == "smallest":  # fp16's subnormals; bf16 above its own
        x *= 2e-7 if dtype == FP16 else 1e-34
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("kind", ["borders", "spread", "outlier", "empty blocks", "largest",
                                  "smallest"])
def test_queries_whose_parts_split_unevenly(dtype, kind):
    """Rows of a few keys under a scale that leaves the scores' errors in
    sight: reach is 8 at most."""
    gen = torch.Generator().manual_seed(63)
    lens = [2, 3, 5, 2, 2, 4]
    host, dev = H.filled(gen, 7, HK, BLOCK)
    tables = H.tables_of(gen, lens, BLOCK, 7)
    q = _queries(kind, len(lens), dtype, gen)
    _, _, reach = _want(q, host, tables, lens, 1.0)
    scale = float(np.float32(8 / reach.max()))
    want = _want(q, host, tables, lens, scale)
    for form, weights, got in _both(q, dev, tables, lens, scale):
        H.check(got, *want, dtype, max(lens), host[3].max(), weights)
