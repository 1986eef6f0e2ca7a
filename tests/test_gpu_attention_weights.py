"""Attention weights of cached tokens (a decode that keeps them, windows of
queries) against the definition in 64 bits."""

import numpy as np
import pytest
import torch

import microserve_amd as M
from oracle import weights_oracle as W
from tests import weights_helpers as H

pytestmark = pytest.mark.gpu
D = 128


def _setup(seed, lens, hq, hk, block, dtype, width=0, extra=3, gain=1.0):
    gen = torch.Generator().manual_seed(seed)
    pages = sum(-(-n // block) for n in lens) + extra
    host, dev = H.pool(gen, pages, hk, block, k_gain=gain)
    tables = H.tables_of(gen, lens, block, pages, width)
    weights = torch.rand(pages, hk, block, generator=gen)
    return gen, host, dev, tables, weights


def _decode_case(seed, lens, hq, hk, block, dtype, width=0, start=0, scale=D ** -0.5, gain=1.0,
                 spoil=None):
    gen, host, dev, tables, old = _setup(seed, lens, hq, hk, block, dtype, width, gain=gain)
    if spoil is not None:
        spoil(tables)
    q = torch.randn(len(lens), hq, D, generator=gen).to(dtype)
    weights = old.to(H.DEV)
    starts = list(start) if isinstance(start, (list, tuple)) else [start] * len(lens)
    given = H.gpu(starts) if isinstance(start, (list, tuple)) else start
    out = M.fp8_decode_attention_weights(q.to(H.DEV), *dev, H.gpu(lens), H.gpu(tables), scale,
                                         weights, start=given)
    plain = M.fp8_decode_attention(q.to(H.DEV), *dev, H.gpu(lens), H.gpu(tables), scale)
    torch.cuda.synchronize()
    assert torch.equal(out, plain)  # the same kernels' walk
    want = old.double().numpy()
    touched = np.zeros(want.shape, bool)
    reach, keys = 0.0, max(lens, default=0)
    for b, n in enumerate(lens):
        n = min(n, tables.shape[1] * block)
        if n <= 0:
            continue
        k, ok = W.rows_of(host[0], host[2], tables[b], n, block)
        p = W.probabilities(q[b:b + 1].double().numpy(), k, ok, scale, [n])
        sums = W.by_kv_head(p, hk)
        W.record(want, sums, ok, tables[b], starts[b], lambda t: t < n - 1)
        W.record(touched, np.ones(sums.shape, bool), ok, tables[b], starts[b], lambda t: False)
        reach = max(reach, H.reach_of(q[b].double().numpy(), k, scale))
    got = weights.cpu().numpy()
    assert np.array_equal(got[~touched], old.numpy()[~touched]), "an entry beside the tokens"
    H.check_weights(got, want, np.where(touched, 0.0, want), reach, keys, hq // hk)
    return got


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,hq,hk,block,width", [
    ([1], 4, 1, 32, 0), ([0], 8, 8, 256, 1), ([700], 16, 8, 256, 16), ([33, 0, 1, 256, 257], 32, 8, 256, 0),
    ([1500, 7, 1024, 0], 40, 8, 128, 40), ([95, 96, 97], 12, 4, 96, 3), ([2000, 31], 40, 2, 512, 4),
    ([300] * 5, 17, 1, 256, 2), ([5000], 24, 1, 256, 64)])
def test_decode_weights(dtype, lens, hq, hk, block, width):
    _decode_case(sum(lens) + hq, lens, hq, hk, block, dtype, width)


@pytest.mark.parametrize("start", [0, 5, 256, 258, 5000, [0, 300, 299, 511]])
def test_decode_weights_from_a_start(start):
    _decode_case(7, [300, 300, 300, 512], 8, 2, 256, torch.bfloat16, start=start)


def test_decode_weights_in_work_items_and_long_tables():
    rng = np.random.default_rng(3)
    lens = [int(x) for x in np.exp(rng.uniform(np.log(1), np.log(3000), 40))]
    lens[0] = 9000
    assert M.decode_num_splits(len(lens), 8, 8, 128, 256) * len(lens) > 512
    _decode_case(4, lens, 8, 8, 256, torch.float16, width=128)


def test_decode_weights_of_invalid_pages_and_tables_end():
    def spoil(tables):
        tables[0, 0] = -1
        tables[1, 1] = 10 ** 6
        tables[2, :] = -1
    _decode_case(5, [600, 600, 100, 40], 8, 4, 256, torch.float16, spoil=spoil)
    _decode_case(6, [64, 200], 8, 4, 64, torch.float16)
    gen, host, dev, tables, old = _setup(9, [512, 256], 8, 4, 256, torch.float16)
    lens = [5000, 256]  # past the table's width: its tokens alone
    q = torch.randn(2, 8, D, generator=gen).half().to(H.DEV)
    a, b = (old.to(H.DEV) for _ in range(2))
    M.fp8_decode_attention_weights(q, *dev, H.gpu(lens), H.gpu(tables), 0.1, a)
    M.fp8_decode_attention_weights(q, *dev, H.gpu([512, 256]), H.gpu(tables), 0.1, b)
    torch.cuda.synchronize()
    assert torch.equal(a, b)


def test_decode_weights_of_large_scores():
    """Scores of thousands: one token takes everything, the others nothing."""
    got = _decode_case(8, [500, 100], 8, 2, 256, torch.bfloat16, scale=3.0, gain=30.0)
    assert np.isfinite(got).all()


def test_decode_weights_without_room_for_scores():
    """Tables so wide that a step's scores would pass 1 GiB: K is read again."""
    from microserve_amd import _lib
    lib, width = _lib.load(), 1 << 15
    assert lib.mskv_decode_weights_workspace_bytes(3, 16, 4, 256, width) < 3 * 16 * width * 256 * 4
    _decode_case(11, [700, 0, 257], 16, 4, 256, torch.float16, width=width)
    _decode_case(12, [1, 513, 40], 16, 4, 256, torch.bfloat16, width=width, start=[0, 300, 2])


def test_nan_in_a_query_stays_in_its_sequence():
    gen, host, dev, tables, old = _setup(13, [300, 200], 4, 2, 256, torch.float16)
    q = torch.randn(2, 4, D, generator=gen).half()
    q[0, 1, 5] = float("nan")  # kv head 0 of sequence 0
    w = old.to(H.DEV)
    M.fp8_decode_attention_weights(q.to(H.DEV), *dev, H.gpu([300, 200]), H.gpu(tables), 0.1, w)
    got = w.cpu()
    for page, n in ((tables[0, 0], 256), (tables[0, 1], 44)):
        assert got[page, 0, :n].isnan().all() and got[page, 1].isfinite().all()
    assert got[tables[1, 0]].isfinite().all()


def _window_case(seed, new, lens, hq, hk, block, dtype, accumulate, width=0, start=0,
                 scale=D ** -0.5, max_k=True, spoil=None, spare=0):
    gen, host, dev, tables, old = _setup(seed, lens, hq, hk, block, dtype, width)
    if spoil is not None:
        spoil(tables)
    q = torch.randn(sum(new) + spare, hq, D, generator=gen).to(dtype)
    cu_q, cu_k = np.cumsum([0, *new]), np.cumsum([0, *lens])
    weights = old.to(H.DEV)
    got = M.fp8_window_attention_weights(
        q.to(H.DEV), dev[0], dev[2], H.gpu(tables), H.gpu(cu_q), H.gpu(cu_k), max(new, default=0),
        scale, weights, accumulate=accumulate, start=start,
        max_seqlen_k=max(lens, default=1) if max_k else None)
    assert got is weights
    torch.cuda.synchronize()
    want, touched = old.double().numpy(), np.zeros(old.shape, bool)
    reach = 0.0
    for b, (n, lq) in enumerate(zip(lens, new)):
        if n == 0:
            continue
        k, ok = W.rows_of(host[0], host[2], tables[b], n, block)
        rows = q[cu_q[b]:cu_q[b + 1]].double().numpy()
        p = W.probabilities(rows, k, ok, scale, n - lq + 1 + np.arange(lq))
        sums = W.by_kv_head(p, hk)
        W.record(want, sums, ok, tables[b], start, lambda t: accumulate)
        W.record(touched, np.ones(sums.shape, bool), ok, tables[b], start, lambda t: False)
        reach = max(reach, H.reach_of(rows, k, scale))
    got = got.cpu().numpy()
    assert np.array_equal(got[~touched], old.numpy()[~touched]), "an entry beside the tokens"
    H.check_weights(got, want, np.where(touched & ~np.bool_(False), 0.0, want), reach,
                    max(lens, default=0), hq // hk * max(new, default=0))


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new,lens,hq,hk,block,width", [
    ([1], [1], 8, 8, 128, 0), ([16], [600], 16, 8, 256, 0), ([32, 5, 1], [1000, 5, 300], 32, 8, 256, 9),
    ([64, 0, 3], [64, 77, 0], 4, 1, 256, 0), ([33], [257], 40, 8, 128, 0), ([7, 40], [700, 511], 17, 1, 512, 0),
    ([100], [300], 12, 4, 128, 0), ([3], [2500], 64, 2, 256, 0), ([5, 9], [3, 4], 8, 2, 256, 0)])
def test_window_weights(new, lens, hq, hk, block, width, dtype, accumulate):
    _window_case(sum(lens) + hq, new, lens, hq, hk, block, dtype, accumulate, width)


@pytest.mark.parametrize("group", [4, 13])
def test_window_weights_of_many_sequences(group):
    """More sequences than a wave has lanes, some without queries, some without
    tokens; rows of one turn and of several side by side."""
    rng = np.random.default_rng(group)
    lens = [int(x) for x in rng.integers(0, 300, 90)]
    lens[7], lens[70] = 2000, 1300
    new = [int(rng.integers(0, min(n, 40) + 1)) for n in lens]
    new[7], new[70] = 33, 1
    _window_case(group, new, lens, 2 * group, 2, 128, torch.bfloat16, False, 0)


def test_window_weights_from_a_start_and_without_a_bound():
    _window_case(3, [8, 8], [600, 300], 8, 2, 256, torch.bfloat16, True, start=290, max_k=False)
    _window_case(4, [8], [600], 8, 2, 256, torch.float16, False, start=10 ** 6)


def test_window_weights_of_invalid_pages_and_padded_queries():
    def spoil(tables):
        tables[0, 1] = -1
        tables[1, 0] = 10 ** 6
    _window_case(5, [20, 20], [700, 200], 8, 2, 256, torch.float16, False, spoil=spoil)
    _window_case(6, [9, 4], [500, 50], 8, 2, 128, torch.bfloat16, True, spare=30)


def test_window_of_no_sequences_and_no_queries():
    _window_case(7, [0, 0], [300, 9], 8, 2, 256, torch.float16, False)
    _window_case(8, [0, 0], [300, 9], 8, 2, 256, torch.float16, True)
    w = M.allocate_attention_weights(2, 128, 2)
    kv, sc = torch.zeros(2, 128, 2, D, device=H.DEV).to(torch.float8_e4m3fn), torch.ones(2, 128, 2, device=H.DEV)
    q = torch.zeros(0, 4, D, device=H.DEV).half()
    empty = torch.zeros(0, 1, dtype=torch.int32, device=H.DEV)
    zero = torch.zeros(1, dtype=torch.int32, device=H.DEV)
    M.fp8_window_attention_weights(q, kv, sc, empty, zero, zero, 0, 0.1, w)
    M.fp8_decode_attention_weights(q, kv, kv, sc, sc, zero[:0], empty, 0.1, w)
    assert not w.any()


def test_window_of_one_query_is_the_decode():
    gen, host, dev, tables, old = _setup(21, [900, 40], 8, 2, 256, torch.bfloat16)
    q = torch.randn(2, 8, D, generator=gen).bfloat16().to(H.DEV)
    a, b = torch.zeros_like(old).to(H.DEV), torch.zeros_like(old).to(H.DEV)
    M.fp8_decode_attention_weights(q, *dev, H.gpu([900, 40]), H.gpu(tables), 0.09, a)
    M.fp8_window_attention_weights(q, dev[0], dev[2], H.gpu(tables), H.gpu([0, 1, 2]),
                                   H.gpu([0, 900, 940]), 1, 0.09, b)
    assert torch.allclose(a, b, rtol=1e-4, atol=1e-30)  # (two orders of the same sums)
    assert abs(float(a.sum()) - 2 * 8) < 1e-3


def test_captured_decode_weights_replay():
    gen, host, dev, tables, old = _setup(31, [900, 300, 0], 8, 2, 256, torch.float16, width=8)
    q = torch.randn(3, 8, D, generator=gen).half().to(H.DEV)
    lens, t = H.gpu([900, 300, 0]), H.gpu(tables)
    w, eager = old.to(H.DEV), old.to(H.DEV)
    call = lambda x: M.fp8_decode_attention_weights(q, *dev, lens, t, 0.1, x)  # noqa: E731
    call(torch.zeros_like(w))
    torch.cuda.synchronize()
    graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=s):
        out = call(w)
    for step in range(3):
        lens.copy_(torch.tensor([900 - step, 300, step], dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        want = call(eager)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(w, eager), f"replay {step}"
