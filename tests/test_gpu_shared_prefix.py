"""Decode over shared prefixes against the definition in 64 bits and against the
decode that reads every sequence's pages."""

import numpy as np
import pytest
import torch

import microserve_amd as M
from oracle import weights_oracle as W
from tests import weights_helpers as H

pytestmark = pytest.mark.gpu
D = 128


def _batch(gen, sizes, prefixes, tails, block, width=0, extra=2):
    """(lens, tables, pool): groups of `sizes` sequences over prefixes of whole
    pages, each with a tail of its own."""
    lens, rows, used = [], [], 0
    tails = list(tails)
    for n, p in zip(sizes, prefixes):
        shared = list(range(used, used + p // block))
        used += len(shared)
        for _ in range(n):
            length = p + tails.pop(0)
            own = -(-length // block) - len(shared)
            rows.append(shared + list(range(used, used + own)))
            used += own
            lens.append(length)
    pool = used + extra
    order = torch.randperm(pool, generator=gen).numpy()
    tables = np.full((len(rows), max([width, 1, *map(len, rows)])), -1, np.int32)
    for i, r in enumerate(rows):
        tables[i, :len(r)] = order[r]
    return lens, tables, pool


def _check(gen, lens, tables, pool, sizes, prefixes, hq, hk, block, dtype, scale=D ** -0.5,
           bound=None, gain=1.0, spoil=None, cu=None):
    host, dev = H.pool(gen, pool, hk, block, k_gain=gain)
    if spoil is not None:
        spoil(tables)
    q = torch.randn(len(lens), hq, D, generator=gen).to(dtype)
    cu = np.cumsum([0, *sizes]) if cu is None else cu
    args = (q.to(H.DEV), *dev, H.gpu(lens), H.gpu(tables), scale)
    out = M.fp8_shared_prefix_decode_attention(*args, H.gpu(cu), H.gpu(prefixes),
                                               max_prefix_len=bound)
    torch.cuda.synchronize()
    reach, keys = 0.0, max(lens, default=0)
    want, weight = (np.zeros((len(lens), hq, D)) for _ in range(2))
    for b, n in enumerate(lens):
        n = min(n, tables.shape[1] * block)
        if n <= 0:
            continue
        k, ok = W.rows_of(host[0], host[2], tables[b], n, block)
        v, _ = W.rows_of(host[1], host[3], tables[b], n, block)
        p = W.probabilities(q[b:b + 1].double().numpy(), k, ok, scale, [n])[0]
        for h in range(hq):
            want[b, h] = p[h] @ v[:, h * hk // hq]
            weight[b, h] = p[h] @ np.abs(v[:, h * hk // hq])
        reach = max(reach, H.reach_of(q[b].double().numpy(), k, scale))
    H.check_out(out, want, weight, reach, dtype, keys, host[3].max(), 1)
    return out, args


CASES = [
    # sizes, prefixes, tails, hq, hk, block, table width
    ([1], [256], [1], 8, 8, 256, 0), ([2], [128], [1, 5], 4, 1, 128, 0),
    ([4], [1024], [60, 1, 61, 300], 16, 8, 256, 32), ([3, 2], [512, 0], [5, 6, 7, 300, 2], 32, 8, 256, 0),
    ([33], [768], [40] * 33, 32, 8, 256, 0), ([40, 1, 9], [512, 256, 1536], range(50), 40, 8, 128, 0),
    ([65], [256], range(1, 66), 17, 1, 256, 0), ([5, 6], [640, 384], [700] * 11, 12, 4, 128, 20),
    ([3, 3], [2048, 256], [1, 0, 0, 0, 0, 3], 40, 2, 256, 0), ([12] * 5, [256] * 5, [90] * 60, 24, 1, 256, 0)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("sizes,prefixes,tails,hq,hk,block,width", CASES)
def test_shared_prefix(sizes, prefixes, tails, hq, hk, block, width, dtype):
    gen = torch.Generator().manual_seed(sum(sizes) + hq)
    lens, tables, pool = _batch(gen, sizes, prefixes, tails, block, width)
    _check(gen, lens, tables, pool, sizes, prefixes, hq, hk, block, dtype)


@pytest.mark.parametrize("bound", [0, 100, 256, 1000, 10 ** 9])
def test_bounds_below_and_above_the_prefix(bound):
    gen = torch.Generator().manual_seed(bound % 97)
    lens, tables, pool = _batch(gen, [3, 4], [768, 512], [30] * 7, 256)
    _check(gen, lens, tables, pool, [3, 4], [768, 512], 8, 2, 256, torch.float16, bound=bound)


@pytest.mark.parametrize("prefixes", [[300, 511], [1, 0], [-5, 10 ** 8]])
def test_prefixes_that_are_no_whole_tiles(prefixes):
    gen = torch.Generator().manual_seed(5)
    lens, tables, pool = _batch(gen, [3, 4], [768, 512], [30] * 7, 256)
    # (as long as a prefix is at most what the tables share, it may say less;
    # past the shortest sequence it is cut)
    if max(prefixes) > 768:
        lens, tables, pool = _batch(gen, [3, 4], [768, 512], [0] * 7, 256)
    _check(gen, lens, tables, pool, [3, 4], prefixes, 8, 2, 256, torch.bfloat16)


def test_padding_sequences_and_groups():
    """Rows of no tokens and -1 tables, first and last of a group; empty groups;
    sequences outside every group; a sequence shorter than its group's prefix."""
    gen = torch.Generator().manual_seed(6)
    lens, tables, pool = _batch(gen, [6, 3], [512, 256], [9, 300, 10, 11, 12, 13, 5, 6, 7], 256)
    for b in (0, 4, 8):
        lens[b], tables[b] = 0, -1
    out, _ = _check(gen, lens, tables, pool, [6, 3], [512, 256], 16, 4, 256, torch.float16)
    assert not out[[0, 4, 8]].any()
    lens[2] = 200
    _check(gen, lens, tables, pool, None, [512, 0, 256, 256], 16, 4, 256, torch.float16,
           cu=[1, 5, 5, 6, 8])
    _check(gen, lens, tables, pool, None, [], 16, 4, 256, torch.float16, cu=[0])
    _check(gen, [0] * 9, tables, pool, [9], [512], 16, 4, 256, torch.float16)


def test_groups_that_do_not_ascend_end():
    """No result is promised; every read stays inside, and the next call is right."""
    gen = torch.Generator().manual_seed(21)
    sizes, prefixes = [3, 4], [256, 512]
    lens, tables, pool = _batch(gen, sizes, prefixes, range(20, 27), 128)
    _, args = _check(gen, lens, tables, pool, sizes, prefixes, 8, 2, 128, torch.float16)
    want = M.fp8_shared_prefix_decode_attention(*args, H.gpu([0, 3, 7]), H.gpu(prefixes))
    for cu in ([7, 3, 0], [0, 7, 3], [5, 5, 5], [-9, 99, 2], [3, 0, 7]):
        M.fp8_shared_prefix_decode_attention(*args, H.gpu(cu), H.gpu(prefixes))
        torch.cuda.synchronize()
    got = M.fp8_shared_prefix_decode_attention(*args, H.gpu([0, 3, 7]), H.gpu(prefixes))
    assert torch.equal(got, want)


def test_invalid_pages_are_skipped():
    def spoil(tables):
        tables[:3, 1] = -1      # of a prefix
        tables[3, 3] = 10 ** 6  # of a tail
        tables[4:, 0] = 10 ** 6
    gen = torch.Generator().manual_seed(7)
    lens, tables, pool = _batch(gen, [3, 1, 2], [768, 512, 512], [30, 40, 50, 700, 1, 2], 256)
    _check(gen, lens, tables, pool, [3, 1, 2], [768, 512, 512], 8, 2, 256, torch.bfloat16,
           spoil=spoil)
    lens, tables, pool = _batch(gen, [2], [512], [0, 0], 256)
    tables[:] = -1
    out, _ = _check(gen, lens, tables, pool, [2], [512], 8, 2, 256, torch.float16)
    assert not out.any()


def test_large_scores_and_many_groups():
    gen = torch.Generator().manual_seed(8)
    lens, tables, pool = _batch(gen, [5], [512], [100] * 5, 128)
    _check(gen, lens, tables, pool, [5], [512], 8, 2, 128, torch.bfloat16, scale=2.0, gain=30.0)
    sizes = [1, 2, 3] * 100
    lens, tables, pool = _batch(gen, sizes, [128] * 300, [3] * 600, 128)
    _check(gen, lens, tables, pool, sizes, [128] * 300, 4, 1, 128, torch.float16)


def test_of_no_sequences_and_into_out():
    gen = torch.Generator().manual_seed(9)
    lens, tables, pool = _batch(gen, [2], [256], [4, 5], 256)
    got, args = _check(gen, lens, tables, pool, [2], [256], 8, 2, 256, torch.float16)
    out = torch.empty_like(got)
    cu, pre = H.gpu([0, 2]), H.gpu([256])
    assert M.fp8_shared_prefix_decode_attention(*args, cu, pre, out=out) is out
    assert torch.equal(out, got)
    e = H.gpu(np.zeros((0,)))
    none = M.fp8_shared_prefix_decode_attention(args[0][:0], *args[1:5], args[5][:0], args[6][:0],
                                                0.1, H.gpu([0]), e)
    assert none.shape == (0, 8, D)


def test_nan_in_a_query_stays_in_its_row_and_scores_of_nan_keys_in_their_group():
    gen = torch.Generator().manual_seed(10)
    lens, tables, pool = _batch(gen, [3, 2], [512, 256], [30] * 5, 256)
    host, dev = H.pool(gen, pool, 2, 256)
    q = torch.randn(5, 8, D, generator=gen).half()
    q[1, 3, 7] = float("nan")
    dev[2][int(tables[3, 0]), 5, 1] = float("nan")  # a key scale of group 1's prefix, kv head 1
    out = M.fp8_shared_prefix_decode_attention(q.to(H.DEV), *dev, H.gpu(lens), H.gpu(tables), 0.1,
                                               H.gpu([0, 3, 5]), H.gpu([512, 256])).cpu()
    bad = torch.zeros(5, 8, dtype=torch.bool)
    bad[1, 3], bad[3:, 4:] = True, True
    assert out[bad].isnan().all() and out[~bad].isfinite().all()


def test_captured_replays_follow_lengths_and_groups():
    gen = torch.Generator().manual_seed(11)
    lens, tables, pool = _batch(gen, [3, 2, 1], [512, 768, 256], [30] * 6, 256, width=8)
    host, dev = H.pool(gen, pool, 2, 256)
    q = torch.randn(6, 8, D, generator=gen).half().to(H.DEV)
    n, t = H.gpu(lens), H.gpu(tables)
    cu, pre = H.gpu([0, 3, 5, 6]), H.gpu([512, 768, 256])
    call = lambda: M.fp8_shared_prefix_decode_attention(q, *dev, n, t, 0.1, cu, pre, 1024)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=s):
        out = call()
    for new, bounds, shared in ((lens, [0, 3, 5, 6], [512, 768, 256]),
                                ([520, 600, 540, 0, 790, 1], [0, 2, 3, 6], [256, 512, 0]),
                                ([513] * 3 + [769] * 2 + [300], [0, 0, 5, 6], [0, 0, 256])):
        n.copy_(torch.tensor(new, dtype=torch.int32))
        cu.copy_(torch.tensor(bounds, dtype=torch.int32))
        pre.copy_(torch.tensor(shared, dtype=torch.int32))
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        full = M.fp8_decode_attention(q, *dev, n, t, 0.1)
        # (two roundings of half a step to fp16, of outputs below 4, and weights')
        assert (out.float() - full.float()).abs().max() < 2 ** -8


def test_two_streams_at_once():
    gen = torch.Generator().manual_seed(12)
    work = []
    for i in range(2):
        lens, tables, pool = _batch(gen, [20, 9], [1024, 512], [100 + i] * 29, 256)
        host, dev = H.pool(gen, pool, 4, 256)
        q = torch.randn(29, 16, D, generator=gen).bfloat16().to(H.DEV)
        args = (q, *dev, H.gpu(lens), H.gpu(tables), 0.1, H.gpu([0, 20, 29]), H.gpu([1024, 512]))
        work.append((args, M.fp8_shared_prefix_decode_attention(*args), torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, (args, _, stream) in enumerate(work):
            with torch.cuda.stream(stream):
                outs[i].append(M.fp8_shared_prefix_decode_attention(*args))
    torch.cuda.synchronize()
    for i, (_, want, _) in enumerate(work):
        assert all(torch.equal(o, want) for o in outs[i])
