"""Decode and prefill attention over the 4-bit cache against the oracle in 64
bits, and a run of a layer's steps over one."""

import numpy as np
import pytest
import torch

import microserve_amd as M
from microserve_amd import _lib
from oracle import fp4_oracle as O
from tests import fp4_helpers as H

pytestmark = pytest.mark.gpu

SCALE = 128 ** -0.5
BF16, FP16 = torch.bfloat16, torch.float16


def _i32(x):
    return torch.as_tensor(x, dtype=torch.int32, device=H.DEV)


def _decode_want(q, caches, lens, tables, scale):
    outs = []
    for i, n in enumerate(lens):
        n = min(n, tables.shape[1] * caches[1].shape[2])
        k, v = O.rows(caches, tables[i], n)
        seen = ~np.isnan(k[0, :, 0])[None]  # (pages outside the pool are not seen)
        outs.append(O.attend(q[i:i + 1].float().numpy(), k, v, scale, seen))
    return [np.concatenate(x) for x in zip(*outs)]


def _decode(seed, lens, hq, hk, block, dtype, width=0, scale=SCALE, extra=1):
    gen = torch.Generator().manual_seed(seed)
    pool = sum(-(-n // block) for n in lens) + extra
    host, dev = H.filled(gen, pool, hk, block)
    tables = H.tables_of(gen, lens, block, pool, width)
    q = torch.randn(len(lens), hq, 128, generator=gen).to(dtype)
    return host, dev, tables, q


def _check_decode(host, dev, tables, q, lens, scale=SCALE):
    got = M.fp4_decode_attention(q.to(H.DEV), *dev, _i32(lens), _i32(tables), scale)
    want = _decode_want(q, host, lens, tables, scale)
    H.check(got, *want, q.dtype, max(lens, default=1), np.nanmax(host[3]), 1)
    for i, n in enumerate(lens):
        if n == 0:
            assert (got[i] == 0).all()
    return got


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lens,hq,hk,block,width", [
    ([1], 8, 8, 128, 0), ([2], 4, 1, 256, 3), ([63, 64, 65], 8, 2, 128, 0),
    ([0, 127, 128, 129], 16, 8, 128, 0), ([0], 4, 4, 128, 2), ([255, 1, 0, 257], 32, 8, 256, 128),
    ([700], 16, 8, 256, 128), ([1000, 3], 40, 8, 384, 0), ([511], 24, 1, 256, 0),
    ([500, 130], 34, 2, 128, 16), ([2100], 12, 4, 256, 0)])
def test_decode_matches_the_oracle(dtype, lens, hq, hk, block, width):
    _check_decode(*_decode(1 + len(lens), lens, hq, hk, block, dtype, width), lens)


@pytest.mark.parametrize("lens,hq,hk,block,width,kind", [
    ([1, 64, 65, 128, 129, 0, 255, 256, 257, 511, 512, 513, 1000, 1024], 34, 2, 128, 8,
     "joined, with idle lanes"),
    ([1, 320, 64] * 23, 8, 8, 128, 0, "joined"),
    ([8192, 70] + [300] * 15, 16, 16, 256, 0, "joined, the longest"),
    ([90, 128, 1] * 40, 32, 32, 128, 0, "a wave each"),
    ([100, 0, 128] * 400, 8, 8, 128, 0, "a wave each, of more workgroups"),
    ([130] * 63 + [5000], 8, 8, 256, 64, "splits of the shape"),
    ([40, 900, 3, 0, 260] * 24, 4, 4, 128, 66, "work items of few heads"),
    ([60, 1500, 2, 0, 128, 700] * 24, 8, 8, 128, 65, "work items"),
    ([5000, 70, 1, 0], 8, 1, 128, 64, "splits that follow the lengths"),
    ([9000], 2, 2, 128, 70, "the wide merge")])
def test_decode_of_every_launch_form(lens, hq, hk, block, width, kind):
    _check_decode(*_decode(41, lens, hq, hk, block, BF16, width), lens)


def test_decode_lengths_past_the_table_are_cut():
    host, dev, tables, q = _decode(5, [128, 256], 8, 2, 128, FP16)
    _check_decode(host, dev, tables, q, [5000, 300])


# tables of a few pages: a workgroup takes a head's whole sequence; of many: the
# sequences are split and merged
WIDTHS = pytest.mark.parametrize("width", [8, 60])


@WIDTHS
def test_decode_skips_blocks_outside_the_pool(width):
    host, dev, tables, q = _decode(6, [300, 400, 100], 8, 2, 128, BF16, width)
    tables[0, 0], tables[1, 2], tables[2, 0] = 999, -7, -1
    got = _check_decode(host, dev, tables, q, [300, 400, 100])
    assert (got[2] == 0).all()


@WIDTHS
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.5])
def test_decode_of_any_scale(scale, width):
    host, dev, tables, q = _decode(7, [200, 70], 8, 2, 128, FP16, width)
    _check_decode(host, dev, tables, q, [200, 70], scale)


@WIDTHS
@pytest.mark.parametrize("ratio", [1e3, 1e5, 1e-5])
def test_values_of_very_different_sizes(ratio, width):
    """One key a step whose V is `ratio` times the others', with a low score:
    the others keep their precision."""
    gen = torch.Generator().manual_seed(14)
    host, dev = H.filled(gen, 4, 2, 128, v_gain=0.01 if ratio > 1 else 10.0)
    tables = np.full((1, width), -1, np.int32)
    tables[0, :3] = 2, 0, 3
    q = torch.randn(1, 8, 128, generator=gen).to(BF16)
    for page in tables[0, :3]:
        host[3][page, :, 5::64] *= np.float32(ratio)
        host[0][page, :, 0::4, :, 5] = 0  # score 0 by codes of 0
    dev = H.to_gpu(host)
    want = _decode_want(q, host, [380], tables, 4 * SCALE)
    got = M.fp4_decode_attention(q.to(H.DEV), *dev, _i32([380]), _i32(tables), 4 * SCALE)
    H.check(got, *want, BF16, 380, host[3].max(), 1)
    row = M.fp4_chunk_prefill_attention(q.to(H.DEV), *dev, _i32(tables[0]), 379, 4 * SCALE)
    H.check(row, *want, BF16, 380, host[3].max(), 4)


@WIDTHS
@pytest.mark.parametrize("where", ["query", "key", "value"])
def test_a_nan_reaches_the_rows_that_see_it_and_no_other(where, width):
    lens = [200, 500, 70]
    host, dev, tables, q = _decode(8, lens, 8, 2, 128, FP16, width)
    page = tables[1, 2]
    if where == "query":
        q[1, 4, 100] = float("nan")
        q[1, 5, 0] = float("inf")
        q[1, 6:8] = float("nan")
    elif where == "key":
        host[2][page, 1, 0, 2, 9, 1] = O.NAN_SCALE
    else:
        host[3][page, 1, 25] = np.nan
    dev = H.to_gpu(host)
    got = M.fp4_decode_attention(q.to(H.DEV), *dev, _i32(lens), _i32(tables), SCALE).cpu()
    bad = got.isnan()
    assert bad[1, 4:].all() and bad.sum() == bad[1, 4:].numel()
    chunk = torch.stack([q[1]] * 300).to(H.DEV)
    got = M.fp4_chunk_prefill_attention(chunk, *dev, _i32(tables[1]), 200, SCALE).cpu()
    first = {"query": 0, "key": 256 + 16 + 9 - 200, "value": 256 + 25 - 200}[where]
    bad = got.isnan()
    assert bad[first:, 4:].all() and not bad[:first].any() and not bad[:, :4].any()


@WIDTHS
def test_garbage_behind_the_last_token_is_not_seen(width):
    """Scales of NaN and infinity, and any codes, behind the sequence's end
    and in its unused pages."""
    for n in (1, 60, 64, 100, 128, 190):
        host, dev, tables, q = _decode(15, [n], 8, 2, 128, BF16, width, extra=2)
        want = _decode_want(q, host, [n], tables, SCALE)
        pages = -(-n // 128)
        used = np.zeros((host[1].shape[0], 128), bool)
        for i in range(pages):
            used[tables[0, i], :min(128, n - 128 * i)] = True
        host[3][~used[:, None].repeat(2, 1)] = np.nan
        host[1][~used[:, None].repeat(2, 1)] = 0xFF
        t = np.arange(128)
        for page in range(len(used)):
            for tok in t[~used[page]]:
                host[2][page, :, tok // 64, :, tok % 16, tok // 16 % 4] = 254 + tok % 2
        dev = H.to_gpu(host)
        got = M.fp4_decode_attention(q.to(H.DEV), *dev, _i32([n]), _i32(tables), SCALE)
        H.check(got, *want, BF16, n, 1.0, 1)
        got = M.fp4_chunk_prefill_attention(q.to(H.DEV), *dev, _i32(tables[0]), n - 1, SCALE)
        H.check(got, *want, BF16, n, 1.0, 4)


@WIDTHS
def test_decode_graph_replays_with_new_lengths_beside_eager_calls(width):
    lens = [300, 900, 0, 64]
    host, dev, tables, q = _decode(16, lens, 8, 2, 128, BF16, width)
    q, lens_t, tables_t = q.to(H.DEV), _i32(lens), _i32(tables)
    out = torch.empty_like(q)

    def step():
        M.fp4_decode_attention(q, *dev, lens_t, tables_t, SCALE, out=out)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for new in ([300, 900, 0, 64], [1, 2, 3, 4], [384, 1024, 128, 128], [0, 0, 0, 0]):
        new = [min(n, 128 * int((tables[i] >= 0).sum())) for i, n in enumerate(new)]
        lens_t.copy_(_i32(new))
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        eager = M.fp4_decode_attention(q, *dev, lens_t, tables_t, SCALE)
        assert torch.equal(got, eager)


def test_calls_on_two_streams_at_once():
    cases = [_decode(20 + i, lens, 16, 2, 128, BF16, width=30)
             for i, lens in enumerate(([3000], [1, 900, 2500]))]
    lens = [[3000], [1, 900, 2500]]
    args = [(q.to(H.DEV), *dev, _i32(n), _i32(t), SCALE) for (_, dev, t, q), n in zip(cases, lens)]
    want = [M.fp4_decode_attention(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].append(M.fp4_decode_attention(*args[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])


def test_no_sequences_and_caches_that_start_on_an_odd_byte():
    host, dev, tables, q = _decode(31, [200, 130], 8, 2, 128, FP16)
    none = M.fp4_decode_attention(q[:0].to(H.DEV), *dev, _i32([]), _i32(tables[:0]), SCALE)
    assert none.shape == (0, 8, 128)
    none = M.fp4_varlen_prefill_attention(q[:0].to(H.DEV), *dev, _i32(tables[:0]), _i32([0]),
                                          _i32([0]), 0, SCALE)
    assert none.shape == (0, 8, 128)
    flat = torch.zeros(dev[0].numel() + 4, dtype=torch.uint8, device=H.DEV)
    odd = flat[1:1 + dev[0].numel()].view(dev[0].shape)
    with pytest.raises(Exception, match="status -1"):
        M.fp4_decode_attention(q.to(H.DEV), odd, *dev[1:], _i32([200, 130]), _i32(tables), SCALE)
    with pytest.raises(Exception, match="status -1"):
        M.fp4_chunk_prefill_attention(q.to(H.DEV), odd, *dev[1:], _i32(tables[0]), 3, SCALE)


def test_out_and_views():
    lens = [100, 90]
    host, dev, tables, q = _decode(22, lens, 8, 2, 128, FP16)
    args = (*dev, _i32(lens), _i32(tables), SCALE)
    want = M.fp4_decode_attention(q.to(H.DEV), *args)
    out = torch.empty_like(want)
    assert M.fp4_decode_attention(q.to(H.DEV), *args, out=out) is out and torch.equal(out, want)
    wide = torch.zeros(2, 16, 128, dtype=FP16, device=H.DEV)
    wide[:, ::2] = q.to(H.DEV)
    assert torch.equal(M.fp4_decode_attention(wide[:, ::2], *args), want)
    flat = torch.zeros(2 * 8 * 128 + 3, dtype=FP16, device=H.DEV)
    flat[3:] = q.to(H.DEV).flatten()
    assert torch.equal(M.fp4_decode_attention(flat[3:].view(2, 8, 128), *args), want)
    with pytest.raises(AssertionError):
        M.fp4_decode_attention(q.to(H.DEV), *args, out=out[:1])
    with pytest.raises(AssertionError):
        M.fp4_decode_attention(q.to(H.DEV).float(), *args)
    with pytest.raises(AssertionError):
        M.fp4_decode_attention(q.to(H.DEV), *dev, _i32(lens), _i32(tables).long(), SCALE)
    assert M.fp4_decode_attention(q[:0].to(H.DEV), *dev, _i32([]), _i32(tables[:0]),
                                  SCALE).shape == (0, 8, 128)


# ------------------------------------------------------------------ prefill --

def _prefill_want(q, caches, tables, lq, lk, scale):
    outs, at = [], 0
    for i, (n, m) in enumerate(zip(lq, lk)):
        k, v = O.rows(caches, tables[i], max(m, 0))
        seen = np.arange(max(m, 0))[None] < (m - n + 1 + np.arange(n))[:, None]
        seen &= ~np.isnan(k[0, :, 0])[None]
        outs.append(O.attend(q[at:at + n].float().numpy(), k, v, scale, seen))
        at += n
    return [np.concatenate(x) for x in zip(*outs)]


def _cu(x):
    return _i32(np.concatenate(([0], np.cumsum(x))))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lq,lc,hq,hk,block", [
    ([1], [0], 4, 4, 128), ([1, 2, 1], [0, 127, 128], 8, 2, 128), ([31], [273], 16, 8, 256),
    ([130, 5, 64], [0, 500, 63], 8, 2, 128), ([33, 1], [95, 1000], 5, 1, 256),
    ([20, 7], [300, 2], 24, 1, 128), ([200], [56], 12, 4, 384), ([9], [2500], 8, 1, 128)])
def test_prefill_matches_the_oracle(dtype, lq, lc, hq, hk, block):
    gen = torch.Generator().manual_seed(31 + len(lq))
    lk = [a + b for a, b in zip(lq, lc)]
    pool = sum(-(-n // block) for n in lk) + 1
    host, dev = H.filled(gen, pool, hk, block)
    tables = H.tables_of(gen, lk, block, pool)
    q = torch.randn(sum(lq), hq, 128, generator=gen).to(dtype)
    want = _prefill_want(q, host, tables, lq, lk, SCALE)
    args = (q.to(H.DEV), *dev, _i32(tables), _cu(lq), _cu(lk), max(lq), SCALE)
    got = M.fp4_varlen_prefill_attention(*args, max_seqlen_k=max(lk))
    H.check(got, *want, dtype, max(lk), host[3].max(), 4)
    H.check(M.fp4_varlen_prefill_attention(*args), *want, dtype, max(lk), host[3].max(), 4)
    if len(lq) == 1:
        one = M.fp4_chunk_prefill_attention(q.to(H.DEV), *dev, _i32(tables[0]), lc[0], SCALE)
        assert torch.equal(one, got)


def test_prefill_rows_without_keys_and_rows_behind():
    """More new tokens than cached ones (the first see nothing), an empty
    sequence, rows behind the last sequence left as they were, and blocks
    outside the pool."""
    gen = torch.Generator().manual_seed(35)
    host, dev = H.filled(gen, 6, 2, 128)
    lq, lk = [5, 0, 4, 200], [2, 3, 0, 300]
    tables = H.tables_of(gen, [2, 3, 1, 300], 128, 6)
    tables[3, 1] = 77
    q = torch.randn(sum(lq) + 10, 8, 128, generator=gen).to(FP16)
    got = M.fp4_varlen_prefill_attention(q.to(H.DEV), *dev, _i32(tables), _cu(lq), _cu(lk), 200,
                                         SCALE)
    want = _prefill_want(q, host, tables, lq, lk, SCALE)
    H.check(got[:sum(lq)], *want, FP16, 300, host[3].max(), 4)
    assert (got[:3] == 0).all() and (got[5:9] == 0).all()
    lib, sentinel = _lib.load(), torch.full_like(got, 3)
    s = torch.cuda.current_stream().cuda_stream
    cu_q, cu_k, tb, qd = _cu(lq), _cu(lk), _i32(tables), q.to(H.DEV)
    assert lib.mskv_fp4_prefill_attention(
        qd.data_ptr(), *(t.data_ptr() for t in dev), tb.data_ptr(), cu_q.data_ptr(),
        cu_k.data_ptr(), 0, sentinel.data_ptr(), 4, len(q), 200, 0, 8, 2, 128, 128, 6,
        tables.shape[1], SCALE, 0, None, 0, s) == 0
    torch.cuda.synchronize()
    assert (sentinel[sum(lq):] == 3).all()
    H.check(sentinel[:sum(lq)], *want, FP16, 300, host[3].max(), 4)


def test_prefill_graph_with_split_keys():
    gen = torch.Generator().manual_seed(36)
    host, dev = H.filled(gen, 40, 2, 128)
    table = _i32(torch.randperm(40, generator=gen))
    q = torch.randn(30, 16, 128, generator=gen).to(BF16).to(H.DEV)
    lib = _lib.load()
    assert lib.mskv_fp8_prefill_bounded_workspace_bytes(1, 30, 30, 5000, 16, 2, 128, 128, 40) > 0

    def call():
        return M.fp4_chunk_prefill_attention(q, *dev, table, 4970, SCALE)

    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for seed in range(3):
        q.copy_(torch.randn(30, 16, 128, generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, call())
    tab = table.cpu().numpy()[None]
    want = _prefill_want(q.cpu()[:3], host, tab, [3], [4973], SCALE)
    H.check(got[:3], *want, BF16, 5000, host[3].max(), 4)


def test_native_paths_and_wrappers_agree(monkeypatch):
    lens = [300, 70]
    host, dev, tables, q = _decode(45, lens, 8, 2, 128, BF16)
    q, n, t = q.to(H.DEV), _i32(lens), _i32(tables)
    gen = torch.Generator().manual_seed(46)
    rows = torch.randn(40, 2, 128, generator=gen).to(BF16).to(H.DEV)
    slots = torch.arange(40, device=H.DEV)

    def calls():
        M.store_fp4_kvcache(rows, rows, *dev, slots)
        cu = _cu([1, 1])
        return [M.fp4_decode_attention(q, *dev, n, t, SCALE),
                *M.load_fp4_kvcache(*dev, slots, torch.float16),
                M.fp4_chunk_prefill_attention(q, *dev, t[0], 100, SCALE),
                M.fp4_varlen_prefill_attention(q, *dev, t, cu, _cu(lens), 1, SCALE)] + [
                    c.clone() for c in dev]

    before = [c.clone() for c in dev]
    native = calls()
    for c, old in zip(dev, before):
        c.copy_(old)

    class Off:
        def __getattr__(self, name):
            return lambda *a: None

    monkeypatch.setattr(_lib, "fast", Off())
    for a, b in zip(native, calls()):
        assert torch.equal(a, b)


# --------------------------------------------------------------- together --

def test_a_layers_steps_over_a_pool_that_forks_and_is_compacted():
    """Prefill, a chunk, a fork with its copied page, decode steps of parent
    and child, a compaction, and a decode over the moved pages, through the
    Attention layer, against the oracle over the tokens themselves."""
    gen = torch.Generator().manual_seed(50)
    hq, hk, bs, pool = 8, 2, 128, 24
    caches = M.allocate_fp4_kvcache(pool, bs, hk)
    layer = M.Attention(hq, 128, SCALE, hk)
    layer.kv_cache_dtype = "fp4_e2m1"
    layer.k_cache, layer.v_cache, layer.k_scale_cache, layer.v_scale_cache = caches

    def rows(n):
        return [torch.randn(n, h, 128, generator=gen).to(BF16) for h in (hq, hk, hk)]

    def step(mode, q, k, v, **ctx):
        M.set_context(M.Context(mode=mode, **ctx))
        return layer(*(x.to(H.DEV) for x in (q, k, v)))

    def slots(table, a, b):
        return torch.tensor([table[p // bs] * bs + p % bs for p in range(a, b)], device=H.DEV)

    # one sequence: 150 tokens fresh, then a chunk of 100
    table = [19, 7]
    q, k, v = rows(150)
    cu = _i32([0, 150])
    got = step(M.AttentionMode.PREFILL, q, k, v, slot_mapping=slots(table, 0, 150), cu_seqlens_q=cu,
               cu_seqlens_k=cu, max_seqlen_q=150, max_seqlen_k=150)
    assert torch.equal(got, M.varlen_attention(q.to(H.DEV), k.to(H.DEV), v.to(H.DEV), cu, cu, 150,
                                               softmax_scale=SCALE))
    keys, vals = [k], [v]
    q, k, v = rows(100)
    got = step(M.AttentionMode.CHUNK_PREFILL, q, k, v, slot_mapping=slots(table, 150, 250),
               block_tables=_i32([table]), prefix_len=150, query_len=100)
    keys.append(k), vals.append(v)

    def stored(keys, vals):
        """The oracle's own pages of these tokens."""
        k, v = (torch.cat(x).float().numpy() for x in (keys, vals))
        n = len(k)
        host = H.empty(-(-n // bs), hk, bs)
        O.store(k, v, host, np.arange(n))
        return host, n

    host, n = stored(keys, vals)
    seq = np.arange(len(host[1]))[None]
    want = _prefill_want(q, host, seq, [100], [250], SCALE)
    H.check(got, *want, BF16, 250, host[3].max(), 4)

    # fork: the full page is shared, the other one copied
    child = [19, 22]
    M.copy_kv_blocks(caches, [7], [22])
    keys, vals = [list(keys), list(keys)], [list(vals), list(vals)]
    tabs = [table, child]
    for i in range(8):
        if 250 + i == 256:  # both take a new page
            tabs[0].append(12), tabs[1].append(23)
        q, k, v = rows(2)
        at = torch.cat([slots(t, 250 + i, 251 + i) for t in tabs])
        got = step(M.AttentionMode.DECODE, q, k, v, slot_mapping=at, block_tables=_i32(tabs),
                   cache_seqlens=_i32([251 + i] * 2))
        for b in range(2):
            keys[b].append(k[b:b + 1]), vals[b].append(v[b:b + 1])
    for b in range(2):
        host, n = stored(keys[b], vals[b])
        want = _decode_want(q[b:b + 1], host, [n], np.arange(len(host[1]))[None], SCALE)
        H.check(got[b:b + 1], *want, BF16, n, host[3].max(), 1)

    # the five live pages to the front; the next step reads them there
    moved, remap, live = M.compact_kv_blocks(caches, _i32(tabs))
    assert live.item() == 5 and sorted(set(moved.flatten().tolist())) == [0, 1, 2, 3, 4]
    lens = _i32([n, n])
    before = got
    again = M.fp4_decode_attention(q.to(H.DEV), *caches, lens, moved, SCALE)
    assert torch.equal(again, before)
    M.reset_context()
