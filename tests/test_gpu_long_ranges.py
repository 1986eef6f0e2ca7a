"""Shared prefixes, attention weights and eviction where a workgroup's range is
longer than one tile, a wave's scores fill its LDS before its range ends, and a
workgroup moves several heads.  Each case says by the launch's own rules that it
gets there.  References are in 64 bits, on the GPU for their size."""

import numpy as np
import pytest
import torch

import microserve_amd as M
from microserve_amd import _lib
from tests import weights_helpers as H

pytestmark = pytest.mark.gpu
D = 128


def _pool(gen, pages, heads, block, k_scales=None, v_scales=None):
    """Caches of random bytes (no NaN) and scales, [pages] factors on the scales."""
    dev = torch.Generator(H.DEV).manual_seed(int(torch.randint(1 << 30, (1,), generator=gen)))
    out, scales = [], []
    for factor in (k_scales, v_scales):
        x = torch.randint(0, 0x77, (pages, block, heads, D), generator=dev, device=H.DEV,
                          dtype=torch.uint8)
        x |= torch.randint(0, 2, x.shape, generator=dev, device=H.DEV, dtype=torch.uint8) << 7
        s = 0.004 * (1 + torch.rand(pages, block, heads, generator=dev, device=H.DEV))
        if factor is not None:
            s *= torch.as_tensor(factor, dtype=torch.float32, device=H.DEV)[:, None, None]
        out.append(x.view(torch.float8_e4m3fn))
        scales.append(s)
    return [*out, *scales]


def _rows(cache, scales, table, n):
    """[heads, n, 128] of a sequence in 64 bits, and which tokens exist."""
    block = cache.shape[1]
    t = torch.arange(n, device=H.DEV)
    blk = torch.as_tensor(np.asarray(table), device=H.DEV).long()[t // block]
    ok = (blk >= 0) & (blk < cache.shape[0])
    at = blk * ok
    x = cache.view(torch.uint8)[at, t % block].view(torch.float8_e4m3fn).double()
    x = x * scales[at, t % block].double()[..., None] * ok[:, None, None]
    return x.permute(1, 0, 2).contiguous(), ok


def _attend(q, k, ok, scale, sees):
    """Probabilities [heads, rows, keys], the rows query by query, of q [Lq, Hq, 128]."""
    lq, hq, _ = q.shape
    hk = k.shape[0]
    rows = q.double().view(lq, hk, hq // hk, D).transpose(0, 1).reshape(hk, -1, D).contiguous()
    s = torch.bmm(rows, k.transpose(1, 2).contiguous()) * scale
    sees = torch.as_tensor(np.asarray(sees), device=H.DEV).repeat_interleave(hq // hk)
    seen = ok[None] & (torch.arange(k.shape[1], device=H.DEV)[None] < sees[:, None])
    s = s.masked_fill(~seen[None], -float("inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - top.masked_fill(top == -float("inf"), 0.0))
    return p / p.sum(-1, keepdim=True).clamp_min(1e-300)


def _reach(q, k, scale):
    return scale * float(q.double().norm(dim=-1).max() * k.norm(dim=-1).max())


def _put(weights, sums, table, keep):
    """weights [pages, H, block] in 64 bits: keep(first, count) * entry + sums."""
    block = weights.shape[2]
    for p in range(-(-sums.shape[1] // block)):
        if 0 <= table[p] < weights.shape[0]:
            part = sums[:, p * block:(p + 1) * block]
            place = weights[int(table[p]), :, :part.shape[1]]
            place.copy_(place * keep(p * block, part.shape[1]) + part)


# ------------------------------------------------------------ shared prefixes --

def _tiles_of_a_range(batch, tiles, blocks, steps, hq, hk):
    """per_a of the plan of one group (`steps`: of each sequence's tail)."""
    units = hk * -(-(hq // hk) // 16)
    chain = (tiles * blocks * units * 3.6 + sum(steps) * -(-units // 4) * 2.2) / 512
    return int(np.ceil(chain / 3.6))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size,tiles,hq,hk,tails,spoiled,per", [
    (5, 40, 64, 32, [30, 1, 0, 200, 129], (), 3),         # ranges of 3, the last of 1
    (3, 17, 32, 32, [5, 6, 7], (), 2),                    # of 2, the last of 1
    (9, 64, 64, 64, [0] * 9, (), 8), (4, 50, 68, 34, [40] * 4, (0, 5, 6, 49), 4),
    (40, 34, 32, 8, [64] * 40, (3, 33), 2),               # two blocks of 128 rows
    (2, 36, 128, 32, [700, 3], tuple(range(36)), 3)])     # no page of the prefix exists
def test_ranges_of_several_tiles(size, tiles, hq, hk, tails, spoiled, per, dtype):
    gen = torch.Generator().manual_seed(size + tiles)
    block, scale = 128, 0.02
    own = [-(-n // block) for n in tails]
    pages = tiles + sum(own) + 1
    order = torch.randperm(pages, generator=gen).numpy()
    tables = np.full((size, tiles + max(max(own), 1)), -1, np.int32)
    tables[:, :tiles] = order[:tiles]
    tables[:, list(spoiled)] = np.where(np.arange(len(spoiled)) % 2, -1, 10 ** 6)
    at = tiles
    for b, n in enumerate(own):
        tables[b, tiles:tiles + n] = order[at:at + n]
        at += n
    # scores and v_scales that grow from tile to tile: the running maximum and the
    # weights' power of two move inside a range
    k_factor, v_factor = np.ones(pages), np.ones(pages)
    k_factor[order[:tiles]] = 1 + 1.5 * np.arange(tiles) / tiles
    v_factor[order[:tiles]] = 2.0 ** (12 * np.arange(tiles) / tiles)
    cache = _pool(gen, pages, hk, block, k_factor, v_factor)
    q = torch.randn(size, hq, D, generator=gen).to(H.DEV, dtype)
    lens = [tiles * block + n for n in tails]
    group = hq // hk
    rows = 8 * (16 // min(group, 16))
    assert _tiles_of_a_range(size, tiles, -(-size // rows), [-(-n // 32) for n in tails],
                             hq, hk) == per >= 2
    call = lambda: M.fp8_shared_prefix_decode_attention(  # noqa: E731
        q, *cache, H.gpu(lens), H.gpu(tables), scale, H.gpu([0, size]), H.gpu([tiles * block]))
    out = call()
    want, weight = (np.zeros((size, hq, D)) for _ in range(2))
    reach = 0.0
    for b, n in enumerate(lens):
        k, ok = _rows(cache[0], cache[2], tables[b], n)
        v, _ = _rows(cache[1], cache[3], tables[b], n)
        p = _attend(q[b:b + 1], k, ok, scale, [n])
        want[b] = torch.bmm(p, v).reshape(hq, D).cpu().numpy()
        weight[b] = torch.bmm(p, v.abs()).reshape(hq, D).cpu().numpy()
        reach = max(reach, _reach(q[b], k, scale))
    H.check_out(out, want, weight, reach, dtype, max(lens), float(cache[3].max()), 1)
    assert torch.equal(call(), out)  # nothing depends on timing


def test_one_long_prefix_in_a_large_batch():
    """The ranges that a prefix may have shrink with the batch: two sequences over
    40 tiles, beside 1022 of five tokens in no group."""
    gen = torch.Generator().manual_seed(1)
    batch, heads, block, scale, tiles = 1024, 8, 128, 0.05, 40
    pages = tiles + batch + 1
    cache = _pool(gen, pages, heads, block)
    order = torch.randperm(pages, generator=gen).numpy()
    tables = np.full((batch, tiles + 1), -1, np.int32)
    tables[:2, :tiles] = order[:tiles]
    tables[:2, tiles] = order[tiles:tiles + 2]
    tables[2:, 0] = order[tiles + 2:tiles + batch]
    lens = [tiles * block + 1] * 2 + [5] * (batch - 2)
    q = torch.randn(batch, heads, D, generator=gen).half().to(H.DEV)
    out = M.fp8_shared_prefix_decode_attention(q, *cache, H.gpu(lens), H.gpu(tables), scale,
                                               H.gpu([0, 2]), H.gpu([tiles * block]))
    for b in (0, 1, 2, 500, batch - 1):
        k, ok = _rows(cache[0], cache[2], tables[b], lens[b])
        v, _ = _rows(cache[1], cache[3], tables[b], lens[b])
        p = _attend(q[b:b + 1], k, ok, scale, [lens[b]])
        H.check_out(out[b], torch.bmm(p, v).reshape(heads, D).cpu().numpy(),
                    torch.bmm(p, v.abs()).reshape(heads, D).cpu().numpy(), _reach(q[b], k, scale),
                    torch.float16, lens[b], float(cache[3].max()), 1)


# ------------------------------------------------------------------- windows --

@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new,lens,hq,hk,per", [
    ([20], [5100], 64, 64, 3),                 # rows of one turn
    ([70, 9], [10000, 900], 96, 32, 3),        # 210 rows: two turns of the sums
    ([300, 40], [5000, 700], 64, 64, 3),       # more rows than LDS holds, staged tile by tile
    ([150], [4500], 96, 48, 2)])
def test_windows_of_several_tiles(new, lens, hq, hk, per, dtype, accumulate):
    gen = torch.Generator().manual_seed(sum(new))
    block, scale = 256, 0.03
    tiles = sum(-(-n // 256) for n in lens)
    assert -(-tiles * hk // 512) == per >= 2
    pages = tiles + 2
    cache = _pool(gen, pages, hk, block)
    tables = H.tables_of(gen, lens, block, pages)
    tables[0, 4] = -1
    old = torch.rand(pages, hk, block, generator=gen) * 1e-3
    q = torch.randn(sum(new), hq, D, generator=gen).to(H.DEV, dtype)
    cu_q, cu_k = np.cumsum([0, *new]), np.cumsum([0, *lens])

    def call():
        w = old.to(H.DEV)
        return M.fp8_window_attention_weights(
            q, cache[0], cache[2], H.gpu(tables), H.gpu(cu_q), H.gpu(cu_k), max(new), scale, w,
            accumulate=accumulate, max_seqlen_k=max(lens))
    got = call()
    want, reach = old.double().to(H.DEV), 0.0
    for b, (n, lq) in enumerate(zip(lens, new)):
        k, ok = _rows(cache[0], cache[2], tables[b], n)
        rows = q[cu_q[b]:cu_q[b + 1]]
        p = _attend(rows, k, ok, scale, n - lq + 1 + np.arange(lq))
        _put(want, p.sum(1), tables[b], lambda *a: float(accumulate))
        reach = max(reach, _reach(rows, k, scale))
    before = old if accumulate else torch.where(want.cpu() == old.double(), old, 0.0)
    H.check_weights(got.cpu().numpy(), want.cpu().numpy(), before.numpy(), reach, max(lens),
                    hq // hk * max(new))
    assert torch.equal(call(), got)


# ------------------------------------------------------------ tracking decode --

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch,least,most,hq,hk,block,width", [
    (2, 1500, 2000, 8, 2, 2048, 1), (3, 500, 1024, 32, 2, 1024, 1), (1, 4090, 4096, 3, 3, 4096, 1),
    (2, 993, 2048, 40, 2, 2048, 1),    # groups of 20: 16 heads and four
    (16, 3000, 8192, 128, 8, 256, 32),  # splits that follow the lengths
    (300, 100, 1024, 16, 1, 256, 4),    # work items
    (520, 200, 512, 16, 1, 512, 1)])    # workgroups of four waves
def test_scores_that_fill_lds_inside_a_range(batch, least, most, hq, hk, block, width, dtype):
    gen = torch.Generator().manual_seed(batch)
    scale, group = 0.03, hq // hk
    lens = torch.randint(least, most + 1, (batch,), generator=gen).tolist()
    lens[-1] = most
    splits = M.decode_num_splits(batch, hq, hk, width, block)
    room = 3968 // (min(group, 16) * 32) * 32
    assert -(-width // splits) * block > room and most > room
    pages = sum(-(-n // block) for n in lens)
    cache = _pool(gen, pages, hk, block)
    tables = H.tables_of(gen, lens, block, pages, width)
    q = torch.randn(batch, hq, D, generator=gen).to(H.DEV, dtype)
    old = torch.rand(pages, hk, block, generator=gen) * 1e-3
    args = (q, *cache, H.gpu(lens), H.gpu(tables), scale)

    def call():
        w = old.to(H.DEV)
        return M.fp8_decode_attention_weights(*args, w), w
    out, got = call()
    assert torch.equal(out, M.fp8_decode_attention(*args))
    want, before, reach = old.double().to(H.DEV), old.double().to(H.DEV), 0.0
    for b, n in enumerate(lens):
        k, ok = _rows(cache[0], cache[2], tables[b], n)
        p = _attend(q[b:b + 1], k, ok, scale, [n])
        keep = lambda first, count: (  # noqa: E731
            torch.arange(first, first + count, device=H.DEV) < n - 1).double()
        _put(want, p.sum(1), tables[b], keep)
        _put(before, torch.zeros_like(p.sum(1)), tables[b], keep)
        reach = max(reach, _reach(q[b], k, scale))
    H.check_weights(got.cpu().numpy(), want.cpu().numpy(), before.cpu().numpy(), reach, most, group)
    for a, b in zip(call(), (out, got)):
        assert torch.equal(a, b)


# ------------------------------------------------------------------ eviction --

def _heads_of(heads, units):
    n = max(1, min(heads, units))
    while heads % n:
        n -= 1
    return n


@pytest.mark.parametrize("batch,heads,scale_heads,row_heads", [
    (64, 8, 8, 2), (64, 12, 12, 3), (300, 5, 5, 5), (120, 5, 5, 1), (64, 40, 40, 10),
    (40, 14, 14, 2), (300, 6, 6, 6), (100, 9, 9, 3)])
def test_heads_that_move_together(batch, heads, scale_heads, row_heads):
    assert _heads_of(heads, batch * heads // 32) == scale_heads
    assert _heads_of(heads, batch * 2 * heads // 512) == row_heads
    gen = torch.Generator().manual_seed(batch + heads)
    block, budget = 32, 150
    lens = torch.randint(1, 400, (batch,), generator=gen).tolist()
    pages = sum(-(-n // block) for n in lens) + 2
    cache = _pool(gen, pages, heads, block)
    tables = H.tables_of(gen, lens, block, pages)
    tables[3, 0] = -1
    w = torch.rand(pages, heads, block, generator=gen).to(H.DEV)
    kept, n = M.select_kv_tokens(w, H.gpu(lens), H.gpu(tables), budget, 20, 3)
    arrays = [x.view(torch.uint8).cpu().numpy() if x.element_size() == 1 else x.cpu().numpy()
              for x in cache] + [w.permute(0, 2, 1).cpu().numpy()]
    old = [np.ascontiguousarray(x) for x in arrays]
    want = [x.copy() for x in old]
    for b in range(batch):
        m, of_heads = int(n[b]), kept[b].cpu().numpy()
        to = np.arange(m)
        for h in range(heads):
            src = of_heads[h, :m]
            here, there = tables[b, to // block], tables[b, src // block]
            ok = (here >= 0) & (there >= 0)
            for x, o in zip(want, old):
                x[here[ok], to[ok] % block, h] = o[there[ok], src[ok] % block, h]
    M.evict_kv_tokens(*cache, kept, n, H.gpu(tables), w)
    got = [*H.to_cpu(cache), w.permute(0, 2, 1).cpu().numpy()]
    for g, x, name in zip(got, want, ("k", "v", "k_scale", "v_scale", "weights")):
        assert np.ascontiguousarray(g).tobytes() == x.tobytes(), name


@pytest.mark.parametrize("new,lens,hq,hk", [
    ([16, 3], [3000, 700], 32, 32), ([40], [9000], 64, 64), ([130, 1], [5000, 6000], 48, 48)])
def test_windows_under_tables_wider_than_their_ranges(new, lens, hq, hk):
    """The partials follow what runs at once, not a table of 64 k tokens; a
    workspace of just that size is not overrun."""
    gen = torch.Generator().manual_seed(3)
    block, scale, width = 256, 0.03, 256
    pages = sum(-(-n // 256) for n in lens) + 2
    cache = _pool(gen, pages, hk, block)
    tables = H.tables_of(gen, lens, block, pages, width)
    q = torch.randn(sum(new), hq, D, generator=gen).half().to(H.DEV)
    cu_q, cu_k = (H.gpu(np.cumsum([0, *x])) for x in (new, lens))
    lib, t, w = _lib.load(), H.gpu(tables), torch.zeros(pages, hk, block, device=H.DEV)
    need = lib.mskv_window_weights_bounded_workspace_bytes(sum(new), max(new), 0, hq, hk, block,
                                                           width)
    turns = -(-max(new) * hq // hk // 128)
    assert need == sum(new) * hq * (-(-512 // (hk * turns)) + 1) * 4 + 4
    ws = torch.zeros(need + 4096, dtype=torch.uint8, device=H.DEV)
    ws[need:] = 77
    status = lib.mskv_fp8_window_attention_weights(
        q.data_ptr(), cache[0].data_ptr(), cache[2].data_ptr(), t.data_ptr(), cu_q.data_ptr(),
        cu_k.data_ptr(), w.data_ptr(), None, 0, 0, len(new), sum(new), max(new), 0, hq, hk, D,
        block, pages, width, scale, 0, ws.data_ptr(), need, _lib.stream_of(q))
    torch.cuda.synchronize()
    assert status == 0 and bool((ws[need:] == 77).all())
    want, reach = torch.zeros_like(w).double(), 0.0
    at = np.cumsum([0, *new])
    for b, (n, lq) in enumerate(zip(lens, new)):
        k, ok = _rows(cache[0], cache[2], tables[b], n)
        rows = q[at[b]:at[b + 1]]
        p = _attend(rows, k, ok, scale, n - lq + 1 + np.arange(lq))
        _put(want, p.sum(1), tables[b], lambda *a: 0.0)
        reach = max(reach, _reach(rows, k, scale))
    H.check_weights(w.cpu().numpy(), want.cpu().numpy(), 0.0, reach, max(lens),
                    hq // hk * max(new))
