"""Choosing the tokens that stay and moving their rows, against plain
restatements; a run of the operators as they are used."""

import numpy as np
import pytest
import torch

import microserve_amd as M
from oracle import weights_oracle as W
from tests import weights_helpers as H

pytestmark = pytest.mark.gpu
D = 128


def _weights(gen, pages, heads, block, kind):
    w = torch.randn(pages, heads, block, generator=gen)
    if kind == "ties":
        w = (w * 2).round() * 0.5  # few values, zeros of both signs
    elif kind == "equal":
        w = torch.zeros_like(w)
    elif kind == "specials":
        w[torch.rand(w.shape, generator=gen) < 0.3] = float("nan")
        w[torch.rand(w.shape, generator=gen) < 0.1] = float("inf")
        w[torch.rand(w.shape, generator=gen) < 0.1] = -float("inf")
        w[torch.rand(w.shape, generator=gen) < 0.1] = torch.finfo(torch.float32).min
        w[torch.rand(w.shape, generator=gen) < 0.1] = 1e-45
    else:
        w = torch.exp(2 * w)
    return w


def _select(w, lens, tables, budget, recent, starts, start=None):
    given = H.gpu(starts) if start is None else start
    kept, n = M.select_kv_tokens(w.to(H.DEV), H.gpu(lens), H.gpu(tables), budget, recent, given)
    torch.cuda.synchronize()
    for b, length in enumerate(lens):
        want, new = W.select(w.numpy(), length, tables[b].tolist(), budget, recent, starts[b])
        assert int(n[b]) == new, b
        got = kept[b].cpu().numpy()
        assert np.array_equal(got, want), (b, np.argwhere(got != want)[:3])
    return kept, n


@pytest.mark.parametrize("kind", ["random", "ties", "equal", "specials"])
@pytest.mark.parametrize("lens,heads,block,budget,recent,start", [
    ([1], 1, 32, 1, 0, 0), ([0, 5, 6, 7], 2, 128, 6, 2, 1), ([300, 255, 257], 8, 256, 256, 64, 4),
    ([1000, 2049], 3, 256, 1, 0, 0), ([2500, 100], 2, 256, 2000, 500, 700),
    ([700], 1, 32, 699, 699, 0), ([700], 1, 96, 100, 300, 60), ([1024, 1023, 1025], 2, 512, 512, 0, 0)])
def test_select(lens, heads, block, budget, recent, start, kind):
    gen = torch.Generator().manual_seed(sum(lens) + budget)
    pages = sum(-(-n // block) for n in lens) + 1
    tables = H.tables_of(gen, lens, block, pages, width=2)
    w = _weights(gen, pages, heads, block, kind)
    _select(w, lens, tables, budget, recent, [start] * len(lens), start)


@pytest.mark.parametrize("width", [12, 40, 200])  # the forms by the tables' width
def test_select_in_long_tables(width):
    gen = torch.Generator().manual_seed(width)
    lens = [width * 256 - 77, 300, 9000 if width > 36 else 2900]
    pages = sum(-(-n // 256) for n in lens) + 1
    tables = H.tables_of(gen, lens, 256, pages, width)
    for kind in ("random", "ties"):
        w = _weights(gen, pages, 1, 256, kind)
        _select(w, lens, tables, 700, 33, [0, 2, 5])


def test_select_with_invalid_pages_and_lengths_past_the_table():
    gen = torch.Generator().manual_seed(2)
    tables = H.tables_of(gen, [512, 512, 512], 128, 12)
    tables[0, 1], tables[1, :] = -1, 99
    w = _weights(gen, 12, 2, 128, "random")
    _select(w, [512, 400, 10 ** 6], tables, 300, 7, [3, 0, 0])
    kept, n = M.select_kv_tokens(w.to(H.DEV), H.gpu([-4]), H.gpu(tables[:1]), 5)
    assert int(n) == 0 and (kept == -1).all()


def _evict(gen, lens, heads, block, budget, recent, start, kind="random", width=0, spoil=None):
    pages = sum(-(-n // block) for n in lens) + 2
    host, dev = H.pool(gen, pages, heads, block)
    tables = H.tables_of(gen, lens, block, pages, width)
    if spoil is not None:
        spoil(tables)
    w = _weights(gen, pages, heads, block, kind)
    wd, t = w.to(H.DEV), H.gpu(tables)
    kept, n = M.select_kv_tokens(wd, H.gpu(lens), t, budget, recent, start)
    M.evict_kv_tokens(*dev, kept, n, t, weights=wd)
    torch.cuda.synchronize()
    rows = w.permute(0, 2, 1).contiguous().numpy()
    arrays = [*host, rows]
    for b in range(len(lens)):
        W.evict(arrays, kept[b].cpu().numpy(), int(n[b]), tables[b], block)
    for got, want, name in zip([*H.to_cpu(dev), wd.permute(0, 2, 1).cpu().numpy()], arrays,
                               ("k", "v", "k_scale", "v_scale", "weights")):
        assert got.tobytes() == want.tobytes(), name


@pytest.mark.parametrize("lens,heads,block,budget,recent,start", [
    ([1], 1, 32, 1, 0, 0), ([300, 255, 0, 257], 8, 256, 256, 64, 4), ([1000, 2049], 5, 128, 700, 30, 0),
    ([3000, 1500], 2, 256, 1400, 1400, 0), ([900], 1, 96, 37, 0, 0), ([2000, 1999], 1, 512, 1998, 900, 256),
    ([600] * 9, 3, 32, 64, 3, 5)])
def test_evict(lens, heads, block, budget, recent, start):
    gen = torch.Generator().manual_seed(sum(lens) + budget)
    _evict(gen, lens, heads, block, budget, recent, start)


def test_evict_without_weights_leaves_them_and_invalid_pages_are_skipped():
    gen = torch.Generator().manual_seed(5)

    def spoil(tables):
        tables[0, 1], tables[1, 0] = -1, 77

    _evict(gen, [600, 600, 600], 2, 128, 300, 10, 0, spoil=spoil)


def test_evict_of_lengths_past_the_table():
    """More places than the pages have: those behind the last page are left out."""
    gen = torch.Generator().manual_seed(9)
    block, heads, cap = 128, 2, 256
    host, dev = H.pool(gen, 6, heads, block)
    tables = H.tables_of(gen, [cap, cap], block, 6)
    kept = np.full((2, heads, 700), -1, np.int32)
    kept[0, :, :cap - 3] = np.arange(3, cap)
    kept[1, :, :600] = np.arange(600)
    kept[1, 1, 100:cap] = np.minimum(np.arange(100, cap) + 7, cap + 5)
    M.evict_kv_tokens(*dev, H.gpu(kept), H.gpu([700, 600]), H.gpu(tables))
    torch.cuda.synchronize()
    for b in range(2):
        now = kept[b, :, :cap].copy()
        now[now >= cap] = -1
        for h in range(heads):
            moved = np.flatnonzero((now[h] >= 0) & (now[h] != np.arange(cap)))
            src, dst = now[h][moved], moved
            slot = lambda t: tables[b][t // block] * block + t % block
            for x in host:
                rows = x.reshape(6 * block, heads, -1)
                rows[slot(dst), h] = rows[slot(src), h]
    for got, want in zip(H.to_cpu(dev), host):
        assert got.tobytes() == want.tobytes()


def test_evict_of_rows_past_32_bits_of_bytes():
    """A pool of 4.3 GB a cache, the sequence's pages at its ends."""
    gen = torch.Generator().manual_seed(6)
    block, heads, pages = 256, 8, (1 << 32) // (256 * 8 * 128) + 2
    kc = torch.zeros(pages, block, heads, D, dtype=torch.uint8, device=H.DEV)
    vc, ks, vs = torch.zeros_like(kc), torch.zeros(pages, block, heads, device=H.DEV), None
    vs = torch.zeros_like(ks)
    order = [pages - 1, 0, pages - 2]
    for i, p in enumerate(order):
        kc[p] = torch.randint(0, 255, kc[p].shape, generator=gen, dtype=torch.uint8).to(H.DEV)
        vc[p] = torch.randint(0, 255, kc[p].shape, generator=gen, dtype=torch.uint8).to(H.DEV)
        ks[p] = torch.rand(block, heads, generator=gen).to(H.DEV)
        vs[p] = torch.rand(block, heads, generator=gen).to(H.DEV)
    old = [torch.cat([x[p] for p in order]) for x in (kc, vc, ks, vs)]
    kept = torch.stack([torch.randperm(700, generator=gen)[:500].sort()[0] for _ in range(heads)])
    f8 = torch.float8_e4m3fn
    M.evict_kv_tokens(kc.view(f8), vc.view(f8), ks, vs, H.gpu(kept[None]), H.gpu([500]),
                      H.gpu([order]))
    new = [torch.cat([x[p] for p in order]) for x in (kc, vc, ks, vs)]
    kept = kept.to(H.DEV)
    for a, b in zip(old, new):
        for h in range(heads):
            assert torch.equal(b[:500, h], a[kept[h], h]) and torch.equal(b[500:, h], a[500:, h])


def test_a_prompt_is_cut_and_the_decode_goes_on():
    """Store, window weights of the prompt, eviction, decode steps that keep
    weights, eviction again: the attention over what is left is that of the kept
    tokens, whatever their places."""
    gen = torch.Generator().manual_seed(8)
    hq, hk, block, lens = 8, 2, 128, [500, 260]
    tables = H.tables_of(gen, [640, 640], block, 12)
    pages = 12
    kc = torch.zeros(pages, block, hk, D, dtype=torch.float8_e4m3fn, device=H.DEV)
    vc = torch.zeros_like(kc)
    ks, vs = (torch.ones(pages, block, hk, device=H.DEV) for _ in range(2))
    caches, t = (kc, vc, ks, vs), H.gpu(tables)
    weights = M.allocate_attention_weights(pages, block, hk)

    def slots(b, positions):
        return torch.tensor([int(tables[b, p // block]) * block + p % block for p in positions])

    at = torch.cat([slots(b, range(n)) for b, n in enumerate(lens)]).to(H.DEV)
    k = torch.randn(len(at), hk, D, generator=gen).half().to(H.DEV)
    M.store_fp8_kvcache(k, k * 0.5, *caches, at)
    q = torch.randn(16, hq, D, generator=gen).half().to(H.DEV)
    M.fp8_window_attention_weights(q, kc, ks, t, H.gpu([0, 8, 16]), H.gpu([0, 500, 760]), 8, 0.09,
                                   weights)
    before = [x.clone() for x in caches]
    kept, n = M.select_kv_tokens(weights, H.gpu(lens), t, 300, recent=16, start=2)
    M.evict_kv_tokens(*caches, kept, n, t, weights=weights)
    assert n.tolist() == [300, 260]
    # the attention of the kept tokens of each head, out of the old cache
    qd = torch.randn(2, hq, D, generator=gen).half()
    for step in range(3):
        out = M.fp8_decode_attention_weights(qd.to(H.DEV), *caches, n, t, 0.09, weights)
        if step == 0:
            host = H.to_cpu(before)
            for b, m in enumerate(n.tolist()):
                full = lens[b]
                kk, ok = W.rows_of(host[0], host[2], tables[b], full, block)
                vv, _ = W.rows_of(host[1], host[3], tables[b], full, block)
                for h in range(hq):
                    live = kept[b, h // 4, :m].cpu().numpy()
                    p = W.probabilities(qd[b:b + 1, h:h + 1].double().numpy(), kk[live][:, h // 4:h // 4 + 1],
                                        ok[live], 0.09, [m])[0, 0]
                    want = p @ vv[live, h // 4]
                    reach = H.reach_of(qd[b, h:h + 1].double().numpy(), kk, 0.09)
                    H.check_out(out[b, h], want, np.abs(p) @ np.abs(vv[live, h // 4]), reach,
                                torch.float16, full, host[3].max(), 1)
        n = n + 1  # the next token
        new = torch.randn(2, hk, D, generator=gen).half().to(H.DEV)
        at = torch.cat([slots(b, [int(n[b]) - 1]) for b in range(2)]).to(H.DEV)
        M.store_fp8_kvcache(new, new, *caches, at)
    # the tables hold 640 tokens: pages behind the lengths are free
    kept, n = M.select_kv_tokens(weights, n, t, 256, recent=16, start=2)
    M.evict_kv_tokens(*caches, kept, n, t, weights=weights)
    assert n.tolist() == [256, 256] and (kept[:, :, -16:].diff() == 1).all()
