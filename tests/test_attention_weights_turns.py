"""The entries of tokens that a prompt or a turn stores: 0 until a query looks at
them, whatever their places held before."""

import numpy as np
import pytest
import torch

import microserve_amd as M
from microserve_amd import _lib
from microserve_amd import attention as layer
from microserve_amd.context import AttentionMode, Context, reset_context, set_context
from oracle import weights_oracle as W
from tests import weights_helpers as H

D = 128


@pytest.mark.parametrize("mode", list(AttentionMode))
@pytest.mark.parametrize("dtype", ["fp8_e4m3", "fp4_e2m1"])
@pytest.mark.parametrize("fused", [False, True])
def test_a_prefill_of_the_layer_clears_what_it_stores(monkeypatch, mode, dtype, fused):
    if fused and dtype == "fp4_e2m1":
        return
    attn = M.Attention(8, D, 0.1, 2)
    attn.k_cache = attn.v_cache = torch.zeros(4, 128, 2, D)
    attn.kv_cache_dtype = dtype
    seen = []
    for name in ("store_fp8_kvcache", "store_fp4_kvcache", "clear_attention_weights"):
        monkeypatch.setattr(layer, name, lambda *a, name=name: seen.append((name, a)))
    monkeypatch.setattr(layer, "qk_norm_rope_store",
                        lambda *a, **k: seen.append(("store", a)) or (a[1], a[2]))
    monkeypatch.setattr(attn, "_attend", lambda *a: seen.append(("attend", a)))
    slots = torch.arange(3)
    set_context(Context(mode=mode, slot_mapping=slots))
    x = torch.zeros(3, 2, D)
    try:
        for weights in (None, torch.zeros(4, 2, 128)):
            seen.clear()
            attn.attention_weights = weights
            if fused:
                attn.forward_fused(x, x, x, x, None, None, 1e-6, x, x)
            else:
                attn.forward(x, x, x)
            names = [n for n, _ in seen]
            clears = weights is not None and dtype == "fp8_e4m3" and mode is not AttentionMode.DECODE
            assert names[1:] == ["clear_attention_weights"] * clears + ["attend"]
            if clears:
                assert seen[1][1][0] is weights and seen[1][1][1] is slots
    finally:
        reset_context()


def test_refusals(monkeypatch):
    w, slots = torch.zeros(4, 2, 128), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(AssertionError, match="GPU"):
        M.clear_attention_weights(w, slots)
    monkeypatch.setattr(_lib, "on_device", lambda *a: None)
    for a, b in ((w[0], slots), (w.double(), slots), (w.transpose(1, 2), slots),
                 (w, slots.float()), (w, slots.short())):
        with pytest.raises(AssertionError):
            M.clear_attention_weights(a, b)
    p = 1 << 20

    def call(w=p, slots=p, dtype=_lib.INT64, n=2, hk=8, bs=256, nb=4):
        return _lib.load().mskv_clear_attention_weights(w, slots, dtype, n, hk, bs, nb, None)
    assert call(w=None) == call(slots=None) == call(dtype=9) == call(n=-1) == call(hk=0) == -1
    assert call(bs=0) == call(nb=-1) == -1
    assert call(hk=1 << 16) == call(n=1 << 31) == call(nb=1 << 31) == -2
    assert call(n=0, w=None, slots=None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("heads,block,tokens", [(1, 32, 1), (8, 256, 700), (5, 96, 257), (2, 128, 0)])
def test_clear(heads, block, tokens, dtype):
    gen = torch.Generator().manual_seed(tokens + heads)
    pages = 5
    w = torch.rand(pages, heads, block, generator=gen) + 1
    w[0, 0, 0] = float("nan")
    slots = torch.randint(-3, pages * block + 3, (tokens,), generator=gen)
    if tokens > 8:  # the same twice, both ends, far outside
        slots[:8] = torch.tensor([7, 7, 0, pages * block - 1, -1, pages * block, -2 ** 31, 2 ** 31 - 1])
    got = w.to(H.DEV)
    M.clear_attention_weights(got, slots.to(H.DEV, dtype))
    want = w.clone()
    live = slots[(slots >= 0) & (slots < pages * block)]
    want[live // block, :, live % block] = 0
    assert torch.equal(got.cpu().nan_to_num(9.0), want.nan_to_num(9.0))
    again = w.to(H.DEV)  # slots with strides
    M.clear_attention_weights(again, torch.stack([slots, slots], 1)[:, 0].to(H.DEV, dtype))
    assert torch.equal(again.nan_to_num(9.0), got.nan_to_num(9.0))


def _sums(q, keys, ok, scale, lk, hk):
    """A turn's probabilities [hk, lk] of queries at the end of lk tokens."""
    lq = len(q)
    p = W.probabilities(q.double().numpy(), keys, ok, scale, lk - lq + 1 + np.arange(lq))
    return W.by_kv_head(p, hk)


@pytest.mark.gpu
def test_a_turn_after_an_eviction():
    """A context cut to its budget takes a turn that is longer than its window: the
    entries of the turn's tokens are the window's probabilities alone, where the
    evicted tokens' were."""
    gen = torch.Generator().manual_seed(4)
    hq, hk, block, scale, length, budget, turn, window = 8, 2, 128, 0.09, 600, 200, 90, 20
    host, cache = H.pool(gen, 6, hk, block)
    tables = H.tables_of(gen, [768], block, 6)
    weights = (torch.rand(6, hk, block, generator=gen) + 5).to(H.DEV)
    t = H.gpu(tables)
    kept, n = M.select_kv_tokens(weights, H.gpu([length]), t, budget, recent=10)
    M.evict_kv_tokens(*cache, kept, n, t, weights)
    positions = np.arange(budget, budget + turn)
    slots = torch.as_tensor(tables[0][positions // block].astype(np.int64) * block
                            + positions % block).to(H.DEV)
    new = torch.randn(turn, hk, D, generator=gen).half().to(H.DEV)
    M.store_fp8_kvcache(new, new, *cache, slots)
    M.clear_attention_weights(weights, slots)
    old = weights.cpu().double().numpy()
    q = torch.randn(window, hq, D, generator=gen).half()
    lk = budget + turn
    M.fp8_window_attention_weights(q.to(H.DEV), cache[0], cache[2], t, H.gpu([0, window]),
                                   H.gpu([0, lk]), window, scale, weights, accumulate=True)
    now = H.to_cpu(cache)
    k, ok = W.rows_of(now[0], now[2], tables[0], lk, block)
    sums = _sums(q, k, ok, scale, lk, hk)
    want = old.copy()
    W.record(want, sums, ok, tables[0], 0, lambda p: p < budget)
    H.check_weights(weights.cpu().numpy(), want, old, H.reach_of(q.double().numpy(), k, scale), lk,
                    hq // hk * window)


@pytest.mark.gpu
@pytest.mark.parametrize("fused", [False, True])
def test_a_prompt_in_pages_of_a_former_owner(fused):
    """The layer stores a prompt in used pages, then decodes: entries are sums of the
    decode steps' probabilities."""
    gen = torch.Generator().manual_seed(6)
    hq, hk, block, scale, n = 8, 2, 128, 0.09, 300
    attn = M.Attention(hq, D, scale, hk)
    host, (attn.k_cache, attn.v_cache, attn.k_scale_cache, attn.v_scale_cache) = H.pool(
        gen, 4, hk, block)
    attn.attention_weights = (torch.rand(4, hk, block, generator=gen) * 100).to(H.DEV)
    before = attn.attention_weights.clone()
    table = np.array([[2, 0, 3]], np.int32)
    at = np.arange(n + 2)
    slots = torch.as_tensor(table[0][at // block].astype(np.int64) * block + at % block).to(H.DEV)
    cos = torch.ones(1024, D, device=H.DEV).half()

    def step(ctx, tokens):
        q = torch.randn(tokens, hq, D, generator=gen).half().to(H.DEV)
        k = torch.randn(tokens, hk, D, generator=gen).half().to(H.DEV)
        set_context(ctx)
        try:
            if fused:
                attn.forward_fused(torch.arange(tokens, device=H.DEV), q, k, k, None, None, 1e-6,
                                   cos, torch.zeros_like(cos))
            else:
                attn.forward(q, k, k)
        finally:
            reset_context()
        return q
    cu = H.gpu([0, n])
    step(Context(mode=AttentionMode.PREFILL, cu_seqlens_q=cu, cu_seqlens_k=cu, max_seqlen_q=n,
                 max_seqlen_k=n, slot_mapping=slots[:n]), n)
    want = before.cpu().double().numpy()
    places = (table[0][at // block], slice(None), at % block)
    want[table[0][at[:n] // block], :, at[:n] % block] = 0
    assert np.array_equal(attn.attention_weights.cpu().numpy(), want)
    zero, reach = want.copy(), 0.0
    for m in (n + 1, n + 2):
        q = step(Context(mode=AttentionMode.DECODE, cache_seqlens=H.gpu([m]),
                         block_tables=H.gpu(table), slot_mapping=slots[m - 1:m]), 1)
        now = H.to_cpu((attn.k_cache, attn.v_cache, attn.k_scale_cache, attn.v_scale_cache))
        k, ok = W.rows_of(now[0], now[2], table[0], m, block)
        W.record(want, _sums(q.cpu(), k, ok, scale, m, hk), ok, table[0], 0, lambda p: p < m - 1)
        reach = max(reach, H.reach_of(q.cpu().double().numpy(), k, scale))
    zero[places] = 0
    H.check_weights(attn.attention_weights.cpu().numpy(), want, zero, reach, n + 2,
                    2 * hq // hk)
