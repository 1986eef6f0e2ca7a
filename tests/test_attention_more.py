"""The attention layer's decode with attention weights and with shared prefixes."""

import pytest
import torch

import microserve_amd as M
from microserve_amd import attention as layer
from microserve_amd.context import AttentionMode, Context, reset_context, set_context


def _layer(dtype="fp8_e4m3"):
    attn = M.Attention(8, 128, 0.1, 2)
    attn.k_cache = attn.v_cache = torch.zeros(4, 128, 2, 128).to(torch.float8_e4m3fn)
    attn.k_scale_cache = attn.v_scale_cache = torch.ones(4, 128, 2)
    attn.kv_cache_dtype = dtype
    return attn


@pytest.fixture
def calls(monkeypatch):
    seen = []
    for name in ("fp8_decode_attention", "fp8_decode_attention_weights",
                 "fp8_shared_prefix_decode_attention", "store_fp8_kvcache",
                 "store_fp4_kvcache"):
        monkeypatch.setattr(layer, name,
                            lambda *a, name=name: seen.append((name, a)) or torch.zeros(1))
    yield seen
    reset_context()


def _step(attn, **groups):
    lens, tables = torch.ones(3, dtype=torch.int32), torch.zeros(3, 1, dtype=torch.int32)
    set_context(Context(mode=AttentionMode.DECODE, cache_seqlens=lens, block_tables=tables,
                        slot_mapping=torch.arange(3), **groups))
    x = torch.zeros(3, 2, 128)
    attn.forward(torch.zeros(3, 8, 128), x, x)
    return lens, tables


def test_a_plain_decode_stays_as_it_was(calls):
    _step(_layer())
    assert [c[0] for c in calls] == ["store_fp8_kvcache", "fp8_decode_attention"]


def test_weights_and_groups_choose_the_call(calls):
    attn = _layer()
    cu, pre = torch.tensor([0, 3], dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    lens, tables = _step(attn, cu_groups=cu, prefix_lens=pre, max_prefix_len=128)
    name, args = calls[-1]
    assert name == "fp8_shared_prefix_decode_attention"
    assert args[5] is lens and args[6] is tables and args[8] is cu and args[9] is pre
    assert args[10] == 128
    attn.attention_weights, attn.attention_weights_start = torch.zeros(4, 2, 128), 5
    _step(attn, cu_groups=cu, prefix_lens=pre)
    name, args = calls[-1]
    assert name == "fp8_decode_attention_weights"
    assert args[8] is attn.attention_weights and args[9] == 5


@pytest.mark.parametrize("what", ["weights", "groups"])
def test_a_4_bit_cache_has_neither(calls, what):
    attn = _layer("fp4_e2m1")
    cu = torch.tensor([0, 3], dtype=torch.int32) if what == "groups" else None
    if what == "weights":
        attn.attention_weights = torch.zeros(4, 2, 128)
    with pytest.raises(NotImplementedError):
        _step(attn, cu_groups=cu, prefix_lens=cu)


@pytest.mark.gpu
def test_decode_steps_of_the_layer():
    """Three sequences behind one page: the layer with groups, with weights and
    plain give one another's results, and the weights sum to the steps."""
    gen = torch.Generator().manual_seed(5)
    heads, group, block = 2, 4, 256
    attn = M.Attention(heads * group, 128, 0.09, heads).cuda()
    attn.k_cache = torch.zeros(8, block, heads, 128, device="cuda").to(torch.float8_e4m3fn)
    attn.v_cache = attn.k_cache.clone()
    attn.k_scale_cache = torch.ones(8, block, heads, device="cuda")
    attn.v_scale_cache = torch.ones(8, block, heads, device="cuda")
    old = torch.randn(4 * block, heads, 128, generator=gen).half().cuda()
    M.store_fp8_kvcache(old, old.flip(0), attn.k_cache, attn.v_cache, attn.k_scale_cache,
                        attn.v_scale_cache, torch.arange(4 * block, device="cuda"))
    tables = torch.tensor([[0, 1], [0, 2], [0, 3]], dtype=torch.int32)
    lens = torch.tensor([300, 257, 500], dtype=torch.int32)
    order, cu, prefixes = M.group_by_prefix(tables.tolist(), block)
    assert order == [0, 1, 2] and cu == [0, 3] and prefixes == [block]
    ctx = Context(mode=AttentionMode.DECODE, cache_seqlens=lens.cuda(), block_tables=tables.cuda())
    ctx.slot_mapping = (tables[:, 1].long() * block + lens - 1 - block).cuda()
    q = torch.randn(3, heads * group, 128, generator=gen).half().cuda()
    k = torch.randn(3, heads, 128, generator=gen).half().cuda()
    set_context(ctx)
    try:
        plain = attn.forward(q, k, k)
        ctx.cu_groups = torch.tensor(cu, dtype=torch.int32, device="cuda")
        ctx.prefix_lens = torch.tensor(prefixes, dtype=torch.int32, device="cuda")
        shared = attn.forward(q, k, k)
        attn.attention_weights = M.allocate_attention_weights(8, block, heads, device="cuda")
        attn.attention_weights_start = block
        tracked = attn.forward(q, k, k)
        torch.cuda.synchronize()
    finally:
        reset_context()
    assert torch.equal(tracked, plain)
    # two orders of the same sums: half a step of fp16 in the output of each and in
    # the probabilities by which each weighs the values (relative, so of the largest
    # value at most), and another for the fp32 sums behind them
    top = max(float(old.float().abs().max()), float(k.float().abs().max()))
    assert float((shared.float() - plain.float()).abs().max()) <= 5 * 2.0 ** -11 * top
    w = attn.attention_weights
    assert float(w[0].abs().max()) == 0 and float(w[4:].abs().max()) == 0
    assert float(w.sum()) <= 3 * heads * group * (1 + 1e-5)
    assert bool((w[1, :, 300 - block:] == 0).all()) and bool((w[1, :, :300 - block] > 0).all())
