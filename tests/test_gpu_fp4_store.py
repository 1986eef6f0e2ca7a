"""The 4-bit cache's store and read-back against the oracle, byte for byte."""

import numpy as np
import pytest
import torch

import microserve_amd as M
from oracle import fp4_oracle as O
from tests import fp4_helpers as H

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _same(caches, want):
    for got, w in zip(caches, want):
        np.testing.assert_array_equal(got.cpu().numpy(), w)


def _marked(num_blocks, heads, block):
    """Caches whose every byte is known, so that strays show."""
    want = H.empty(num_blocks, heads, block)
    for i, c in enumerate(want):
        c[...] = 0.5 if i == 3 else 0x5A
    return want, H.to_gpu(want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,heads,block,slot", [
    (1, 8, 256, torch.int64), (7, 1, 128, torch.int32), (8, 3, 128, torch.int64),
    (9, 8, 256, torch.int32), (64, 2, 384, torch.int64), (301, 5, 256, torch.int64),
    (1000, 8, 256, torch.int32)])
def test_store_matches_the_oracle(dtype, n, heads, block, slot):
    gen = torch.Generator().manual_seed(n + heads)
    blocks = -(-n // block) + 2
    key = (torch.randn(n, heads, 128, generator=gen)
           * torch.exp2(torch.randint(-12, 12, (n, heads, 1), generator=gen))).to(dtype)
    value = torch.randn(n, heads, 128, generator=gen).to(dtype)
    slots = torch.randperm(blocks * block, generator=gen)[:n]
    if n > 40:  # consecutive ones, as a prefill has them
        slots[20:n] = torch.arange(20, n) + 3
        slots[:20] = blocks * block - 1 - torch.arange(20)
    if n > 6:  # tokens without a slot
        slots[2], slots[5] = -1, blocks * block
    slots = slots.to(slot)
    want, caches = _marked(blocks, heads, block)
    M.store_fp4_kvcache(key.to(H.DEV), value.to(H.DEV), *caches, slots.to(H.DEV))
    O.store(key.float().numpy(), value.float().numpy(), want, slots.numpy())
    _same(caches, want)
    for out in TYPES:
        k, v = M.load_fp4_kvcache(*caches, slots.to(H.DEV), out)
        assert k.shape == v.shape == (n, heads, 128) and k.dtype == v.dtype == out
        rk, rv = _read(want, slots.tolist(), heads)
        assert torch.equal(k.cpu(), torch.from_numpy(rk).to(out))
        assert torch.equal(v.cpu(), torch.from_numpy(rv).to(out))


def _read(caches, slots, heads):
    """code * scale in fp32; zeros outside the cache."""
    nb, _, bs = caches[1].shape[:3]
    rk, rv = np.zeros((2, len(slots), heads, 128), np.float32)
    every = {}
    for i, s in enumerate(slots):
        if 0 <= s < nb * bs:
            page = s // bs
            if page not in every:
                every[page] = O.rows([c if j < 3 else c for j, c in enumerate(caches)], [page], bs)
            k = every[page][0][:, s % bs]
            codes = O.decode(O.unpack(caches[1][page, :, s % bs])).astype(np.float32)
            with np.errstate(over="ignore"):
                rk[i] = k.astype(np.float32)
                rv[i] = codes * caches[3][page, :, s % bs][:, None]
    return rk, rv


@pytest.mark.parametrize("dtype", TYPES)
def test_every_16_bit_pattern_and_the_edges(dtype):
    """Rows of neighbouring patterns (subnormals, zeros of both signs), ties
    of every scale, rows of one value, zeros, infinities and NaN."""
    if dtype == torch.float32:
        gen = torch.Generator().manual_seed(8)
        x = torch.randn(512, 128, generator=gen) * torch.exp2(
            torch.randint(-126, 127, (512, 1), generator=gen).float())
        x[3, :64] = 3.4e38
        x[4] = 1e-40
    else:
        p = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(dtype)
        x = p.view(512, 128).clone()
    gen = torch.Generator().manual_seed(9)
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 6.996])
    ties = mids[torch.randint(0, 10, (512, 128), generator=gen)]
    ties *= torch.sign(torch.randn(512, 128, generator=gen))
    ties *= torch.exp2(torch.randint(-12, 9, (512, 1), generator=gen).float())
    x = torch.cat((x, ties.to(dtype), torch.zeros(8, 128, dtype=dtype), -torch.zeros(8, 128, dtype=dtype)))
    x[-1, 33] = float("nan")
    x[-2, 127] = float("inf")
    x[-3, 0] = -float("inf")
    n = len(x) // 8
    rows = x.view(n, 8, 128)
    want, caches = _marked(2, 8, 128)
    slots = torch.arange(n) + 60
    M.store_fp4_kvcache(rows.to(H.DEV), rows.to(H.DEV), *caches, slots.to(H.DEV))
    O.store(rows.float().numpy(), rows.float().numpy(), want, slots.numpy())
    # the codes under a NaN scale stand for nothing
    ok_k, ok_v = want[2] != O.NAN_SCALE, ~np.isnan(want[3])
    got = [c.cpu().numpy() for c in caches]
    np.testing.assert_array_equal(got[2], want[2])
    np.testing.assert_array_equal(got[3], want[3])
    np.testing.assert_array_equal(got[1][ok_v], want[1][ok_v])
    ok_k = ok_k.transpose(0, 1, 2, 5, 3, 4).reshape(want[0].shape[:-1])
    np.testing.assert_array_equal(got[0][ok_k], want[0][ok_k])
    k, v = M.load_fp4_kvcache(*caches, slots.to(H.DEV), torch.float32)
    bad = ~torch.isfinite(rows.float()).unflatten(-1, (4, 32)).all(-1)
    assert torch.equal(k.cpu().unflatten(-1, (4, 32)).isnan().all(-1), bad)
    assert torch.equal(k.cpu().unflatten(-1, (4, 32)).isnan().any(-1), bad)
    assert torch.equal(v.cpu().isnan().all(-1), bad.any(-1))


def test_views_of_a_projection_and_other_strides():
    gen = torch.Generator().manual_seed(11)
    n, heads = 77, 4
    qkv = torch.randn(n, 3, heads, 128, generator=gen).half()
    odd = torch.randn(n, heads, 256, generator=gen).half()
    slots = torch.randperm(256, generator=gen)[:n]
    for key, value in ((qkv[:, 1], qkv[:, 2]),  # tokens apart, heads together
                       (odd[..., ::2], odd[..., 1::2]),  # elements apart
                       (odd[..., 3:131], qkv[:, 0]),  # rows off 16 bytes
                       (odd.transpose(0, 1)[:, :heads, :128], odd.transpose(0, 1)[:, :heads, 128:])):
        m = key.shape[0]
        want, caches = _marked(2, key.shape[1], 128)
        dev = qkv.to(H.DEV), odd.to(H.DEV)
        like = {qkv.data_ptr(): dev[0], odd.data_ptr(): dev[1]}
        views = []
        for t in (key, value):
            base = like[qkv.data_ptr() if t.untyped_storage().data_ptr() == qkv.data_ptr()
                        else odd.data_ptr()]
            views.append(base.as_strided(t.shape, t.stride(), t.storage_offset()))
        M.store_fp4_kvcache(*views, *caches, slots[:m].to(H.DEV))
        O.store(key.float().numpy(), value.float().numpy(), want, slots[:m].numpy())
        _same(caches, want)
    pad = torch.full((2 * n,), 255)
    pad[::2] = slots
    want, caches = _marked(2, heads, 128)
    M.store_fp4_kvcache(qkv[:, 1].to(H.DEV), qkv[:, 2].to(H.DEV), *caches, pad.to(H.DEV)[::2])
    O.store(qkv[:, 1].float().numpy(), qkv[:, 2].float().numpy(), want, slots.numpy())
    _same(caches, want)


def test_no_tokens():
    _, caches = _marked(1, 2, 128)
    z = torch.zeros(0, 2, 128, dtype=torch.float16, device=H.DEV)
    slots = torch.zeros(0, dtype=torch.int64, device=H.DEV)
    M.store_fp4_kvcache(z, z, *caches, slots)
    k, v = M.load_fp4_kvcache(*caches, slots)
    assert k.shape == v.shape == (0, 2, 128)


def test_pages_past_32_bits_of_bytes():
    """A pool of 6 GB of codes each for K and V: store, read and attend at its
    last page."""
    nb, heads, bs = 46000, 8, 256
    assert nb * heads * bs * 64 > 1 << 32
    caches = tuple(torch.empty(s, dtype=torch.float32 if i == 3 else torch.uint8, device=H.DEV)
                   for i, s in enumerate(M.fp4_cache_shapes(nb, bs, heads)))
    gen = torch.Generator().manual_seed(12)
    n = 200
    key, value = (torch.randn(n, heads, 128, generator=gen).half() for _ in range(2))
    slots = torch.arange(n) + (nb - 1) * bs
    M.store_fp4_kvcache(key.to(H.DEV), value.to(H.DEV), *caches, slots.to(H.DEV))
    k, v = M.load_fp4_kvcache(*caches, slots.to(H.DEV), torch.float32)
    small = H.empty(1, heads, bs)
    O.store(key.float().numpy(), value.float().numpy(), small, np.arange(n))
    rk, rv = _read(small, range(n), heads)
    assert torch.equal(k.cpu(), torch.from_numpy(rk)) and torch.equal(v.cpu(), torch.from_numpy(rv))
    q = torch.randn(1, 16, 128, generator=gen).half().to(H.DEV)
    lens = torch.tensor([n], dtype=torch.int32, device=H.DEV)
    far = torch.tensor([[nb - 1]], dtype=torch.int32, device=H.DEV)
    near = H.to_gpu(small)
    o = M.fp4_decode_attention(q, *caches, lens, far, 0.1)
    assert torch.equal(o, M.fp4_decode_attention(q, *near, lens, far * 0, 0.1))
    c = M.fp4_chunk_prefill_attention(q, *caches, far[0], n - 1, 0.1)
    assert torch.equal(c, M.fp4_chunk_prefill_attention(q, *near, far[0] * 0, n - 1, 0.1))
