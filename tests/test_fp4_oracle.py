"""The 4-bit cache's definition against brute force and closed forms, and the
refusals of its entry points and of the page moves: all on the CPU."""

import ctypes

import numpy as np
import pytest
import torch

import microserve_amd as M
from microserve_amd import _lib
from oracle import fp4_oracle as O

RNG = np.random.default_rng(5)


def test_encode_is_the_nearest_value_with_ties_to_even():
    y = np.concatenate([RNG.normal(size=4000) * 3, O.GRID, -O.GRID,
                        (O.GRID[1:] + O.GRID[:-1]) / 2, [7, 100, -1e30]])
    got = O.decode(O.encode(y))
    dist = np.abs(np.clip(y, -6, 6)[:, None] - np.concatenate([O.GRID, -O.GRID]))
    np.testing.assert_array_equal(np.abs(got - np.clip(y, -6, 6)), dist.min(1))
    # 0.25 0.75 1.25 1.75 2.5 3.5 5: codes 0 2 2 4 4 6 6
    ties = (O.GRID[1:] + O.GRID[:-1]) / 2
    np.testing.assert_array_equal(O.encode(ties), [0, 2, 2, 4, 4, 6, 6])
    assert O.encode(-0.0) == 8 and O.encode(0.0) == 0


def test_k_scale_is_the_smallest_power_of_two_that_holds_the_block():
    x = RNG.normal(size=(500, 128)) * np.exp2(RNG.integers(-20, 20, (500, 1)))
    codes, e = O.quantize_k(x)
    amax = np.abs(x.reshape(500, 4, 32)).max(-1)
    scale = np.exp2(e.astype(float) - 127)
    assert (amax < 7 * scale).all() and (amax >= 3.5 * scale).all()
    err = np.abs(O.decode(codes).reshape(500, 4, 32) * scale[..., None] - x.reshape(500, 4, 32))
    assert (err <= 1.0 * scale[..., None]).all()  # half of the last step, 4 to 6
    for a, want in ((7.0, 1), (np.nextafter(7.0, 0), 0), (6.0, 0), (3.5, 0), (3.49, -1)):
        row = np.zeros(128)
        row[5] = a
        assert O.quantize_k(row)[1][0] == 127 + want, a
    assert O.quantize_k(np.zeros(128))[1].tolist() == [1] * 4


def test_v_scale_takes_the_largest_value_to_six():
    x = RNG.normal(size=(300, 128)).astype(np.float32)
    codes, s = O.quantize_v(x)
    assert (O.decode(codes).max(-1) == 6).any()
    assert (np.abs(O.decode(codes)).max(-1) == 6).all()
    np.testing.assert_allclose(s * 6, np.abs(x).max(-1), rtol=2e-7)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_v_codes_of_16_bit_rows_are_those_of_exact_arithmetic(dtype):
    """24 |x| against k amax in whole numbers, k the midpoints' quarters: no
    rounding anywhere, ties included."""
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(4000, 128, generator=gen).to(dtype).float().numpy()
    codes, _ = O.quantize_v(x)
    step = 2.0 ** -30
    xi = np.abs(x.astype(np.float64)) / step
    ai = xi.max(-1, keepdims=True)
    assert (xi == np.round(xi)).all()
    mids = (1, 3, 5, 7, 10, 14, 20)
    exact = np.zeros(x.shape, int)
    ties = 0
    for c, k in enumerate(mids):
        left, right = 24 * xi, k * ai
        ties += int((left == right).sum())
        exact += (left > right) | ((left == right) & (c % 2 == 1))
    assert ties > 100
    np.testing.assert_array_equal(codes & 7, exact)


def test_blocks_and_rows_without_a_finite_scale():
    x = np.ones((3, 128), np.float32)
    x[0, 40] = np.nan
    x[1, 0] = -np.inf
    assert O.quantize_k(x)[1].tolist() == [[125, 255, 125, 125], [255, 125, 125, 125], [125] * 4]
    assert np.isnan(O.quantize_v(x)[1]).tolist() == [True, True, False]


def test_rows_give_back_what_was_stored():
    caches = [np.zeros(s, np.float32 if i == 3 else np.uint8)
              for i, s in enumerate(M.fp4_cache_shapes(3, 128, 2))]
    key, value = RNG.normal(size=(2, 200, 2, 128)).astype(np.float32)
    pages = [2, 0]
    slots = [pages[t // 128] * 128 + t % 128 for t in range(200)]
    O.store(key, value, caches, slots)
    k, v = O.rows(caches, pages, 200)
    kc, ke = O.quantize_k(key)
    want = O.decode(kc).reshape(200, 2, 4, 32) * np.exp2(ke.astype(float) - 127)[..., None]
    np.testing.assert_array_equal(k.transpose(1, 0, 2), want.reshape(200, 2, 128))
    vc, vs = O.quantize_v(value)
    np.testing.assert_array_equal(v.transpose(1, 0, 2), O.decode(vc) * vs.astype(float)[..., None])


# ---------------------------------------------------------------- refusals --

def _caches(nb=2, h=2, bs=128):
    return M.allocate_fp4_kvcache(nb, bs, h, device="cpu")


def test_shapes_and_allocation():
    kc, vc, ks, vs = M.allocate_fp4_kvcache(3, 256, 8, num_layers=2, device="cpu")
    assert kc.shape == (2, 3, 8, 16, 4, 16, 16) and vc.shape == (2, 3, 8, 256, 64)
    assert ks.shape == (2, 3, 8, 4, 4, 16, 4) and vs.shape == (2, 3, 8, 256)
    assert kc.dtype == ks.dtype == torch.uint8 and vs.dtype == torch.float32
    assert sum(t[0, 0, 0].numel() * t.element_size() for t in (kc, vc, ks, vs)) == 256 * 136
    for bs in (0, 64, 100, -128):
        with pytest.raises(AssertionError):
            M.fp4_cache_shapes(3, bs, 8)


def _calls(q, k, caches, lens, tables, cu):
    return [
        lambda: M.store_fp4_kvcache(k, k, *caches, lens),
        lambda: M.load_fp4_kvcache(*caches, lens),
        lambda: M.fp4_decode_attention(q, *caches, lens, tables, 0.1),
        lambda: M.fp4_chunk_prefill_attention(q, *caches, tables[0], 0, 0.1),
        lambda: M.fp4_varlen_prefill_attention(q, *caches, tables[:1], cu, cu, 2, 0.1),
    ]


def test_host_tensors_are_refused():
    q, k = torch.zeros(2, 4, 128).half(), torch.zeros(2, 2, 128).half()
    lens, tables = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 1, dtype=torch.int32)
    for call in _calls(q, k, _caches(), lens, tables, lens):
        with pytest.raises(AssertionError, match="GPU|must be on"):
            call()
    with pytest.raises(AssertionError, match="GPU"):
        M.copy_kv_blocks(_caches(), [0], [1])
    with pytest.raises(AssertionError, match="GPU"):
        M.compact_kv_blocks(_caches(), tables)


def test_caches_of_other_shapes_and_types_are_refused():
    q, k = torch.zeros(2, 4, 128).half(), torch.zeros(2, 2, 128).half()
    lens, tables = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 1, dtype=torch.int32)
    good = _caches()
    for i, bad in ((0, good[0].float()), (0, good[0][..., :8]), (1, good[1][:, :1]),
                   (1, good[1][..., :32]), (2, good[2].view(torch.int8)), (2, good[2][:1]),
                   (3, good[3].double()), (3, good[3][:, :, :64]),
                   (1, good[1].transpose(0, 1).contiguous().transpose(0, 1))):
        caches = list(good)
        caches[i] = bad
        for call in _calls(q, k, caches, lens, tables, lens):
            with pytest.raises(AssertionError):
                call()


FAKE = 1 << 20  # a pointer that nothing reads: every call here is refused first


def test_the_c_entries_refuse_before_any_launch():
    lib = _lib.load()
    E, U, W = -1, -2, -3

    def store(tokens=4, hk=2, d=128, bs=128, nb=4, dt=0, ks=256, vs=256, key=FAKE, slot=1,
              kc=FAKE):
        return lib.mskv_store_fp4_kvcache(key, ks, FAKE, vs, kc, FAKE, FAKE, FAKE, FAKE, slot,
                                          tokens, hk, d, bs, nb, dt, None)

    assert store(tokens=0) == 0
    assert store(tokens=-1) == E and store(hk=0) == E and store(nb=-1) == E and store(bs=0) == E
    assert store(d=64) == U and store(bs=64) == U and store(bs=1 << 25) == U
    assert store(nb=1 << 60) == U
    assert store(dt=3) == E and store(slot=2) == E and store(ks=248) == E and store(vs=260) == E
    assert store(key=None) == E and store(key=FAKE + 8) == E and store(kc=FAKE + 8) == E

    def load(tokens=4, out=FAKE, dt=1):
        return lib.mskv_load_fp4_kvcache(FAKE, FAKE, FAKE, FAKE, FAKE, 0, out, FAKE, tokens, 2,
                                         128, 128, 4, dt, None)

    assert load(tokens=0) == 0 and load(tokens=-1) == E and load(dt=5) == E
    assert load(out=None) == E and load(out=FAKE + 2) == E

    def decode(b=2, hq=4, hk=2, d=128, bs=128, w=4, splits=None, dt=0, ws=None, n=0, kc=FAKE):
        if splits is None:
            splits = lib.mskv_fp4_decode_num_splits(b, hq, hk, w, bs)
        return lib.mskv_fp4_decode_attention(FAKE, kc, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, b, hq,
                                             hk, d, bs, 8, w, 0.1, dt, splits, ws, n, None)

    assert decode(b=0) == 0
    assert decode(hq=5) == E and decode(dt=2) == E and decode(w=0) == E and decode(hk=0) == E
    assert decode(d=64) == U and decode(bs=64) == U and decode(bs=192) == U
    assert decode(w=1 << 23) == U
    assert decode(splits=999) == E and decode(w=1, kc=None) == E
    assert lib.mskv_fp4_decode_num_splits(2, 4, 2, 90, 128) > 1 and decode(w=90) == W
    assert lib.mskv_fp4_decode_num_splits(2, 4, 2, 4, 128) == 1  # (no workspace)

    def prefill(seqs=1, total=4, cu=None, scale=0.1, bs=128, d=128, hq=4, prefix=0, kc=FAKE,
                ks=FAKE, dt=0):
        return lib.mskv_fp4_prefill_attention(FAKE, kc, FAKE, ks, FAKE, FAKE, cu, cu, prefix, FAKE,
                                              seqs, total, total, 0, hq, 2, d, bs, 8, 4, scale, dt,
                                              None, 0, None)

    assert prefill(total=0) == 0
    assert prefill(seqs=2) == E and prefill(hq=5) == E and prefill(prefix=-1) == E
    assert prefill(dt=2) == E and prefill(kc=None) == E and prefill(kc=FAKE + 8) == E
    assert prefill(ks=FAKE + 2) == E
    for scale in (0.0, -0.1, float("inf"), float("nan")):
        assert prefill(scale=scale) == U
    assert prefill(bs=64) == U and prefill(d=64) == U and prefill(seqs=70000, cu=FAKE) == U


def test_attention_refuses_other_alignments_and_tables_past_an_int():
    lib = _lib.load()
    splits = lib.mskv_fp4_decode_num_splits(2, 4, 2, 1, 128)
    for at in range(5):  # query, K, V and the two scales
        ptrs = [FAKE + (2 if i == at else 0) for i in range(5)]
        assert lib.mskv_fp4_decode_attention(*ptrs, FAKE, FAKE, FAKE, 2, 4, 2, 128, 128, 8, 1, 0.1,
                                             0, splits, FAKE, 1 << 20, None) == -1
        assert lib.mskv_fp4_prefill_attention(*ptrs, FAKE, None, None, 0, FAKE, 1, 4, 4, 0, 4, 2,
                                              128, 128, 8, 4, 0.1, 0, None, 0, None) == -1
    assert lib.mskv_fp4_prefill_attention(*[FAKE] * 6, None, None, 0, FAKE, 1, 4, 4, 0, 4, 2, 128,
                                          128, 8, 1 << 24, 0.1, 0, None, 0, None) == -2


def _pool(n=1, base=FAKE, planes=2, stride=None, page=256, blocks=8):
    stride = blocks * page if stride is None else stride
    return (n, (ctypes.c_void_p * n)(*[base] * n), (ctypes.c_int64 * n)(*[planes] * n),
            (ctypes.c_int64 * n)(*[stride] * n), (ctypes.c_int64 * n)(*[page] * n), blocks)


def _i32(x):
    return (ctypes.c_int32 * max(1, len(x)))(*x)


def test_page_moves_refuse_before_any_launch():
    lib = _lib.load()
    E, U = -1, -2

    def copy(src=(0,), dst=(1,), n=None, **pool):
        return lib.mskv_copy_kv_blocks(*_pool(**pool), _i32(src), _i32(dst),
                                       len(src) if n is None else n, None)

    assert copy(src=(), dst=()) == 0
    assert copy(n=-1) == E and copy(src=(8,)) == E and copy(dst=(-1,)) == E and copy(dst=(8,)) == E
    assert copy(src=(0, 1), dst=(2, 2)) == E  # written twice
    assert copy(src=(0, 1), dst=(2, 0)) == E  # written and read
    assert copy(src=(3,), dst=(3,)) == E
    assert copy(src=(0,) * 9, dst=tuple(range(9))) == E
    assert copy(base=None) == E and copy(planes=0) == E and copy(page=0) == E
    assert copy(stride=256) == E and copy(stride=-16) == E  # planes that overlap
    assert copy(page=264) == U and copy(base=FAKE + 4) == U
    assert copy(n=1, base=FAKE, page=16 << 40, blocks=1 << 30) == E
    assert copy(page=(1 << 24) * 16384, blocks=8) == U
    assert lib.mskv_copy_kv_blocks(0, None, None, None, None, 8, _i32((0,)), _i32((1,)), 1,
                                   None) == E
    assert lib.mskv_copy_kv_blocks(*_pool(n=9), _i32((0,)), _i32((1,)), 1, None) == E

    def compact(tables=FAKE, n=4, new=2 * FAKE, remap=FAKE, **pool):
        return lib.mskv_compact_kv_blocks(*_pool(**pool), tables, n, new, remap, FAKE, None)

    assert compact(n=-1) == E and compact(tables=None) == E and compact(remap=None) == E
    assert compact(new=None) == E and compact(new=FAKE) == E  # tables that others still read
    assert compact(new=FAKE + 12) == E and compact(new=FAKE - 12) == E
    assert compact(remap=FAKE + 12) == E  # written over the tables
    assert compact(blocks=0) == E and compact(blocks=1 << 19) == U
    assert compact(page=8) == U


def test_copies_refuse_ids_in_python_too(monkeypatch):
    """Before the library is reached, whatever the device."""
    monkeypatch.setattr(_lib, "on_device", lambda *a: None)
    pool = torch.zeros(2, 8, 64)
    for src, dst in (([0], [8]), ([-1], [0]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([1], [1]),
                     ([0], [1, 2]), ([1 << 40], [0])):
        with pytest.raises(AssertionError):
            M.copy_kv_blocks(pool, src, dst, block_dim=1)
    M.copy_kv_blocks(pool, [], [], block_dim=1)
    with pytest.raises(AssertionError, match="same blocks"):
        M.copy_kv_blocks((pool, pool[:, :4].contiguous()), [0], [1], block_dim=1)
    with pytest.raises(AssertionError, match="contiguous"):
        M.copy_kv_blocks(pool[:, ::2], [0], [1], block_dim=1)
    for n in (0, 9, -1):
        with pytest.raises(AssertionError, match="num_blocks"):
            M.compact_kv_blocks(pool, torch.zeros(3, dtype=torch.int32), n, block_dim=1)


def test_the_layer_takes_either_cache():
    layer = M.Attention(4, 128, 0.1, 2)
    layer.k_cache = torch.zeros(1)
    layer.kv_cache_dtype = "int8"
    with pytest.raises(NotImplementedError):
        layer._check_cache()
    layer.kv_cache_dtype = "fp4_e2m1"
    layer._check_cache()
    with pytest.raises(NotImplementedError, match="forward"):
        layer.forward_fused(*[None] * 9)


def test_native_paths_leave_other_calls_to_the_wrappers():
    f = _lib.fast
    q, k = torch.zeros(2, 4, 128).half(), torch.zeros(2, 2, 128).half()
    caches, i32 = _caches(), torch.zeros(2, dtype=torch.int32)
    assert f.store4(k, k, *caches, i32) is None
    assert f.load4(*caches, i32, torch.float16) is None
    assert f.decode4(q, *caches, i32, i32.view(-1, 1), 0.1, None, None) is None
    assert f.prefill4(q, *caches, i32, None, None, 0, 2, 0, 0.1) is None
    pool = torch.zeros(3, 64)
    assert f.copy_blocks(pool, [0], [1], 0) is None and f.copy_blocks((pool,), [0], [1], 0) is None
    assert f.compact_blocks([pool], i32, None, 0) is None
    for fn in (f.copy_blocks, f.compact_blocks):
        assert fn() is None and fn(*[None] * 4) is None and fn(*["x"] * 4) is None
        assert fn((), [], [], 0) is None and fn((3, "y"), (1 << 40,), [1.5], -1) is None
    for fn in (f.store4, f.load4, f.decode4, f.prefill4):
        assert fn() is None
        assert fn(*[None] * 6) is None and fn(*[None] * 7) is None and fn(*["x"] * 12) is None
