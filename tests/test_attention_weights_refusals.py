"""What the weights' and eviction's entries refuse, before any launch."""

import pytest
import torch

import microserve_amd as M
from microserve_amd import _lib

NB, H, BS, B = 4, 2, 128, 2


@pytest.fixture
def cpu(monkeypatch):
    """Tensors on the CPU, and a library whose launches fail the test."""
    class Lib:
        def __getattr__(self, name):
            if name.endswith("workspace_bytes"):
                return lambda *a: 0
            raise AssertionError(f"{name} was launched")
    monkeypatch.setattr(_lib, "load", Lib)
    monkeypatch.setattr(_lib, "on_device", lambda *a: None)
    monkeypatch.setattr(_lib, "current", lambda t: __import__("contextlib").nullcontext())
    monkeypatch.setattr(_lib, "stream_of", lambda t: 0)


def _caches():
    kv = torch.zeros(NB, BS, H, 128).to(torch.float8_e4m3fn)
    return kv, kv.clone(), torch.ones(NB, BS, H), torch.ones(NB, BS, H)


def _ints(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def _decode(**k):
    q = k.pop("q", torch.zeros(B, 4, 128).half())
    w = k.pop("weights", M.allocate_attention_weights(NB, BS, H, device="cpu"))
    return M.fp8_decode_attention_weights(q, *k.pop("caches", _caches()), k.pop("lens", _ints(B)),
                                          k.pop("tables", _ints(B, 3)), 0.1, w, **k)


def _window(**k):
    q = k.pop("q", torch.zeros(B, 4, 128).half())
    w = k.pop("weights", M.allocate_attention_weights(NB, BS, H, device="cpu"))
    kc, _, ks, _ = _caches()
    return M.fp8_window_attention_weights(q, kc, ks, k.pop("tables", _ints(B, 3)),
                                          k.pop("cu_q", _ints(B + 1)), k.pop("cu_k", _ints(B + 1)),
                                          1, 0.1, w, **k)


def _select(**k):
    w = k.pop("weights", M.allocate_attention_weights(NB, BS, H, device="cpu"))
    return M.select_kv_tokens(w, k.pop("lens", _ints(B)), k.pop("tables", _ints(B, 3)),
                              k.pop("budget", 5), **k)


def _evict(**k):
    return M.evict_kv_tokens(*k.pop("caches", _caches()), k.pop("kept", _ints(B, H, 5)),
                             k.pop("lens", _ints(B)), k.pop("tables", _ints(B, 3)), **k)


W = torch.zeros
REFUSED = [
    (_decode, dict(weights=W(NB, BS, H))), (_decode, dict(weights=W(NB, H, BS).double())),
    (_decode, dict(weights=W(NB, BS, H).transpose(1, 2))), (_decode, dict(start=-1)),
    (_decode, dict(start=torch.zeros(B))), (_decode, dict(start=_ints(B + 1))),
    (_decode, dict(lens=_ints(B + 1))), (_decode, dict(tables=_ints(B + 1, 3))),
    (_decode, dict(q=torch.zeros(B, 3, 128).half())), (_decode, dict(q=torch.zeros(B, 4, 128))),
    (_decode, dict(out=torch.zeros(B, 4, 128))),
    (_window, dict(weights=W(NB, H, BS + 1))), (_window, dict(cu_k=_ints(B))),
    (_window, dict(tables=_ints(B))), (_window, dict(q=torch.zeros(B, 4, 64).half())),
    (_window, dict(cu_q=torch.zeros(B + 1, dtype=torch.int64))), (_window, dict(start=-3)),
    (_select, dict(budget=0)), (_select, dict(recent=-1)), (_select, dict(start=-1)),
    (_select, dict(weights=W(NB, H, BS).half())), (_select, dict(weights=W(NB, H))),
    (_select, dict(lens=torch.zeros(B, dtype=torch.int64))), (_select, dict(tables=_ints(B + 1, 3))),
    (_evict, dict(kept=_ints(B, H + 1, 5))), (_evict, dict(kept=_ints(B, 5))),
    (_evict, dict(kept=torch.zeros(B, H, 5))), (_evict, dict(weights=W(NB, BS, H))),
    (_evict, dict(tables=_ints(B + 1, 3))),
    (_evict, dict(caches=tuple(t.transpose(1, 2) for t in _caches()))),
]


@pytest.mark.parametrize("call,args", REFUSED)
def test_refused_by_the_wrapper(cpu, call, args):
    with pytest.raises(AssertionError) as e:
        call(**args)
    assert "was launched" not in str(e.value)


def test_tensors_off_the_gpu_are_refused():
    for call in (_decode, _window, _select, _evict):
        with pytest.raises(AssertionError, match="GPU"):
            call()


def test_refused_by_the_c_abi():
    lib = _lib.load()
    p = 1 << 20  # never read: the arguments are refused first

    def decode(weights=p, bs=256, hq=32, hk=8, d=128, w=4, start=0, dtype=0, ws=p, nbytes=1 << 40,
               batch=2):
        return lib.mskv_fp8_decode_attention_weights(
            p, p, p, p, p, p, p, weights, None, start, p, batch, hq, hk, d, bs, 8, w, 0.1, dtype,
            ws, nbytes, None)
    assert decode(weights=None) == decode(weights=p + 4) == decode(start=-1) == -1
    assert decode(hq=30) == decode(dtype=2) == decode(batch=-1) == decode(w=0) == -1
    assert decode(d=64) == decode(bs=100) == -2
    assert decode(ws=None) == decode(nbytes=16) == -3
    # past 1 GiB of scores K is read again, in pages of whole 128s
    assert decode(bs=96, w=1 << 16, batch=2) == -2

    def window(hq=32, hk=8, d=128, bs=256, dtype=0, start=0, ws=p, q=p, cu_q=p, weights=p, mq=2):
        return lib.mskv_fp8_window_attention_weights(
            q, p, p, p, cu_q, p, weights, None, start, 0, 2, 4, mq, 0, hq, hk, d, bs, 8, 4, 0.1,
            dtype, ws, 1 << 40, None)
    assert window(hq=30) == window(dtype=2) == window(start=-1) == window(q=None) == -1
    assert window(cu_q=None) == window(weights=None) == window(q=p + 2) == window(mq=-1) == -1
    assert window(d=64) == window(bs=96) == window(mq=1 << 30) == -2
    assert window(ws=None) == -3

    def select(weights=p, kept=p, budget=4, start=0, recent=0, bs=256, w=4, hk=8):
        return lib.mskv_select_kv_tokens(weights, p, p, None, start, recent, budget, kept, p, 2,
                                         hk, bs, 8, w, None)
    assert select(weights=None) == select(kept=None) == select(budget=0) == select(start=-1) == -1
    assert select(recent=-1) == select(bs=0) == select(hk=0) == -1
    assert select(w=1 << 22) == select(hk=1 << 17) == -2

    def evict(kc=p, kept=p, d=128, budget=4, w=4):
        return lib.mskv_evict_kv_tokens(kc, p, p, p, None, kept, p, p, 2, 8, d, 256, 8, w, budget,
                                        None)
    assert evict(kc=None) == evict(kc=p + 8) == evict(kept=None) == evict(budget=0) == -1
    assert evict(d=64) == evict(w=1 << 22) == -2


def test_workspaces_follow_the_shapes():
    lib = _lib.load()
    scores = 64 * 32 * (16 * 256 + 32) * 4
    splits = lib.mskv_decode_num_splits(64, 32, 8, 16, 256)
    part = (64 * 32 * splits * 129 * 4 + 255) // 256 * 256
    assert lib.mskv_decode_weights_workspace_bytes(64, 32, 8, 256, 16) == part + scores
    # the largest tables: no scores in memory
    wide = lib.mskv_decode_weights_workspace_bytes(256, 32, 8, 256, 512)
    assert wide < 256 * 32 * 512 * 256 * 4
    # partials of four and of two tiles, the logarithms, and the tiles of a range
    assert lib.mskv_window_weights_workspace_bytes(32, 1000, 32, 256, 128) == 32 * 32 * 5 * 4 + 4
    assert lib.mskv_window_weights_workspace_bytes(32, 0, 32, 256, 2) == 32 * 32 * 3 * 4 + 4
