"""Groups of sequences by their first pages, and what the decode over shared
prefixes refuses."""

import pytest
import torch

import microserve_amd as M
from microserve_amd import _lib


def test_groups_by_their_first_pages():
    tables = [[5, 6, 7], [1, 2], [5, 6, 9, 4], [8], [5, 6], [1, 3]]
    order, cu, prefixes = M.group_by_prefix(tables, 16)
    assert order == [1, 5, 0, 2, 4, 3] and cu == [0, 2, 5, 6] and prefixes == [16, 32, 0]
    assert M.group_by_prefix([], 16) == ([], [0], [])
    assert M.group_by_prefix([[], [3], []], 16)[1:] == ([0, 1, 2, 3], [0, 0, 0])
    assert M.group_by_prefix([[2, 4], [2, 4]], 8) == ([0, 1], [0, 2], [16])


def _call(**k):
    kv = torch.zeros(4, 128, 2, 128).to(torch.float8_e4m3fn)
    sc = torch.ones(4, 128, 2)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    return M.fp8_shared_prefix_decode_attention(
        k.pop("q", torch.zeros(3, 4, 128).half()), kv, kv, sc, k.pop("v_scale", sc),
        k.pop("lens", i32(3)), k.pop("tables", i32(3, 2)), 0.1, k.pop("cu", i32(3)),
        k.pop("prefixes", i32(2)), **k)


@pytest.mark.parametrize("args", [
    dict(cu=torch.zeros(2, dtype=torch.int32)), dict(cu=torch.zeros(3)),
    dict(prefixes=torch.zeros(2, dtype=torch.int64)), dict(max_prefix_len=-1),
    dict(cu=torch.zeros(1026, dtype=torch.int32), prefixes=torch.zeros(1025, dtype=torch.int32)),
    dict(lens=torch.zeros(2, dtype=torch.int32)), dict(tables=torch.zeros(2, 2, dtype=torch.int32)),
    dict(q=torch.zeros(3, 3, 128).half()), dict(q=torch.zeros(3, 4, 128)),
    dict(v_scale=torch.ones(4, 128, 3)), dict(out=torch.zeros(3, 4, 128))])
def test_refused_by_the_wrapper(monkeypatch, args):
    monkeypatch.setattr(_lib, "on_device", lambda *a: None)
    with pytest.raises(AssertionError):
        _call(**args)


def test_tensors_off_the_gpu_are_refused():
    with pytest.raises(AssertionError, match="GPU"):
        _call()


def test_refused_by_the_c_abi():
    lib, p = _lib.load(), 1 << 20

    def call(q=p, cu=p, bound=512, batch=4, groups=2, hq=32, hk=8, d=128, bs=256, w=8, dtype=0,
             ws=p, nbytes=1 << 40, kc=p):
        return lib.mskv_fp8_shared_prefix_decode_attention(
            q, kc, p, p, p, p, p, cu, p, bound, p, batch, groups, hq, hk, d, bs, 9, w, 0.1, dtype,
            ws, nbytes, None)
    assert call(q=None) == call(cu=None) == call(bound=-1) == call(groups=-1) == call(dtype=2) == -1
    assert call(hq=30) == call(kc=p + 8) == call(w=0) == call(batch=-1) == -1
    assert call(d=64) == call(bs=192) == call(groups=1025) == call(w=1 << 22) == -2
    assert call(batch=1 << 20) == call(batch=60000, w=1 << 14) == -2
    assert call(ws=None) == call(nbytes=100) == -3
    assert call(batch=0, q=None) == 0


def test_the_workspace_follows_the_shapes():
    lib = _lib.load()
    size = lambda *a: lib.mskv_shared_decode_workspace_bytes(*a)  # noqa: E731
    assert size(64, 1, 32, 8, 256, 34, 8192) < 256 << 20
    assert size(64, 1, 32, 8, 256, 34, 8192) > size(64, 1, 32, 8, 256, 34, 0) > 64 * 32 * 129 * 4
    assert size(0, 1, 32, 8, 256, 34, 8192) == size(4, 1, 30, 8, 256, 34, 0) == 0
