"""A pool of more tensors than one launch takes is refused whole: no launch
has moved anything when a later tensor turns out not to be supported."""

import contextlib

import pytest
import torch

import microserve_amd as M
from microserve_amd import _lib
from microserve_amd.kv_blocks import MAX_POOLS

PAGES = 6


class _Recorded:
    """The library with its two moves noted instead of launched: they answer as
    the library does to a pool that it does not take."""

    def __init__(self, lib):
        self._lib, self.moved = lib, []

    def __getattr__(self, name):
        return getattr(self._lib, name)

    def _move(self, pool):
        status = self._lib.mskv_copy_kv_blocks(*pool, None, None, 0, None)
        if status == 0:
            self.moved.append(pool[0])
        return status

    def mskv_copy_kv_blocks(self, *args):
        return self._move(args[:6])

    def mskv_compact_kv_blocks(self, *args):
        return self._move(args[:6])


@pytest.fixture
def recorded(monkeypatch):
    lib = _Recorded(_lib.load())
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(_lib, "on_device", lambda *a: None)
    monkeypatch.setattr(_lib, "current", lambda t: contextlib.nullcontext())
    monkeypatch.setattr(_lib, "stream_of", lambda t: None)
    return lib


def _bad(kind):
    if kind == "page":  # of 12 bytes
        return torch.zeros(PAGES, 3)
    flat = torch.zeros(PAGES * 4 + 8)
    at = 1 + (-flat.data_ptr() // 4) % 4  # one element past 16 bytes
    return flat[at:at + PAGES * 4].view(PAGES, 4)


@pytest.mark.parametrize("kind", ["page", "start"])
@pytest.mark.parametrize("at", [0, MAX_POOLS - 1, MAX_POOLS, 2 * MAX_POOLS])
def test_no_tensor_moves_beside_one_that_is_refused(recorded, kind, at):
    pools = [torch.zeros(PAGES, 8) for _ in range(2 * MAX_POOLS + 1)]
    pools[at] = _bad(kind)
    with pytest.raises(RuntimeError, match="not supported"):
        M.copy_kv_blocks(pools, [0], [1])
    with pytest.raises(RuntimeError, match="not supported"):
        M.compact_kv_blocks(pools, torch.tensor([[4, 1]], dtype=torch.int32))
    assert recorded.moved == []


def test_pools_of_several_launches_move_whole(recorded):
    pools = [torch.zeros(PAGES, 8) for _ in range(2 * MAX_POOLS + 1)]
    M.copy_kv_blocks(pools, [0], [1])
    assert recorded.moved == [MAX_POOLS, MAX_POOLS, 1]
    M.compact_kv_blocks(pools, torch.tensor([[4, 1]], dtype=torch.int32))
    assert recorded.moved == 2 * [MAX_POOLS, MAX_POOLS, 1]


def test_too_many_pages_are_refused_before_any_move(recorded):
    pools = [torch.zeros((1 << 18) + 1, 4) for _ in range(MAX_POOLS + 1)]
    tables = torch.tensor([[4, 1]], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="not supported"):
        M.compact_kv_blocks(pools, tables)
    assert recorded.moved == []
    M.compact_kv_blocks(pools, tables, 1 << 18)
    assert recorded.moved == [MAX_POOLS, 1]


def test_the_check_answers_as_the_calls_do():
    import ctypes
    lib, at = _lib.load(), 1 << 20

    def pool(n=1, base=at, planes=2, stride=None, page=256, blocks=8):
        stride = blocks * page if stride is None else stride
        return (n, (ctypes.c_void_p * n)(*[base] * n), (ctypes.c_int64 * n)(*[planes] * n),
                (ctypes.c_int64 * n)(*[stride] * n), (ctypes.c_int64 * n)(*[page] * n), blocks)

    for compact in (0, 1):
        assert lib.mskv_check_kv_blocks(*pool(), compact) == 0
        for args, status in ((dict(base=None), -1), (dict(planes=0), -1), (dict(stride=256), -1),
                             (dict(n=MAX_POOLS + 1), -1), (dict(page=264), -2),
                             (dict(base=at + 4), -2)):
            assert lib.mskv_check_kv_blocks(*pool(**args), compact) == status, (args, compact)
    assert lib.mskv_check_kv_blocks(*pool(blocks=1 << 19), 0) == 0
    assert lib.mskv_check_kv_blocks(*pool(blocks=1 << 19), 1) == -2
    assert lib.mskv_check_kv_blocks(*pool(blocks=0), 1) == -1
