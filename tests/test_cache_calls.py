"""The decode over shared prefixes, the attention weights and the eviction launch
with their tensors' GPU as the current device, in the wrappers and in the native
paths, and the native paths leave what they cannot take to the wrappers."""

import contextlib
import os
import re

import pytest
import torch

import microserve_amd as M
from microserve_amd import _lib

HERE = os.path.dirname(os.path.abspath(__file__))
NATIVE = os.path.join(HERE, "..", "microserve_amd", "csrc", "host", "cache_calls.h")


class _Lib:
    """The library, with launches noted by the device that is current."""

    def __init__(self, lib):
        self._lib, self.inside, self.launches = lib, None, []

    def __getattr__(self, name):
        if name.endswith("workspace_bytes"):
            return getattr(self._lib, name)

        def launch(*args):
            self.launches.append((name, self.inside))
            return 0
        return launch


@pytest.fixture
def lib(monkeypatch):
    lib = _Lib(_lib.load())

    @contextlib.contextmanager
    def current(t):
        before, lib.inside = lib.inside, t.device
        yield
        lib.inside = before

    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(_lib, "on_device", lambda *a: None)
    monkeypatch.setattr(_lib, "current", current)
    monkeypatch.setattr(_lib, "stream_of", lambda t: 0)
    return lib


def _arguments():
    n, hq, hk, bs = 3, 8, 2, 128
    q = torch.zeros(n, hq, 128).half()
    kv = torch.zeros(4, bs, hk, 128).to(torch.float8_e4m3fn)
    sc = torch.ones(4, bs, hk)
    lens, tables = torch.zeros(n, dtype=torch.int32), torch.zeros(n, 2, dtype=torch.int32)
    return q, (kv, kv, sc, sc), lens, tables, torch.zeros(4, hk, bs)


def test_the_wrappers_launch_on_their_tensors_device(lib):
    q, cache, lens, tables, w = _arguments()
    cu = torch.arange(4, dtype=torch.int32)
    groups = torch.tensor([0, 3], dtype=torch.int32)
    M.fp8_shared_prefix_decode_attention(q, *cache, lens, tables, 0.1, groups, lens[:1])
    M.fp8_decode_attention_weights(q, *cache, lens, tables, 0.1, w)
    M.fp8_window_attention_weights(q, cache[0], cache[2], tables, cu, cu, 1, 0.1, w)
    M.evict_kv_tokens(*cache, *M.select_kv_tokens(w, lens, tables, 4), tables, w)
    assert [name for name, _ in lib.launches] == [
        "mskv_fp8_shared_prefix_decode_attention", "mskv_fp8_decode_attention_weights",
        "mskv_fp8_window_attention_weights", "mskv_select_kv_tokens", "mskv_evict_kv_tokens"]
    assert all(device == q.device for _, device in lib.launches)


def test_the_native_paths_launch_inside_the_device_scope():
    text = open(NATIVE).read()
    launches = list(re.finditer(r"status = api\.(\w+)\(", text))
    assert sorted(m.group(1) for m in launches) == ["choose", "evict", "shared", "track", "window"]
    scopes = [m.start() for m in re.finditer(r"const OnDevice on\(in\.device\);", text)]
    for m in launches:
        opened = max(p for p in scopes if p < m.start())
        body = text[text.rindex("{", 0, opened):m.start()]
        assert body.count("{") > body.count("}"), "a launch behind the scope's end"
        # outputs and workspaces too come from this device's current stream
        assert "at::empty" not in text[text.rindex("\n}\n", 0, opened):opened]


def test_tensors_that_are_not_on_a_gpu_are_left_to_the_wrappers():
    _lib.load()
    q, cache, lens, tables, w = _arguments()
    cu, kept = torch.arange(4, dtype=torch.int32), torch.zeros(3, 2, 4, dtype=torch.int32)
    fast = _lib.fast
    assert fast.shared(q, *cache, lens, tables, 0.1, cu, lens, None, None) is None
    assert fast.track(q, *cache, lens, tables, 0.1, w, 0, None) is None
    assert fast.window(q, cache[0], cache[2], tables, cu, cu, 1, 0.1, w, False, 0, None) is None
    assert fast.choose(w, lens, tables, 4, 0, 0) is None
    assert fast.evict(*cache, kept, lens, tables, w) is None
    for call in (fast.shared, fast.track, fast.window, fast.choose, fast.evict):
        assert call(1, 2) is None
