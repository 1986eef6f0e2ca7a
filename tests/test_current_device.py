"""Attention, stores, the prologue and the page moves launch with their
tensors' GPU as the current device, whichever was current at the call: in the
wrappers by the guard they hold at the moment of the launch, in the native
paths by the scope that launches need."""

import contextlib
import os
import re

import pytest
import torch

import microserve_amd as M
from microserve_amd import _lib

HERE = os.path.dirname(os.path.abspath(__file__))
NATIVE = os.path.join(HERE, "..", "microserve_amd", "csrc", "host", "fast_calls.cpp")
HOST_ONLY = ("workspace_bytes", "num_splits", "check_kv_blocks", "status_string")


class _Lib:
    """The library, with launches noted by the device that is current."""

    def __init__(self, lib):
        self._lib, self.inside, self.launches = lib, None, []

    def __getattr__(self, name):
        if name.endswith(HOST_ONLY):
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


def test_the_wrappers_launch_on_their_tensors_device(lib):
    n, hq, hk, bs = 3, 8, 2, 128
    q, k = torch.zeros(n, hq, 128).half(), torch.zeros(n, hk, 128).half()
    i32, tables = torch.zeros(n, dtype=torch.int32), torch.zeros(n, 70, dtype=torch.int32)
    cu, slots = torch.arange(n + 1, dtype=torch.int32), torch.arange(n)
    kv = torch.zeros(4, bs, hk, 128).to(torch.float8_e4m3fn)
    sc = torch.ones(4, bs, hk)
    eight, four = (kv, kv, sc, sc), M.allocate_fp4_kvcache(4, bs, hk, device="cpu")
    cos = torch.ones(16, 128).half()
    calls = {
        "store": lambda: (M.store_fp8_kvcache(k, k, *eight, slots),
                          M.store_fp4_kvcache(k, k, *four, slots),
                          M.load_fp4_kvcache(*four, slots)),
        "decode": lambda: (M.fp8_decode_attention(q, *eight, i32, tables, 0.1),
                           M.fp4_decode_attention(q, *four, i32, tables, 0.1)),
        "prefill": lambda: (
            M.fp8_chunk_prefill_attention(q, *eight, tables[0], 5, 0.1),
            M.fp8_varlen_prefill_attention(q, *eight, tables, cu, cu, 1, 0.1),
            M.fp4_chunk_prefill_attention(q, *four, tables[0], 5, 0.1),
            M.fp4_varlen_prefill_attention(q, *four, tables, cu, cu, 1, 0.1),
            M.varlen_attention(q, k, k, cu, cu, 1)),
        "prologue": lambda: M.qk_norm_rope_store(slots, q, k, k, None, None, 1e-6, cos, cos,
                                                 *eight, slots),
        "pages": lambda: (M.copy_kv_blocks(four, [0], [1]), M.compact_kv_blocks(four, tables)),
    }
    for what, call in calls.items():
        lib.launches.clear()
        call()
        assert lib.launches, what
        for name, device in lib.launches:
            assert device == q.device, f"{name} was launched beside its device's guard"


def test_the_native_paths_release_the_lock_only_under_the_device():
    """One scope does both, and every launch of the bound entries lies in one."""
    text = open(NATIVE).read()
    assert len(re.findall(r"PyEval_SaveThread", text)) == 1
    scope = re.search(r"struct (\w+) \{\n  const c10::DeviceGuard guard;", text).group(1)
    launches = re.findall(r"(?:status = api\.|status = call\(api\.)(\w+)", text)
    assert set(launches) == {"store", "store4", "load4", "decode", "decode4", "prefill",
                             "prefill4", "fresh", "prologue", "copy", "compact"}
    scopes = [m.start() for m in re.finditer(scope + r" on\(in\.device\);", text)]
    for m in re.finditer(r"status = (?:api\.\w+|call\(api\.)", text):
        opened = max(p for p in scopes if p < m.start())
        body = text[text.rindex("{", 0, opened):m.start()]
        assert body.count("{") > body.count("}"), "a launch behind the scope's end"
