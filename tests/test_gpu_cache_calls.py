"""The native call paths of shared prefixes, attention weights and eviction give
what their wrappers' own paths give, and refuse what those refuse."""

import numpy as np
import pytest
import torch

import microserve_amd as M
from microserve_amd import _lib
from tests import weights_helpers as H

pytestmark = pytest.mark.gpu
SCALE = 0.09


class _None:
    """Native paths that take nothing."""

    def __getattr__(self, name):
        return lambda *a: None


@pytest.fixture
def both(monkeypatch):
    """Runs a call on both paths; the results, and that the native one was taken."""
    native = _lib.fast

    def run(name, call):
        seen = []

        class Noted:
            def __getattr__(self, attr):
                def f(*a):
                    res = getattr(native, attr)(*a)
                    seen.append((attr, res is not None))
                    return res
                return f
        monkeypatch.setattr(_lib, "fast", Noted())
        first = call()
        assert (name, True) in seen, f"{name} was left to the wrapper"
        monkeypatch.setattr(_lib, "fast", _None())
        return first, call()
    return run


def _batch(dtype):
    gen = torch.Generator().manual_seed(3)
    lens, heads, block = [300, 1, 517], 2, 256
    _, cache = H.pool(gen, 8, heads, block)
    tables = H.tables_of(gen, lens, block, 8)
    q = torch.randn(3, 4 * heads, 128, generator=gen).to(H.DEV, dtype)
    w = torch.rand(8, heads, block, generator=gen).to(H.DEV)
    return q, cache, H.gpu(lens), H.gpu(tables), w


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tensor_start", [False, True])
def test_both_paths_agree(both, dtype, tensor_start):
    _lib.load()
    q, cache, lens, tables, w = _batch(dtype)
    start = H.gpu([2, 0, 5]) if tensor_start else 3

    def track(out=None):
        x = w.clone()
        return M.fp8_decode_attention_weights(q, *cache, lens, tables, SCALE, x, start, out), x
    for a, b in zip(*both("track", track)):
        assert torch.equal(a, b)
    out = torch.empty_like(q)
    (a, _), (b, _) = both("track", lambda: track(out))
    assert a is out and b is out

    cu, cu_k = H.gpu([0, 1, 2, 3]), torch.cumsum(torch.nn.functional.pad(lens, (1, 0)), 0).int()
    for accumulate in (False, True):
        for bound in (None, 520):
            def window():
                x = w.clone()
                assert M.fp8_window_attention_weights(q, cache[0], cache[2], tables, cu, cu_k, 1,
                                                      SCALE, x, accumulate, start, bound) is x
                return x
            a, b = both("window", window)
            assert torch.equal(a, b)

    def evict():
        kept, n = M.select_kv_tokens(w, lens, tables, 100, 10, start)
        c, x = [t.clone() for t in cache], w.clone()
        assert M.evict_kv_tokens(*c, kept, n, tables, x) is None
        M.evict_kv_tokens(*c, kept, n, tables)
        return [kept, n, x] + [t.view(torch.uint8) if t.element_size() == 1 else t for t in c]
    for a, b in zip(*both("evict", evict)):
        assert torch.equal(a, b)

    cu_groups, prefix = H.gpu([0, 2, 3]), H.gpu([0, 256])
    for bound in (None, 256, 0):
        a, b = both("shared", lambda: M.fp8_shared_prefix_decode_attention(
            q, *cache, lens, tables, SCALE, cu_groups, prefix, bound))
        assert torch.equal(a, b)


def test_what_the_wrappers_refuse():
    q, cache, lens, tables, w = _batch(torch.float16)
    cu, groups, prefix = H.gpu([0, 1, 2, 3]), H.gpu([0, 3]), H.gpu([0])
    kept, n = M.select_kv_tokens(w, lens, tables, 100)
    before = w.clone()
    for call in (
            lambda: M.fp8_decode_attention_weights(q, *cache, lens, tables, SCALE, w[:4]),
            lambda: M.fp8_decode_attention_weights(q, *cache, lens, tables, SCALE, w, start=-1),
            lambda: M.fp8_decode_attention_weights(q, *cache, lens, tables, SCALE, w,
                                                   start=H.gpu([1, 2])),
            lambda: M.fp8_decode_attention_weights(q, *cache, lens[:2], tables, SCALE, w),
            lambda: M.fp8_decode_attention_weights(q, *cache, lens, tables, SCALE, w, 0,
                                                   torch.empty_like(q)[:2]),
            lambda: M.fp8_window_attention_weights(q, cache[0], cache[2], tables, cu, cu[:3], 1,
                                                   SCALE, w),
            lambda: M.fp8_window_attention_weights(q.float(), cache[0], cache[2], tables, cu, cu, 1,
                                                   SCALE, w),
            lambda: M.select_kv_tokens(w, lens, tables, 0),
            lambda: M.select_kv_tokens(w, lens, tables, 4, recent=-1),
            lambda: M.select_kv_tokens(w.half(), lens, tables, 4),
            lambda: M.evict_kv_tokens(*cache, kept[:, :1].contiguous(), n, tables),
            lambda: M.evict_kv_tokens(*cache, kept, n, tables, w[:2]),
            lambda: M.fp8_shared_prefix_decode_attention(q, *cache, lens, tables, SCALE, groups,
                                                         H.gpu([0, 0])),
            lambda: M.fp8_shared_prefix_decode_attention(q, *cache, lens, tables, SCALE, groups,
                                                         prefix, -1),
            lambda: M.fp8_shared_prefix_decode_attention(q, *cache, lens, tables, SCALE, groups,
                                                         prefix.long())):
        with pytest.raises((AssertionError, TypeError, ValueError)):
            call()
    torch.cuda.synchronize()
    assert torch.equal(w, before)


def test_arguments_of_other_layouts_go_to_the_wrapper():
    """Lengths and tables with strides, and a query that starts off 16 bytes."""
    q, cache, lens, tables, w = _batch(torch.bfloat16)
    flat = torch.empty(q.numel() + 1, dtype=q.dtype, device=H.DEV)
    off = flat[1:].view(q.shape).copy_(q)
    l2 = torch.stack([lens, lens], 1)[:, 0]
    t2 = torch.cat([tables, tables], 1)[:, :tables.shape[1]]
    assert not l2.is_contiguous() and not t2.is_contiguous()
    a, b = w.clone(), w.clone()
    x = M.fp8_decode_attention_weights(q, *cache, lens, tables, SCALE, a)
    y = M.fp8_decode_attention_weights(off, *cache, l2, t2, SCALE, b)
    assert torch.equal(x, y) and torch.equal(a, b)
    for got, want in zip(M.select_kv_tokens(a, l2, t2, 50, 5),
                         M.select_kv_tokens(a, lens, tables, 50, 5)):
        assert torch.equal(got, want)
    groups, prefix = H.gpu([0, 1, 3]), H.gpu([256, 0])
    assert torch.equal(
        M.fp8_shared_prefix_decode_attention(off, *cache, l2, t2, SCALE, groups, prefix),
        M.fp8_shared_prefix_decode_attention(q, *cache, lens, tables, SCALE, groups, prefix))


def test_captured_run_replays():
    """A turn's window weights, a decode step that keeps weights, the choice and the
    moving in one graph: each replay, over lengths and caches of its own, is the
    eager run."""
    gen = torch.Generator().manual_seed(12)
    heads, block, scale = 2, 128, 0.1
    _, pool = H.pool(gen, 16, heads, block)
    tables = H.gpu(H.tables_of(gen, [512, 640, 384], block, 16))
    q = torch.randn(3, 8, 128, generator=gen).half().to(H.DEV)
    qw = torch.randn(24, 8, 128, generator=gen).half().to(H.DEV)
    cu_q = H.gpu([0, 10, 10, 24])
    lens, cu_k = H.gpu([1, 1, 1]), H.gpu([0, 1, 2, 3])
    cache, w = [t.clone() for t in pool], torch.zeros(16, heads, block, device=H.DEV)

    def run(c, x):
        M.fp8_window_attention_weights(qw, c[0], c[2], tables, cu_q, cu_k, 14, scale, x)
        out = M.fp8_decode_attention_weights(q, *c, lens, tables, scale, x, 3)
        kept, n = M.select_kv_tokens(x, lens, tables, 200, 20, 3)
        M.evict_kv_tokens(*c, kept, n, tables, x)
        return out, kept, n

    def fill(n):
        lens.copy_(H.gpu(n))
        cu_k.copy_(H.gpu(np.cumsum([0, *n])))

    def bytes_of(c):
        return [t.view(torch.uint8) if t.element_size() == 1 else t for t in c]

    fill([500, 600, 300])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run([t.clone() for t in pool], w.clone())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(cache, w)
    for n in ([500, 600, 300], [20, 0, 384], [512, 640, 1], [201, 200, 199]):
        fill(n)
        for mine, start in zip(bytes_of(cache), bytes_of(pool)):
            mine.copy_(start)
        w.fill_(0.25)
        copy, x = [t.clone() for t in pool], w.clone()
        graph.replay()
        torch.cuda.synchronize()
        want = run(copy, x)
        torch.cuda.synchronize()
        for a, b in zip([*got, w, *bytes_of(cache)], [*want, x, *bytes_of(copy)]):
            assert torch.equal(a, b)


def test_two_streams_at_once():
    """Runs of the operators side by side, each with workspaces of its own."""
    runs = []
    for i in range(2):
        gen = torch.Generator().manual_seed(30 + i)
        lens = [2000 + 300 * i, 900]
        _, cache = H.pool(gen, 28, 2, 128)
        tables = H.gpu(H.tables_of(gen, lens, 128, 28))
        q = torch.randn(2, 16, 128, generator=gen).to(H.DEV, torch.bfloat16)
        runs.append((q, cache, H.gpu(lens), tables, H.gpu(np.cumsum([0, *lens])),
                     torch.rand(28, 2, 128, generator=gen).to(H.DEV)))

    def run(r, x):
        q, cache, lens, tables, cu_k, _ = r
        out = M.fp8_decode_attention_weights(q, *cache, lens, tables, SCALE, x)
        M.fp8_window_attention_weights(q, cache[0], cache[2], tables, H.gpu([0, 1, 2]), cu_k, 1,
                                       SCALE, x, accumulate=True)
        return (out, x, *M.select_kv_tokens(x, lens, tables, 300, 7))
    want = [run(r, r[5].clone()) for r in runs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in runs], [[], []]
    for _ in range(8):
        for i, (s, r) in enumerate(zip(streams, runs)):
            with torch.cuda.stream(s):
                got[i].append(run(r, r[5].clone()))
    torch.cuda.synchronize()
    for w, gs in zip(want, got):
        for g in gs:
            for a, b in zip(w, g):
                assert torch.equal(a, b)
