"""The 4-bit decode in every form that its launch takes, named by the number of
splits that the shape gives: values, and graphs replayed with new lengths."""

import numpy as np
import pytest
import torch

import microserve_amd as M
from microserve_amd import _lib
from oracle import fp4_oracle as O
from tests import fp4_helpers as H

pytestmark = pytest.mark.gpu

BF16, BLOCK = torch.bfloat16, 128


def _i32(x):
    return torch.as_tensor(x, dtype=torch.int32, device=H.DEV)


def _want(q, host, tables, lens, scale):
    outs = []
    for i, n in enumerate(lens):
        k, v = O.rows(host, tables[i], n)
        outs.append(O.attend(q[i:i + 1].double().numpy(), k, v, scale, np.ones((1, n), bool)))
    return [np.concatenate(x) for x in zip(*outs)]


ONE, EACH = "one workgroup a head", "a page each"
FINER, PAGES = "finer than pages", "splits of pages"
FORMS = [  # lens, q heads, kv heads, the table's width, the form
    ([300, 900, 1, 64], 8, 2, 8, ONE),
    ([300, 900, 1, 64], 8, 2, 60, EACH),
    ([9000, 1], 2, 2, 71, FINER),  # more splits than one wave merges
    ([9000, 1], 16, 8, 100, EACH),  # (here too)
    ([1000, 2048, 1, 64], 8, 2, 16, FINER),
    ([2000, 700, 0], 34, 2, 16, FINER),
    ([700], 8, 8, 16, FINER),
    ([9000, 700, 65, 2], 16, 8, 80, PAGES),
    ([2900, 4000, 1, 129, 513, 70, 64, 0], 32, 8, 128, PAGES),
    ([60, 1500, 2, 0, 128, 700] * 12, 8, 8, 65, PAGES)]  # over work items


def _form(splits, width):
    return ONE if splits == 1 else FINER if splits > width else EACH if splits == width else PAGES


def _case(lens, hq, hk, width, seed, dtype=BF16):
    gen = torch.Generator().manual_seed(seed)
    pool = sum(-(-n // BLOCK) for n in lens) + 1
    host, dev = H.filled(gen, pool, hk, BLOCK)
    tables = H.tables_of(gen, lens, BLOCK, pool, width)
    return host, dev, tables, torch.randn(len(lens), hq, 128, generator=gen).to(dtype)


@pytest.mark.parametrize("lens,hq,hk,width,form", FORMS)
def test_decode_of_each_form(lens, hq, hk, width, form):
    """Splits follow the lengths where they are finer than a page, and where more
    than eight hold two pages or more."""
    splits = _lib.load().mskv_fp4_decode_num_splits(len(lens), hq, hk, width, BLOCK)
    assert _form(splits, width) == form and (form != PAGES or splits > 8)
    host, dev, tables, q = _case(lens, hq, hk, width, 64)
    assert tables.shape[1] == width
    scale = 128 ** -0.5
    got = M.fp4_decode_attention(q.to(H.DEV), *dev, _i32(lens), _i32(tables), scale)
    live = [i for i, n in enumerate(lens) if n]
    want = _want(q[live], host, tables[live], [lens[i] for i in live], scale)
    H.check(got[live], *want, BF16, max(lens), host[3].max(), 1)
    for i, n in enumerate(lens):
        assert n or (got[i] == 0).all()


@pytest.mark.parametrize("lens,hq,hk,width,form", FORMS)
def test_each_forms_graph_replays_with_new_lengths(lens, hq, hk, width, form):
    host, dev, tables, q = _case(lens, hq, hk, width, 65)
    q, lens_t, tables_t = q.to(H.DEV), _i32(lens), _i32(tables)
    out, scale = torch.empty_like(q), 128 ** -0.5

    def step(out):
        return M.fp4_decode_attention(q, *dev, lens_t, tables_t, scale, out=out)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(out)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(out)
    for part in (1, 0.4, 0.01, 0.7, 0, 1):
        new = [min(n, max(1, int(n * part))) if part else 0 for n in lens]
        lens_t.copy_(_i32(new))
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, step(None))
        live = [i for i, n in enumerate(new) if n]
        if live:
            want = _want(q.cpu()[live], host, tables[live], [new[i] for i in live], scale)
            H.check(got[live], *want, BF16, max(new), host[3].max(), 1)
        for i, n in enumerate(new):
            assert n or (got[i] == 0).all()
