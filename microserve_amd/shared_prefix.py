"""Decode attention for sequences that share prefixes (requests that hit the
block manager's prefix cache, samples of one prompt, forks): the shared pages
are read once for a whole group."""

from __future__ import annotations

import torch

from microserve_amd import _lib

MAX_GROUPS = 1024


def _most_saving_groups(tables):
    """The partition of the sequences whose groups save the most reads of pages: a
    group of m saves m - 1 reads of each of its common first pages.

    In the tree of common beginnings a sequence belongs to the deepest group that
    is open above it.  ``best[node][j]``: the most that the sequences below a node
    save, if the j-th node above it is the nearest group (each member counts its
    depth, an open group pays its own once); node 0 above all has depth 0.
    """
    order = sorted(range(len(tables)), key=lambda i: (tables[i], i))
    # the nodes, from the common beginnings of neighbours: (depth, children),
    # children numbers of nodes, or ~i for sequence i
    nodes, stack = [], [(0, [])]

    def close(depth):
        while stack[-1][0] > depth:
            nodes.append(stack.pop())
            if stack[-1][0] < depth:
                stack.append((depth, []))
            stack[-1][1].append(len(nodes) - 1)

    for i, at in zip(order, order[1:] + [None]):
        if at is None:
            common = 0
        else:
            a, b = tables[i], tables[at]
            most = min(len(a), len(b))
            common = most if a[:most] == b[:most] else next(
                j for j in range(most) if a[j] != b[j])
        if stack[-1][0] < common:
            stack.append((common, []))
        stack[-1][1].append(~i)
        close(common)
    nodes.append(stack.pop())  # the root, last; a node comes behind its children

    # each node's depths of the nodes above it, from the root on
    above = [None] * len(nodes)
    above[-1] = []
    for x in range(len(nodes) - 1, -1, -1):
        for c in nodes[x][1]:
            if c >= 0:
                above[c] = above[x] + [x]
    best, sums = [None] * len(nodes), [None] * len(nodes)
    for x, (depth, children) in enumerate(nodes):
        leaves = sum(c < 0 for c in children)
        sums[x] = [leaves * nodes[y][0] + sum(best[c][j] for c in children if c >= 0)
                   for j, y in enumerate(above[x] + [x])]
        opened = sums[x][-1] - depth
        best[x] = [max(v, opened) for v in sums[x][:-1]]
    members, nearest = {}, {len(nodes) - 1: 0}  # (the root is a group of depth 0)
    for x in range(len(nodes) - 1, -1, -1):
        j = nearest[x]
        if x < len(nodes) - 1 and sums[x][-1] - nodes[x][0] > sums[x][j]:
            j = len(above[x])
        group = (above[x] + [x])[j]
        for c in nodes[x][1]:
            if c < 0:
                members.setdefault(group, []).append(~c)
            else:
                nearest[c] = j
    alone = members.pop(len(nodes) - 1, [])
    return [sorted(m) for m in members.values()] + [[i] for i in alone]


def _common(tables, group):
    """The pages that all of a group name first (one alone shares none)."""
    if len(group) == 1:
        return 0
    a, b = (f((tables[i] for i in group)) for f in (min, max))
    return next((j for j, (x, y) in enumerate(zip(a, b)) if x != y), min(len(a), len(b)))


def group_by_prefix(block_tables, block_size: int):
    """Groups of sequences that name the same first pages.

    ``block_tables`` is the sequences' lists of pages (the block manager's).
    Returns ``(order, cu_groups, prefix_lens)``, lists of host integers: the
    order in which the batch must be built so that a group's sequences follow
    one another, the groups' boundaries in it, and the tokens of each group's
    shared pages.  The groups are those that save the most reads of pages: a few
    sequences that share less than the others do not shorten their prefix.  A
    sequence alone has a prefix of 0; where there are more than ``MAX_GROUPS``
    groups, those that save the least are one group, the last, with a prefix of 0.
    """
    tables = [list(t) for t in block_tables]
    groups = [(m, _common(tables, m)) for m in _most_saving_groups(tables)] if tables else []
    groups.sort(key=lambda g: (tables[g[0][0]][:1], g[0][0]))
    if len(groups) > MAX_GROUPS:
        first = sorted(groups, key=lambda g: -(len(g[0]) - 1) * g[1])[:MAX_GROUPS - 1]
        kept = {g[0][0] for g in first}
        rest = sorted(i for m, _ in groups if m[0] not in kept for i in m)
        groups = [g for g in groups if g[0][0] in kept] + [(rest, 0)]
    order, cu = [], [0]
    for members, _ in groups:
        order += members
        cu.append(len(order))
    return order, cu, [pages * block_size for _, pages in groups]


def fp8_shared_prefix_decode_attention(
    query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
    k_scale_cache: torch.Tensor, v_scale_cache: torch.Tensor,
    cache_seqlens: torch.Tensor, block_tables: torch.Tensor, softmax_scale: float,
    cu_groups: torch.Tensor, prefix_lens: torch.Tensor, max_prefix_len: int | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``fp8_decode_attention`` where groups of sequences share their first pages.

    The first ``prefix_lens[g]`` tokens of sequences ``cu_groups[g]`` to
    ``cu_groups[g + 1] - 1`` lie in the same pages (int32 tensors on the GPU,
    ``cu_groups`` ascending).  ``cache_seqlens`` and ``block_tables`` describe
    whole contexts, as for ``fp8_decode_attention``, and the result is that
    call's.  ``max_prefix_len``, a host integer, is the longest prefix that is
    read once (default: the tables' width); what a group shares beyond it, past
    its shortest sequence or past a multiple of 128 tokens is read sequence by
    sequence.  It pays where many share much: a group of 16 from about 1024 tokens,
    of eight from 2048, of four from 8192, if that is more than each has of its own
    (32 q heads over 8, bf16); below that ``fp8_decode_attention`` is faster, by up to
    half.  The launch depends on shapes and ``max_prefix_len`` alone, so the
    call can be captured in a HIP graph.
    """
    res = _lib.fast.shared(query, k_cache, v_cache, k_scale_cache, v_scale_cache, cache_seqlens,
                           block_tables, softmax_scale, cu_groups, prefix_lens, max_prefix_len,
                           out)
    if res is not None:
        return res
    what = "fp8_shared_prefix_decode_attention"
    query = _lib.aligned(query)
    cache_seqlens, block_tables = cache_seqlens.contiguous(), block_tables.contiguous()
    cu_groups, prefix_lens = cu_groups.contiguous(), prefix_lens.contiguous()
    batch, num_q_heads, head_dim = query.shape
    assert query.dtype in (torch.float16, torch.bfloat16)
    assert k_cache.dtype == v_cache.dtype == torch.float8_e4m3fn
    assert k_scale_cache.dtype == v_scale_cache.dtype == torch.float32
    assert k_cache.dim() == 4 and v_cache.shape == k_cache.shape
    assert k_scale_cache.shape == v_scale_cache.shape == k_cache.shape[:3]
    for t in (k_cache, v_cache, k_scale_cache, v_scale_cache):
        assert t.is_contiguous(), "caches must be contiguous"
    num_blocks, block_size, num_kv_heads = k_cache.shape[:3]
    for t in (cache_seqlens, block_tables, cu_groups, prefix_lens):
        assert t.dtype == torch.int32
    assert num_q_heads % num_kv_heads == 0 and head_dim == k_cache.shape[3]
    assert block_tables.dim() == 2 and block_tables.shape[0] == batch == cache_seqlens.numel()
    groups = prefix_lens.numel()
    assert cu_groups.numel() == groups + 1, f"{what}: cu_groups must be [groups + 1]"
    assert groups <= MAX_GROUPS, f"{what}: at most {MAX_GROUPS} groups"
    _lib.on_device(what, query, k_cache, v_cache, k_scale_cache, v_scale_cache, cache_seqlens,
                   block_tables, cu_groups, prefix_lens, out)
    width = block_tables.shape[1]
    bound = width * block_size if max_prefix_len is None else int(max_prefix_len)
    assert bound >= 0, f"{what}: max_prefix_len must not be negative"
    if out is None:
        out = torch.empty_like(query)
    else:
        assert out.shape == query.shape and out.dtype == query.dtype and out.is_contiguous()
    lib = _lib.load()
    nbytes = lib.mskv_shared_decode_workspace_bytes(batch, groups, num_q_heads, num_kv_heads,
                                                    block_size, width, bound)
    with _lib.current(query):
        # on the current stream: reused in stream order, and a graph's own
        # under capture
        ws = torch.empty(nbytes, dtype=torch.uint8, device=query.device)
        status = lib.mskv_fp8_shared_prefix_decode_attention(
            query.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale_cache.data_ptr(),
            v_scale_cache.data_ptr(), cache_seqlens.data_ptr(), block_tables.data_ptr(),
            cu_groups.data_ptr(), prefix_lens.data_ptr(), bound, out.data_ptr(), batch, groups,
            num_q_heads, num_kv_heads, head_dim, block_size, num_blocks, width,
            float(softmax_scale), _lib.act_dtype(query), ws.data_ptr(), nbytes,
            _lib.stream_of(query))
    _lib.check(status, what)
    return out
