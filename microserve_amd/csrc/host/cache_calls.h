// Native call paths of the decode over shared prefixes, the attention weights and
// the eviction: part of fast_calls.cpp, whose rules are theirs.
#pragma once

// `start`: a whole number, or an int32 tensor of one entry a sequence
bool start_of(Args& in, PyObject* o, int64_t batch, int& start, const int32_t*& starts) {
  starts = nullptr;
  if (whole(o, start)) return true;
  start = 0;
  const at::Tensor* t = in.next(o);
  if (!in.ok || !dense_of(*t, at::kInt) || t->numel() != batch) return false;
  starts = (const int32_t*)t->data_ptr();
  return true;
}

bool weights_of(const at::Tensor& w, const Dims& m) {
  return dense_of(w, at::kFloat) && w.sizes() == at::IntArrayRef({m.blocks, m.heads, m.block});
}

at::Tensor bytes_like(const at::Tensor& t, size_t bytes) {
  return at::empty({(int64_t)bytes}, t.options().dtype(at::kByte).requires_grad(false));
}

// A decode's arguments: query, k_cache, v_cache, k_scale, v_scale, seqlens, tables
struct DecodeCall {
  const at::Tensor *q, *kc, *vc, *ks, *vs, *len, *bt;
  Dims m;
  int64_t b, hq, d, w;
  int dt;
  bool take(Args& in, PyObject* const* a) {
    q = in.first(a[0]), kc = in.next(a[1]), vc = in.next(a[2]), ks = in.next(a[3]);
    vs = in.next(a[4]), len = in.next(a[5]), bt = in.next(a[6]);
    if (!in.ok || q->dim() != 3 || !q->is_contiguous() || !aligned(*q) || !act(*q, dt) ||
        !dense_of(*len, at::kInt) || bt->dim() != 2 || !dense_of(*bt, at::kInt) ||
        !caches_ok(*kc, *vc, *ks, *vs))
      return false;
    m = dims_of(*kc);
    b = q->size(0), hq = q->size(1), d = q->size(2), w = bt->size(1);
    return fits({b, hq, d, m.heads, m.block, w}) && hq % m.heads == 0 &&
           caches_match(*kc, *vc, *ks, *vs, m.heads, d) && bt->size(0) == b && len->numel() == b;
  }
  bool takes_out(const at::Tensor& out) const {
    return out.sizes() == q->sizes() && out.scalar_type() == q->scalar_type() &&
           out.is_contiguous();
  }
};

// The result of a call whose `out` argument is `given` (or None: `fresh`).
PyObject* out_of(PyObject* given, at::Tensor& fresh) {
  if (given == Py_None) return THPVariable_Wrap(std::move(fresh));
  Py_INCREF(given);
  return given;
}

// shared(query, k_cache, v_cache, k_scale, v_scale, seqlens, tables, scale, cu_groups,
//        prefix_lens, max_prefix_len | None, out | None) -> out | None
PyObject* shared(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in;
    DecodeCall c;
    double scale;
    int bound = 0;
    if (n != 12 || !c.take(in, a) || !number(a[7], scale)) return nullptr;
    const at::Tensor *cu = in.next(a[8]), *pre = in.next(a[9]);
    const at::Tensor* given = in.ok && a[11] != Py_None ? in.next(a[11]) : nullptr;
    if (!in.ok || !dense_of(*cu, at::kInt) || !dense_of(*pre, at::kInt) ||
        cu->numel() != pre->numel() + 1 || (given && !c.takes_out(*given)) ||
        (a[10] != Py_None && !whole(a[10], bound)))
      return nullptr;
    const int groups = (int)pre->numel();
    const int64_t most = a[10] == Py_None ? c.w * c.m.block : bound;
    const size_t bytes = api.shared_bytes((int)c.b, groups, (int)c.hq, (int)c.m.heads,
                                          (int)c.m.block, (int)c.w, most);
    at::Tensor fresh;
    int status;
    {
      const OnDevice on(in.device);
      if (!given) fresh = at::empty(c.q->sizes(), c.q->options().requires_grad(false));
      const at::Tensor ws = bytes_like(*c.q, bytes);
      status = api.shared(c.q->data_ptr(), c.kc->data_ptr(), c.vc->data_ptr(),
                          (float*)c.ks->data_ptr(), (float*)c.vs->data_ptr(),
                          (int32_t*)c.len->data_ptr(), (int32_t*)c.bt->data_ptr(),
                          (int32_t*)cu->data_ptr(), (int32_t*)pre->data_ptr(), most,
                          (given ? *given : fresh).data_ptr(), (int)c.b, groups, (int)c.hq,
                          (int)c.m.heads, (int)c.d, (int)c.m.block, c.m.blocks, (int)c.w,
                          (float)scale, c.dt, ws.data_ptr(), bytes, stream_of(in.device));
    }
    if (status != MSKV_OK) return failed("fp8_shared_prefix_decode_attention", status);
    return out_of(a[11], fresh);
  });
}

// track(query, k_cache, v_cache, k_scale, v_scale, seqlens, tables, scale, weights, start,
//       out | None) -> out | None
PyObject* track(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in;
    DecodeCall c;
    double scale;
    int start;
    const int32_t* starts;
    if (n != 11 || !c.take(in, a) || !number(a[7], scale)) return nullptr;
    const at::Tensor* weights = in.next(a[8]);
    if (!in.ok || !weights_of(*weights, c.m) || !start_of(in, a[9], c.b, start, starts))
      return nullptr;
    const at::Tensor* given = a[10] != Py_None ? in.next(a[10]) : nullptr;
    if (!in.ok || (given && !c.takes_out(*given))) return nullptr;
    const size_t bytes =
        api.track_bytes((int)c.b, (int)c.hq, (int)c.m.heads, (int)c.m.block, (int)c.w);
    at::Tensor fresh;
    int status;
    {
      const OnDevice on(in.device);
      if (!given) fresh = at::empty(c.q->sizes(), c.q->options().requires_grad(false));
      const at::Tensor ws = bytes_like(*c.q, bytes);
      status = api.track(c.q->data_ptr(), c.kc->data_ptr(), c.vc->data_ptr(),
                         (float*)c.ks->data_ptr(), (float*)c.vs->data_ptr(),
                         (int32_t*)c.len->data_ptr(), (int32_t*)c.bt->data_ptr(),
                         (float*)weights->data_ptr(), starts, start,
                         (given ? *given : fresh).data_ptr(), (int)c.b, (int)c.hq,
                         (int)c.m.heads, (int)c.d, (int)c.m.block, c.m.blocks, (int)c.w,
                         (float)scale, c.dt, ws.data_ptr(), bytes, stream_of(in.device));
    }
    if (status != MSKV_OK) return failed("fp8_decode_attention_weights", status);
    return out_of(a[10], fresh);
  });
}

// window(query, k_cache, k_scale, tables, cu_q, cu_k, max_q, scale, weights, accumulate,
//        start, max_k | None) -> weights | None
PyObject* window(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 12 || !PyBool_Check(a[9])) return nullptr;
    Args in;
    const at::Tensor *q = in.first(a[0]), *kc = in.next(a[1]), *ks = in.next(a[2]),
                     *bt = in.next(a[3]), *cq = in.next(a[4]), *ck = in.next(a[5]),
                     *weights = in.next(a[8]);
    double scale;
    int dt, max_q, start, bound = 0;
    const int32_t* starts;
    if (!in.ok || q->dim() != 3 || !q->is_contiguous() || !aligned(*q) || !act(*q, dt) ||
        !whole(a[6], max_q) || !number(a[7], scale) || !dense_of(*bt, at::kInt) ||
        bt->dim() != 2 || !dense_of(*cq, at::kInt) || !dense_of(*ck, at::kInt) ||
        !caches_ok(*kc, *kc, *ks, *ks) || (a[11] != Py_None && (!whole(a[11], bound) || bound < 1)))
      return nullptr;
    const Dims m = dims_of(*kc);
    const int64_t nq = q->size(0), hq = q->size(1), d = q->size(2), seqs = cq->numel() - 1,
                  w = bt->size(1);
    if (!fits({nq, hq, d, m.heads, m.block, w, seqs}) || hq % m.heads != 0 ||
        !caches_match(*kc, *kc, *ks, *ks, m.heads, d) || ck->numel() != seqs + 1 ||
        bt->size(0) != seqs || !weights_of(*weights, m) ||
        !start_of(in, a[10], seqs, start, starts))
      return nullptr;
    const size_t bytes =
        api.window_bytes(nq, max_q, bound, (int)hq, (int)m.heads, (int)m.block, (int)w);
    int status;
    {
      const OnDevice on(in.device);
      const at::Tensor ws = bytes_like(*q, bytes);
      status = api.window(q->data_ptr(), kc->data_ptr(), (float*)ks->data_ptr(),
                          (int32_t*)bt->data_ptr(), (int32_t*)cq->data_ptr(),
                          (int32_t*)ck->data_ptr(), (float*)weights->data_ptr(), starts, start,
                          a[9] == Py_True, (int)seqs, nq, max_q, bound, (int)hq, (int)m.heads,
                          (int)d, (int)m.block, m.blocks, (int)w, (float)scale, dt, ws.data_ptr(),
                          bytes, stream_of(in.device));
    }
    if (status != MSKV_OK) return failed("fp8_window_attention_weights", status);
    Py_INCREF(a[8]);
    return a[8];
  });
}

// choose(weights, seqlens, tables, budget, recent, start) -> (kept, seqlens) | None
PyObject* choose(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 6) return nullptr;
    Args in;
    const at::Tensor *weights = in.first(a[0]), *len = in.next(a[1]), *bt = in.next(a[2]);
    int budget, recent, start;
    const int32_t* starts;
    if (!in.ok || weights->dim() != 3 || !dense_of(*weights, at::kFloat) ||
        !dense_of(*len, at::kInt) || bt->dim() != 2 || !dense_of(*bt, at::kInt) ||
        !whole(a[3], budget) || !whole(a[4], recent))
      return nullptr;
    const int64_t b = len->numel(), heads = weights->size(1), block = weights->size(2),
                  w = bt->size(1);
    if (!fits({b, heads, block, w, budget}) || bt->size(0) != b ||
        !start_of(in, a[5], b, start, starts))
      return nullptr;
    at::Tensor kept, fresh;
    int status;
    {
      const OnDevice on(in.device);
      const auto opts = len->options().requires_grad(false);
      kept = at::empty({b, heads, budget}, opts);
      fresh = at::empty({b}, opts);
      status = api.choose((float*)weights->data_ptr(), (int32_t*)len->data_ptr(),
                          (int32_t*)bt->data_ptr(), starts, start, recent, budget,
                          (int32_t*)kept.data_ptr(), (int32_t*)fresh.data_ptr(), (int)b,
                          (int)heads, (int)block, weights->size(0), (int)w,
                          stream_of(in.device));
    }
    if (status != MSKV_OK) return failed("select_kv_tokens", status);
    PyObject* k = THPVariable_Wrap(std::move(kept));
    return Py_BuildValue("(NN)", k, THPVariable_Wrap(std::move(fresh)));
  });
}

// evict(k_cache, v_cache, k_scale, v_scale, kept, seqlens, tables, weights | None)
//   -> True | None
PyObject* evict(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 8) return nullptr;
    Args in;
    const at::Tensor *kc = in.first(a[0]), *vc = in.next(a[1]), *ks = in.next(a[2]),
                     *vs = in.next(a[3]), *kept = in.next(a[4]), *len = in.next(a[5]),
                     *bt = in.next(a[6]);
    const at::Tensor* weights = in.ok && a[7] != Py_None ? in.next(a[7]) : nullptr;
    if (!in.ok || !caches_ok(*kc, *vc, *ks, *vs) || kept->dim() != 3 ||
        !dense_of(*kept, at::kInt) || !dense_of(*len, at::kInt) || bt->dim() != 2 ||
        !dense_of(*bt, at::kInt))
      return nullptr;
    const Dims m = dims_of(*kc);
    const int64_t b = len->numel(), w = bt->size(1), budget = kept->size(2);
    if (!caches_match(*kc, *vc, *ks, *vs, m.heads, m.d) ||
        !fits({b, m.heads, m.d, m.block, w, budget}) ||
        kept->size(0) != b || kept->size(1) != m.heads || bt->size(0) != b ||
        (weights && !weights_of(*weights, m)))
      return nullptr;
    int status;
    {
      const OnDevice on(in.device);
      status = api.evict(kc->data_ptr(), vc->data_ptr(), (float*)ks->data_ptr(),
                         (float*)vs->data_ptr(), weights ? (float*)weights->data_ptr() : nullptr,
                         (int32_t*)kept->data_ptr(), (int32_t*)len->data_ptr(),
                         (int32_t*)bt->data_ptr(), (int)b, (int)m.heads, (int)m.d, (int)m.block,
                         m.blocks, (int)w, (int)budget, stream_of(in.device));
    }
    if (status != MSKV_OK) return failed("evict_kv_tokens", status);
    Py_RETURN_TRUE;
  });
}
