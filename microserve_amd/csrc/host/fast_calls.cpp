// Native call paths of the hot entry points (CPython extension module
// microserve_amd._fast_calls).
//
// A decode step of a small batch is bound by the host: the Python wrappers
// spend 10 to 20 us per call on tensor attributes, checks and a ctypes call of
// up to 30 arguments, several times the kernels' launches.  Each function
// here takes its wrapper's arguments, and if every tensor is an ordinary one
// that the kernel can read in place (exact class, this GPU, the dtypes,
// shapes and strides the wrapper asserts) it allocates the outputs and calls
// the C ABI directly.  Anything else, arguments that the C ABI rejects
// included (a negative status, before any launch), returns None without
// effect, and the wrapper's own path, the only place where arguments are
// converted and checked, runs as if this module did not exist.  A launch
// that failed (a positive status) raises here: the runtime forgets an error
// once it has been read, so a second try could pass in silence.
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <vector>

#include "../../../include/mskv.h"

namespace {

struct Api {
  decltype(&mskv_store_fp8_kvcache_strided) store = nullptr;
  decltype(&mskv_decode_num_splits) num_splits = nullptr;
  decltype(&mskv_decode_workspace_bytes) decode_bytes = nullptr;
  decltype(&mskv_fp8_decode_attention) decode = nullptr;
  decltype(&mskv_fp8_prefill_bounded_workspace_bytes) prefill_bytes = nullptr;
  decltype(&mskv_fp8_prefill_attention_bounded) prefill = nullptr;
  decltype(&mskv_prefill_attention_strided) fresh = nullptr;
  decltype(&mskv_qk_norm_rope_store) prologue = nullptr;
  decltype(&mskv_store_fp4_kvcache) store4 = nullptr;
  decltype(&mskv_load_fp4_kvcache) load4 = nullptr;
  decltype(&mskv_fp4_decode_num_splits) num_splits4 = nullptr;
  decltype(&mskv_fp4_decode_attention) decode4 = nullptr;
  decltype(&mskv_fp4_prefill_attention) prefill4 = nullptr;
  decltype(&mskv_copy_kv_blocks) copy = nullptr;
  decltype(&mskv_compact_kv_blocks) compact = nullptr;
  decltype(&mskv_shared_decode_workspace_bytes) shared_bytes = nullptr;
  decltype(&mskv_fp8_shared_prefix_decode_attention) shared = nullptr;
  decltype(&mskv_decode_weights_workspace_bytes) track_bytes = nullptr;
  decltype(&mskv_fp8_decode_attention_weights) track = nullptr;
  decltype(&mskv_window_weights_bounded_workspace_bytes) window_bytes = nullptr;
  decltype(&mskv_fp8_window_attention_weights) window = nullptr;
  decltype(&mskv_select_kv_tokens) choose = nullptr;
  decltype(&mskv_evict_kv_tokens) evict = nullptr;
  decltype(&mskv_status_string) text = nullptr;
  bool bound = false;
} api;

PyObject* g_device;  // "device"

// The tensor, if it is a plain one in GPU memory: no subclass, no wrapper
// of a transform (vmap, functional or fake tensors carry other keys).
const at::Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined()) return nullptr;
  static const c10::DispatchKeySet allowed(
      {c10::DispatchKey::CUDA, c10::DispatchKey::AutogradCUDA, c10::DispatchKey::AutocastCUDA,
       c10::DispatchKey::ADInplaceOrView});
  if ((t.key_set().raw_repr() & ~allowed.raw_repr()) != 0 || !t.is_cuda() || !t.has_storage())
    return nullptr;
  return &t;
}

// Plain tensors that must share `ref`'s GPU.
struct Args {
  c10::Device device{c10::DeviceType::CPU};
  bool ok = api.bound && !at::impl::torch_function_mode_enabled();
  const at::Tensor* first(PyObject* o) {
    const at::Tensor* t = ok ? plain(o) : nullptr;
    if (t) device = t->device();
    ok = t != nullptr;
    return t;
  }
  const at::Tensor* next(PyObject* o) {
    const at::Tensor* t = ok ? plain(o) : nullptr;
    ok = t && t->device() == device;
    return t;
  }
};

bool act(const at::Tensor& t, int& code) {
  const auto d = t.scalar_type();
  code = d == at::kHalf ? MSKV_FLOAT16 : d == at::kBFloat16 ? MSKV_BFLOAT16 : -1;
  return code >= 0;
}

bool dense_of(const at::Tensor& t, at::ScalarType d) {
  return t.scalar_type() == d && t.is_contiguous();
}

bool slots_of(const at::Tensor& t, int64_t n, int& code) {
  const auto d = t.scalar_type();
  code = d == at::kLong ? MSKV_INT64 : d == at::kInt ? MSKV_INT32 : -1;
  return code >= 0 && t.is_contiguous() && t.numel() == n;
}

// the four caches, as every wrapper asserts them
bool caches_ok(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks,
               const at::Tensor& vs) {
  return kc.dim() == 4 && dense_of(kc, at::kFloat8_e4m3fn) && dense_of(vc, at::kFloat8_e4m3fn) &&
         dense_of(ks, at::kFloat) && dense_of(vs, at::kFloat);
}
bool caches_match(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks,
                  const at::Tensor& vs, int64_t hk, int64_t d) {
  return kc.size(2) == hk && kc.size(3) == d && vc.sizes() == kc.sizes() &&
         ks.sizes() == kc.sizes().slice(0, 3) && vs.sizes() == ks.sizes();
}

struct Dims {
  int64_t blocks, block, heads, d;
};
// the FP8 cache's, from k_cache (the others are checked by the caller)
Dims dims_of(const at::Tensor& kc) { return {kc.size(0), kc.size(1), kc.size(2), kc.size(3)}; }
// the four 4-bit caches, as fp4_kv_cache.check_fp4_caches asserts them
bool fp4_caches(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks,
                const at::Tensor& vs, Dims& m) {
  if (!dense_of(kc, at::kByte) || !dense_of(vc, at::kByte) || !dense_of(ks, at::kByte) ||
      !dense_of(vs, at::kFloat) || vc.dim() != 4 || vc.size(3) != 64)
    return false;
  const int64_t nb = vc.size(0), h = vc.size(1), bs = vc.size(2);
  m = {nb, bs, h, 128};
  return bs > 0 && bs % 128 == 0 && kc.sizes() == at::IntArrayRef({nb, h, bs / 16, 4, 16, 16}) &&
         ks.sizes() == at::IntArrayRef({nb, h, bs / 64, 4, 16, 4}) &&
         vs.sizes() == at::IntArrayRef({nb, h, bs});
}

// the kernels' vector and direct-to-LDS loads start on 16 bytes
bool aligned(const at::Tensor& t) {
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}

// elements between the tokens of a [tokens, heads, D] tensor read in place
bool token_rows(const at::Tensor& t, int64_t& stride) {
  const int64_t row = t.size(1) * t.size(2);
  if (!aligned(t)) return false;
  if (t.is_contiguous()) {
    stride = row;
    return true;
  }
  stride = t.stride(0);
  return t.stride(2) == 1 && t.stride(1) == t.size(2) && stride >= row && stride <= 1 << 22 &&
         stride * t.element_size() % 16 == 0;
}

bool number(PyObject* o, double& v) {
  if (PyFloat_CheckExact(o)) {
    v = PyFloat_AS_DOUBLE(o);
    return true;
  }
  if (!PyLong_CheckExact(o)) return false;
  v = PyLong_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

bool whole(PyObject* o, int& v) {
  if (!PyLong_CheckExact(o)) return false;
  int over = 0;
  const long long x = PyLong_AsLongLongAndOverflow(o, &over);
  if (over || x < 0 || x > 0x7FFFFFFF) return false;
  v = (int)x;
  return true;
}

void* stream_of(c10::Device d) { return c10::hip::getCurrentHIPStream(d.index()).stream(); }

bool fits(std::initializer_list<int64_t> v) {
  for (const int64_t x : v)
    if (x <= 0 || x > 0x7FFFFFFF) return false;
  return true;
}

// Held around allocations and launches, as torch's and ctypes' own calls do:
// the tensors' GPU is current (a launch goes to the current one, and its
// stream must be that one's), and other threads may run.
struct OnDevice {
  const c10::DeviceGuard guard;
  PyThreadState* state = PyEval_SaveThread();
  explicit OnDevice(c10::Device d) : guard(d) {}
  ~OnDevice() { PyEval_RestoreThread(state); }
};

// The bodies run inside this: a C++ exception (an allocation that failed,
// say) also leaves the call to the wrapper, which raises its own.
template <typename F>
PyObject* guarded(F&& f) {
  try {
    PyObject* r = f();
    if (r) return r;
  } catch (const std::exception&) {
  }
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

// A call's non-zero status: null without an error if the arguments were
// rejected, else with the wrapper's error.
PyObject* failed(const char* what, int status) {
  if (status > 0)
    PyErr_Format(PyExc_RuntimeError, "%s failed: status %d (%s)", what, status, api.text(status));
  return nullptr;
}

// store(key, value, k_cache, v_cache, k_scale, v_scale, slots) -> True | None
PyObject* store(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 7) return nullptr;
    Args in;
    const at::Tensor *key = in.first(a[0]), *value = in.next(a[1]), *kc = in.next(a[2]),
                     *vc = in.next(a[3]), *ks = in.next(a[4]), *vs = in.next(a[5]),
                     *sl = in.next(a[6]);
    if (!in.ok || key->dim() != 3 || value->sizes() != key->sizes() ||
        value->scalar_type() != key->scalar_type() || !caches_ok(*kc, *vc, *ks, *vs) ||
        !caches_match(*kc, *vc, *ks, *vs, key->size(1), key->size(2)) ||
        !fits({key->size(0), key->size(1), key->size(2)}))
      return nullptr;
    int dt = MSKV_FLOAT32, st;
    int64_t k_stride, v_stride;
    if (key->scalar_type() != at::kFloat && !act(*key, dt)) return nullptr;
    if (!slots_of(*sl, key->size(0), st) || !token_rows(*key, k_stride) ||
        !token_rows(*value, v_stride))
      return nullptr;
    int status;
    {
      const OnDevice on(in.device);
      status = api.store(key->data_ptr(), k_stride, value->data_ptr(), v_stride, kc->data_ptr(),
                  vc->data_ptr(), (float*)ks->data_ptr(), (float*)vs->data_ptr(), sl->data_ptr(),
                  st, key->size(0), (int)key->size(1), (int)key->size(2),
                  kc->size(0) * kc->size(1), dt, stream_of(in.device));
    }
    if (status != MSKV_OK) return failed("store_fp8_kvcache", status);
    Py_RETURN_TRUE;
  });
}

// store4: store's arguments over the 4-bit caches
PyObject* store4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 7) return nullptr;
    Args in;
    const at::Tensor *key = in.first(a[0]), *value = in.next(a[1]), *kc = in.next(a[2]),
                     *vc = in.next(a[3]), *ks = in.next(a[4]), *vs = in.next(a[5]),
                     *sl = in.next(a[6]);
    Dims m;
    if (!in.ok || key->dim() != 3 || value->sizes() != key->sizes() ||
        value->scalar_type() != key->scalar_type() || !fp4_caches(*kc, *vc, *ks, *vs, m) ||
        key->size(1) != m.heads || key->size(2) != m.d || !fits({key->size(0), m.heads, m.block}))
      return nullptr;
    int dt = MSKV_FLOAT32, st;
    int64_t k_stride, v_stride;
    if (key->scalar_type() != at::kFloat && !act(*key, dt)) return nullptr;
    if (!slots_of(*sl, key->size(0), st) || !token_rows(*key, k_stride) ||
        !token_rows(*value, v_stride))
      return nullptr;
    int status;
    {
      const OnDevice on(in.device);
      status = api.store4(key->data_ptr(), k_stride, value->data_ptr(), v_stride, kc->data_ptr(),
                          vc->data_ptr(), ks->data_ptr(), (float*)vs->data_ptr(), sl->data_ptr(),
                          st, key->size(0), (int)m.heads, (int)m.d, (int)m.block, m.blocks, dt,
                          stream_of(in.device));
    }
    if (status != MSKV_OK) return failed("store_fp4_kvcache", status);
    Py_RETURN_TRUE;
  });
}

// load4(k_cache, v_cache, k_scale, v_scale, slots, dtype) -> (key, value) | None
PyObject* load4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 6 || !THPDtype_Check(a[5])) return nullptr;
    Args in;
    const at::Tensor *kc = in.first(a[0]), *vc = in.next(a[1]), *ks = in.next(a[2]),
                     *vs = in.next(a[3]), *sl = in.next(a[4]);
    Dims m;
    if (!in.ok || !fp4_caches(*kc, *vc, *ks, *vs, m)) return nullptr;
    const auto type = reinterpret_cast<THPDtype*>(a[5])->scalar_type;
    const int dt = type == at::kHalf       ? MSKV_FLOAT16
                   : type == at::kBFloat16 ? MSKV_BFLOAT16
                   : type == at::kFloat    ? MSKV_FLOAT32
                                           : -1;
    const int64_t tokens = sl->numel();
    int st;
    if (dt < 0 || !slots_of(*sl, tokens, st) || !fits({tokens, m.heads, m.block})) return nullptr;
    at::Tensor key, value;
    int status;
    {
      const OnDevice on(in.device);
      const auto opts = vs->options().dtype(type).requires_grad(false);
      key = at::empty({tokens, m.heads, m.d}, opts);
      value = at::empty({tokens, m.heads, m.d}, opts);
      status = api.load4(kc->data_ptr(), vc->data_ptr(), ks->data_ptr(), (float*)vs->data_ptr(),
                         sl->data_ptr(), st, key.data_ptr(), value.data_ptr(), tokens,
                         (int)m.heads, (int)m.d, (int)m.block, m.blocks, dt,
                         stream_of(in.device));
    }
    if (status != MSKV_OK) return failed("load_fp4_kvcache", status);
    PyObject* k = THPVariable_Wrap(std::move(key));
    return Py_BuildValue("(NN)", k, THPVariable_Wrap(std::move(value)));
  });
}

// decode(query, k_cache, v_cache, k_scale, v_scale, seqlens, tables, scale,
//        out | None, scratch) -> out | None;
// scratch(device, stream, bytes) -> the stream's split-partials tensor
template <bool kFp4>
PyObject* decode_call(PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 10) return nullptr;
    Args in;
    const at::Tensor *q = in.first(a[0]), *kc = in.next(a[1]), *vc = in.next(a[2]),
                     *ks = in.next(a[3]), *vs = in.next(a[4]), *len = in.next(a[5]),
                     *bt = in.next(a[6]);
    const at::Tensor* given = in.ok && a[8] != Py_None ? in.next(a[8]) : nullptr;
    double scale;
    int dt;
    if (!in.ok || q->dim() != 3 || !q->is_contiguous() || !aligned(*q) || !act(*q, dt) || !number(a[7], scale) ||
        !dense_of(*len, at::kInt) || bt->dim() != 2 || !dense_of(*bt, at::kInt))
      return nullptr;
    Dims m;
    if (kFp4 ? !fp4_caches(*kc, *vc, *ks, *vs, m) : !caches_ok(*kc, *vc, *ks, *vs)) return nullptr;
    if (!kFp4) m = dims_of(*kc);
    const int64_t b = q->size(0), hq = q->size(1), d = q->size(2), hk = m.heads, bs = m.block,
                  w = bt->size(1);
    if (!fits({b, hq, d, hk, bs, w}) || hq % hk != 0 || d != m.d || bt->size(0) != b ||
        len->numel() != b)
      return nullptr;
    if (given && (given->sizes() != q->sizes() || given->scalar_type() != q->scalar_type() ||
                  !given->is_contiguous()))
      return nullptr;
    void* stream = stream_of(in.device);
    const int splits =
        (kFp4 ? api.num_splits4 : api.num_splits)((int)b, (int)hq, (int)hk, (int)w, (int)bs);
    const size_t bytes = api.decode_bytes((int)b, (int)hq, (int)hk, (int)d, splits);
    void* ws = nullptr;
    if (bytes) {
      PyObject* dev = PyObject_GetAttr(a[0], g_device);
      if (!dev) return nullptr;
      PyObject* buf =
          PyObject_CallFunction(a[9], "NKn", dev, (unsigned long long)stream, (Py_ssize_t)bytes);
      if (!buf) return nullptr;
      // the caller's table keeps the buffer alive
      if (THPVariable_Check(buf)) ws = THPVariable_Unpack(buf).data_ptr();
      Py_DECREF(buf);
      if (!ws) return nullptr;
    }
    at::Tensor fresh;
    int status;
    {
      const OnDevice on(in.device);
      if (!given) fresh = at::empty(q->sizes(), q->options().requires_grad(false));
      const at::Tensor& out = given ? *given : fresh;
      auto call = [&](auto f) {
        return f(q->data_ptr(), kc->data_ptr(), vc->data_ptr(), (float*)ks->data_ptr(),
                 (float*)vs->data_ptr(), (int32_t*)len->data_ptr(), (int32_t*)bt->data_ptr(),
                 out.data_ptr(), (int)b, (int)hq, (int)hk, (int)d, (int)bs, m.blocks, (int)w,
                 (float)scale, dt, splits, ws, bytes, stream);
      };
      if constexpr (kFp4)
        status = call(api.decode4);
      else
        status = call(api.decode);
    }
    if (status != MSKV_OK)
      return failed(kFp4 ? "fp4_decode_attention" : "fp8_decode_attention", status);
    if (given) {
      Py_INCREF(a[8]);
      return a[8];
    }
    return THPVariable_Wrap(std::move(fresh));
  });
}

PyObject* decode(PyObject*, PyObject* const* a, Py_ssize_t n) { return decode_call<false>(a, n); }
PyObject* decode4(PyObject*, PyObject* const* a, Py_ssize_t n) { return decode_call<true>(a, n); }

// prefill(query, k_cache, v_cache, k_scale, v_scale, tables, cu_q | None,
//         cu_k | None, prefix_len, max_seqlen_q, max_seqlen_k, scale)
//   -> out | None
// (without cu_q, one sequence: max_seqlen_q and max_seqlen_k are not read)
template <bool kFp4>
PyObject* prefill_call(PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 12) return nullptr;
    Args in;
    const at::Tensor *q = in.first(a[0]), *kc = in.next(a[1]), *vc = in.next(a[2]),
                     *ks = in.next(a[3]), *vs = in.next(a[4]), *bt = in.next(a[5]);
    const bool varlen = a[6] != Py_None;
    const at::Tensor *cq = varlen && in.ok ? in.next(a[6]) : nullptr,
                     *ck = varlen && in.ok ? in.next(a[7]) : nullptr;
    double scale;
    int dt, prefix, max_q, bound;
    if (!in.ok || q->dim() != 3 || !q->is_contiguous() || !aligned(*q) || !act(*q, dt) || !whole(a[8], prefix) ||
        !whole(a[9], max_q) || !whole(a[10], bound) || !number(a[11], scale) ||
        !dense_of(*bt, at::kInt))
      return nullptr;
    Dims m;
    if (kFp4 ? !fp4_caches(*kc, *vc, *ks, *vs, m) : !caches_ok(*kc, *vc, *ks, *vs)) return nullptr;
    if (!kFp4) m = dims_of(*kc);
    const int64_t nq = q->size(0), hq = q->size(1), d = q->size(2), hk = m.heads, bs = m.block;
    int64_t seqs = 1, w = bt->numel();
    if (varlen) {
      if (bt->dim() != 2 || !dense_of(*cq, at::kInt) || !dense_of(*ck, at::kInt)) return nullptr;
      seqs = cq->numel() - 1;
      w = bt->size(1);
      if (ck->numel() != seqs + 1 || bt->size(0) != seqs) return nullptr;
    }
    if (!fits({nq, hq, d, hk, bs, w, seqs}) || hq % hk != 0 || d != m.d) return nullptr;
    int64_t max_k = bound;
    if (!varlen) {
      max_q = (int)nq;
      max_k = prefix + nq;
    }
    const size_t bytes = api.prefill_bytes((int)seqs, nq, max_q, max_k, (int)hq, (int)hk, (int)d,
                                           (int)bs, (int)w);
    at::Tensor ws, out;
    int status;
    {
      const OnDevice on(in.device);
      if (bytes) ws = at::empty({(int64_t)bytes}, q->options().dtype(at::kByte).requires_grad(false));
      out = at::empty(q->sizes(), q->options().requires_grad(false));
      auto call = [&](auto f) {
        return f(q->data_ptr(), kc->data_ptr(), vc->data_ptr(), (float*)ks->data_ptr(),
                 (float*)vs->data_ptr(), (int32_t*)bt->data_ptr(),
                 varlen ? (int32_t*)cq->data_ptr() : nullptr,
                 varlen ? (int32_t*)ck->data_ptr() : nullptr, prefix, out.data_ptr(), (int)seqs,
                 nq, max_q, max_k, (int)hq, (int)hk, (int)d, (int)bs, m.blocks, (int)w,
                 (float)scale, dt, bytes ? ws.data_ptr() : nullptr, bytes, stream_of(in.device));
      };
      if constexpr (kFp4)
        status = call(api.prefill4);
      else
        status = call(api.prefill);
    }
    if (status != MSKV_OK) {
      if (kFp4)
        return failed(varlen ? "fp4_varlen_prefill_attention" : "fp4_chunk_prefill_attention",
                      status);
      return failed(varlen ? "fp8_varlen_prefill_attention" : "fp8_chunk_prefill_attention",
                    status);
    }
    return THPVariable_Wrap(std::move(out));
  });
}
PyObject* prefill(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return prefill_call<false>(a, n);
}
PyObject* prefill4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return prefill_call<true>(a, n);
}

// fresh(q, k, v, cu_q, cu_k, max_seqlen_q, scale) -> out | None
PyObject* fresh(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 7) return nullptr;
    Args in;
    const at::Tensor *q = in.first(a[0]), *k = in.next(a[1]), *v = in.next(a[2]),
                     *cq = in.next(a[3]), *ck = in.next(a[4]);
    double scale;
    int dt, max_q;
    int64_t k_stride, v_stride;
    if (!in.ok || q->dim() != 3 || !q->is_contiguous() || !aligned(*q) || !act(*q, dt) || k->dim() != 3 ||
        k->sizes() != v->sizes() || k->scalar_type() != q->scalar_type() ||
        v->scalar_type() != q->scalar_type() || !dense_of(*cq, at::kInt) ||
        !dense_of(*ck, at::kInt) || !whole(a[5], max_q) || !number(a[6], scale))
      return nullptr;
    const int64_t nq = q->size(0), hq = q->size(1), d = q->size(2), nk = k->size(0),
                  hk = k->size(1), seqs = cq->numel() - 1;
    if (!fits({nq, hq, d, nk, hk, seqs}) || k->size(2) != d || hq % hk != 0 ||
        ck->numel() != seqs + 1 || !token_rows(*k, k_stride) || !token_rows(*v, v_stride))
      return nullptr;
    at::Tensor out;
    int status;
    {
      const OnDevice on(in.device);
      out = at::empty(q->sizes(), q->options().requires_grad(false));
      status = api.fresh(q->data_ptr(), k->data_ptr(), k_stride, v->data_ptr(), v_stride, out.data_ptr(),
                  (int32_t*)cq->data_ptr(), (int32_t*)ck->data_ptr(), (int)seqs, nq, nk, max_q,
                  (int)hq, (int)hk, (int)d, (float)scale, dt, stream_of(in.device));
    }
    if (status != MSKV_OK) return failed("varlen_attention", status);
    return THPVariable_Wrap(std::move(out));
  });
}

// prologue(positions, q, k, v, q_weight | None, k_weight | None, eps, cos,
//          sin, k_cache, v_cache, k_scale, v_scale, slots, return_k)
//   -> (q_out, k_out | None) | None
PyObject* prologue(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 15) return nullptr;
    Args in;
    const at::Tensor *q = in.first(a[1]), *k = in.next(a[2]), *v = in.next(a[3]),
                     *pos = in.next(a[0]), *cos = in.next(a[7]), *sin = in.next(a[8]),
                     *kc = in.next(a[9]), *vc = in.next(a[10]), *ks = in.next(a[11]),
                     *vs = in.next(a[12]), *sl = in.next(a[13]);
    const bool norm = a[4] != Py_None;
    const at::Tensor *qw = norm && in.ok ? in.next(a[4]) : nullptr,
                     *kw = norm && in.ok ? in.next(a[5]) : nullptr;
    double eps;
    int dt, st;
    if (!in.ok || (!norm && a[5] != Py_None) || q->dim() != 3 || k->dim() != 3 || !act(*q, dt) ||
        !number(a[6], eps) || !PyBool_Check(a[14]))
      return nullptr;
    const int64_t t = q->size(0), hq = q->size(1), d = q->size(2), hk = k->size(1);
    const auto type = q->scalar_type();
    if (!fits({t, hq, d, hk}) || k->size(0) != t || k->size(2) != d || v->sizes() != k->sizes())
      return nullptr;
    for (const at::Tensor* x : {q, k, v})
      if (x->scalar_type() != type || x->stride(2) != 1 || x->stride(1) != d) return nullptr;
    if (norm)
      for (const at::Tensor* x : {qw, kw})
        if (!dense_of(*x, type) || x->numel() != d) return nullptr;
    if (!dense_of(*cos, type) || !dense_of(*sin, type) || cos->numel() != sin->numel() ||
        cos->numel() == 0 || cos->numel() % d != 0 || !dense_of(*pos, at::kLong) ||
        pos->numel() != t || !slots_of(*sl, t, st) || !caches_ok(*kc, *vc, *ks, *vs) ||
        !caches_match(*kc, *vc, *ks, *vs, hk, d))
      return nullptr;
    const auto opts = q->options().requires_grad(false);
    at::Tensor q_out, k_out;
    const bool with_k = a[14] == Py_True;
    int status;
    {
      const OnDevice on(in.device);
      q_out = at::empty({t, hq, d}, opts);
      if (with_k) k_out = at::empty({t, hk, d}, opts);
      status = api.prologue(q->data_ptr(), k->data_ptr(), v->data_ptr(), q->stride(0), k->stride(0),
                     v->stride(0), (int64_t*)pos->data_ptr(), norm ? qw->data_ptr() : nullptr,
                     norm ? kw->data_ptr() : nullptr, (float)eps, cos->data_ptr(), sin->data_ptr(),
                     cos->numel() / d, q_out.data_ptr(), with_k ? k_out.data_ptr() : nullptr,
                     kc->data_ptr(), vc->data_ptr(), (float*)ks->data_ptr(),
                     (float*)vs->data_ptr(), sl->data_ptr(), st, t, (int)hq, (int)hk, (int)d,
                     kc->size(0) * kc->size(1), dt, stream_of(in.device));
    }
    if (status != MSKV_OK) return failed("mskv_qk_norm_rope_store", status);
    PyObject* qo = THPVariable_Wrap(std::move(q_out));
    PyObject* ko = Py_None;
    if (with_k)
      ko = THPVariable_Wrap(std::move(k_out));
    else
      Py_INCREF(ko);
    return Py_BuildValue("(NN)", qo, ko);
  });
}

// The caches of a call that moves pages, as kv_blocks._pools describes them:
// a tensor or a tuple or list of up to MSKV_MAX_POOLS, dimension `dim` of each
// numbering the same blocks.
struct PoolArgs {
  int count = 0;
  void* bases[MSKV_MAX_POOLS];
  int64_t planes[MSKV_MAX_POOLS], strides[MSKV_MAX_POOLS], pages[MSKV_MAX_POOLS], blocks = -1;
  bool add(Args& in, PyObject* o, int dim) {
    const at::Tensor* t = count ? in.next(o) : in.first(o);
    if (!in.ok || count == MSKV_MAX_POOLS || !t->is_contiguous() || t->dim() <= dim ||
        t->numel() <= 0 || (blocks >= 0 && t->size(dim) != blocks))
      return false;
    blocks = t->size(dim);
    int64_t n = 1;
    for (int i = 0; i < dim; ++i) n *= t->size(i);
    bases[count] = t->data_ptr();
    planes[count] = n;
    pages[count] = t->numel() / (n * blocks) * t->element_size();
    strides[count] = blocks * pages[count];
    ++count;
    return true;
  }
  bool take(Args& in, PyObject* caches, int dim) {
    if (!PyTuple_CheckExact(caches) && !PyList_CheckExact(caches)) return add(in, caches, dim);
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(caches);
    if (n < 1 || n > MSKV_MAX_POOLS) return false;
    for (Py_ssize_t i = 0; i < n; ++i)
      if (!add(in, PySequence_Fast_GET_ITEM(caches, i), dim)) return false;
    return true;
  }
};

// a list or tuple of whole numbers that fit an int
bool ids_of(PyObject* o, std::vector<int32_t>& v) {
  if (!PyTuple_CheckExact(o) && !PyList_CheckExact(o)) return false;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(o);
  v.resize((size_t)n);
  for (Py_ssize_t i = 0; i < n; ++i)
    if (!whole(PySequence_Fast_GET_ITEM(o, i), v[(size_t)i])) return false;
  return true;
}

// copy_blocks(caches, src, dst, block_dim) -> True | None
PyObject* copy_blocks(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    int dim;
    std::vector<int32_t> src, dst;
    if (n != 4 || !whole(a[3], dim) || !ids_of(a[1], src) || !ids_of(a[2], dst) ||
        src.size() != dst.size())
      return nullptr;
    Args in;
    PoolArgs p;
    if (!p.take(in, a[0], dim)) return nullptr;
    int status;
    {
      const OnDevice on(in.device);
      status = api.copy(p.count, p.bases, p.planes, p.strides, p.pages, p.blocks, src.data(),
                        dst.data(), (int64_t)src.size(), stream_of(in.device));
    }
    if (status != MSKV_OK) return failed("copy_kv_blocks", status);
    Py_RETURN_TRUE;
  });
}

// compact_blocks(caches, tables, num_blocks | None, block_dim)
//   -> (tables, remap, num_live) | None
PyObject* compact_blocks(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    int dim, given = 0;
    if (n != 4 || !whole(a[3], dim) || (a[2] != Py_None && !whole(a[2], given))) return nullptr;
    Args in;
    PoolArgs p;
    if (!p.take(in, a[0], dim)) return nullptr;
    const at::Tensor* tables = in.next(a[1]);
    const int64_t blocks = a[2] == Py_None ? p.blocks : given;
    if (!in.ok || !dense_of(*tables, at::kInt) || blocks < 1 || blocks > p.blocks) return nullptr;
    at::Tensor renamed, remap, live;
    int status;
    {
      const OnDevice on(in.device);
      const auto opts = tables->options().requires_grad(false);
      renamed = at::empty(tables->sizes(), opts);
      remap = at::empty({blocks}, opts);
      live = at::empty({1}, opts);
      status = api.compact(p.count, p.bases, p.planes, p.strides, p.pages, blocks,
                           (const int32_t*)tables->data_ptr(), tables->numel(),
                           (int32_t*)renamed.data_ptr(), (int32_t*)remap.data_ptr(),
                           (int32_t*)live.data_ptr(), stream_of(in.device));
    }
    if (status != MSKV_OK) return failed("compact_kv_blocks", status);
    PyObject* t = THPVariable_Wrap(std::move(renamed));
    PyObject* r = THPVariable_Wrap(std::move(remap));
    return Py_BuildValue("(NNN)", t, r, THPVariable_Wrap(std::move(live)));
  });
}

#include "cache_calls.h"

// bind({name: address}): the entry points of the loaded library
PyObject* bind(PyObject*, PyObject* table) {
  auto get = [&](const char* name, auto& fn) {
    PyObject* v = PyDict_Check(table) ? PyDict_GetItemString(table, name) : nullptr;
    void* p = v ? PyLong_AsVoidPtr(v) : nullptr;
    if (!p) return false;
    fn = reinterpret_cast<std::remove_reference_t<decltype(fn)>>(p);
    return true;
  };
  Api f;
  f.bound = get("mskv_store_fp8_kvcache_strided", f.store) &&
            get("mskv_decode_num_splits", f.num_splits) &&
            get("mskv_decode_workspace_bytes", f.decode_bytes) &&
            get("mskv_fp8_decode_attention", f.decode) &&
            get("mskv_fp8_prefill_bounded_workspace_bytes", f.prefill_bytes) &&
            get("mskv_fp8_prefill_attention_bounded", f.prefill) &&
            get("mskv_prefill_attention_strided", f.fresh) &&
            get("mskv_qk_norm_rope_store", f.prologue) &&
            get("mskv_store_fp4_kvcache", f.store4) && get("mskv_load_fp4_kvcache", f.load4) &&
            get("mskv_fp4_decode_num_splits", f.num_splits4) &&
            get("mskv_fp4_decode_attention", f.decode4) &&
            get("mskv_fp4_prefill_attention", f.prefill4) &&
            get("mskv_copy_kv_blocks", f.copy) && get("mskv_compact_kv_blocks", f.compact) &&
            get("mskv_shared_decode_workspace_bytes", f.shared_bytes) &&
            get("mskv_fp8_shared_prefix_decode_attention", f.shared) &&
            get("mskv_decode_weights_workspace_bytes", f.track_bytes) &&
            get("mskv_fp8_decode_attention_weights", f.track) &&
            get("mskv_window_weights_bounded_workspace_bytes", f.window_bytes) &&
            get("mskv_fp8_window_attention_weights", f.window) &&
            get("mskv_select_kv_tokens", f.choose) && get("mskv_evict_kv_tokens", f.evict) &&
            get("mskv_status_string", f.text);
  if (!f.bound) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_KeyError, "an entry point has no address");
    return nullptr;
  }
  api = f;
  Py_RETURN_NONE;
}

#define FAST(f) {#f, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {FAST(store), FAST(decode), FAST(prefill), FAST(fresh), FAST(prologue),
                          FAST(store4), FAST(load4), FAST(decode4), FAST(prefill4),
                          FAST(copy_blocks), FAST(compact_blocks), FAST(shared), FAST(track),
                          FAST(window), FAST(choose), FAST(evict),
                          {"bind", bind, METH_O, nullptr},
                          {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_fast_calls",
                       "Native call paths of the hot entry points.", -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__fast_calls(void) {
  g_device = PyUnicode_InternFromString("device");
  if (!g_device) return nullptr;
  return PyModule_Create(&kModule);
}
