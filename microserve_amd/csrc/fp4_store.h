// Tokens into and out of the 4-bit paged cache (fp4.h has the format).
//
// store: per (token, kv head) row of K and V
//   K, each 32 dimensions: 2^e the smallest power of two with the largest
//   magnitude below 7 * 2^e (at 7 * 2^e the next one): 6 is then off by no
//   more than half of the grid's last step.  e = floor(log2 amax) - 2, one
//   more from 1.75 * 2^floor up, which adding 0.25 to the mantissa carries
//   into the exponent.
//   V, the row: scale = max(amax, 1e-8) / 6.
//   code = e2m1(x / scale), nearest, ties to even, by the hardware convert.
// x / 2^e is exact.  For V the quotient is taken of 0.75 x by 0.125
// max(amax, 1e-8), both exact for 16-bit rows, rather than of x by the
// rounded scale: one value in 200 of such a row lies exactly between two
// codes (6 x / amax = 2.5, say), and the rounded scale would put it on either
// side.  A quotient that is no tie is at least 2^-16 away from one, so the
// fp32 division decides every 16-bit value as exact arithmetic does.
// A block (K) or row (V) that holds an infinity or a NaN gets the scale NaN,
// and reads back as NaN.
//
// Eight lanes own one row, 16 elements each; a wave takes eight tokens of one
// head, whose 16-byte pieces make whole 128-byte lines of the K page where
// their slots are consecutive and start on eight.  HBM-bound: 512 bytes in
// and 136 out a row (load: the reverse).
#pragma once

#include "fp4.h"
#include "fp8_row.h"

namespace mskv {

constexpr int kFp4Tokens = 8;  // of one head, per wave
constexpr int kFp4Waves = 4;

struct Fp4StoreArgs {
  const void *key, *value;  // rows in (store)
  void *key_out, *value_out;  // rows out (load)
  uint8_t *kc, *vc, *ks;
  float* vs;
  const void* slots;
  int64_t tokens, num_slots, key_stride, value_stride;
  int hk, bs;
};

// Where a lane's pieces of slot `slot` of head `head` lie.
struct Fp4Place {
  int64_t k, v, ks, vs;  // K and V codes (8 bytes a lane), scale byte, scale
};
__device__ __forceinline__ Fp4Place fp4_place(int64_t slot, int head, int sub, int hk, int bs) {
  int64_t page;
  int t;
  if (slot <= 0x7FFFFFFF) {  // (a 64-bit division costs five times as much)
    page = (uint32_t)slot / (uint32_t)bs;
    t = (int)((uint32_t)slot - (uint32_t)page * (uint32_t)bs);
  } else {
    page = slot / bs;
    t = (int)(slot - page * bs);
  }
  const int64_t row = (page * hk + head) * bs;
  Fp4Place p;
  p.k = row * kFp4Row + (t >> 4) * 1024 + (sub >> 1) * 256 + (t & 15) * 16 + (sub & 1) * 8;
  p.v = (row + t) * kFp4Row + sub * 8;
  p.ks = row * 4 + (t >> 6) * 256 + (sub >> 1) * 64 + (t & 15) * 4 + ((t >> 4) & 3);
  p.vs = row + t;
  return p;
}

__device__ __forceinline__ uint32_t fp4_pack8(const float* x, float scale) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
  return w;
}

// the largest magnitude's bits: as integers, a NaN is above infinity
__device__ __forceinline__ uint32_t amax_bits16(const float* x) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(x[i]) & 0x7FFFFFFFu);
  return m;
}
template <int kDpp>
__device__ __forceinline__ uint32_t max_dpp_u32(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, kDpp, 0xF, 0xF, false));
}
constexpr uint32_t kInfBits = 0x7F800000u;

template <typename T, typename SlotT>
__global__ __launch_bounds__(64 * kFp4Waves) void store_fp4_kernel(Fp4StoreArgs a) {
  const int lane = threadIdx.x & 63;
  const int sub = lane & 7;
  const int64_t group = (int64_t)blockIdx.x * kFp4Waves + (threadIdx.x >> 6);
  const int64_t tb = group / a.hk;
  const int head = (int)(group - tb * a.hk);
  const int64_t tok = tb * kFp4Tokens + (lane >> 3);
  if (tok >= a.tokens) return;  // whole 8-lane groups leave together
  const int64_t slot = (int64_t)static_cast<const SlotT*>(a.slots)[tok];
  float x[16], y[16];
  load16<T>(a.key, tok * a.key_stride + head * kHeadDim, sub, x);
  load16<T>(a.value, tok * a.value_stride + head * kHeadDim, sub, y);

  const uint32_t kb = max_dpp_u32<0xB1>(amax_bits16(x));  // quad_perm [1,0,3,2]
  const uint32_t e = kb >= kInfBits ? (uint32_t)kE8M0Nan
                                    : (uint32_t)max((int)((kb + 0x200000u) >> 23) - 2, 1);
  const float scale = __uint_as_float(e << 23);
  const u32x2 kq = {fp4_pack8(x, scale), fp4_pack8(x + 8, scale)};

  uint32_t vb = max_dpp_u32<0xB1>(amax_bits16(y));
  vb = max_dpp_u32<0x141>(max_dpp_u32<0x4E>(vb));  // quad_perm [2,3,0,1], row_half_mirror
  const float top = fmaxf(__uint_as_float(vb), 1e-8f);
  const float vscale = vb >= kInfBits ? __uint_as_float(0x7FC00000u) : top / kFp4Max;
  // (RowDivider's conditions hold: the divisor lies in [1.2e-9, 4.3e37], and
  // |0.75 y| is at most six times it)
  const RowDivider div(0.125f * top);
#pragma unroll
  for (int i = 0; i < 16; ++i) y[i] = div(0.75f * y[i]);
  const u32x2 vq = {fp4_pack8(y, 1.0f), fp4_pack8(y + 8, 1.0f)};

  if (slot < 0 || slot >= a.num_slots) return;
  const Fp4Place p = fp4_place(slot, head, sub, a.hk, a.bs);
  *reinterpret_cast<u32x2*>(a.kc + p.k) = kq;
  *reinterpret_cast<u32x2*>(a.vc + p.v) = vq;
  if ((sub & 1) == 0) a.ks[p.ks] = (uint8_t)e;
  if (sub == 0) a.vs[p.vs] = vscale;
}

// eight elements, rounded once to the row's type
template <typename T>
__device__ __forceinline__ void store8(void* base, int64_t at, const float* x) {
  if constexpr (sizeof(T) == 4) {
    f32x4* p = reinterpret_cast<f32x4*>(reinterpret_cast<float*>(base) + at);
    p[0] = f32x4{x[0], x[1], x[2], x[3]};
    p[1] = f32x4{x[4], x[5], x[6], x[7]};
  } else {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = (uint32_t)Act<T>::from_f32(x[2 * i]) |
             ((uint32_t)Act<T>::from_f32(x[2 * i + 1]) << 16);
    __builtin_nontemporal_store(
        v, reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(base) + at));
  }
}

__device__ __forceinline__ void fp4_unpack8(uint32_t w, float scale, float* x) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0);
  const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
  const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2);
  const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
  x[0] = a[0] * scale; x[1] = a[1] * scale;
  x[2] = b[0] * scale; x[3] = b[1] * scale;
  x[4] = c[0] * scale; x[5] = c[1] * scale;
  x[6] = d[0] * scale; x[7] = d[1] * scale;
}

// The eight lanes of a row write whole 128-byte lines: lane l the dimensions
// [8l, 8l + 8) and [64 + 8l, 72 + 8l).  (16 in one run, as the store reads
// them, leave half of every 32 bytes to a second store: 65,536 tokens 134 us.)
template <typename T, typename SlotT>
__global__ __launch_bounds__(64 * kFp4Waves) void load_fp4_kernel(Fp4StoreArgs a) {
  const int lane = threadIdx.x & 63;
  const int sub = lane & 7;
  const int64_t group = (int64_t)blockIdx.x * kFp4Waves + (threadIdx.x >> 6);
  const int64_t tb = group / a.hk;
  const int head = (int)(group - tb * a.hk);
  const int64_t tok = tb * kFp4Tokens + (lane >> 3);
  if (tok >= a.tokens) return;
  const int64_t slot = (int64_t)static_cast<const SlotT*>(a.slots)[tok];
  float x[2][8], y[2][8];
  if (slot >= 0 && slot < a.num_slots) {
    const Fp4Place p = fp4_place(slot, head, 0, a.hk, a.bs);
    const float vscale = a.vs[p.vs];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int block = 2 * h + (sub >> 2);
      const uint32_t kq =
          *reinterpret_cast<const uint32_t*>(a.kc + p.k + 256 * block + 4 * (sub & 3));
      const uint32_t vq = *reinterpret_cast<const uint32_t*>(a.vc + p.v + 32 * h + 4 * sub);
      const uint32_t e = a.ks[p.ks + 64 * block];
      // (2^-127 is a subnormal float)
      const uint32_t bits =
          e == (uint32_t)kE8M0Nan ? 0x7FC00000u : e == 0 ? 0x00400000u : e << 23;
      fp4_unpack8(kq, __uint_as_float(bits), x[h]);
      fp4_unpack8(vq, vscale, y[h]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[0][i] = x[1][i] = y[0][i] = y[1][i] = 0.0f;
  }
  const int64_t at = (tok * a.hk + head) * kHeadDim + 8 * sub;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    store8<T>(a.key_out, at + 64 * h, x[h]);
    store8<T>(a.value_out, at + 64 * h, y[h]);
  }
}

template <bool kStore, typename T, typename SlotT>
static hipError_t launch_fp4_rows(const Fp4StoreArgs& a, unsigned blocks, hipStream_t st) {
  if constexpr (kStore)
    hipLaunchKernelGGL((store_fp4_kernel<T, SlotT>), dim3(blocks), dim3(64 * kFp4Waves), 0, st, a);
  else
    hipLaunchKernelGGL((load_fp4_kernel<T, SlotT>), dim3(blocks), dim3(64 * kFp4Waves), 0, st, a);
  return hipGetLastError();
}

// Checks what both directions share and launches.
template <bool kStore>
static int fp4_rows(Fp4StoreArgs a, int slot_dtype, int head_dim, int64_t num_blocks,
                    int act_dtype, void* stream) {
  if (a.tokens < 0 || a.hk <= 0 || a.bs <= 0 || num_blocks < 0) return MSKV_EINVAL;
  if (slot_dtype != MSKV_INT32 && slot_dtype != MSKV_INT64) return MSKV_EINVAL;
  if (act_dtype != MSKV_FLOAT16 && act_dtype != MSKV_BFLOAT16 && act_dtype != MSKV_FLOAT32)
    return MSKV_EINVAL;
  if (head_dim != kHeadDim || a.bs % 128 != 0 || (int64_t)a.bs * kFp4Row > 0x7FFFFFFFLL)
    return MSKV_EUNSUPPORTED;
  // every byte offset of a cache fits an int64
  if (num_blocks > (INT64_MAX >> 8) / ((int64_t)a.hk * a.bs)) return MSKV_EUNSUPPORTED;
  if (kStore) {
    const int64_t row = (int64_t)a.hk * head_dim;
    const int64_t unit = act_dtype == MSKV_FLOAT32 ? 4 : 8;
    if (a.key_stride < row || a.value_stride < row || a.key_stride % unit != 0 ||
        a.value_stride % unit != 0)
      return MSKV_EINVAL;
  }
  if (a.tokens == 0) return MSKV_OK;
  const void* rows_k = kStore ? a.key : a.key_out;
  const void* rows_v = kStore ? a.value : a.value_out;
  if (!rows_k || !rows_v || !a.kc || !a.vc || !a.ks || !a.vs || !a.slots) return MSKV_EINVAL;
  if (misaligned({rows_k, rows_v, a.kc, a.vc})) return MSKV_EINVAL;
  if (a.tokens > (int64_t)1 << 40) return MSKV_EUNSUPPORTED;
  const int64_t groups = (a.tokens + kFp4Tokens - 1) / kFp4Tokens * a.hk;
  const int64_t blocks = (groups + kFp4Waves - 1) / kFp4Waves;
  if (blocks > 0x7FFFFFFFLL) return MSKV_EUNSUPPORTED;
  a.num_slots = num_blocks * a.bs;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  auto of = [&](auto type) {
    using T = decltype(type);
    return slot_dtype == MSKV_INT64 ? launch_fp4_rows<kStore, T, int64_t>(a, (unsigned)blocks, s)
                                    : launch_fp4_rows<kStore, T, int32_t>(a, (unsigned)blocks, s);
  };
  return (int)(act_dtype == MSKV_BFLOAT16  ? of(__bf16())
               : act_dtype == MSKV_FLOAT16 ? of(_Float16())
                                           : of(float()));
}

}  // namespace mskv

extern "C" int mskv_store_fp4_kvcache(const void* key, int64_t key_stride, const void* value,
                                      int64_t value_stride, void* k_cache, void* v_cache,
                                      void* k_scale_cache, float* v_scale_cache,
                                      const void* slot_mapping, int slot_dtype,
                                      int64_t num_tokens, int num_kv_heads, int head_dim,
                                      int block_size, int64_t num_blocks, int act_dtype,
                                      void* stream) {
  const mskv::Fp4StoreArgs a = {key, value, nullptr, nullptr, (uint8_t*)k_cache,
                                (uint8_t*)v_cache, (uint8_t*)k_scale_cache, v_scale_cache,
                                slot_mapping, num_tokens, 0, key_stride, value_stride,
                                num_kv_heads, block_size};
  return mskv::fp4_rows<true>(a, slot_dtype, head_dim, num_blocks, act_dtype, stream);
}

extern "C" int mskv_load_fp4_kvcache(const void* k_cache, const void* v_cache,
                                     const void* k_scale_cache, const float* v_scale_cache,
                                     const void* slot_mapping, int slot_dtype, void* key,
                                     void* value, int64_t num_tokens, int num_kv_heads,
                                     int head_dim, int block_size, int64_t num_blocks,
                                     int act_dtype, void* stream) {
  const mskv::Fp4StoreArgs a = {nullptr, nullptr, key, value, (uint8_t*)k_cache,
                                (uint8_t*)v_cache, (uint8_t*)k_scale_cache,
                                (float*)v_scale_cache, slot_mapping, num_tokens, 0, 0, 0,
                                num_kv_heads, block_size};
  return mskv::fp4_rows<false>(a, slot_dtype, head_dim, num_blocks, act_dtype, stream);
}
