// The 4-bit paged KV cache shared by its store, load, decode and prefill.
//
// A value is an e2m1 code: 0, 0.5, 1, 1.5, 2, 3, 4 or 6 with a sign in bit 3,
// two to a byte, the even dimension in the low half.
//
// K: a power-of-two scale for each 32 dimensions of a (token, kv head) row,
// held as the byte e + 127 (E8M0; 255 marks a block that held an infinity or
// a NaN).  Those blocks run along the contraction of QK^T, where
// v_mfma_scale_f32_16x16x128_f8f6f4 applies them: no instruction dequantizes
// K.  Pages are laid out in that MFMA's operand order, so lane (g, n) of a
// wave reads its operand from memory with one 16-byte load, 1 KB contiguous
// over the wave:
//   k_cache  [num_blocks, H, BS / 16, 4, 16, 16]: 16 tokens; 32-dimension
//            block g; token n of the 16; its 32 codes
//   k_scale  [num_blocks, H, BS / 64, 4, 16, 4]: 64 tokens; block g; n; the
//            bytes of tokens n, 16 + n, 32 + n and 48 + n, which the MFMA's
//            byte select takes one after the other
// V: one fp32 scale per row, as the FP8 cache has.  PV contracts over tokens,
// so a row's scale belongs to the token's softmax weight; a scale per 32
// dimensions would need four weights per token.  (On normal values the two
// cost the same precision: the largest of 128 is about 2.7 sigma, a unit of
// 0.45 sigma with an exact scale; the largest of 32 about 2.1 sigma, a unit
// of 0.43 sigma on average under a power of two.)
//   v_cache  [num_blocks, H, BS, 64], v_scale [num_blocks, H, BS]
#pragma once

#include "mskv_device.h"

namespace mskv {

constexpr float kFp4Max = 6.0f;
constexpr int kFp4Row = kHeadDim / 2;  // bytes of a row's codes
constexpr int kE8M0Nan = 255;

// e4m3 parts the query is split into against 4-bit keys: bf16's 8
// significant bits take two, fp16's 11 take three
template <typename T> struct Fp4Query { static constexpr int parts = 3; };
template <> struct Fp4Query<__bf16> { static constexpr int parts = 2; };

// S^T += K . Q^T for 16 tokens: A the codes under their block scales (byte
// kByte of `ks`), B a part of the query under its row's scale byte
template <int kByte>
__device__ __forceinline__ f32x4 mfma_fp4(const u32x4& k, uint32_t ks, const i32x8& q,
                                          uint32_t qscale, f32x4 c) {
  const i32x8 a = {(int)k[0], (int)k[1], (int)k[2], (int)k[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, q, c, 4 /* fp4 */, 0 /* e4m3 */,
                                                          kByte, (int)ks, 0, (int)qscale);
}

// The pieces of a query row that lane (g, n) holds in the B operand: the e4m3
// operand's bytes 0-15 meet the dimensions [16g, 16g + 16) and its bytes 16-31
// [64 + 16g, 80 + 16g).
struct QueryRow {
  u32x4 v[4];
};
__device__ __forceinline__ QueryRow load_query(const uint16_t* row, int g) {
  QueryRow q;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    q.v[c] = *reinterpret_cast<const u32x4*>(row + 64 * (c >> 1) + 16 * g + 8 * (c & 1));
  return q;
}

// What the products of a query row's parts come in: the scale byte they are
// multiplied under, and what takes them to q . k.
struct QueryScale {
  uint32_t byte;
  float unit;
};

// The query row of lane (g, n) as the B operand: e4m3 parts of q * f, f the
// power of two that brings the row's largest magnitude near e4m3's (q * f is
// exact; below 2^-117 f stays 2^126).  NaNs for a row that holds an infinity or
// a NaN, zeros where !ok.
// Where f is above 1, the scale byte takes it back out inside the MFMA: keys
// large enough to meet so small a query would overflow the products else (a
// key of 10^34 times 448).  Below 1 the products stay in units of 1 / f, as
// large queries times ordinary keys would overflow without.
template <typename T>
__device__ __forceinline__ QueryScale fp4_query(const QueryRow& row, bool ok,
                                                i32x8 (&qp)[Fp4Query<T>::parts]) {
  using A = Act<T>;
  float x[32];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const u32x4 v = ok ? row.v[c] : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[8 * c + 2 * i] = A::to_f32((uint16_t)(v[i] & 0xFFFFu));
      x[8 * c + 2 * i + 1] = A::to_f32((uint16_t)(v[i] >> 16));
    }
  }
  // the largest magnitude, as bits: a NaN is above infinity
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
  const auto r16 = __builtin_amdgcn_permlane16_swap(top, top, false, false);
  top = max((uint32_t)r16[0], (uint32_t)r16[1]);
  const auto r32 = __builtin_amdgcn_permlane32_swap(top, top, false, false);
  top = max((uint32_t)r32[0], (uint32_t)r32[1]);
  // The clamp below would make a NaN finite: its row gets e4m3 NaNs, set by
  // their bits, since -fno-honor-nans lets the compiler drop a NaN that it
  // sees made.
  const bool finite = top < 0x7F800000u;
  const uint32_t nan = finite ? 0u : 0x7F7F7F7Fu;
  const float amax = finite ? __uint_as_float(top) : 0.0f;
  const float f = fminf(amax > 0.0f ? pow2_floor(kFp8Max / amax) : 1.0f, 0x1p126f);
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = fminf(fmaxf(x[4 * c + i] * f, -kFp8Max), kFp8Max);
    uint32_t h, mi, lo;
    if constexpr (Fp4Query<T>::parts == 2) {
      split_fp8x4(y[0], y[1], y[2], y[3], h, lo);
      qp[0][c] = (int)(h | nan);
      qp[1][c] = (int)lo;
    } else {
      split3_fp8x4(y[0], y[1], y[2], y[3], h, mi, lo);
      qp[0][c] = (int)(h | nan);
      qp[1][c] = (int)mi;
      qp[2][c] = (int)lo;
    }
  }
  // (127 - log2 f, from f's exponent field)
  const bool small = f > 1.0f;
  return {small ? 254u - (__float_as_uint(f) >> 23) : 127u, small ? 1.0f : 1.0f / f};
}

// The query in e2m3 parts, for the prefill: against codes, a 6-bit operand runs
// at 1.6 times e4m3's rate (9.5 and 15.2 ns an MFMA and SIMD), and three of its
// 4 significant bits hold fp16's 11 as three of e4m3 do.
typedef uint32_t u32x6 __attribute__((ext_vector_type(6)));
constexpr int kQ6Parts = 3;

template <int kByte, int kPart>
__device__ __forceinline__ f32x4 mfma_fp4_q6(const u32x4& k, uint32_t ks, const u32x6& q,
                                             uint32_t qscale, f32x4 c) {
  const i32x8 a = {(int)k[0], (int)k[1], (int)k[2], (int)k[3], 0, 0, 0, 0};
  const i32x8 b = {(int)q[0], (int)q[1], (int)q[2], (int)q[3], (int)q[4], (int)q[5], 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4 /* fp4 */, 2 /* e2m3 */,
                                                          kByte, (int)ks, kPart, (int)qscale);
}

// The pieces of a query row that lane (g, n) holds in the e2m3 operand: the
// dimensions [32g, 32g + 32), K's own blocks.
__device__ __forceinline__ QueryRow load_query6(const uint16_t* row, int g) {
  QueryRow q;
#pragma unroll
  for (int c = 0; c < 4; ++c) q.v[c] = *reinterpret_cast<const u32x4*>(row + 32 * g + 8 * c);
  return q;
}

// e2m3 parts of the lane's block under scales 2^e, 2^(e-4) and 2^(e-9) (bytes 0, 1
// and 2 of the returned word), e the smallest with every magnitude at most 7.5 *
// 2^e.  A part leaves at most a quarter of 2^e, then 2^(e-7); the third's step
// is 2^(e-12) at most, and finer where the rest is small: only elements below
// 2^-5 of the block's largest binade lose bits of fp16, at most 2^(e-13).
// Blocks with an infinity or a NaN get a NaN scale, zeros come out where !ok.
template <typename T>
__device__ __forceinline__ uint32_t fp4_query6(const QueryRow& row, bool ok,
                                               u32x6 (&qp)[kQ6Parts]) {
  typedef T x32 __attribute__((ext_vector_type(32)));
  typedef float f32x16 __attribute__((ext_vector_type(16)));
  typedef float f32x32 __attribute__((ext_vector_type(32)));
  typedef uint32_t u32x16 __attribute__((ext_vector_type(16)));
  u32x16 w;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    w[i] = ok ? row.v[i >> 2][i & 3] : 0u;
    // (fp16 and bf16 both order as their bits; a NaN is above infinity)
    top = max(top, max(w[i] & 0x7FFFu, (w[i] >> 16) & 0x7FFFu));
  }
  const uint32_t bits = __float_as_uint(Act<T>::to_f32((uint16_t)top));
  // 1.875 * 2^floor and up start the next power of two
  const uint32_t e = (uint32_t)max((int)((bits + 0x100000u) >> 23) - 2, 16);
  const float s0 = __uint_as_float(e << 23), s1 = __uint_as_float((e - 4) << 23),
              s2 = __uint_as_float((e - 9) << 23);
  const x32 x = __builtin_bit_cast(x32, w);
  // (The wide converts write their result while they still read: keeping the
  // sources live past them keeps the result out of the sources' registers.)
  if constexpr (Act<T>::kId == 1)
    qp[0] = __builtin_amdgcn_cvt_scalef32_pk32_fp6_bf16(x, s0);
  else
    qp[0] = __builtin_amdgcn_cvt_scalef32_pk32_fp6_f16(x, s0);
  asm volatile("" ::"v"(x), "v"(qp[0]));
  f32x32 back = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(qp[0], s0);
  asm volatile("" ::"v"(qp[0]), "v"(back));
  f32x16 even, odd;  // (the fp32 convert interleaves its two sources)
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    even[i] = Act<T>::to_f32((uint16_t)(w[i] & 0xFFFFu)) - back[2 * i];
    odd[i] = Act<T>::to_f32((uint16_t)(w[i] >> 16)) - back[2 * i + 1];
  }
  qp[1] = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(even, odd, s1);
  asm volatile("" ::"v"(even), "v"(odd), "v"(qp[1]));
  back = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(qp[1], s1);
  asm volatile("" ::"v"(qp[1]), "v"(back));
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    even[i] -= back[2 * i];
    odd[i] -= back[2 * i + 1];
  }
  qp[2] = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(even, odd, s2);
  asm volatile("" ::"v"(even), "v"(odd), "v"(qp[2]));
  return bits >= 0x7F800000u ? 0xFFFFFFu : e | (e - 4) << 8 | (e - 9) << 16;
}

// eight codes (a dword) -> eight exact fp16 values
__device__ __forceinline__ f16x8 fp4x8_to_f16(uint32_t w) {
  f16x8 r;
  const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 0);
  const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 1);
  const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 2);
  const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 3);
  r[0] = a[0]; r[1] = a[1]; r[2] = b[0]; r[3] = b[1];
  r[4] = c[0]; r[5] = c[1]; r[6] = d[0]; r[7] = d[1];
  return r;
}

// V tiles in LDS hold 64-byte rows whose 16-byte chunks are XOR-swizzled by
// (row / 16) % 4.  ds_read_b64_tr_b4 hands lane i of each 16 the nibble i of
// the 8 bytes that the 16 lanes name, lane j's as the j-th: lane (g, j) names
// row 16 * (j / 4) + 4g + j % 4, so its result holds, at one dimension, the
// tokens that S^T's accumulators leave in lane group g (tile j / 4, register
// j % 4).  The swizzle gives the 16 rows of a group distinct banks.
__device__ __forceinline__ uint32_t fp4_v_row(int lane) {
  const int g = lane >> 4, j = lane & 15;
  return (uint32_t)(16 * (j >> 2) + 4 * g + (j & 3)) * kFp4Row;
}
// byte offset of dimension tile dt (16 dimensions) inside lane's row
__device__ __forceinline__ uint32_t fp4_v_col(int lane, int dt) {
  return 16u * (uint32_t)((dt >> 1) ^ ((lane >> 2) & 3)) + 8u * (dt & 1);
}
__device__ __forceinline__ i32x2 fp4_v_read(const uint8_t* tile, uint32_t off) {
  return __builtin_amdgcn_ds_read_tr4_b64_v2i32(
      reinterpret_cast<__attribute__((address_space(3))) i32x2*>(
          (__attribute__((address_space(3))) uint8_t*)tile + off));
}

}  // namespace mskv
