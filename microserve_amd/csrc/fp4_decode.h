// The decode's walk over the 4-bit cache (the split kernel's Fp4Cache): a wave
// takes one (sequence, kv head, split), 64 tokens a step.
//
//  * K goes from memory to the matrix unit: the page's layout is the A
//    operand's (fp4.h), the block scales are applied by the MFMA, and the
//    e4m3 parts of the query are the B operand: exact for bf16, fp16 with a
//    2^-12 residual.  No K byte passes through LDS or a conversion.
//  * V rows pass through a per-wave LDS tile and come back transposed
//    (ds_read_b64_tr_b4), 16 tokens a lane at one dimension, and convert to
//    fp16 exactly.
//  * Everything else is the FP8 walk's: online softmax in base 2 with a lazy
//    rescale, weights fp16(p * v_scale * f).
// HBM-bound: 136 bytes a token and kv head against the FP8 cache's 264.
#pragma once

#include "fp4.h"

namespace mskv {

struct Fp4Loads {
  u32x4 k[4];       // lane (g, n): block g of token 16c + n
  u32x4 v[4];       // row 16c + lane / 4, 16-byte chunk lane % 4
  uint32_t kscale;  // lane (g, n): bytes of tokens 16c + n, block g
  float vscale;     // of token `lane`
  int valid;
};

struct Fp4Cache {
  static constexpr int kUnit = 64;
  static constexpr int kPageUnit = 128;  // as the prefill's tiles
  typedef uint8_t Tiles[2][kUnit * kFp4Row];  // V, double-buffered
  typedef float Scales[2][kUnit];             // v_scale * f

  // Issues the loads of the step at token t0, whose page holds block `blk`.
  // An invalid block is read through zero-length resources.
  static __device__ __forceinline__ void load(const DecodeArgs& a, int blk, int kvh, int t0,
                                              int t_end, int lane, Fp4Loads& s) {
    const int off = t0 % a.bs;
    const bool ok = blk >= 0 && (int64_t)blk < a.num_blocks;
    const int64_t row = ((ok ? (int64_t)blk : 0) * a.hk + kvh) * a.bs;
    const uint32_t bytes = ok ? (uint32_t)a.bs * kFp4Row : 0u;
    const uint32_t sbytes = ok ? (uint32_t)a.bs * 4u : 0u;
    const auto kr = make_rsrc(a.kc + row * kFp4Row, bytes);
    const auto vr = make_rsrc(a.vc + row * kFp4Row, bytes);
    const auto ksr = make_rsrc(a.ks + row, sbytes);
    const auto vsr = make_rsrc(a.vs + row, sbytes);
    const uint32_t o = (uint32_t)off * kFp4Row + 16u * lane;
#pragma unroll
    for (int c = 0; c < 4; ++c) s.k[c] = buf_load16_nt(kr, o + 1024u * c);
    s.kscale = __float_as_uint(buf_load_f32(ksr, ((uint32_t)off + lane) * 4u));
#pragma unroll
    for (int c = 0; c < 4; ++c) s.v[c] = buf_load16_nt(vr, o + 1024u * c);
    s.vscale = buf_load_f32(vsr, ((uint32_t)off + lane) * 4u);
    s.valid = ok ? min(kUnit, t_end - t0) : 0;
  }

  template <typename T>
  static __device__ __forceinline__ void attend(const DecodeArgs& a, int b, int kvh, int qh,
                                                bool head_ok, int t_begin, int t_end,
                                                int blk_first, int lane, Tiles& tiles,
                                                Scales& scales, f32x4 (&acc)[8], float& m,
                                                float& l) {
    constexpr int NQ = Fp4Query<T>::parts;
    const int g = lane >> 4;
    i32x8 qp[NQ];
    // scores in log2 units: S^T * qs
    const float qs =
        a.scale_log2 / fp4_query<T>(a.q + ((int64_t)b * a.hq + qh) * kHeadDim, head_ok, g, qp);

#pragma unroll
    for (int dt = 0; dt < 8; ++dt) acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY;
    l = 0.0f;
    // f: the power of two with v_scale * f <= kPvScaleMax for every valid
    // token so far (0 until the first one), as in the FP8 walk
    float f = 0.0f, vseen = 0.0f;

    // Stages one step's V rows and scales into buffer `buf`.  Rows past the
    // end need no zeros: every code is a finite value, and their weights are 0.
    auto stage = [&](const Fp4Loads& s, int buf) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint32_t at = (uint32_t)(16 * c + (lane >> 2)) * kFp4Row + 16u * ((lane & 3) ^ c);
        *reinterpret_cast<u32x4*>(&tiles[buf][at]) = s.v[c];
      }
      const bool vtok = lane < s.valid;
      if (__any(vtok && !(s.vscale * f <= kPvScaleMax)) || f == 0.0f) {
        float vm = vtok ? s.vscale : 0.0f;
        vm = fmaxf(max_xor32(max_xor16(max16_dpp(vm))), vseen);
        const float fnew = vm > 0.0f ? pow2_floor(kPvScaleMax / vm) : 0.0f;
        if (f != 0.0f && fnew < f) {
          const float r = fnew / f;  // a power of two < 1: exact
#pragma unroll
          for (int dt = 0; dt < 8; ++dt) acc[dt] *= r;
        }
        if (fnew > 0.0f && (f == 0.0f || fnew < f)) f = fnew;
        vseen = vm;
      }
      scales[buf][lane] = s.vscale * f;
    };

    const uint32_t vrow = fp4_v_row(lane);
    Fp4Loads cur, nxt;
    load(a, blk_first, kvh, t_begin, t_end, lane, cur);
    stage(cur, 0);
    wave_lds_sync();
    int buf = 0;
    for (int t0 = t_begin; t0 < t_end; t0 += kUnit, buf ^= 1) {
      const int valid = cur.valid;
      const bool more = t0 + kUnit < t_end;
      if (more)
        load(a, a.bt[(int64_t)b * a.w + (t0 + kUnit) / a.bs], kvh, t0 + kUnit, t_end, lane, nxt);

      // lane (g, n): scores of tokens 16c + 4g + r of head n
      f32x4 s[4];
      const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
      s[0] = mfma_fp4<0>(cur.k[0], cur.kscale, qp[0], zero);
      s[1] = mfma_fp4<1>(cur.k[1], cur.kscale, qp[0], zero);
      s[2] = mfma_fp4<2>(cur.k[2], cur.kscale, qp[0], zero);
      s[3] = mfma_fp4<3>(cur.k[3], cur.kscale, qp[0], zero);
#pragma unroll
      for (int p = 1; p < NQ; ++p) {
        s[0] = mfma_fp4<0>(cur.k[0], cur.kscale, qp[p], s[0]);
        s[1] = mfma_fp4<1>(cur.k[1], cur.kscale, qp[p], s[1]);
        s[2] = mfma_fp4<2>(cur.k[2], cur.kscale, qp[p], s[2]);
        s[3] = mfma_fp4<3>(cur.k[3], cur.kscale, qp[p], s[3]);
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) s[c] *= qs;
      if (valid != kUnit) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (!(16 * c + 4 * g + r < valid)) s[c][r] = -INFINITY;
      }
      float tmax = s[0][0];
#pragma unroll
      for (int c = 0; c < 4; ++c)
        tmax = fmaxf(fmaxf(tmax, fmaxf(s[c][0], s[c][1])), fmaxf(s[c][2], s[c][3]));
      tmax = max_xor32(max_xor16(tmax));
      if (__any(tmax > m + kRescaleSlack)) {
        const float m_new = fmaxf(m, tmax);
        const float alpha = m_new == -INFINITY ? 1.0f : exp2_fast(m - m_new);
        l *= alpha;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) acc[dt] *= alpha;
        m = m_new;
      }
      const float m_use = m == -INFINITY ? 0.0f : m;
      const float* vsc = scales[buf];
      f16x8 pt[2];
      float psum = 0.0f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const f32x4 vs4 = *reinterpret_cast<const f32x4*>(vsc + 16 * c + 4 * g);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = exp2_fast(s[c][r] - m_use);
          psum += p;
          float w = p * vs4[r];
          // (a token past the end may carry any scale, NaN included)
          if (valid != kUnit && s[c][r] == -INFINITY) w = 0.0f;
          pt[c >> 1][4 * (c & 1) + r] = (_Float16)w;
        }
      }
      l += psum;

      // O^T += V^T . P^T: 16 dimensions by 32 tokens an MFMA
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) {
        const i32x2 raw = fp4_v_read(tiles[buf], vrow + fp4_v_col(lane, dt));
        acc[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fp4x8_to_f16((uint32_t)raw[0]), pt[0],
                                                         acc[dt], 0, 0, 0);
        acc[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fp4x8_to_f16((uint32_t)raw[1]), pt[1],
                                                         acc[dt], 0, 0, 0);
      }
      if (more) {
        stage(nxt, buf ^ 1);
        cur = nxt;
      }
      wave_lds_sync();
    }
    l = sum_xor32(sum_xor16(l));
    if (f != 0.0f) {
      const float inv_f = 1.0f / f;  // a power of two: exact
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) acc[dt] *= inv_f;
    }
  }
};

}  // namespace mskv
