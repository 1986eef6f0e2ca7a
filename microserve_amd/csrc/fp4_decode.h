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
  // A split of a grid of many rounds holds twice the FP8 cache's pages, its
  // bytes, and a workgroup of work items half the waves (two workgroups a CU,
  // whose starts and ends overlap).  At 4 pages and 8 waves / 8 and 8 / 8 and
  // 4 / 16 and 4, us: 256 x 16 to 32768 tokens 217 / 215 / 208 / 209, 128 x
  // 8192 200 / 190 / 192 / 186, 256 x 16 to 8192 76 to 82 / 80 / 75 / 160.
  static constexpr int kMaxPages = 8;
  // one step is the least of a split: 1 x 700 tokens 10.0 us (two steps 11.8),
  // 8 x 1000 10.4 (12.1)
  static constexpr int kMinSteps = 1;
  static constexpr int kItemWaves = kNarrowWaves;
  // a token whose bytes (64 a token, 31 bits) lie past the end of any page
  static constexpr uint32_t kPastEnd = (1u << 25) - kUnit;
  typedef uint8_t Tiles[2][kUnit * kFp4Row];  // V, double-buffered
  typedef float Scales[2][kUnit];             // v_scale * f

  // The page that loads are issued from: four resources of one kv head's rows
  // (zero-length for an invalid block), and the next step's place in it.
  struct Page {
    __amdgpu_buffer_rsrc_t k, v, ks, vs;
    bool ok;
    int off, index;
  };
  static __device__ __forceinline__ void open(const DecodeArgs& a, int blk, int kvh, Page& p) {
    p.ok = blk >= 0 && (int64_t)blk < a.num_blocks;
    const int64_t row = ((p.ok ? (int64_t)blk : 0) * a.hk + kvh) * a.bs;
    const uint32_t bytes = p.ok ? (uint32_t)a.bs * kFp4Row : 0u;
    const uint32_t sbytes = p.ok ? (uint32_t)a.bs * 4u : 0u;
    p.k = make_rsrc(a.kc + row * kFp4Row, bytes);
    p.v = make_rsrc(a.vc + row * kFp4Row, bytes);
    p.ks = make_rsrc(a.ks + row, sbytes);
    p.vs = make_rsrc(a.vs + row, sbytes);
  }

  template <typename T>
  static __device__ __forceinline__ void attend(const DecodeArgs& a, int b, int kvh, int qh,
                                                bool head_ok, int t_begin, int t_end,
                                                int blk_first, int lane, Tiles& tiles,
                                                Scales& scales, f32x4 (&acc)[8], float& m,
                                                float& l) {
    constexpr int NQ = Fp4Query<T>::parts;
    const int g = lane >> 4;
    // (a wave's own: the compiler takes it to differ from lane to lane)
    kvh = __builtin_amdgcn_readfirstlane(kvh);
    // the block table is read-only: the constant address space keeps its
    // loads scalar
    const auto* table = reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(
        reinterpret_cast<uintptr_t>(a.bt + (int64_t)b * a.w));
    Page page;
    page.index = t_begin / a.bs;
    page.off = t_begin - page.index * a.bs;
    open(a, blk_first, kvh, page);
    // the block after it, read a page ahead
    int blk_next = table[min(page.index + 1, a.w - 1)];
    // Issues the loads of the step at token t0; steps come in order.  Past the
    // end every offset is out of range: the loads read nothing, but they are
    // always issued, so that the waits for the loads before them can be counted.
    auto issue = [&](int t0, Fp4Loads& s) {
      const bool more = t0 < t_end;
      if (more && page.off == a.bs) {
        page.off = 0;
        open(a, blk_next, kvh, page);
        blk_next = table[min(++page.index + 1, a.w - 1)];
      }
      const uint32_t at = more ? (uint32_t)page.off : kPastEnd;
      const uint32_t o = at * kFp4Row + 16u * lane;
#pragma unroll
      for (int c = 0; c < 4; ++c) s.k[c] = buf_load16_nt(page.k, o + 1024u * c);
      const uint32_t so = (at + lane) * 4u;
      s.kscale = __float_as_uint(buf_load_f32(page.ks, so));
#pragma unroll
      for (int c = 0; c < 4; ++c) s.v[c] = buf_load16_nt(page.v, o + 1024u * c);
      s.vscale = buf_load_f32(page.vs, so);
      s.valid = page.ok ? max(min(kUnit, t_end - t0), 0) : 0;
      page.off += kUnit;
    };
    // (the query's row first: waiting for it is then no wait for the steps')
    const QueryRow row = load_query(
        a.q + ((int64_t)b * a.hq + (head_ok ? qh : kvh * a.group)) * kHeadDim, g);
    // Two steps are in flight: the loads of step i + 2 go into the registers
    // of step i once its products are issued (its V lies in LDS by then).
    Fp4Loads even, odd;
    issue(t_begin, even);
    issue(t_begin + kUnit, odd);

    i32x8 qp[NQ];
    // scores in log2 units: S^T * qs
    const float qs = a.scale_log2 / fp4_query<T>(row, head_ok, qp);

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
    // step i, whose V is in buffer `buf`; `cur` holds its K, `nxt` step i + 1
    auto step = [&](int t0, int buf, Fp4Loads& cur, Fp4Loads& nxt, auto last) {
      const int valid = cur.valid;
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
      // (not before the products: the loads would take other registers, and
      // moving those at the loop's end would wait for them)
      if constexpr (!decltype(last)::value) {
        __builtin_amdgcn_sched_barrier(0);
        issue(t0 + 2 * kUnit, cur);
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
      if constexpr (!decltype(last)::value) {
        stage(nxt, buf ^ 1);  // (past the end: nothing, as it was loaded)
        wave_lds_sync();
      }
    };

    stage(even, 0);
    wave_lds_sync();
    // (the last step of an odd number after the loop: a way out of its middle
    // would also lose the count of the loads in flight)
    int t0 = t_begin;
    for (; t0 + kUnit < t_end; t0 += 2 * kUnit) {
      step(t0, 0, even, odd, std::false_type());
      step(t0 + kUnit, 1, odd, even, std::false_type());
    }
    if (t0 < t_end) step(t0, 0, even, odd, std::true_type());
    l = sum_xor32(sum_xor16(l));
    if (f != 0.0f) {
      const float inv_f = 1.0f / f;  // a power of two: exact
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) acc[dt] *= inv_f;
    }
  }
};

}  // namespace mskv
