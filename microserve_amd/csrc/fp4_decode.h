// The decode's walk over the 4-bit cache (the split kernel's Fp4Cache): a wave
// takes one (sequence, kv head, split), 64 tokens a step.
//
//  * K goes from memory to the matrix unit: the page's layout is the A
//    operand's (fp4.h), the block scales are applied by the MFMA, and the
//    e4m3 parts of the query are the B operand.  In units in which the row's
//    largest element lies in [224, 448], a bf16 element from 1/4 up is exact and
//    an fp16 one from 2 up; smaller ones are off by at most 2^-10, half of
//    e4m3's last step, which is 2^-17.8 of the largest.  No K byte passes
//    through LDS or a conversion.
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
  // 4 / 16 and 4, all split, us: 256 x 16 to 32768 tokens 217 / 215 / 208 / 209, 128 x
  // 8192 200 / 190 / 192 / 186, 256 x 16 to 8192 76 to 82 / 80 / 75 / 160.
  static constexpr int kMaxPages = 8;
  // one step is the least of a split: under tables of 128 entries, 1 x 700
  // tokens 10.0 us (two steps 11.8), 8 x 1000 10.4 (12.1)
  static constexpr int kMinSteps = 1;
  static constexpr int kItemWaves = kNarrowWaves;
  static constexpr bool kTrack = false;
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
    const QueryScale qu = fp4_query<T>(row, head_ok, qp);
    // scores in log2 units: S^T * qs
    const float qs = a.scale_log2 * qu.unit;

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
      s[0] = mfma_fp4<0>(cur.k[0], cur.kscale, qp[0], qu.byte, zero);
      s[1] = mfma_fp4<1>(cur.k[1], cur.kscale, qp[0], qu.byte, zero);
      s[2] = mfma_fp4<2>(cur.k[2], cur.kscale, qp[0], qu.byte, zero);
      s[3] = mfma_fp4<3>(cur.k[3], cur.kscale, qp[0], qu.byte, zero);
#pragma unroll
      for (int p = 1; p < NQ; ++p) {
        s[0] = mfma_fp4<0>(cur.k[0], cur.kscale, qp[p], qu.byte, s[0]);
        s[1] = mfma_fp4<1>(cur.k[1], cur.kscale, qp[p], qu.byte, s[1]);
        s[2] = mfma_fp4<2>(cur.k[2], cur.kscale, qp[p], qu.byte, s[2]);
        s[3] = mfma_fp4<3>(cur.k[3], cur.kscale, qp[p], qu.byte, s[3]);
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

// The whole of a (sequence, kv head) in one workgroup: its four waves take
// equal runs of the sequence's steps and join their results in LDS, in one
// launch and without partials in memory.  Two such workgroups run on a CU at
// once, 512 on the chip, and start and end apart from each other.  Which
// shapes take it, and what it measured, stands at joined_of.  (Eight waves of
// half the steps were no faster up to 2048 tokens: 64 x 4096 51.8 against 47
// us, 32 x 2048 16.4 against 14.8, 8 x 4096 17.9 against 19.4.)
constexpr int kJoinWaves = 4;
constexpr int64_t kJoinMaxTokens = 8192;
static_assert(kJoinMaxTokens / Fp4Cache::kPageUnit <= 64, "a table's entries fit a wave's lanes");

template <typename T>
__global__ __launch_bounds__(64 * kJoinWaves)
__attribute__((amdgpu_waves_per_eu(2, 8)))
void decode_fp4_joined_kernel(DecodeArgs a) {
  using A = Act<T>;
  constexpr int W = kJoinWaves;
  // a wave's tiles, then its output: 16 heads of 128 dimensions, 16-byte chunks
  // XOR-swizzled by the head
  __shared__ __attribute__((aligned(16))) Fp4Cache::Tiles tiles[W];
  __shared__ __attribute__((aligned(16))) Fp4Cache::Scales scales[W];
  __shared__ float s_m[W][16], s_l[W][16];
  static_assert(sizeof(Fp4Cache::Tiles) >= 16 * kHeadDim * sizeof(float), "");
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int g = lane >> 4, n = lane & 15;
  const int unit = blockIdx.x, b = blockIdx.z;
  // (the length and the block ids, 64 at most, in one round trip)
  const int32_t* row = a.bt + (int64_t)b * a.w;
  const int entry = row[min(lane, a.w - 1)];
  const int L = min(__builtin_amdgcn_readfirstlane(a.seqlens[b]), a.w * a.bs);
  const int kvh = unit / a.qgroups;
  const int first = (unit - kvh * a.qgroups) * 16;  // head within the group
  const int heads = min(16, a.group - first);
  const int qh0 = kvh * a.group + first;
  const int steps = (max(L, 0) + Fp4Cache::kUnit - 1) / Fp4Cache::kUnit;
  const int per = (steps + W - 1) / W * Fp4Cache::kUnit;
  const int t_begin = wave * per, t_end = min(L, t_begin + per);
  f32x4 acc[8];
  float m = -INFINITY, l = 0.0f;
  if (t_begin < t_end) {
    const int blk = __builtin_amdgcn_readlane(entry, t_begin / a.bs);
    Fp4Cache::attend<T>(a, b, kvh, qh0 + n, n < heads, t_begin, t_end, blk, lane, tiles[wave],
                        scales[wave], acc, m, l);
  } else {
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  wave_lds_sync();
  auto* part = reinterpret_cast<f32x4(*)[16][kHeadDim / 4]>(&tiles[0][0][0]);
  if (n < heads) {
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) part[wave][n][(4 * dt + g) ^ n] = acc[dt];
  }
  if (g == 0) {
    s_m[wave][n] = m;
    s_l[wave][n] = l;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * (kHeadDim / 4); i += 64 * W) {
    const int h = i / (kHeadDim / 4), c = i % (kHeadDim / 4);
    float top = s_m[0][h];
#pragma unroll
    for (int w = 1; w < W; ++w) top = fmaxf(top, s_m[w][h]);
    // (no token seen: every weight 2^-inf, of zeros or of NaNs)
    if (top == -INFINITY) top = 0.0f;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    float den = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float p = exp2_fast(s_m[w][h] - top);
      sum += part[w][h][c ^ h] * p;
      den += s_l[w][h] * p;
    }
    sum *= den > 0.0f ? 1.0f / den : 0.0f;
    const uint32_t lo = (uint32_t)A::from_f32(sum[0]) | ((uint32_t)A::from_f32(sum[1]) << 16);
    const uint32_t hi = (uint32_t)A::from_f32(sum[2]) | ((uint32_t)A::from_f32(sum[3]) << 16);
    *reinterpret_cast<u32x2*>(a.out + ((int64_t)b * a.hq + qh0 + h) * kHeadDim + 4 * c) =
        u32x2{lo, hi};
  }
}

}  // namespace mskv
