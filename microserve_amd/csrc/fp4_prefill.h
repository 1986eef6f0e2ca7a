// Varlen causal prefill over the 4-bit paged cache (fp4.h has the format):
// query i of a sequence with Lq new tokens and Lk cached ones (new ones
// included) sees positions p < (Lk - Lq) + i + 1.
//
// The FP8 kernel's decomposition (a workgroup of four waves takes 128 rows of
// one (sequence, kv head, block of query tokens), tiles of 128 keys, longest
// blocks first, keys split over workgroups where the grid is small), with
// half of its LDS traffic and without its work on the scales:
//  * A tile of one head is contiguous: K is copied to LDS in the operand
//    order that it has in memory and read back 16 bytes a lane, free of
//    bank conflicts.
//  * QK^T: v_mfma_scale_f32_16x16x128_f8f6f4 takes the codes and their block
//    scales as stored, and the query in three e2m3 parts under scales of their
//    own; the scores need no scaling by key.  (Two e4m3 parts of a bf16 query
//    took the same time, three of an fp16 one 9% more of the whole kernel.)
//  * PV: v_mfma_f32_16x16x32_f16; V^T from ds_read_b64_tr_b4 converts to fp16
//    exactly; weights fp16(p) * fp16(v_scale * fw) as in the FP8 kernel.
#pragma once

#include "fp4.h"

namespace mskv {

template <int N> using Int = std::integral_constant<int, N>;

// What a row's exponents are taken against, from its running maximum m of the
// unscaled scores: exponent = (score - base) * scale - log.  With base 0, log
// is m * scale, whose rounding the row's keys share, and the exponent is one
// fma.  Past kPFar in log2 units that rounding would show (from 2^27 up by more
// than 2^3, and weights would leave fp16's range): such scores are
// subtracted before the scale.  A row without a key (-FLT_MAX) is none of those.
constexpr float kPFar = 1 << 20;
struct Level {
  float base, log;
};
__device__ __forceinline__ Level level_of(float m, float scale) {
  const float log = fmaxf(m * scale, -FLT_MAX);
  const bool far = fabsf(log) > kPFar && m != -FLT_MAX;
  return {far ? m : 0.0f, far ? 0.0f : log};
}

// kSplit: the workgroup takes one of a.splits ranges of the keys (whole
// tiles, from the actual key count) and leaves partials for the merge.
template <typename T, bool kSplit>
__global__ __launch_bounds__(PShape::threads, 2) void prefill_fp4_kernel(PrefillArgs a) {
  using A = Act<T>;
  constexpr int kPBlocks = PShape::blocks;
  constexpr int kPWaves = PShape::waves;
  constexpr int kKeys = kPStep;  // of a tile
  constexpr int kGroups = kKeys / 16;  // S^T tiles
  constexpr int kChunks = kKeys / 32;  // P^T chunks
  constexpr int kHalves = kKeys / 64;  // V^T reads
  // two tile buffers as separate objects, and a loop unrolled by two, as in
  // the FP8 kernel: direct loads into one then never alias the other's reads
  __shared__ __attribute__((aligned(16))) uint8_t k_lds0[kKeys * kFp4Row];
  __shared__ __attribute__((aligned(16))) uint8_t v_lds0[kKeys * kFp4Row];
  __shared__ __attribute__((aligned(16))) uint8_t k_lds1[kKeys * kFp4Row];
  __shared__ __attribute__((aligned(16))) uint8_t v_lds1[kKeys * kFp4Row];
  __shared__ __attribute__((aligned(16))) uint32_t sc_lds0[2][kKeys];
  __shared__ __attribute__((aligned(16))) uint32_t sc_lds1[2][kKeys];
  // each wave's v_scale * fw of the current tile's keys
  constexpr bool kFp16 = A::kId == 0;
  typedef typename std::conditional<kFp16, float, _Float16>::type VScale;
  typedef VScale vscale4 __attribute__((ext_vector_type(4)));
  __shared__ __attribute__((aligned(16))) VScale vsf_lds[kPWaves][kKeys];

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int g = lane >> 4, n = lane & 15;
  // grid (kv head units, sequences, query blocks): the query block varies
  // slowest and runs last-first, so every sequence's longest blocks are
  // dispatched before any shorter ones (longest-first across the whole
  // grid, not within each sequence): bf16 5.4%, fp16 3.9% faster than
  // query blocks varying fastest
  const int s = blockIdx.y;
  const int unit = blockIdx.x;
  const int kvh = unit / a.qgroups;
  const int qgi = unit - kvh * a.qgroups;

  // query rows are clamped to [0, total_q) and positions to the table width,
  // so inconsistent cu_seqlens cannot address memory outside the tensors
  const int64_t tq = a.total_q;
  const int q_begin = a.cu_q ? (int)min((int64_t)max(a.cu_q[s], 0), tq) : 0;
  const int q_end = a.cu_q ? (int)min((int64_t)max(a.cu_q[s + 1], q_begin), tq) : (int)tq;
  const int lq = q_end - q_begin;
  const int lk = a.cu_k ? a.cu_k[s + 1] - a.cu_k[s] : a.prefix_len + lq;
  const int prefix = lk - lq;
  const int wave_tok = kPBlocks * a.tpr;  // query tokens per wave
  const int wg_tok = kPWaves * wave_tok;
  // grid z: query blocks, of a.splits key ranges each
  int zb = (int)(gridDim.z - 1 - blockIdx.z), split = 0;
  if constexpr (kSplit) {
    split = zb % a.splits;
    zb /= a.splits;
  }
  const int wg_q0 = zb * wg_tok;
  if (wg_q0 >= lq || lq <= 0) return;
  const int wg_qlast = min(lq, wg_q0 + wg_tok) - 1;
  int kv_end = min(min(lk, prefix + wg_qlast + 1), a.w * a.bs);
  int kv_begin = 0;
  if constexpr (kSplit) {
    const int tiles = (kv_end + kPStep - 1) / kPStep;
    const int per = max((tiles + a.splits - 1) / a.splits, kPMinSplitTiles);
    const bool whole = tiles <= per;  // one range holds all the keys
    kv_begin = split * per * kPStep;
    kv_end = min(kv_end, kv_begin + per * kPStep);
    // a range without keys (unless it is the only one: it writes the rows,
    // zeros if there are no keys at all) leaves empty partials
    if (kv_begin >= kv_end && !(whole && split == 0)) {
      if (whole) return;
      for (int r = tid; r < kPWaves * kPBlocks * 16; r += PShape::threads) {
        const int rn = r & 15;
        const int rq = (rn * a.gc_magic) >> 8;
        const int qi = wg_q0 + (r >> 4) * a.tpr + rq;
        const int h = qgi * 16 + rn - rq * a.gc;
        if (rn < a.tpr * a.gc && qi < lq && h < a.group)
          a.part_lse[((int64_t)(q_begin + qi) * a.hq + kvh * a.group + h) * a.splits + split] =
              -INFINITY;
      }
      return;
    }
    if (whole) split = -1;  // the rows are written here, not merged
  }
  // keys below w_all are visible to every row of this wave; no row of it
  // sees keys at or above w_none
  const int w_q0 = wg_q0 + wave * wave_tok;
  const int w_all = prefix + w_q0 + 1;
  const int w_none = w_q0 < lq ? prefix + min(lq, w_q0 + wave_tok) : 0;

  // rows: block b, lane n -> query token w_q0 + b * tpr + n / gc, head n % gc
  int lim[kPBlocks];
  bool row_ok[kPBlocks];
  int qh[kPBlocks];
  u32x6 qp[kPBlocks][kQ6Parts];
  uint32_t qe[kPBlocks];  // the parts' scale bytes
#pragma unroll
  for (int b = 0; b < kPBlocks; ++b) {
    const int nq = (n * a.gc_magic) >> 8;  // n / gc
    const int qi = w_q0 + b * a.tpr + nq;
    // a unit of a group above 16 that is not a multiple of 16 has idle
    // lanes past the group's last head
    row_ok[b] = n < a.tpr * a.gc && qi < lq && qgi * 16 + n - nq * a.gc < a.group;
    qh[b] = kvh * a.group + qgi * 16 + n - nq * a.gc;
    lim[b] = row_ok[b] ? prefix + qi + 1 : 0;
    const int64_t row = row_ok[b] ? (int64_t)(q_begin + qi) * a.hq + qh[b] : 0;
    qe[b] = fp4_query6<T>(load_query6(a.q + row * kHeadDim, g), row_ok[b], qp[b]);
  }

  // acc: O^T in units of fw, the power-of-two scale applied to v_scale (0
  // until the first tile with a stored token sets it); lacc: the softmax
  // denominator, as the output tile of an all-ones A operand against P^T,
  // so every row of it holds its column's sum of the fp16 probabilities
  f32x4 acc[kPBlocks][8], lacc[kPBlocks];
  float m[kPBlocks];  // the running maxima, of the scores before the scale
#pragma unroll
  for (int b = 0; b < kPBlocks; ++b) {
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) acc[b][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    lacc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
    // -FLT_MAX rather than -inf: a row that has seen no key yet keeps it,
    // and its masked (-inf) scores still give p = 0 with no select; the
    // first finite score raises it like any other growth (an idle lane's row
    // needs none)
    m[b] = row_ok[b] ? -FLT_MAX : 0.0f;
  }
  float fw = 0.0f;
  f16x8 ones;
#pragma unroll
  for (int i = 0; i < 8; ++i) ones[i] = (_Float16)1.0f;

  const uint32_t vrow = fp4_v_row(lane);

  // the block table is read-only: the constant address space keeps its
  // loads scalar
  const auto* btc = reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(
      reinterpret_cast<uintptr_t>(a.bt));

  // Stages tile t0 with direct loads; returns the number of keys holding real
  // tokens.  A tile of one head is contiguous in memory: 8 KB of K in operand
  // order, copied as it is, and 8 KB of V rows, whose 16-byte chunks are
  // swizzled on the way (lane i lands in slot i of its kilobyte, and reads
  // the chunk that belongs there).  Wave w loads kilobytes w and 4 + w.
  // Keys past the last valid one keep whatever the page holds: every code is
  // a finite value and their scores are masked.  Their v_scale reads as zero,
  // since 0 * NaN would not.
  auto stage_tile = [&](int t0, uint8_t* kt, uint8_t* vt, uint32_t (*sct)[kKeys]) {
    const int page = t0 / a.bs;
    const int off = t0 - page * a.bs;
    const int blk = btc[(int64_t)s * a.w + page];
    const bool ok = blk >= 0 && (int64_t)blk < a.num_blocks;
    const int valid = ok ? min(kKeys, lk - t0) : 0;
    const int64_t row = ((ok ? (int64_t)blk : 0) * a.hk + kvh) * a.bs + off;
    const uint32_t bytes = valid > 0 ? kKeys * kFp4Row : 0u;
    const auto kr = make_rsrc(a.kc + row * kFp4Row, bytes);
    const auto vr = make_rsrc(a.vc + row * kFp4Row, bytes);
    // waves 0 to kHalves - 1 load the block scales of K, the next the v_scales
    const bool of_k = wave < kHalves;
    const int half = of_k ? wave : wave - kHalves;
    const auto sr = make_rsrc((of_k ? a.ks : a.vs) + row,
                              valid > 0 ? (of_k ? kKeys : valid) * 4u : 0u);
#pragma unroll
    for (int j = 0; j < kKeys / 16 / kPWaves; ++j) {
      const int kb = kPWaves * j + wave;
      lds_load16(kr, kt + 1024 * kb, 1024u * kb + 16u * lane);
      lds_load16(vr, vt + 1024 * kb, 1024u * kb + 16u * (lane ^ (kb & 3)));
    }
    if (wave < 2 * kHalves)
      lds_load4(sr, &sct[of_k ? 0 : 1][64 * half], 256u * half + 4u * lane);
    return valid;
  };

  // one tile of work for this wave: QK^T, softmax, PV
  auto compute_tile = [&](int t0, int valid, const uint8_t* kt, const uint8_t* vt,
                          const uint32_t (*sct)[kKeys]) {
    if (t0 < w_none) {
      const float* vss = reinterpret_cast<const float*>(sct[1]);
      // S^T = K . Q^T: lane (g, n) gets keys 16tt + 4g + r of row n
      f32x4 st[kPBlocks][kGroups];
      uint32_t ksw[kHalves];
#pragma unroll
      for (int i = 0; i < kHalves; ++i) ksw[i] = sct[0][64 * i + lane];
      u32x4 ka[kGroups];
#pragma unroll
      for (int tt = 0; tt < kGroups; ++tt)
        ka[tt] = *reinterpret_cast<const u32x4*>(kt + 1024 * tt + 16 * lane);
      // One part of the query at a time over 64 keys: an MFMA follows the one
      // whose sum it continues at a distance of eight.
      auto qk = [&](auto half, auto part) {
        constexpr int h = decltype(half)::value, p = decltype(part)::value;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int b = 0; b < kPBlocks; ++b) {
          auto one = [&](auto tile) {
            constexpr int t = decltype(tile)::value;
            const f32x4 c = p == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : st[b][4 * h + t];
            st[b][4 * h + t] =
                mfma_fp4_q6<t, p>(ka[4 * h + t], ksw[h], qp[b][p], qe[b], c);
          };
          one(Int<0>()), one(Int<1>()), one(Int<2>()), one(Int<3>());
        }
      };
      qk(Int<0>(), Int<0>()), qk(Int<0>(), Int<1>()), qk(Int<0>(), Int<2>());
      qk(Int<1>(), Int<0>()), qk(Int<1>(), Int<1>()), qk(Int<1>(), Int<2>());
      __builtin_amdgcn_sched_barrier(0);
      // masked keys -> -inf on tiles that need masks
      const bool full = t0 + kKeys <= w_all && valid == kKeys;
      // The barrier after each row of keys keeps the scheduler from hoisting
      // all 64 lane-mask compares ahead of their selects.  Hoisted, their
      // SGPR pairs overflow the SGPR file, and the allocator then spills
      // SGPRs through VGPR lanes in every tile, masked or not (~50
      // v_readlane/v_writelane per full tile): 4.7-4.9% of kernel time.
      if (!full) {
#pragma unroll
        for (int tt = 0; tt < kGroups; ++tt) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int key = 16 * tt + 4 * g + r;
#pragma unroll
            for (int b = 0; b < kPBlocks; ++b)
              if (!(key < valid && t0 + key < lim[b])) st[b][tt][r] = -INFINITY;
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      // Row maxima (the scale is positive: they keep their order).  Each lane tests its own
      // 32 scores against the row's running max: a row's maximum is the
      // largest of its four lanes', and the positive scale keeps the order,
      // so the wave vote equals the test on the row maxima, and the
      // cross-lane reduction runs only when the vote passes.
      // Maxima past kPFar take that way with every tile.
      float lm[kPBlocks], ml[kPBlocks];  // (ml: of m, as the exponents below take it)
      bool grow = false;
#pragma unroll
      for (int b = 0; b < kPBlocks; ++b) {
        float v = fmaxf(fmaxf(st[b][0][0], st[b][0][1]), fmaxf(st[b][0][2], st[b][0][3]));
#pragma unroll
        for (int tt = 1; tt < kGroups; ++tt)
          v = fmaxf(fmaxf(v, st[b][tt][0]), fmaxf(fmaxf(st[b][tt][1], st[b][tt][2]), st[b][tt][3]));
        lm[b] = v;
        ml[b] = fmaxf(m[b] * a.scale_log2, -FLT_MAX);
        grow |= v * a.scale_log2 > ml[b] + kPSlack || fabsf(ml[b]) > kPFar;
      }
      if (__any(grow)) {
        float base[kPBlocks];
        bool far = false;
#pragma unroll
        for (int b = 0; b < kPBlocks; ++b) {
          const float m_new = fmaxf(m[b], max_xor32(max_xor16(lm[b])));
          const Level was = level_of(m[b], a.scale_log2), is = level_of(m_new, a.scale_log2);
          const float alpha = exp2_fast(fmaf(was.base - is.base, a.scale_log2, was.log - is.log));
          ml[b] = is.log;
          base[b] = is.base;
          far |= is.base != 0.0f;
          lacc[b] *= alpha;
#pragma unroll
          for (int dt = 0; dt < 8; ++dt) acc[b][dt] *= alpha;
          m[b] = m_new;
        }
        if (__any(far)) {
#pragma unroll
          for (int b = 0; b < kPBlocks; ++b)
#pragma unroll
            for (int tt = 0; tt < kGroups; ++tt) st[b][tt] -= base[b];
        }
      }
      // The PV product runs on v_mfma_f32_16x16x32_f16.  V converts to fp16
      // exactly, and each weight is fp16(p) * fp16(v_scale * fw), formed in
      // pairs by v_pk_mul_f16.  fw is a power of two per wave, set from the
      // largest v_scale the wave has seen: v_scale * fw <= kPVScaleMax, so
      // with p <= 2^8 (the lazy rescale's slack) no weight leaves fp16's
      // range (the bound on the smaller keys' precision is in the header).
      // It only ever shrinks, and the accumulator is then rescaled
      // by the exact ratio; the output is divided by it at the end.
      // A wave vote on the lanes' own keys skips the tile's v_scale maximum
      // while every key fits under fw (a NaN scale fails the test and takes
      // the exact path, whose maximum ignores it).
      {
        const float v0 = vss[lane], v1 = vss[64 + lane];
        if (__any(!(v0 * fw <= kPVScaleMax) || !(v1 * fw <= kPVScaleMax)) || fw == 0.0f) {
          const float vm = max_xor32(max_xor16(max16_dpp(fmaxf(v0, v1))));
          if (vm > 0.0f && (fw == 0.0f || vm * fw > kPVScaleMax)) {
            const float fnew = pow2_floor(kPVScaleMax / vm);
            if (fw != 0.0f) {
              const float r = fnew / fw;  // a power of two: exact
#pragma unroll
              for (int b = 0; b < kPBlocks; ++b)
#pragma unroll
                for (int dt = 0; dt < 8; ++dt) acc[b][dt] *= r;
            }
            fw = fnew;
          }
        }
      }
      // v_scale * fw of the tile's keys, computed once per key by
      // this wave (lane i: keys i and 64 + i) and read back in groups of
      // four; the wave reads only its own writes, so a wave-level barrier
      // orders them
      VScale* vsw = vsf_lds[wave];
      vsw[lane] = (VScale)(vss[lane] * fw);
      vsw[64 + lane] = (VScale)(vss[64 + lane] * fw);
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      // The wave raises its priority over the P loop and the PV MFMAs and
      // drops it after.
      __builtin_amdgcn_s_setprio(1);
      // P^T for the f16 MFMA: 32-key chunk c of the tile is S^T tiles 2c and
      // 2c + 1, so lane (g, n) holds keys 32c + 4g + r and 32c + 16 + 4g + r
      // of row n -- the order in which ds_read_b64_tr_b4 hands it V^T.
      // Each 16-key group's scales are read once for both blocks, one group
      // ahead: read per block and group, every read's LDS latency was
      // exposed.  The denominator's MFMA for a chunk follows its probabilities.
      // An fp16 output sees the weights' roundings: there the scale stays in
      // 32 bits and a weight is rounded once, as in the decode (error against
      // 64 bits 2.9e-4 instead of 3.7e-4, of which the output's own rounding
      // is 2.1e-4).
      f16x8 pw[kPBlocks][kChunks];
      vscale4 vsf_next = *reinterpret_cast<const vscale4*>(vsw + 4 * g);
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        f16x8 pc[kPBlocks];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int tt = 2 * c + h;
          const vscale4 vf = vsf_next;
          if (tt < kGroups - 1) vsf_next = *reinterpret_cast<const vscale4*>(vsw + 16 * (tt + 1) + 4 * g);
#pragma unroll
          for (int b = 0; b < kPBlocks; ++b) {
            float pf[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) pf[r] = exp2_fast(fmaf(st[b][tt][r], a.scale_log2, -ml[b]));
            const f16x2 p01 = {(_Float16)pf[0], (_Float16)pf[1]};
            const f16x2 p23 = {(_Float16)pf[2], (_Float16)pf[3]};
            f16x2 w01, w23;
            if constexpr (kFp16) {
              w01 = f16x2{(_Float16)(pf[0] * vf[0]), (_Float16)(pf[1] * vf[1])};
              w23 = f16x2{(_Float16)(pf[2] * vf[2]), (_Float16)(pf[3] * vf[3])};
            } else {
              w01 = p01 * f16x2{vf[0], vf[1]};
              w23 = p23 * f16x2{vf[2], vf[3]};
            }
            pc[b][4 * h + 0] = p01[0];
            pc[b][4 * h + 1] = p01[1];
            pc[b][4 * h + 2] = p23[0];
            pc[b][4 * h + 3] = p23[1];
            pw[b][c][4 * h + 0] = w01[0];
            pw[b][c][4 * h + 1] = w01[1];
            pw[b][c][4 * h + 2] = w23[0];
            pw[b][c][4 * h + 3] = w23[1];
          }
        }
#pragma unroll
        for (int b = 0; b < kPBlocks; ++b)
          lacc[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pc[b], lacc[b], 0, 0, 0);
      }
      // A masked key's p is 0, but its v_scale may be no number: where a tile
      // that needs masks holds such a scale, the masked weights are set to 0.
      if (!full) {
        const uint32_t v0 = sct[1][lane], v1 = sct[1][64 + lane];
        if (__any((v0 & 0x7F800000u) == 0x7F800000u || (v1 & 0x7F800000u) == 0x7F800000u)) {
          // (the rows' ends again from the lane id: kept live so far, they spill)
          int ln = lane;
          asm volatile("" : "+v"(ln));
          const int first = 4 * (ln >> 4);
          const int end0 = prefix + w_q0 + (((ln & 15) * a.gc_magic) >> 8) + 1 - t0;
#pragma unroll
          for (int i = 0; i < kKeys / 4; ++i) {
            const int key = 16 * (i >> 2) + (i & 3) + first;
#pragma unroll
            for (int b = 0; b < kPBlocks; ++b)
              if (!(key < min(valid, end0 + b * a.tpr))) pw[b][i >> 3][i & 7] = (_Float16)0.0f;
            __builtin_amdgcn_sched_barrier(0);  // (as in the masks above)
          }
        }
      }
      // O^T += V^T . P^T, one 16-wide d tile and 32-key chunk per MFMA; a read
      // brings a lane 16 tokens of 64, two chunks.  The reads of d tile dt + 1
      // are issued before the MFMAs of tile dt.
      i32x2 raw[kHalves];
#pragma unroll
      for (int c = 0; c < kHalves; ++c) raw[c] = fp4_v_read(vt + 64 * kFp4Row * c, vrow + fp4_v_col(lane, 0));
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) {
        i32x2 nxt[kHalves];
#pragma unroll
        for (int c = 0; c < kHalves; ++c)
          nxt[c] = fp4_v_read(vt + 64 * kFp4Row * c, vrow + fp4_v_col(lane, dt < 7 ? dt + 1 : dt));
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const f16x8 va = fp4x8_to_f16((uint32_t)raw[c >> 1][c & 1]);
#pragma unroll
          for (int b = 0; b < kPBlocks; ++b)
            acc[b][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pw[b][c], acc[b][dt], 0, 0, 0);
        }
#pragma unroll
        for (int c = 0; c < kHalves; ++c) raw[c] = nxt[c];
      }
      __builtin_amdgcn_s_setprio(0);
    }
  };

  int valid = stage_tile(kv_begin, k_lds0, v_lds0, sc_lds0);
  __syncthreads();
  for (int t0 = kv_begin; t0 < kv_end; t0 += 2 * kKeys) {
    {
      const bool more = t0 + kKeys < kv_end;
      const int valid_next = more ? stage_tile(t0 + kKeys, k_lds1, v_lds1, sc_lds1) : 0;
      compute_tile(t0, valid, k_lds0, v_lds0, sc_lds0);
      __syncthreads();  // also waits for this wave's direct loads
      valid = valid_next;
      if (!more) break;
    }
    {
      const int t1 = t0 + kKeys;
      const bool more = t1 + kKeys < kv_end;
      const int valid_next = more ? stage_tile(t1 + kKeys, k_lds0, v_lds0, sc_lds0) : 0;
      compute_tile(t1, valid, k_lds1, v_lds1, sc_lds1);
      __syncthreads();
      valid = valid_next;
    }
  }

  // The rows' coordinates are recomputed from the lane id rather than kept
  // live across the loop, which would spill them.
  int n_out = lane & 15;
  asm volatile("" : "+v"(n_out));
  // A split workgroup also reads the arguments again: held in scalar
  // registers across the loop, they spill.
  int hq = a.hq, group = a.group, gc = a.gc, gc_magic = a.gc_magic, tpr = a.tpr;
  uint16_t* out = a.out;
  float *part_o = nullptr, *part_lse = nullptr;
  int splits = 1;
  if constexpr (kSplit) {
    typedef const __attribute__((address_space(4))) PrefillArgs* KernArgs;
    KernArgs ka = (KernArgs)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(ka));
    hq = ka->hq, group = ka->group, gc = ka->gc, gc_magic = ka->gc_magic, tpr = ka->tpr;
    out = ka->out;
    part_o = ka->part_o, part_lse = ka->part_lse, splits = ka->splits;
  }
#pragma unroll
  for (int b = 0; b < kPBlocks; ++b) {
    const float lt = lacc[b][0];
    const int nq = (n_out * gc_magic) >> 8;  // n / gc
    const int qi = w_q0 + b * tpr + nq;
    if (!(n_out < tpr * gc && qi < lq && qgi * 16 + n_out - nq * gc < group)) continue;
    // acc is in units of fw (a power of two): 1 / fw is exact
    const float scale = lt > 0.0f && fw > 0.0f ? (1.0f / lt) * (1.0f / fw) : 0.0f;
    const int qhb = kvh * group + qgi * 16 + n_out - nq * gc;
    const int64_t row = (int64_t)(q_begin + qi) * hq + qhb;
    if constexpr (kSplit) {
      // (with a NaN denominator the partial is NaN: it gets the largest
      // weight, so the merged row is NaN, as the unsplit kernel's is, and
      // the range is not taken for an empty one)
      if (g == 0)
        part_lse[row * splits + max(split, 0)] = split < 0      ? kPWritten
                                                 : is_nan(lt)   ? FLT_MAX
                                                 : lt > 0.0f    ? m[b] * a.scale_log2 + __log2f(lt)
                                                                : -INFINITY;
      if (split >= 0) {
        float* po = part_o + (row * splits + split) * kHeadDim;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt)
          *reinterpret_cast<f32x4*>(po + 16 * dt + 4 * g) = acc[b][dt] * scale;
        continue;
      }
    }
    uint16_t* op = out + row * kHeadDim;
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) {
      const f32x4 o = acc[b][dt] * scale;
      const uint32_t lo = (uint32_t)A::from_f32(o[0]) | ((uint32_t)A::from_f32(o[1]) << 16);
      const uint32_t hi = (uint32_t)A::from_f32(o[2]) | ((uint32_t)A::from_f32(o[3]) << 16);
      *reinterpret_cast<u32x2*>(op + 16 * dt + 4 * g) = u32x2{lo, hi};
    }
  }
}

}  // namespace mskv
