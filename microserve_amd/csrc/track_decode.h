// The FP8 decode's walk that keeps its scores (the split kernel's
// TrackedFp8Cache), for the attention weights of cached tokens.
//
// The products, softmax and weights are the FP8 walk's, on the same tokens in the
// same order.  The scores, in log2 units, are 4 bytes a (q head, token) against
// 264 of a token's K and V, but written step by step they cost the read stream
// far more than their bytes: 64 x 4096 tokens, 33.5 MB of scores, 85 us without
// the stores, 110 with them, whatever their shape or cache policy, 99 in bursts
// of 512 tokens, 92 in bursts of 1024.  So a wave keeps its scores in LDS and
// writes them when that is full or the range ends, all waves of a round at about
// the same time.  The room comes from the tiles: K and V of a step pass through
// one 4 KB tile, one after the other (LDS executes a wave's instructions in
// order), instead of two tiles of each.
#pragma once

namespace mskv {

struct WalkLoads {
  u32x4 k[4], v[4];      // rows 8c + lane/8, 16-byte chunk lane%8
  float kscale, vscale;  // scales of token lane & 31
  int valid;
};

// A wave's LDS of this walk.
constexpr int kScoreFloats = 3968;  // 992 tokens of four heads
template <bool kTrack>
struct WalkTiles {
  uint8_t tile[kStep * kHeadDim];
};
template <>
struct WalkTiles<true> {
  uint8_t tile[kStep * kHeadDim];
  float scores[kScoreFloats];
};
typedef float WalkScales[2 * kStep];

// One wave's online softmax over tokens [t_begin, t_end) of sequence b, as
// attend_range's.  kTrack: the scores are kept.  Else two steps of loads are in
// flight (for grids that have few of these waves on a CU: four of them read 3 us
// a step with one step ahead), those of step i + 2 going into the registers of
// step i once its V lies in LDS; past the end they are issued out of range, where
// they read nothing, so that the waits for the ones before can be counted.
template <typename T, bool kTrack>
__device__ __forceinline__ void walk_range(const DecodeArgs& a, int b, int kvh, int qh,
                                           bool head_ok, int t_begin, int t_end, int blk_first,
                                           int lane, WalkTiles<kTrack>& lds, WalkScales& scales,
                                           f32x4 (&acc)[8], float& m, float& l) {
  using A = Act<T>;
  using x8 = typename A::x8;
  const int g = lane >> 4, n = lane & 15;
  kvh = __builtin_amdgcn_readfirstlane(kvh);
  const auto* table = reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(
      reinterpret_cast<uintptr_t>(a.bt + (int64_t)b * a.w));
  const uint32_t rstride = (uint32_t)a.hk * kHeadDim;
  // Issues the loads of the step at t0, what is needed first first.
  auto load = [&](int blk, int t0, WalkLoads& s) {
    const int off = t0 % a.bs;
    const bool ok = blk >= 0 && (int64_t)blk < a.num_blocks && t0 < t_end;
    const int64_t row = (ok ? (int64_t)blk : 0) * a.bs * a.hk;
    const uint32_t page_bytes = ok ? (uint32_t)a.bs * rstride : 0u;
    const uint32_t spage_bytes = ok ? (uint32_t)a.bs * a.hk * 4u : 0u;
    const auto kr = make_rsrc(a.kc + row * kHeadDim, page_bytes);
    const auto vr = make_rsrc(a.vc + row * kHeadDim, page_bytes);
    const auto ksr = make_rsrc(a.ks + row, spage_bytes);
    const auto vsr = make_rsrc(a.vs + row, spage_bytes);
    const uint32_t rb = ((uint32_t)off + (lane >> 3)) * rstride + (uint32_t)kvh * kHeadDim +
                        16u * (lane & 7);
    const uint32_t so = (((uint32_t)off + (lane & 31)) * a.hk + kvh) * 4u;
    s.kscale = buf_load_f32(ksr, so);
#pragma unroll
    for (int c = 0; c < 4; ++c) s.k[c] = buf_load16_nt(kr, rb + 8u * c * rstride);
    s.vscale = buf_load_f32(vsr, so);
#pragma unroll
    for (int c = 0; c < 4; ++c) s.v[c] = buf_load16_nt(vr, rb + 8u * c * rstride);
    s.valid = ok ? min(kStep, t_end - t0) : 0;
  };
  auto block_at = [&](int t0) { return table[min(t0, t_end - 1) / a.bs]; };

  x8 qop[4];
  {
    // (first, so that waiting for it is no wait for the steps)
    u32x4 v[4] = {};
    if (head_ok) {
      const u32x4* p = reinterpret_cast<const u32x4*>(a.q + ((int64_t)b * a.hq + qh) * kHeadDim);
      v[0] = p[2 * g], v[1] = p[2 * g + 1], v[2] = p[8 + 2 * g], v[3] = p[9 + 2 * g];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) qop[j] = __builtin_bit_cast(x8, v[j]);
  }
  WalkLoads even, odd;
  load(blk_first, t_begin, even);
  if constexpr (!kTrack) load(block_at(t_begin + kStep), t_begin + kStep, odd);

  // kTrack: the unit's heads, the tokens of each that LDS holds (whole steps),
  // and this lane's place in the first head's row, in vector registers (scalar
  // ones are short here, and would spill)
  int heads = 0, room = 0;
  float* rows = nullptr;
  int64_t row_stride = 0;
  if constexpr (kTrack) {
    const int first_head = __builtin_amdgcn_readfirstlane(qh - n);
    heads = min(16, kvh * a.group + a.group - first_head);
    room = kScoreFloats / (heads * kStep) * kStep;
    rows = a.scores + ((int64_t)b * a.hq + first_head) * score_stride(a.w, a.bs) + 4 * lane;
    row_stride = score_stride(a.w, a.bs);
    asm volatile("" : "+v"(rows), "+v"(row_stride));
  }
  int held_from = t_begin;  // the first token whose scores LDS holds

#pragma unroll
  for (int dt = 0; dt < 8; ++dt) acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  m = -INFINITY;
  l = 0.0f;
  float f = 0.0f, vseen = 0.0f;  // as in attend_range

  const int i16 = lane & 15;
  const int slot = i16 >> 1;
  const int trow = slot < 4 ? 4 * g + slot : 16 + 4 * g + (slot - 4);
  const uint32_t tr_base = (uint32_t)trow * kHeadDim + 8u * (i16 & 1);
  const uint32_t tr_swz = 16u * (uint32_t)((trow >> 1) & 7);
  const uint32_t k_lo = tile_off(n, g), k_hi = tile_off(n, 4 + g);

  auto step = [&](int t0, WalkLoads& cur) {
    const int valid = cur.valid;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      *reinterpret_cast<u32x4*>(&lds.tile[tile_off(8 * c + (lane >> 3), lane & 7)]) = cur.k[c];
    if (lane < 32) scales[lane] = cur.kscale * a.scale_log2;
    wave_lds_sync();
    if constexpr (kTrack) {
      if (t0 + kStep < t_end) load(block_at(t0 + kStep), t0 + kStep, odd);
    }

    const uint8_t* kt = lds.tile;
    const u32x4 k0a = *reinterpret_cast<const u32x4*>(kt + k_lo);
    const u32x4 k0b = *reinterpret_cast<const u32x4*>(kt + k_hi);
    const u32x4 k1a = *reinterpret_cast<const u32x4*>(kt + 16 * kHeadDim + k_lo);
    const u32x4 k1b = *reinterpret_cast<const u32x4*>(kt + 16 * kHeadDim + k_hi);
    const f32x4 ksc0 = *reinterpret_cast<const f32x4*>(scales + 4 * g);
    const f32x4 ksc1 = *reinterpret_cast<const f32x4*>(scales + 16 + 4 * g);
    f32x4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = {0.f, 0.f, 0.f, 0.f};
    x8 ka;
    A::fp8x4_to(k0a[0], ka, 0); A::fp8x4_to(k0a[1], ka, 4); s0 = A::mfma(ka, qop[0], s0);
    A::fp8x4_to(k0a[2], ka, 0); A::fp8x4_to(k0a[3], ka, 4); s0 = A::mfma(ka, qop[1], s0);
    A::fp8x4_to(k0b[0], ka, 0); A::fp8x4_to(k0b[1], ka, 4); s0 = A::mfma(ka, qop[2], s0);
    A::fp8x4_to(k0b[2], ka, 0); A::fp8x4_to(k0b[3], ka, 4); s0 = A::mfma(ka, qop[3], s0);
    A::fp8x4_to(k1a[0], ka, 0); A::fp8x4_to(k1a[1], ka, 4); s1 = A::mfma(ka, qop[0], s1);
    A::fp8x4_to(k1a[2], ka, 0); A::fp8x4_to(k1a[3], ka, 4); s1 = A::mfma(ka, qop[1], s1);
    A::fp8x4_to(k1b[0], ka, 0); A::fp8x4_to(k1b[1], ka, 4); s1 = A::mfma(ka, qop[2], s1);
    A::fp8x4_to(k1b[2], ka, 0); A::fp8x4_to(k1b[3], ka, 4); s1 = A::mfma(ka, qop[3], s1);
    wave_lds_sync();

    // V takes K's place; rows past the end are zeroed, as in attend_range
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int row = 8 * c + (lane >> 3);
      *reinterpret_cast<u32x4*>(&lds.tile[tile_off(row, lane & 7)]) =
          row < valid ? cur.v[c] : u32x4{0u, 0u, 0u, 0u};
    }
    const bool vtok = lane >= 32 && lane - 32 < valid;
    if (__any(vtok && !(cur.vscale * f <= kPvScaleMax)) || f == 0.0f) {
      float vm = vtok ? cur.vscale : 0.0f;
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
    if (lane >= 32) scales[lane] = cur.vscale * f;
    if constexpr (!kTrack) {
      __builtin_amdgcn_sched_barrier(0);
      load(block_at(t0 + 2 * kStep), t0 + 2 * kStep, cur);
    }

    float x[8];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      x[r] = s0[r] * ksc0[r];
      x[4 + r] = s1[r] * ksc1[r];
    }
    if (valid != kStep) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (!(4 * g + r < valid)) x[r] = -INFINITY;
        if (!(16 + 4 * g + r < valid)) x[4 + r] = -INFINITY;
      }
    }
    if constexpr (kTrack) {
      if (n < heads) {
        float* to = &lds.scores[n * room + (t0 - held_from) + 4 * g];
        *reinterpret_cast<f32x4*>(to) = f32x4{x[0], x[1], x[2], x[3]};
        *reinterpret_cast<f32x4*>(to + 16) = f32x4{x[4], x[5], x[6], x[7]};
      }
    }
    float tmax = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])),
                       fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
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
    wave_lds_sync();
    const f32x4 vsc0 = *reinterpret_cast<const f32x4*>(scales + 32 + 4 * g);
    const f32x4 vsc1 = *reinterpret_cast<const f32x4*>(scales + 48 + 4 * g);
    float psum = 0.0f;
    f16x8 pt;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float p = exp2_fast(x[e] - m_use);
      psum += p;
      pt[e] = (_Float16)(p * (e < 4 ? vsc0[e] : vsc1[e - 4]));
    }
    if (valid != kStep) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (x[e] == -INFINITY) pt[e] = (_Float16)0.0f;
    }
    l += psum;
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) {
      const i32x2 raw = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
          reinterpret_cast<__attribute__((address_space(3))) i32x2*>(
              (__attribute__((address_space(3))) uint8_t*)lds.tile + tr_base +
              ((16u * dt) ^ tr_swz)));
      const f16x8 vt = fp8x8_to_f16((uint32_t)raw[0], (uint32_t)raw[1]);
      acc[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, pt, acc[dt], 0, 0, 0);
    }
    wave_lds_sync();
    if constexpr (kTrack) {
      const int held = t0 + kStep - held_from;
      if (held == room || t0 + kStep >= t_end) {  // LDS is full, or the range ends
        float* row = rows + held_from;
        for (int h = 0; h < heads; ++h, row += row_stride) {
          float* to = row;
          for (int i = 4 * lane; i < held; i += 256, to += 256)
            *reinterpret_cast<f32x4*>(to) =
                *reinterpret_cast<const f32x4*>(&lds.scores[h * room + i]);
        }
        wave_lds_sync();
        held_from = t0 + kStep;
      }
    }
  };
  if constexpr (kTrack) {
    for (int t0 = t_begin; t0 < t_end; t0 += kStep) {
      step(t0, even);
      even = odd;
    }
  } else {
    for (int t0 = t_begin; t0 < t_end; t0 += 2 * kStep) {
      step(t0, even);
      if (t0 + kStep >= t_end) break;
      step(t0 + kStep, odd);
    }
  }
  l = sum_xor32(sum_xor16(l));
  if (f != 0.0f) {
    const float inv_f = 1.0f / f;  // a power of two: exact
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) acc[dt] *= inv_f;
  }
}

struct TrackedFp8Cache : Fp8Cache {
  static constexpr bool kTrack = true;
  typedef WalkTiles<true> Tiles;
  typedef WalkScales Scales;
  template <typename T>
  static __device__ __forceinline__ void attend(const DecodeArgs& a, int b, int kvh, int qh,
                                                bool head_ok, int t_begin, int t_end,
                                                int blk_first, int lane, Tiles& tiles,
                                                Scales& scales, f32x4 (&acc)[8], float& m,
                                                float& l) {
    walk_range<T, true>(a, b, kvh, qh, head_ok, t_begin, t_end, blk_first, lane, tiles, scales,
                        acc, m, l);
  }
};

}  // namespace mskv
