// Decode attention for a batch whose sequences share prefixes: the pages of a
// group's prefix are attended once for all of its sequences.
//
// out = softmax over the prefix's and the sequence's own tokens: the prefix's
// part (o, log-sum-exp) of every row comes from one pass over its keys by all of
// the group's rows, the rest from the decode's walk over the sequence's own
// tokens, and a merge weighs the parts by 2^lse.
//
//  * A prefix item: a workgroup covers 128 rows (sequence of the group, q head
//    of the kv head) and a range of keys, tile by tile of 128.  K and V come to
//    LDS by direct loads, double-buffered, and serve four waves of two 16-row
//    blocks; products, transposes and weights are the decode's (K converted
//    exactly, one rounding a weight).
//  * A tail item: four waves of the decode's walk over one range of a sequence's
//    own tokens, a kv head unit each.
//  * Both lie in one grid, prefix items first, so that the matrix units work
//    while the tails stream.  Two workgroups (67 KB of LDS) run on a CU.
//  * What the items are follows the lengths on the device: every workgroup
//    makes the plan for itself.  The launch is a function of shapes alone.
//  * A group's shared part ends at the shortest of its sequences (of those that
//    have tokens) and at a whole tile, so that no score of it is masked; the
//    tokens behind belong to the tails.
//
// Bound by what a SIMD issues: a prefix tile's conversions, exponentials and
// products take about 5750 cycles of its wave, a tail's step 2500; the plan takes
// 4 us of every workgroup.  64 sequences over a prefix of 8192 tokens with 512
// each of their own, 32 heads over 8: 32 us and 5 of the merge, 35 in all (the
// decode, which reads 64 x 8704 tokens for them, 120); 128 in eight groups over 512
// to 6144 tokens, 16 to 2048 of their own: 54 in all.
#pragma once

namespace mskv {

constexpr int kSharedThreads = 256;
constexpr int kSharedTile = 128;  // keys
constexpr int kSharedMaxGroups = 1024;
constexpr int kSharedWorkgroups = 512;  // that run at once: two a CU

struct SharedArgs {
  DecodeArgs d;  // part_o, part_lse: [batch * hq, d.splits]
  const int32_t *cu_groups, *prefix_lens;
  int* counts;  // partials of each sequence's rows; -1: its rows are written
  int groups, max_prefix;  // max_prefix: whole tiles' tokens
  int gc, tpr;             // heads of a unit, sequences of a 16-row block
  int sa, sb;              // most ranges of a prefix, of a tail
};

// What a workgroup is to do.
struct SharedItem {
  int kind;         // 0: nothing, 1: of a prefix, 2: of a tail
  int first, size;  // prefix: the group's sequences; tail: the sequence, -
  int row0;         // prefix: first sequence of its 128 rows
  int source;       // prefix: the sequence whose table names the pages
  int begin, end;   // tokens
  int slot, count;  // its partial, and all of the sequence's (tail)
};

struct SharedPlan {
  int cu[kSharedMaxGroups + 1], shared[kSharedMaxGroups], source[kSharedMaxGroups];
  int sums[4][4], scans[4][2];
  SharedItem item;
};

// Time of a prefix item's tile and of a tail item's step beside another
// workgroup, in the same unit (us): what the ranges are balanced by.
constexpr float kSharedTileTime = 3.6f, kSharedStepTime = 2.2f;

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Finds workgroup `index`'s item and its unit: items of prefixes first (`units`
// workgroups each), then those of tails (`tail_units` each), then none.
//
// The ranges are as long as lets all of them run at once, a prefix's and a
// tail's taking about as long: a second round would pay for the plan, the first
// loads and the last stores again.  (64 sequences over a prefix of 8192 tokens:
// 44 us in two rounds of ranges sized apart, 32 in one.)
__device__ __forceinline__ int shared_plan(const SharedArgs& a, int index, int units,
                                           int tail_units, SharedPlan& p) {
  const int tid = threadIdx.x, wave = tid >> 6;
  const int batch = a.d.batch;
  const int cap = a.d.w * a.d.bs;
  // (a thread's first length is read with the groups, and kept)
  const int own_raw = tid < batch ? a.d.seqlens[tid] : 0;
  if (tid == 0) p.item.kind = 0;
  for (int g = tid; g <= a.groups; g += kSharedThreads)
    p.cu[g] = min(max(a.cu_groups[g], 0), batch);
  for (int g = tid; g < a.groups; g += kSharedThreads) {
    p.shared[g] = min(max(a.prefix_lens[g], 0), a.max_prefix);
    p.source[g] = 0x7FFFFFFF;
  }
  __syncthreads();
  // the last group that starts at or before a sequence, if it holds it
  auto group_of = [&](int b) {
    int lo = 0, hi = a.groups;  // cu[lo] <= b < cu[hi], if any
    if (a.groups == 0 || p.cu[0] > b) return -1;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.cu[mid] <= b)
        lo = mid;
      else
        hi = mid;
    }
    return b < p.cu[lo + 1] ? lo : -1;
  };
  auto length = [&](int b) {
    return max(0, min(b == tid ? own_raw : a.d.seqlens[b], cap));
  };
  const int own_group = tid < batch ? group_of(tid) : -1;
  auto group = [&](int b) { return b == tid ? own_group : group_of(b); };
  for (int b = tid; b < batch; b += kSharedThreads) {
    const int g = group(b), len = length(b);
    if (g >= 0 && len > 0) {
      atomicMin(&p.shared[g], len);
      atomicMin(&p.source[g], b);
    }
  }
  __syncthreads();
  // (a group without tokens has nothing to share)
  auto tiles_of = [&](int g) {
    return p.source[g] == 0x7FFFFFFF ? 0 : p.shared[g] / kSharedTile;
  };
  const int rows = 8 * a.tpr;  // sequences of a workgroup's 128 rows
  auto blocks_of = [&](int g) { return ceil_div(max(p.cu[g + 1] - p.cu[g], 0), rows); };
  auto prefix_of = [&](int b) {  // tiles that a sequence shares
    const int g = group(b);
    return g >= 0 && length(b) > 0 ? tiles_of(g) : 0;
  };
  auto steps_of = [&](int b) { return ceil_div(length(b) - prefix_of(b) * kSharedTile, kStep); };
  int work = 0, longest = 0, steps = 0, most = 0;
  for (int g = tid; g < a.groups; g += kSharedThreads) {
    const int t = tiles_of(g);
    work += t * blocks_of(g);
    longest = max(longest, t);
  }
  for (int b = tid; b < batch; b += kSharedThreads) {
    const int s = steps_of(b);
    steps += s;
    most = max(most, s);
  }
  work = wave_sum_i32(work), steps = wave_sum_i32(steps);
  longest = wave_max_u31(longest), most = wave_max_u31(most);
  if ((tid & 63) == 0) {
    p.sums[wave][0] = work, p.sums[wave][1] = longest;
    p.sums[wave][2] = steps, p.sums[wave][3] = most;
  }
  __syncthreads();
  work = longest = steps = most = 0;
#pragma unroll
  for (int i = 0; i < kSharedThreads / 64; ++i) {
    work += p.sums[i][0], longest = max(longest, p.sums[i][1]);
    steps += p.sums[i][2], most = max(most, p.sums[i][3]);
  }
  const float chain = ((float)work * units * kSharedTileTime +
                       (float)steps * tail_units * kSharedStepTime) / kSharedWorkgroups;
  // tiles of a prefix's range, steps of a tail's (no more than the longest has, so
  // that a range's tokens stay an int)
  const int per_a =
      max(min(max((int)ceilf(chain / kSharedTileTime), ceil_div(longest, a.sa)), longest), 1);
  const int per_b = max(min(max((int)ceilf(chain / kSharedStepTime), ceil_div(most, a.sb)), most),
                        kMinSplitSteps);

  // each thread's groups and sequences, one after the other, and the items
  // before them
  const int each_g = ceil_div(a.groups, kSharedThreads);
  const int g0 = min(tid * each_g, a.groups), g1 = min(g0 + each_g, a.groups);
  const int each_b = ceil_div(batch, kSharedThreads);
  const int b0 = min(tid * each_b, batch), b1 = min(b0 + each_b, batch);
  int na = 0, nb = 0;
  for (int g = g0; g < g1; ++g) na += blocks_of(g) * ceil_div(tiles_of(g), per_a);
  // (a sequence without a tail has an item too, which notes its partials)
  for (int b = b0; b < b1; ++b) nb += max(1, ceil_div(steps_of(b), per_b));
  int at_a = wave_scan_i32(na), at_b = wave_scan_i32(nb);
  if ((tid & 63) == 63) p.scans[wave][0] = at_a, p.scans[wave][1] = at_b;
  __syncthreads();
  at_a -= na, at_b -= nb;
  int items_a = 0;
#pragma unroll
  for (int i = 0; i < kSharedThreads / 64; ++i) {
    if (i < wave) at_a += p.scans[i][0], at_b += p.scans[i][1];
    items_a += p.scans[i][0];
  }
  const bool tail = index >= items_a * units;
  if (tail) index -= items_a * units;
  const int item = index / (tail ? tail_units : units);
  const int unit = index - item * (tail ? tail_units : units);
  if (!tail && item >= at_a && item < at_a + na) {
    for (int g = g0; g < g1; ++g) {
      const int blocks = blocks_of(g), ranges = ceil_div(tiles_of(g), per_a);
      if (item < at_a + blocks * ranges) {
        // (a range's row blocks one after the other: they read the same keys)
        const int range = (item - at_a) / blocks, rb = item - at_a - range * blocks;
        p.item = SharedItem{1, p.cu[g], p.cu[g + 1] - p.cu[g], rb * rows, p.source[g],
                            range * per_a * kSharedTile,
                            min((range + 1) * per_a, tiles_of(g)) * kSharedTile, range, 0};
        break;
      }
      at_a += blocks * ranges;
    }
  }
  if (tail && item >= at_b && item < at_b + nb) {
    for (int b = b0; b < b1; ++b) {
      const int ranges = ceil_div(steps_of(b), per_b), i = item - at_b;
      if (i < max(1, ranges)) {
        const int tiles = prefix_of(b), ahead = ceil_div(tiles, per_a), len = length(b);
        const int begin = tiles * kSharedTile + i * per_b * kStep;
        p.item = SharedItem{2, b, 0, i, 0, begin, min(begin + per_b * kStep, len), ahead + i,
                            ahead + ranges};
        break;
      }
      at_b += max(1, ranges);
    }
  }
  __syncthreads();
  return unit;
}

// The LDS of a workgroup: tiles of K and V, double-buffered (separate objects,
// so that the compiler sees that loads into one never alias reads of the
// other), and the tiles' scales.
typedef uint8_t SharedTile[kSharedTile * kHeadDim];
typedef float SharedScales[2][kSharedTile];

template <typename T>
__device__ __forceinline__ void shared_prefix(const SharedArgs& s, const SharedItem& e, int unit,
                                              SharedTile& k_lds0, SharedTile& v_lds0,
                                              SharedTile& k_lds1, SharedTile& v_lds1,
                                              SharedScales& sc_lds0, SharedScales& sc_lds1) {
  using A = Act<T>;
  using x8 = typename A::x8;
  const DecodeArgs& a = s.d;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, n = lane & 15;
  const int kvh = unit / a.qgroups, qgi = unit - kvh * a.qgroups;

  // rows: block k, lane n -> sequence row0 + (2 wave + k) tpr + n / gc of the
  // group, head n % gc of the unit
  x8 qop[2][4];
  int64_t row[2];
  const int hig = qgi * 16 + n % s.gc;
  const int seq0 = e.row0 + 2 * wave * s.tpr;
  const bool active = seq0 < e.size;  // else no row of this wave exists
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int i = seq0 + k * s.tpr + n / s.gc;
    const bool ok = n < s.tpr * s.gc && i < e.size && hig < a.group;
    row[k] = ok ? (int64_t)(e.first + i) * a.hq + kvh * a.group + hig : -1;
    u32x4 v[4] = {};
    if (ok) {
      const u32x4* p = reinterpret_cast<const u32x4*>(a.q + row[k] * kHeadDim);
      v[0] = p[2 * g], v[1] = p[2 * g + 1], v[2] = p[8 + 2 * g], v[3] = p[9 + 2 * g];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) qop[k][j] = __builtin_bit_cast(x8, v[j]);
  }

  f32x4 acc[2][8];
  float m[2], l[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) acc[k][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    m[k] = -INFINITY;
    l[k] = 0.0f;
  }
  float f = 0.0f;  // v_scale's power of two, as in the decode's walk

  // operand reads out of a tile (the swizzle of rows 16t + n is row n's)
  const uint32_t k_lo = tile_off(n, g), k_hi = tile_off(n, 4 + g);
  const int i16 = lane & 15;
  const int tr_r0 = 16 * (i16 >> 3) + 4 * g + ((i16 >> 1) & 3);
  const uint32_t tr_row = (uint32_t)tr_r0 * kHeadDim + 8u * (i16 & 1);
  const uint32_t tr_swz = 16u * (uint32_t)((tr_r0 >> 1) & 7);

  const uint32_t page_bytes = (uint32_t)a.bs * a.hk * kHeadDim;
  const uint32_t rstride = (uint32_t)a.hk * kHeadDim;
  const auto* table = reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(
      reinterpret_cast<uintptr_t>(a.bt + (int64_t)e.source * a.w));
  auto stage = [&](int t0, uint8_t* kt, uint8_t* vt, SharedScales& sct) {
    const int page = t0 / a.bs, off = t0 - page * a.bs;
    const int blk = table[page];
    const bool ok = blk >= 0 && (int64_t)blk < a.num_blocks;
    const int64_t bo = ok ? blk : 0;
    const auto kr = make_rsrc(a.kc + bo * page_bytes, ok ? page_bytes : 0u);
    const auto vr = make_rsrc(a.vc + bo * page_bytes, ok ? page_bytes : 0u);
    const auto sr = make_rsrc((wave < 2 ? a.ks : a.vs) + bo * a.bs * a.hk,
                              ok ? (uint32_t)a.bs * a.hk * 4u : 0u);
    const uint32_t base = (uint32_t)off * rstride + (uint32_t)kvh * kHeadDim;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = 8 * (4 * j + wave) + (lane >> 3);
      const int c = (lane & 7) ^ ((r >> 1) & 7);
      const uint32_t o = base + (uint32_t)r * rstride + 16u * c;
      lds_load16(kr, kt + 1024 * (4 * j + wave), o);
      lds_load16(vr, vt + 1024 * (4 * j + wave), o);
    }
    lds_load4(sr, &sct[wave >> 1][64 * (wave & 1)],
              (((uint32_t)off + 64 * (wave & 1) + lane) * a.hk + kvh) * 4u);
    return ok;
  };

  auto compute = [&](const uint8_t* kt, const uint8_t* vt, const SharedScales& sct) {
    f32x4 st[2][8];
#pragma unroll
    for (int tt = 0; tt < 8; ++tt) {
      const u32x4 lo = *reinterpret_cast<const u32x4*>(kt + 16 * tt * kHeadDim + k_lo);
      const u32x4 hi = *reinterpret_cast<const u32x4*>(kt + 16 * tt * kHeadDim + k_hi);
      x8 ka[4];
      A::fp8x4_to(lo[0], ka[0], 0); A::fp8x4_to(lo[1], ka[0], 4);
      A::fp8x4_to(lo[2], ka[1], 0); A::fp8x4_to(lo[3], ka[1], 4);
      A::fp8x4_to(hi[0], ka[2], 0); A::fp8x4_to(hi[1], ka[2], 4);
      A::fp8x4_to(hi[2], ka[3], 0); A::fp8x4_to(hi[3], ka[3], 4);
      const f32x4 ksc = *reinterpret_cast<const f32x4*>(&sct[0][16 * tt + 4 * g]) * a.scale_log2;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        st[k][tt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) st[k][tt] = A::mfma(ka[j], qop[k][j], st[k][tt]);
        st[k][tt] *= ksc;
      }
    }
    float top[2];
    bool grow = false;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float v = st[k][0][0];
#pragma unroll
      for (int tt = 0; tt < 8; ++tt)
        v = fmaxf(fmaxf(v, fmaxf(st[k][tt][0], st[k][tt][1])), fmaxf(st[k][tt][2], st[k][tt][3]));
      top[k] = v;
      grow |= v > m[k] + kRescaleSlack;
    }
    if (__any(grow)) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float m_new = fmaxf(m[k], max_xor32(max_xor16(top[k])));
        const float alpha = m_new == -INFINITY ? 1.0f : exp2_fast(m[k] - m_new);
        l[k] *= alpha;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) acc[k][dt] *= alpha;
        m[k] = m_new;
      }
    }
    // f: a power of two with v_scale * f <= kPvScaleMax for every token seen
    {
      const float v0 = sct[1][lane], v1 = sct[1][64 + lane];
      if (__any(!(v0 * f <= kPvScaleMax) || !(v1 * f <= kPvScaleMax)) || f == 0.0f) {
        const float vm = max_xor32(max_xor16(max16_dpp(fmaxf(v0, v1))));
        if (vm > 0.0f && (f == 0.0f || vm * f > kPvScaleMax)) {
          const float fnew = pow2_floor(kPvScaleMax / vm);
          if (f != 0.0f) {
            const float r = fnew / f;  // a power of two: exact
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
              for (int dt = 0; dt < 8; ++dt) acc[k][dt] *= r;
          }
          f = fnew;
        }
      }
    }
    f16x8 pt[2][4];
#pragma unroll
    for (int tt = 0; tt < 8; ++tt) {
      const f32x4 vsc = *reinterpret_cast<const f32x4*>(&sct[1][16 * tt + 4 * g]) * f;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float ref = m[k] == -INFINITY ? 0.0f : m[k];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = exp2_fast(st[k][tt][r] - ref);
          l[k] += p;
          pt[k][tt >> 1][4 * (tt & 1) + r] = (_Float16)(p * vsc[r]);
        }
      }
    }
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const i32x2 raw = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
            reinterpret_cast<__attribute__((address_space(3))) i32x2*>(
                (__attribute__((address_space(3))) uint8_t*)vt +
                (tr_row + ((16u * dt) ^ tr_swz)) + 4096u * c));
        const f16x8 va = fp8x8_to_f16((uint32_t)raw[0], (uint32_t)raw[1]);
#pragma unroll
        for (int k = 0; k < 2; ++k)
          acc[k][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pt[k][c], acc[k][dt], 0, 0, 0);
      }
    }
  };

  bool ok = stage(e.begin, k_lds0, v_lds0, sc_lds0);
  __syncthreads();
  for (int t0 = e.begin; t0 < e.end; t0 += 2 * kSharedTile) {
    {
      const bool more = t0 + kSharedTile < e.end;
      const bool next = more && stage(t0 + kSharedTile, k_lds1, v_lds1, sc_lds1);
      if (active && ok) compute(k_lds0, v_lds0, sc_lds0);
      __syncthreads();  // also waits for this wave's direct loads
      ok = next;
      if (!more) break;
    }
    {
      const bool more = t0 + 2 * kSharedTile < e.end;
      const bool next = more && stage(t0 + 2 * kSharedTile, k_lds0, v_lds0, sc_lds0);
      if (active && ok) compute(k_lds1, v_lds1, sc_lds1);
      __syncthreads();
      ok = next;
    }
  }
  const float inv_f = f != 0.0f ? 1.0f / f : 1.0f;  // a power of two: exact
  // (the arguments read again: held in scalar registers across the loop, they
  // spill)
  typedef const __attribute__((address_space(4))) SharedArgs* KernArgs;
  KernArgs ka = (KernArgs)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(ka));
  float *part_o = ka->d.part_o, *part_lse = ka->d.part_lse;
  const int splits = ka->d.splits;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float den = sum_xor32(sum_xor16(l[k]));
    if (row[k] < 0) continue;
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) acc[k][dt] *= inv_f;
    const int64_t at = row[k] * splits + e.slot;
    write_partial(part_o + at * kHeadDim, part_lse + at, acc[k], m[k], den, g);
  }
}

template <typename T>
__device__ __forceinline__ void shared_tail(const SharedArgs& s, const SharedItem& e, int unit,
                                            WalkTiles<false>& tiles, WalkScales& scales) {
  const DecodeArgs& a = s.d;
  const int lane = threadIdx.x & 63;
  const int g = lane >> 4, n = lane & 15;
  const int b = e.first;
  const int kvh = unit / a.qgroups;
  const int hig = (unit - kvh * a.qgroups) * 16 + n;
  const bool head_ok = hig < a.group;
  const int64_t row = (int64_t)b * a.hq + kvh * a.group + hig;
  if (unit == 0 && lane == 0 && e.row0 == 0)
    s.counts[b] = e.count == 0 || (e.count == 1 && e.begin < e.end) ? -1 : e.count;
  if (e.count == 0) {  // no tokens
    if (head_ok) {
#pragma unroll
      for (int dt = 0; dt < 8; ++dt)
        *reinterpret_cast<u32x2*>(a.out + row * kHeadDim + 16 * dt + 4 * g) = u32x2{0u, 0u};
    }
    return;
  }
  if (e.begin >= e.end) return;  // the prefix is all there is
  f32x4 acc[8];
  float m, l;
  const int blk = a.bt[(int64_t)b * a.w + e.begin / a.bs];
  walk_range<T, false>(a, b, kvh, kvh * a.group + hig, head_ok, e.begin, e.end, blk, lane, tiles,
                       scales, acc, m, l);
  if (!head_ok) return;
  if (e.count == 1) {
    write_output<T>(a.out + row * kHeadDim, acc, l, g);
    return;
  }
  const int64_t at = row * a.splits + e.slot;
  write_partial(a.part_o + at * kHeadDim, a.part_lse + at, acc, m, l, g);
}

template <typename T>
__global__ __launch_bounds__(kSharedThreads, 2) void shared_decode_kernel(SharedArgs a) {
  __shared__ __attribute__((aligned(16))) SharedTile k_lds0, v_lds0, k_lds1, v_lds1;
  __shared__ __attribute__((aligned(16))) SharedScales sc_lds0, sc_lds1;
  static_assert(sizeof(SharedTile) >= sizeof(WalkTiles<false>), "a wave's tile fits a tile");
  static_assert(sizeof(SharedPlan) <= sizeof(SharedTile), "the plan fits a tile");
  const int units = a.d.hk * a.d.qgroups;
  SharedPlan& plan = *reinterpret_cast<SharedPlan*>(k_lds0);
  const int own = shared_plan(a, blockIdx.x, units, (units + 3) / 4, plan);
  SharedItem e = plan.item;
  __syncthreads();  // (the tiles take its place)
  // the same for every lane: page resources and table reads stay scalar
  static_assert(sizeof(SharedItem) % sizeof(int) == 0, "");
#pragma unroll
  for (int i = 0; i < (int)(sizeof(SharedItem) / sizeof(int)); ++i)
    reinterpret_cast<int*>(&e)[i] = __builtin_amdgcn_readfirstlane(reinterpret_cast<int*>(&e)[i]);
  if (!e.kind) return;
  if (e.kind == 1) {
    shared_prefix<T>(a, e, __builtin_amdgcn_readfirstlane(own), k_lds0, v_lds0, k_lds1, v_lds1,
                     sc_lds0, sc_lds1);
    return;
  }
  const int wave = threadIdx.x >> 6;
  const int unit = own * 4 + wave;
  if (unit >= units) return;
  uint8_t* tile = wave == 0 ? k_lds0 : wave == 1 ? v_lds0 : wave == 2 ? k_lds1 : v_lds1;
  float* scales = wave < 2 ? sc_lds0[wave] : sc_lds1[wave - 2];
  shared_tail<T>(a, e, unit, *reinterpret_cast<WalkTiles<false>*>(tile),
                 *reinterpret_cast<WalkScales*>(scales));
}

// out = the merge of a row's partials, one wave a row.
template <typename T>
__global__ __launch_bounds__(64) void shared_merge_kernel(SharedArgs s) {
  const DecodeArgs& a = s.d;
  const int row = blockIdx.x;
  const int lane = threadIdx.x, j = lane >> 5, i = lane & 31;
  // (boundaries that do not ascend may leave a sequence without an item, and its
  // count unwritten)
  const int n = min(s.counts[row / a.hq], a.splits);
  if (n < 0) return;
  const float* lse = a.part_lse + (int64_t)row * a.splits;
  const float* po = a.part_o + (int64_t)row * a.splits * kHeadDim + 4 * i;
  float m = -INFINITY, den = 0.0f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int base = 0; base < n; base += 2 * kLoopK)
    merge_splits<kLoopK>(m, den, o, lse, po, base + j, 2, n);
  merge_across<true>(m, den, o);
  if (j == 0) write_merged<T>(a.out + (int64_t)row * kHeadDim + 4 * i, den, o);
}

// What a shape's launch is made of.
struct SharedShape {
  int max_prefix, gc, tpr, sa, sb;
  int64_t grid;
};

static SharedShape shared_shape(int batch, int groups, int hq, int hk, int w, int bs,
                                int64_t max_prefix_len) {
  SharedShape s;
  const int group = hq / hk, units = hk * qgroups_of(group), tail_units = (units + 3) / 4;
  const int64_t cap = (int64_t)w * bs;
  s.max_prefix = groups > 0 ? (int)(std::min(cap, max_prefix_len) / kSharedTile * kSharedTile) : 0;
  s.gc = group < 16 ? group : 16;
  s.tpr = 16 / s.gc;
  // Ranges of a prefix: four times as many as run at once where all of the batch
  // shares it (512 sequences of 32 heads: 16 for 8192 tokens, partials of 203 MB
  // where 64 took 609), so that a few sequences' long prefix beside many others
  // is still spread.
  const int64_t rows = (batch + 8 * s.tpr - 1) / (8 * s.tpr);
  const int64_t at_once = std::max(1, kSharedWorkgroups / units);
  s.sa = (int)std::max<int64_t>(1, std::min({(int64_t)s.max_prefix / kSharedTile, at_once,
                                             (int64_t)64, 4 * ((at_once + rows - 1) / rows)}));
  // (many sequences: partials of a few ranges each)
  const int64_t slots = kSharedWorkgroups / tail_units;
  const int64_t most = std::max<int64_t>(1, std::min(slots, 8 * ((slots + batch - 1) / batch)));
  s.sb = (int)std::max<int64_t>(1, std::min(most, cap / (kMinSplitSteps * kStep)));
  // Items of ranges that all run at once, and of each sequence's and group's
  // last range (a group's last 128 rows may be few; a group needs a sequence)
  const int64_t blocks =
      s.max_prefix == 0 ? 0 : std::min<int64_t>(batch, batch / (8 * s.tpr) + groups);
  const int64_t least =
      std::min<int64_t>(blocks * s.sa * units, blocks * units + kSharedWorkgroups) +
      std::min<int64_t>((int64_t)batch * s.sb * tail_units,
                        (int64_t)batch * tail_units + kSharedWorkgroups);
  s.grid = std::min<int64_t>(least, (blocks * units + (int64_t)batch * tail_units) +
                                        kSharedWorkgroups + units + tail_units);
  return s;
}

static size_t shared_bytes(int batch, int hq, const SharedShape& s) {
  return partials_bytes(batch, hq, s.sa + s.sb) + (size_t)batch * sizeof(int);
}

template <typename T>
static hipError_t launch_shared(const SharedArgs& a, const SharedShape& s, hipStream_t st) {
  hipLaunchKernelGGL(shared_decode_kernel<T>, dim3((unsigned)s.grid), dim3(kSharedThreads), 0, st,
                     a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(shared_merge_kernel<T>, dim3((unsigned)(a.d.batch * a.d.hq)), dim3(64), 0, st,
                     a);
  return hipGetLastError();
}

}  // namespace mskv

extern "C" size_t mskv_shared_decode_workspace_bytes(int batch, int num_groups, int num_q_heads,
                                                     int num_kv_heads, int block_size,
                                                     int max_blocks_per_seq,
                                                     int64_t max_prefix_len) {
  using namespace mskv;
  if (batch <= 0 || num_groups < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || block_size <= 0 ||
      num_q_heads % num_kv_heads != 0 || max_blocks_per_seq <= 0 || max_prefix_len < 0)
    return 0;
  return shared_bytes(batch, num_q_heads,
                      shared_shape(batch, num_groups, num_q_heads, num_kv_heads,
                                   max_blocks_per_seq, block_size, max_prefix_len));
}

extern "C" int mskv_fp8_shared_prefix_decode_attention(
    const void* query, const void* k_cache, const void* v_cache, const float* k_scale_cache,
    const float* v_scale_cache, const int32_t* cache_seqlens, const int32_t* block_tables,
    const int32_t* cu_groups, const int32_t* prefix_lens, int64_t max_prefix_len, void* out,
    int batch, int num_groups, int num_q_heads, int num_kv_heads, int head_dim, int block_size,
    int64_t num_blocks, int max_blocks_per_seq, float softmax_scale, int act_dtype,
    void* workspace, size_t workspace_bytes, void* stream) {
  using namespace mskv;
  if (batch < 0 || num_groups < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || block_size <= 0 ||
      num_blocks < 0 || max_blocks_per_seq <= 0 || max_prefix_len < 0)
    return MSKV_EINVAL;
  if (act_dtype != MSKV_FLOAT16 && act_dtype != MSKV_BFLOAT16) return MSKV_EINVAL;
  if (num_q_heads % num_kv_heads != 0) return MSKV_EINVAL;
  if (head_dim != kHeadDim || block_size % kSharedTile != 0) return MSKV_EUNSUPPORTED;
  if ((int64_t)block_size * num_kv_heads * head_dim > 0x7FFFFFFFLL) return MSKV_EUNSUPPORTED;
  if ((int64_t)max_blocks_per_seq * block_size >= (1LL << 30)) return MSKV_EUNSUPPORTED;
  // (sums over the batch of 32-token steps, and the merge's grid, stay within
  // an int)
  if (num_groups > kSharedMaxGroups || batch > 65535 || num_kv_heads > 1024 ||
      (int64_t)batch * num_q_heads > 0x7FFFFFFF / 64 ||
      (int64_t)batch * max_blocks_per_seq * block_size / kStep > 0x3FFFFFFF)
    return MSKV_EUNSUPPORTED;
  if (batch == 0) return MSKV_OK;
  if (!query || !k_cache || !v_cache || !k_scale_cache || !v_scale_cache || !cache_seqlens ||
      !block_tables || !out || (num_groups > 0 && (!cu_groups || !prefix_lens)))
    return MSKV_EINVAL;
  if (misaligned({query, k_cache, v_cache, out, workspace}) ||
      (((uintptr_t)k_scale_cache | (uintptr_t)v_scale_cache) & 3))
    return MSKV_EINVAL;
  const SharedShape s = shared_shape(batch, num_groups, num_q_heads, num_kv_heads,
                                     max_blocks_per_seq, block_size, max_prefix_len);
  if (s.grid > 0x3FFFFF) return MSKV_EUNSUPPORTED;  // (a grid's threads fit 32 bits)
  if (!workspace || workspace_bytes < shared_bytes(batch, num_q_heads, s)) return MSKV_EWORKSPACE;
  SharedArgs a = {};
  a.d.q = (const uint16_t*)query;
  a.d.kc = (const uint8_t*)k_cache;
  a.d.vc = (const uint8_t*)v_cache;
  a.d.ks = k_scale_cache;
  a.d.vs = v_scale_cache;
  a.d.seqlens = cache_seqlens;
  a.d.bt = block_tables;
  a.d.out = (uint16_t*)out;
  a.d.splits = s.sa + s.sb;
  a.d.part_o = (float*)workspace;
  a.d.part_lse = a.d.part_o + (size_t)batch * num_q_heads * a.d.splits * kHeadDim;
  a.d.batch = batch;
  a.d.hq = num_q_heads;
  a.d.hk = num_kv_heads;
  a.d.group = num_q_heads / num_kv_heads;
  a.d.qgroups = qgroups_of(a.d.group);
  a.d.bs = block_size;
  a.d.w = max_blocks_per_seq;
  a.d.num_blocks = num_blocks;
  a.d.scale_log2 = softmax_scale * kLog2e;
  a.counts = (int*)((uint8_t*)workspace + partials_bytes(batch, num_q_heads, a.d.splits));
  a.cu_groups = cu_groups;
  a.prefix_lens = prefix_lens;
  a.groups = num_groups;
  a.max_prefix = s.max_prefix;
  a.gc = s.gc;
  a.tpr = s.tpr;
  a.sa = s.sa;
  a.sb = s.sb;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return (int)(act_dtype == MSKV_BFLOAT16 ? launch_shared<__bf16>(a, s, st)
                                          : launch_shared<_Float16>(a, s, st));
}
