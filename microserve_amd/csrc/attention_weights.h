// The attention weight of each cached token: sums of softmax probabilities over
// the queries that read its kv head, added to a tensor [num_blocks, H, BS] that
// lies beside the caches (fp32, a head's tokens of a page in a row).
//
//  * A decode that tracks its weights (track_weights_kernel): the split kernel
//    leaves each score in memory, 4 bytes a (q head, token), and the splits'
//    log-sum-exps; this kernel adds 2^(score - lse) over a kv head's q heads.
//    HBM-bound: the scores are 8 bytes a q head and token (written and read
//    once), 32 at a group of four, where reading K again for them is 132.  64 x
//    4096 tokens of 32 heads: 50 MB, 14 us.
//  * The last queries of prompts (window_lse_kernel, window_sum_kernel): many
//    rows a kv head, whose scores would be more bytes than K.  The scores are
//    computed twice, first for each row's log-sum-exp, then for the sums.  32
//    queries over 32768 tokens at 32 heads over 8 (8.6 GFLOP a pass): 37 us in all;
//    under the profiler, which times a kernel from its dispatch, 20 each.  A
//    workgroup's two tiles take 4 us each, issue-bound (a SIMD issues vector
//    instructions 20 k cycles of about 40 k and multiplies 8 k; waves wait 30% of
//    theirs for memory, 30 to 35% for the issue slot); 6 to 7 us go by before, in the
//    chain of lengths, table, rows and first tile (17 MB at once), and 3 between the
//    launches.  8 x 20 to 8192 tokens, 64 queries: 33 us.
#pragma once

namespace mskv {

struct TrackArgs {
  DecodeArgs d;
  float* weights;
  const int32_t* starts;
  int start;
  int merge_blocks, turns;
};

// The log-sum-exp of a row from those of its first n splits (+inf for a row
// without tokens: 2^(score - lse) is then 0).
__device__ __forceinline__ float merged_lse(const float* lse, int n, int lane) {
  float m = -INFINITY;
  for (int i = lane; i < n; i += 64) m = fmaxf(m, lse[i]);
  m = max_xor32(max_xor16(max16_dpp(m)));
  if (m == -INFINITY) return INFINITY;
  float l = 0.0f;
  for (int i = lane; i < n; i += 64) l += exp2_fast(lse[i] - m);
#pragma unroll
  for (int d = 1; d < 16; d *= 2) l += __shfl_xor(l, d);
  l = sum_xor32(sum_xor16(l));
  return m + __log2f(l);
}

constexpr int kTrackThreads = 256;
constexpr int kTrackTokens = 4 * kTrackThreads;  // of a workgroup's turn
constexpr int kTrackFew = 8;                     // splits that are loaded all at once

// One grid: workgroups that merge the splits of four rows each (merge_blocks of
// them; the decode's own merges, to the same bits), then the weights' ones, (sequence, kv
// head, turn of its tokens) with the turns varying fastest.  A page is whole
// steps of 32 tokens, so a thread's four lie in one page.
template <typename T, bool kRule>
__global__ __launch_bounds__(kTrackThreads) void track_weights_kernel(TrackArgs t) {
  const DecodeArgs& a = t.d;
  extern __shared__ float s_lse[];  // of the group's heads
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int own = kRule ? lane_length(a.seqlens, a.rule) : 0;
  auto valid_splits = [&](int L) {
    const int split_tokens =
        kRule ? split_tokens_of<kStep>(own, L, a.seqlens, a.rule) : a.rule.fixed;
    return L <= 0 ? 0 : min(a.splits, (L + split_tokens - 1) / split_tokens);
  };
  if ((int)blockIdx.x < t.merge_blocks) {
    const int row = blockIdx.x * (kTrackThreads / 64) + wave;
    if (row >= a.batch * a.hq) return;
    const float* lse = a.part_lse + (int64_t)row * a.splits;
    const float* po = a.part_o + (int64_t)row * a.splits * kHeadDim;
    const int len = min(a.seqlens[row / a.hq], a.w * a.bs);
    if (a.splits <= kTrackFew) {  // in order, as decode_combine_small_kernel
      float ls[kTrackFew];
      float2 pv[kTrackFew];
#pragma unroll
      for (int i = 0; i < kTrackFew; ++i) {
        const int at = min(i, a.splits - 1);
        ls[i] = lse[at];
        pv[i] = *reinterpret_cast<const float2*>(po + (int64_t)at * kHeadDim + 2 * lane);
      }
      const int nvalid = valid_splits(len);
      if (nvalid == 1) return;  // written by the split kernel
      float top = -INFINITY, o0 = 0.0f, o1 = 0.0f, den = 0.0f;
#pragma unroll
      for (int i = 0; i < kTrackFew; ++i)
        if (i < nvalid) top = fmaxf(top, ls[i]);
#pragma unroll
      for (int i = 0; i < kTrackFew; ++i) {
        if (i < nvalid && top != -INFINITY) {
          const float p = exp2_fast(ls[i] - top);
          o0 += p * pv[i].x;
          o1 += p * pv[i].y;
          den += p;
        }
      }
      const float inv = den > 0.0f ? 1.0f / den : 0.0f;
      *reinterpret_cast<uint32_t*>(a.out + (int64_t)row * kHeadDim + 2 * lane) =
          (uint32_t)Act<T>::from_f32(o0 * inv) | ((uint32_t)Act<T>::from_f32(o1 * inv) << 16);
      return;
    }
    const int nvalid = valid_splits(len);
    if (nvalid == 1) return;  // written by the split kernel
    const int j = lane >> 5, i = lane & 31;
    po += 4 * i;
    float m = -INFINITY, den = 0.0f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int base = 0; base < nvalid; base += 2 * kLoopK)
      merge_splits<kLoopK>(m, den, o, lse, po, base + j, 2, nvalid);
    merge_across<true>(m, den, o);
    if (j == 0) write_merged<T>(a.out + (int64_t)row * kHeadDim + 4 * i, den, o);
    return;
  }
  const int at0 = blockIdx.x - t.merge_blocks;
  const int turn = at0 % t.turns, pair = at0 / t.turns;
  const int b = pair / a.hk, kvh = pair - b * a.hk;
  const int L = min(a.seqlens[b], a.w * a.bs);
  if (turn * kTrackTokens >= L) return;
  const int nvalid = valid_splits(L);
  const int64_t row0 = (int64_t)b * a.hq + kvh * a.group;
  for (int h = wave; h < a.group; h += kTrackThreads / 64) {
    const float lse = merged_lse(a.part_lse + (row0 + h) * a.splits, nvalid, lane);
    if (lane == 0) s_lse[h] = lse;
  }
  __syncthreads();
  const int64_t cap = score_stride(a.w, a.bs);
  const int first = max(t.starts ? t.starts[b] : t.start, 0);
  for (int at = turn * kTrackTokens; at < L; at += t.turns * kTrackTokens) {
    const int tok = at + 4 * threadIdx.x;
    if (tok >= L || tok + 4 <= first) continue;
    const int page = tok / a.bs;
    const int blk = a.bt[(int64_t)b * a.w + page];
    if (blk < 0 || (int64_t)blk >= a.num_blocks) continue;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    const float* s = a.scores + row0 * cap + tok;
    for (int h = 0; h < a.group; ++h) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(s + h * cap);
#pragma unroll
      for (int r = 0; r < 4; ++r) sum[r] += exp2_fast(x[r] - s_lse[h]);
    }
    float* to = t.weights + ((int64_t)blk * a.hk + kvh) * a.bs + (tok - page * a.bs);
    if (tok >= first && tok + 4 < L) {
      *reinterpret_cast<f32x4*>(to) += sum;
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (tok + r >= first && tok + r < L)  // the newest token's entry starts here
          to[r] = tok + r < L - 1 ? to[r] + sum[r] : sum[r];
    }
  }
}

// ------------------------------------------------------- windows of queries --

struct WindowArgs {
  const uint16_t* q;
  const uint8_t* kc;
  const float* ks;
  const int32_t *bt, *cu_q, *cu_k;  // cu_q null: one query a sequence, lengths in cu_k
  const int32_t* starts;
  float *weights, *part, *lse;
  int* per;  // tiles of a range of window_lse_kernel, for the merge
  int64_t total_q, num_blocks;
  float scale_log2;
  int num_seqs, hq, hk, group, bs, w, start, ranges, rows;
  int most_keys;  // of a sequence: the table's width or the caller's bound
  int parts;      // most ranges of a sequence in window_lse_kernel
  Divider by_group;
  bool add, set_new;
};

constexpr int kWinThreads = 256;
constexpr int kWinTile = 256;  // keys of a workgroup's turn, 64 a wave
constexpr int kWinRows = 128;  // (query, q head of the group) rows of a turn
// Workgroups that should run at once, two a CU
constexpr int kWinSlots = 512;

// A sequence's queries and keys, clamped to the tensors.  What query 0 sees of
// the past, lk - lq, follows the whole length: keys past the table or the bound
// are not counted, but the queries stay where they are.  (Without cu_q the
// length is the table's at most, as the decode takes it.)
struct WindowSeq {
  int q_begin, lq, lk, rows, past;
};
__device__ __forceinline__ int window_length(const WindowArgs& a, int s) {
  return a.cu_q ? a.cu_k[s + 1] - a.cu_k[s] : min(a.cu_k[s], a.w * a.bs);
}
__device__ __forceinline__ int window_keys_of(const WindowArgs& a, int s) {
  return max(0, min(window_length(a, s), a.most_keys));
}
__device__ __forceinline__ WindowSeq window_seq(const WindowArgs& a, int s) {
  WindowSeq w;
  const int64_t tq = a.total_q;
  if (a.cu_q) {
    w.q_begin = (int)min((int64_t)max(a.cu_q[s], 0), tq);
    w.lq = (int)min((int64_t)max(a.cu_q[s + 1], w.q_begin), tq) - w.q_begin;
  } else {
    w.q_begin = s;
    w.lq = 1;
  }
  const int length = window_length(a, s);
  w.lk = max(0, min(length, a.most_keys));
  w.past = length - w.lq;
  w.rows = (int)min((int64_t)w.lq * a.group, (int64_t)a.rows);
  return w;
}

// The workgroup's range of keys: the sequences' tiles are spread over the
// workgroups that run at once, from the lengths (`units` workgroups take a range:
// kv heads, turns of rows), and the ranges with keys come first in the grid.
// (By sequence and chunk, with a grid as wide as the longest one, workgroups
// without keys left the others on a fraction of the CUs: 8 sequences of 20 to
// 8192 tokens took 63 us where eight of 8192 took 75.)
struct WindowRange {
  int s, index, per;  // the sequence (-1: none), its range, tiles of a range
};
__device__ __forceinline__ WindowRange window_range(const WindowArgs& a, int item, int units) {
  const int lane = threadIdx.x & 63;
  auto tiles_of = [&](int s) {
    return s < a.num_seqs ? (window_keys_of(a, s) + kWinTile - 1) / kWinTile : 0;
  };
  const int own = tiles_of(lane);
  int total = own;  // (the host keeps the sum within an int)
  for (int s = 64 + lane; s < a.num_seqs; s += 64) total += tiles_of(s);
  const int tiles = __builtin_amdgcn_readfirstlane(wave_sum_i32(total));
  WindowRange r = {-1, 0, 0};
  // (no more than the longest sequence may have: a range's tokens stay an int)
  r.per = max(1, (int)min(((int64_t)tiles * units + kWinSlots - 1) / kWinSlots,
                          (int64_t)a.ranges));
  for (int base = 0; base < a.num_seqs; base += 64) {
    const int n = ((base == 0 ? own : tiles_of(base + lane)) + r.per - 1) / r.per;
    const int upto = wave_scan_i32(n);
    const uint64_t hit = __ballot(item < upto);
    if (hit) {
      const int at = __ffsll((unsigned long long)hit) - 1;
      r.s = base + at;
      r.index = item - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(n, at));
      return r;
    }
    item -= __builtin_amdgcn_readlane(upto, 63);
  }
  return r;
}

// The wave's 64 keys from t0 on (16 kg + n of lane (g, n)) in the decode's order
// of dimensions: [16g, 16g + 16) and [64 + 16g, 64 + 16g + 16).  Zeros past the
// sequence's end and for an invalid page.
struct WindowLoads {
  u32x4 lo[4], hi[4];
  float scale;  // of key `lane`
  int valid;
};
__device__ __forceinline__ void window_load(const WindowArgs& a, int s, int kvh, int t0, int lk,
                                            int lane, WindowLoads& x) {
  const int g = lane >> 4, n = lane & 15;
  const int page = t0 / a.bs, off = t0 - page * a.bs;
  typedef const __attribute__((address_space(4))) int32_t* Table;  // (stays scalar)
  const int blk =
      t0 < lk ? ((Table)reinterpret_cast<uintptr_t>(a.bt))[(int64_t)s * a.w + page] : -1;
  const bool ok = blk >= 0 && (int64_t)blk < a.num_blocks;
  const int64_t bo = ok ? blk : 0;
  x.valid = ok ? min(64, lk - t0) : 0;
  const uint32_t stride = (uint32_t)a.hk * kHeadDim;
  const auto kr =
      make_rsrc(a.kc + bo * a.bs * stride, ok ? (uint32_t)(off + x.valid) * stride : 0u);
  const auto sr =
      make_rsrc(a.ks + bo * a.bs * a.hk, ok ? (uint32_t)(off + x.valid) * a.hk * 4u : 0u);
#pragma unroll
  for (int kg = 0; kg < 4; ++kg) {
    const uint32_t o = (uint32_t)(off + 16 * kg + n) * stride + (uint32_t)kvh * kHeadDim + 16u * g;
    x.lo[kg] = buf_load16(kr, o);
    x.hi[kg] = buf_load16(kr, o + 64u);
  }
  x.scale = buf_load_f32(sr, (((uint32_t)off + lane) * a.hk + kvh) * 4u);
}
template <typename T>
__device__ __forceinline__ void window_operand(const WindowLoads& x,
                                               typename Act<T>::x8 (&kop)[4][4]) {
  using A = Act<T>;
#pragma unroll
  for (int kg = 0; kg < 4; ++kg) {
    A::fp8x4_to(x.lo[kg][0], kop[kg][0], 0); A::fp8x4_to(x.lo[kg][1], kop[kg][0], 4);
    A::fp8x4_to(x.lo[kg][2], kop[kg][1], 0); A::fp8x4_to(x.lo[kg][3], kop[kg][1], 4);
    A::fp8x4_to(x.hi[kg][0], kop[kg][2], 0); A::fp8x4_to(x.hi[kg][1], kop[kg][2], 4);
    A::fp8x4_to(x.hi[kg][2], kop[kg][3], 0); A::fp8x4_to(x.hi[kg][3], kop[kg][3], 4);
  }
}

// 128 rows of a kv head from row0 on, on their way into LDS: all the loads
// before the first wait (row by row, each load waited for before the next, the
// two kernels took 22 and 31 us, together 20 and 26).  In LDS rows of 256 bytes, 16-byte chunks
// XOR-swizzled by the row, zeros past the last one; and each row's number of
// visible keys.
struct WindowRows {
  static constexpr int kEach = kWinRows * 16 / kWinThreads;
  u32x4 v[kEach];
  int lim[kEach];
  __device__ __forceinline__ void load(const WindowArgs& a, const WindowSeq& w, int kvh, int row0) {
    const int c = threadIdx.x & 15;
    const uint16_t* q = a.q + ((int64_t)w.q_begin * a.hq + kvh * a.group) * kHeadDim + 8 * c;
#pragma unroll
    for (int i = 0; i < kEach; ++i) v[i] = u32x4{0u, 0u, 0u, 0u}, lim[i] = 0;
    if (row0 >= w.rows) return;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int row = min(row0 + ((i * kWinThreads + (int)threadIdx.x) >> 4), w.rows - 1);
      const int qi = a.by_group(row);
      v[i] = *reinterpret_cast<const u32x4*>(
          q + (row + (int64_t)qi * (a.hq - a.group)) * kHeadDim);
      lim[i] = w.past + qi + 1;
    }
  }
  __device__ __forceinline__ void store(const WindowSeq& w, int row0, uint8_t* q_lds,
                                        int* s_lim) const {
    const int c = threadIdx.x & 15;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int r = (i * kWinThreads + threadIdx.x) >> 4;
      const bool ok = row0 + r < w.rows;
      *reinterpret_cast<u32x4*>(q_lds + r * 256 + 16 * (c ^ (r & 15))) =
          ok ? v[i] : u32x4{0u, 0u, 0u, 0u};
      if (c == 0) s_lim[r] = ok ? lim[i] : 0;
    }
  }
};
template <typename T>
__device__ __forceinline__ void window_query(const uint8_t* q_lds, int rb, int lane,
                                             typename Act<T>::x8 (&qop)[4]) {
  const int g = lane >> 4, n = lane & 15;
  const uint8_t* row = q_lds + (16 * rb + n) * 256;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c = (j & 2) * 4 + 2 * g + (j & 1);
    qop[j] = __builtin_bit_cast(typename Act<T>::x8,
                                *reinterpret_cast<const u32x4*>(row + 16 * (c ^ n)));
  }
}

// A row's place in the partials: a kv head's rows side by side, so that they are
// read 64 at a time.
__device__ __forceinline__ int64_t window_row(const WindowArgs& a, const WindowSeq& w, int kvh,
                                              int row) {
  return ((int64_t)kvh * a.total_q + w.q_begin) * a.group + row;
}

// The log-sum-exp of each of 128 rows over the workgroup's range of keys.
// S^T = K . Q^T: a lane holds 16 keys of one row, for which it keeps a running
// maximum and sum of its own; they meet at the end.
// grid: ranges x (kv heads x turns of rows)
template <typename T>
__global__ __launch_bounds__(kWinThreads, 2) void window_lse_kernel(WindowArgs a, int units) {
  using A = Act<T>;
  constexpr int kBlocks = kWinRows / 16;
  __shared__ __attribute__((aligned(16))) uint8_t q_lds[kWinRows * 256];
  __shared__ __attribute__((aligned(16))) float s_scale[4][64];
  __shared__ int s_lim[kWinRows];
  __shared__ float s_m[4][kWinRows], s_l[4][kWinRows];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, n = lane & 15;
  const int unit = blockIdx.x % units;
  const WindowRange range = window_range(a, blockIdx.x / units, units);
  if (blockIdx.x == 0 && tid == 0) *a.per = range.per;
  if (range.s < 0) return;
  const int s = range.s, kvh = unit % a.hk, row0 = unit / a.hk * kWinRows;
  const WindowSeq w = window_seq(a, s);
  if (row0 >= w.rows) return;
  const int first = range.index * range.per * kWinTile;
  const int end = min(w.lk, first + range.per * kWinTile);
  WindowRows q;
  q.load(a, w, kvh, row0);
  WindowLoads next;
  window_load(a, s, kvh, first + 64 * wave, w.lk, lane, next);
  q.store(w, row0, q_lds, s_lim);
  __syncthreads();
  const int blocks = (min(kWinRows, w.rows - row0) + 15) / 16;
  int index = range.index;
  asm("" : "+v"(index));  // (kept in a vector register: the scalar ones are short)
  float m[kBlocks], l[kBlocks];
#pragma unroll
  for (int rb = 0; rb < kBlocks; ++rb) m[rb] = -INFINITY, l[rb] = 0.0f;
  for (int t0 = first; t0 < end; t0 += kWinTile) {
    const int k0 = t0 + 64 * wave;
    typename A::x8 kop[4][4];
    window_operand<T>(next, kop);
    const int valid = next.valid;
    s_scale[wave][lane] = next.scale * a.scale_log2;
    wave_lds_sync();
    f32x4 ksc[4];
#pragma unroll
    for (int kg = 0; kg < 4; ++kg)
      ksc[kg] = *reinterpret_cast<const f32x4*>(&s_scale[wave][16 * kg + 4 * g]);
    if (t0 + kWinTile < end) window_load(a, s, kvh, k0 + kWinTile, w.lk, lane, next);
    if (valid > 0) {
      const bool all = valid == 64 && k0 + 64 <= w.past + 1;  // every row sees every key
#pragma unroll
      for (int rb = 0; rb < kBlocks; ++rb) {
        if (rb < blocks) {
          typename A::x8 qop[4];
          window_query<T>(q_lds, rb, lane, qop);
          f32x4 x[4];
#pragma unroll
          for (int kg = 0; kg < 4; ++kg) x[kg] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int kg = 0; kg < 4; ++kg) x[kg] = A::mfma(kop[kg][j], qop[j], x[kg]);
#pragma unroll
          for (int kg = 0; kg < 4; ++kg) x[kg] *= ksc[kg];
          if (!all) {
            const int lim = min(s_lim[16 * rb + n] - k0, valid);
#pragma unroll
            for (int kg = 0; kg < 4; ++kg)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (!(16 * kg + 4 * g + r < lim)) x[kg][r] = -INFINITY;
          }
          float top = m[rb];
#pragma unroll
          for (int kg = 0; kg < 4; ++kg)
            top = fmaxf(fmaxf(top, fmaxf(x[kg][0], x[kg][1])), fmaxf(x[kg][2], x[kg][3]));
          const float ref = top == -INFINITY ? 0.0f : top;
          float sum = 0.0f;
#pragma unroll
          for (int kg = 0; kg < 4; ++kg)
#pragma unroll
            for (int r = 0; r < 4; ++r) sum += exp2_fast(x[kg][r] - ref);
          l[rb] = l[rb] * exp2_fast(m[rb] - ref) + sum;
          m[rb] = top;
        }
      }
    }
    wave_lds_sync();  // (the scales are read before the next ones are written)
  }
#pragma unroll
  for (int rb = 0; rb < kBlocks; ++rb) {
    const float top = max_xor32(max_xor16(m[rb]));
    const float ref = top == -INFINITY ? 0.0f : top;
    const float sum = sum_xor32(sum_xor16(l[rb] * exp2_fast(m[rb] - ref)));
    if (g == 0) {
      s_m[wave][16 * rb + n] = top;
      s_l[wave][16 * rb + n] = sum;
    }
  }
  __syncthreads();
  if (tid >= kWinRows || row0 + tid >= w.rows) return;
  float top = s_m[0][tid];
#pragma unroll
  for (int i = 1; i < 4; ++i) top = fmaxf(top, s_m[i][tid]);
  const float ref = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) sum += s_l[i][tid] * exp2_fast(s_m[i][tid] - ref);
  a.part[index * (a.total_q * a.hq) + window_row(a, w, kvh, row0 + tid)] =
      partial_lse(top, sum);
}

// A row's log-sum-exp from the ranges that hold keys, by kThreads neighbouring
// lanes; +inf where no key is seen.
template <int kThreads>
__device__ __forceinline__ float window_row_lse(const WindowArgs& a, const WindowSeq& w, int64_t at,
                                                int lane) {
  constexpr int kBatch = 16;  // loads in flight a lane
  const int64_t stride = a.total_q * a.hq;
  const int keys = *a.per * kWinTile;
  const int n = min(a.parts, (w.lk + keys - 1) / keys);
  float m = -INFINITY, l = 0.0f;
  const float* p = a.part + at + min(lane, max(n - 1, 0)) * stride;
  for (int base = lane; base < n; base += kBatch * kThreads) {
    float x[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      x[i] = *p;
      p += base + (i + 1) * kThreads < n ? kThreads * stride : 0;
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      x[i] = base + i * kThreads < n ? x[i] : -INFINITY;
      top = fmaxf(top, x[i]);
    }
    const float ref = top == -INFINITY ? 0.0f : top;
    l *= exp2_fast(m - ref);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) l += exp2_fast(x[i] - ref);
    m = top;
  }
#pragma unroll
  for (int d = 1; d < kThreads; d *= 2) {
    const float mo = __shfl_xor(m, d), lo = __shfl_xor(l, d);
    const float top = fmaxf(m, mo), ref = top == -INFINITY ? 0.0f : top;
    l = l * exp2_fast(m - ref) + lo * exp2_fast(mo - ref);
    m = top;
  }
  return m == -INFINITY ? INFINITY : m + __log2f(l);
}

// lse[row], where a sequence has more rows than window_sum_kernel holds at once:
// grid (rows of a kv head / 256 x kv heads, sequences)
__global__ __launch_bounds__(kWinThreads) void window_merge_kernel(WindowArgs a) {
  const WindowSeq w = window_seq(a, blockIdx.y);
  const int kvh = blockIdx.x % a.hk, row = blockIdx.x / a.hk * kWinThreads + threadIdx.x;
  if (w.rows <= 2 * kWinRows || row >= w.rows || w.lk == 0) return;
  const int64_t at = window_row(a, w, kvh, row);
  a.lse[at] = window_row_lse<1>(a, w, at, 0);
}

// The sums over the rows of 2^(score - lse) at the workgroup's range of keys.
// S = Q . K^T: a lane holds four rows of one key, whose sum needs no exchange
// until all the rows are in.  grid: ranges x kv heads.  kRows: rows in LDS at
// once; more of them are staged again for every tile.
template <typename T, int kRows>
__global__ __launch_bounds__(kWinThreads, 2) void window_sum_kernel(WindowArgs a) {
  using A = Act<T>;
  __shared__ __attribute__((aligned(16))) uint8_t q_lds[kRows * 256];
  __shared__ __attribute__((aligned(16))) int s_lim[kRows];
  __shared__ __attribute__((aligned(16))) float s_lse[kRows];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, n = lane & 15;
  const int kvh = blockIdx.x % a.hk;
  const WindowRange range = window_range(a, blockIdx.x / a.hk, a.hk);
  if (range.s < 0) return;
  const int s = range.s;
  const WindowSeq w = window_seq(a, s);
  const int from = max(a.starts ? a.starts[s] : a.start, 0);
  WindowRows q;
  auto rows = [&](int row0) {  // into LDS (the first 128 are in q), with their log-sum-exps
    if (w.rows > kRows) {
      const int row = row0 + tid;
      if (tid < kRows) s_lse[tid] = row < w.rows ? a.lse[window_row(a, w, kvh, row)] : INFINITY;
    } else {
      constexpr int kOf = kWinThreads / kRows;
      const int row = tid / kOf;
      const float lse = row < w.rows
          ? window_row_lse<kOf>(a, w, window_row(a, w, kvh, row), tid % kOf) : INFINITY;
      if (tid % kOf == 0) s_lse[row] = lse;
    }
    q.store(w, row0, q_lds, s_lim);
#pragma unroll
    for (int more = kWinRows; more < kRows; more += kWinRows) {
      q.load(a, w, kvh, row0 + more);
      q.store(w, row0 + more, q_lds + 256 * more, s_lim + more);
    }
  };
  const int first = range.index * range.per * kWinTile;
  const int end = min(w.lk, first + range.per * kWinTile);
  q.load(a, w, kvh, 0);
  WindowLoads next;
  window_load(a, s, kvh, first + 64 * wave, w.lk, lane, next);
  rows(0);
  __syncthreads();
  for (int t0 = first; t0 < end; t0 += kWinTile) {
    const int k0 = t0 + 64 * wave;
    typename A::x8 kop[4][4];
    window_operand<T>(next, kop);
    const int valid = next.valid;
    float ksc[4], sum[4];
#pragma unroll
    for (int kg = 0; kg < 4; ++kg) {
      ksc[kg] = __shfl(next.scale, 16 * kg + n) * a.scale_log2;
      sum[kg] = 0.0f;
    }
    if (t0 + kWinTile < end) window_load(a, s, kvh, k0 + kWinTile, w.lk, lane, next);
    const bool all = valid == 64 && k0 + 64 <= w.past + 1;  // every row sees every key
    for (int row0 = 0; row0 < w.rows; row0 += kRows) {
      if (w.rows > kRows && (row0 > 0 || t0 > first)) {
        q.load(a, w, kvh, row0);
        __syncthreads();
        rows(row0);
        __syncthreads();
      }
      if (valid == 0) continue;
      const int blocks = (min(kRows, w.rows - row0) + 15) / 16;
      auto add_block = [&](int rb, bool masked) {
        typename A::x8 qop[4];
        window_query<T>(q_lds, rb, lane, qop);
        const f32x4 lse = *reinterpret_cast<const f32x4*>(&s_lse[16 * rb + 4 * g]);
        f32x4 x[4];
#pragma unroll
        for (int kg = 0; kg < 4; ++kg) x[kg] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int kg = 0; kg < 4; ++kg) x[kg] = A::mfma(qop[j], kop[kg][j], x[kg]);
        // row r sees the keys 16 kg + n with 16 kg < sees[r] (with each limit read and
        // branched on by itself, the workgroup of a sequence's last keys took 20 us of
        // its kernel's 28)
        int sees[4];
        if (masked) {
          const u32x4 lim = *reinterpret_cast<const u32x4*>(&s_lim[16 * rb + 4 * g]);
#pragma unroll
          for (int r = 0; r < 4; ++r) sees[r] = min((int)lim[r] - k0, valid) - n;
        }
#pragma unroll
        for (int kg = 0; kg < 4; ++kg) {
          f32x4 p;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            p[r] = exp2_fast(fmaf(x[kg][r], ksc[kg], -lse[r]));
            if (masked) p[r] = 16 * kg < sees[r] ? p[r] : 0.0f;
          }
          sum[kg] += (p[0] + p[1]) + (p[2] + p[3]);
        }
      };
      if (all) {
#pragma unroll 2
        for (int rb = 0; rb < blocks; ++rb) add_block(rb, false);
      } else {
#pragma unroll 2
        for (int rb = 0; rb < blocks; ++rb) add_block(rb, true);
      }
    }
#pragma unroll
    for (int kg = 0; kg < 4; ++kg) sum[kg] = sum_xor32(sum_xor16(sum[kg]));
    const float own = g == 0 ? sum[0] : g == 1 ? sum[1] : g == 2 ? sum[2] : sum[3];
    const int tok = k0 + lane;  // key 16 g + n of the wave's
    if (lane < valid && tok >= from) {
      const int page = k0 / a.bs;
      float* to = a.weights + ((int64_t)a.bt[(int64_t)s * a.w + page] * a.hk + kvh) * a.bs +
                  (tok - page * a.bs);
      const bool add = a.add && !(a.set_new && tok >= w.past);
      *to = add ? *to + own : own;
    }
  }
}

// [parts, total_q * hq] partial log-sum-exps, [total_q * hq] final ones, then
// the tiles of a range
static size_t window_bytes(int64_t total_q, int hq, int64_t parts) {
  return ((size_t)total_q * hq * (parts + 1) + 1) * sizeof(float);
}

// Turns of rows of a sequence, and the most ranges that window_lse_kernel makes of
// its keys: a range holds at least the batch's tiles times the units over the
// workgroups that run at once (window_range).
static int64_t window_turns(int64_t rows) { return (rows + kWinRows - 1) / kWinRows; }
static int64_t window_parts(int64_t tiles, int64_t rows, int hk) {
  const int64_t units = hk * std::max<int64_t>(1, window_turns(rows));
  return std::min(tiles, (kWinSlots + units - 1) / units);
}

template <typename T>
static hipError_t launch_window(const WindowArgs& a, hipStream_t st) {
  // ranges with keys: at most the workgroups that run at once over `units`, and
  // one more a sequence
  auto grid = [&](int64_t units) {
    const int64_t most = (kWinSlots + units - 1) / units + a.num_seqs;
    return dim3((unsigned)(std::min(most, (int64_t)a.ranges * a.num_seqs) * units));
  };
  if (a.rows > 0) {  // (without queries there are only zeros to write)
    const int units = a.hk * (int)window_turns(a.rows);
    hipLaunchKernelGGL(window_lse_kernel<T>, grid(units), dim3(kWinThreads), 0, st, a, units);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (a.rows > 2 * kWinRows) {
      hipLaunchKernelGGL(window_merge_kernel,
                         dim3((unsigned)((a.rows + kWinThreads - 1) / kWinThreads * a.hk),
                              (unsigned)a.num_seqs),
                         dim3(kWinThreads), 0, st, a);
      e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
  }
  if (a.rows <= kWinRows)
    hipLaunchKernelGGL((window_sum_kernel<T, kWinRows>), grid(a.hk), dim3(kWinThreads), 0, st, a);
  else
    hipLaunchKernelGGL((window_sum_kernel<T, 2 * kWinRows>), grid(a.hk), dim3(kWinThreads), 0, st,
                       a);
  return hipGetLastError();
}

// Keys, and tiles of them, of the longest sequence of a window call.
static int64_t window_keys(int64_t max_seqlen_k, int block_size, int w) {
  const int64_t keys = (int64_t)w * block_size;
  return max_seqlen_k > 0 ? std::min(keys, max_seqlen_k) : keys;
}
static int64_t window_tiles(int64_t max_seqlen_k, int block_size, int w) {
  return (window_keys(max_seqlen_k, block_size, w) + kWinTile - 1) / kWinTile;
}

// Most bytes of scores that a tracking decode asks for; past it K is read again
// instead.
constexpr size_t kTrackMaxScores = (size_t)1 << 30;

}  // namespace mskv

extern "C" size_t mskv_window_weights_workspace_bytes(int64_t total_q, int64_t max_seqlen_k,
                                                      int num_q_heads, int block_size,
                                                      int max_blocks_per_seq) {
  using namespace mskv;
  if (total_q <= 0 || num_q_heads <= 0 || block_size <= 0 || max_blocks_per_seq <= 0) return 0;
  // (of any number of kv heads and queries)
  return window_bytes(total_q, num_q_heads,
                      window_parts(window_tiles(max_seqlen_k, block_size, max_blocks_per_seq), 1,
                                   1));
}

extern "C" size_t mskv_window_weights_bounded_workspace_bytes(
    int64_t total_q, int max_seqlen_q, int64_t max_seqlen_k, int num_q_heads, int num_kv_heads,
    int block_size, int max_blocks_per_seq) {
  using namespace mskv;
  if (total_q <= 0 || max_seqlen_q < 0 || num_q_heads <= 0 || num_kv_heads <= 0 ||
      num_q_heads % num_kv_heads != 0 || block_size <= 0 || max_blocks_per_seq <= 0)
    return 0;
  const int64_t rows = std::min<int64_t>(max_seqlen_q, total_q) * (num_q_heads / num_kv_heads);
  return window_bytes(total_q, num_q_heads,
                      window_parts(window_tiles(max_seqlen_k, block_size, max_blocks_per_seq),
                                   rows, num_kv_heads));
}

namespace mskv {

// (the launches' workgroups, and the sum of the tiles, stay within an int)
static bool window_fits(int num_seqs, int64_t total_q, int64_t rows, int num_kv_heads,
                        int block_size, int max_blocks_per_seq) {
  const int64_t turns = window_turns(rows);
  return num_seqs <= 65535 && total_q <= 0x7FFFFFFFLL && rows <= 0x7FFFFFFFLL &&
         (num_seqs + kWinSlots) * turns * num_kv_heads <= 0x7FFFFF &&
         num_seqs * ((int64_t)max_blocks_per_seq * block_size / kWinTile + 1) <= 0x7FFFFFFF;
}

// Validates a window call and launches it.  Without cu_seqlens_q: one query a
// sequence, its length in cu_seqlens_k, the newest token's entry set.
static int window_checked(
    const void* query, const void* k_cache, const float* k_scale_cache,
    const int32_t* block_tables, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
    float* weights, const int32_t* starts, int start, bool accumulate, int num_seqs,
    int64_t total_q, int max_seqlen_q, int64_t max_seqlen_k, int num_q_heads, int num_kv_heads,
    int head_dim, int block_size, int64_t num_blocks, int max_blocks_per_seq, float softmax_scale,
    int act_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (num_seqs < 0 || total_q < 0 || max_seqlen_q < 0 || num_q_heads <= 0 || num_kv_heads <= 0 ||
      block_size <= 0 || num_blocks < 0 || max_blocks_per_seq <= 0 || start < 0)
    return MSKV_EINVAL;
  if (act_dtype != MSKV_FLOAT16 && act_dtype != MSKV_BFLOAT16) return MSKV_EINVAL;
  if (num_q_heads % num_kv_heads != 0) return MSKV_EINVAL;
  if (head_dim != kHeadDim || block_size % 128 != 0) return MSKV_EUNSUPPORTED;
  if ((int64_t)block_size * num_kv_heads * head_dim > 0x7FFFFFFFLL) return MSKV_EUNSUPPORTED;
  if ((int64_t)max_blocks_per_seq * block_size >= (1LL << 30)) return MSKV_EUNSUPPORTED;
  const int group = num_q_heads / num_kv_heads;
  const int64_t rows = (int64_t)max_seqlen_q * group;
  if (!window_fits(num_seqs, total_q, rows, num_kv_heads, block_size, max_blocks_per_seq))
    return MSKV_EUNSUPPORTED;
  if (num_seqs == 0) return MSKV_OK;
  if (!k_cache || !k_scale_cache || !block_tables || !cu_seqlens_k || !weights)
    return MSKV_EINVAL;
  if (total_q > 0 && !query) return MSKV_EINVAL;
  if (misaligned({query, k_cache})) return MSKV_EINVAL;
  WindowArgs a = {};
  a.ranges = (int)window_tiles(max_seqlen_k, block_size, max_blocks_per_seq);
  a.most_keys = (int)window_keys(max_seqlen_k, block_size, max_blocks_per_seq);
  const size_t need = mskv_window_weights_bounded_workspace_bytes(
      total_q, max_seqlen_q, max_seqlen_k, num_q_heads, num_kv_heads, block_size,
      max_blocks_per_seq);
  if (need > 0 && (!workspace || workspace_bytes < need)) return MSKV_EWORKSPACE;
  a.q = (const uint16_t*)query;
  a.kc = (const uint8_t*)k_cache;
  a.ks = k_scale_cache;
  a.bt = block_tables;
  a.cu_q = cu_seqlens_q;
  a.cu_k = cu_seqlens_k;
  a.starts = starts;
  a.start = start;
  a.weights = weights;
  a.part = (float*)workspace;
  a.rows = total_q > 0 ? (int)std::min<int64_t>(rows, total_q * group) : 0;
  a.parts = (int)window_parts(a.ranges, a.rows, num_kv_heads);
  a.lse = a.part + (size_t)total_q * num_q_heads * a.parts;
  a.per = (int*)(a.lse + (size_t)total_q * num_q_heads);
  a.total_q = total_q;
  a.num_blocks = num_blocks;
  a.scale_log2 = softmax_scale * kLog2e;
  a.num_seqs = num_seqs;
  a.hq = num_q_heads;
  a.hk = num_kv_heads;
  a.group = group;
  a.by_group = divider_of(group);
  a.bs = block_size;
  a.w = max_blocks_per_seq;
  a.add = accumulate;
  a.set_new = cu_seqlens_q == nullptr;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return (int)(act_dtype == MSKV_BFLOAT16 ? launch_window<__bf16>(a, s)
                                          : launch_window<_Float16>(a, s));
}

}  // namespace mskv

extern "C" int mskv_fp8_window_attention_weights(
    const void* query, const void* k_cache, const float* k_scale_cache,
    const int32_t* block_tables, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
    float* weights, const int32_t* starts, int start, int accumulate, int num_seqs,
    int64_t total_q, int max_seqlen_q, int64_t max_seqlen_k, int num_q_heads, int num_kv_heads,
    int head_dim, int block_size, int64_t num_blocks, int max_blocks_per_seq, float softmax_scale,
    int act_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (num_seqs > 0 && !cu_seqlens_q) return MSKV_EINVAL;
  return mskv::window_checked(query, k_cache, k_scale_cache, block_tables, cu_seqlens_q,
                              cu_seqlens_k, weights, starts, start, accumulate != 0, num_seqs,
                              total_q, max_seqlen_q, max_seqlen_k, num_q_heads, num_kv_heads,
                              head_dim, block_size, num_blocks, max_blocks_per_seq, softmax_scale,
                              act_dtype, workspace, workspace_bytes, stream);
}

namespace mskv {

// The entries of stored tokens, 0: thread x takes a token of head y (neighbouring
// tokens' entries of a head lie side by side).
template <typename SlotT>
__global__ __launch_bounds__(kWinThreads) void clear_weights_kernel(
    float* __restrict__ weights, const SlotT* __restrict__ slots, int64_t num_tokens, int hk,
    int bs, int64_t num_slots) {
  const int64_t t = (int64_t)blockIdx.x * kWinThreads + threadIdx.x;
  if (t >= num_tokens) return;
  const int64_t slot = (int64_t)slots[t];
  if (slot < 0 || slot >= num_slots) return;
  const int64_t page = slot / bs;
  weights[(page * hk + blockIdx.y) * bs + (slot - page * bs)] = 0.0f;
}

// Whether a tracking decode of this shape leaves its scores in memory.
static bool track_scores(int batch, int hq, int w, int block_size) {
  return track_scores_bytes(batch, hq, w, block_size) <= kTrackMaxScores;
}

}  // namespace mskv

extern "C" int mskv_clear_attention_weights(float* weights, const void* slot_mapping,
                                            int slot_dtype, int64_t num_tokens, int num_kv_heads,
                                            int block_size, int64_t num_blocks, void* stream) {
  using namespace mskv;
  if (num_tokens < 0 || num_kv_heads <= 0 || block_size <= 0 || num_blocks < 0) return MSKV_EINVAL;
  if (slot_dtype != MSKV_INT32 && slot_dtype != MSKV_INT64) return MSKV_EINVAL;
  if (num_kv_heads > 65535 || num_blocks > 0x7FFFFFFFLL || num_tokens > 0x7FFFFFFFLL)
    return MSKV_EUNSUPPORTED;
  if (num_tokens == 0) return MSKV_OK;
  if (!weights || !slot_mapping) return MSKV_EINVAL;
  const dim3 grid((unsigned)((num_tokens + kWinThreads - 1) / kWinThreads),
                  (unsigned)num_kv_heads);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  auto run = [&](auto* slots) {
    using SlotT = std::remove_const_t<std::remove_pointer_t<decltype(slots)>>;
    hipLaunchKernelGGL(clear_weights_kernel<SlotT>, grid, dim3(kWinThreads), 0, s, weights, slots,
                       num_tokens, num_kv_heads, block_size, num_blocks * block_size);
    return (int)hipGetLastError();
  };
  return slot_dtype == MSKV_INT64 ? run((const int64_t*)slot_mapping)
                                  : run((const int32_t*)slot_mapping);
}

extern "C" size_t mskv_decode_weights_workspace_bytes(int batch, int num_q_heads, int num_kv_heads,
                                                      int block_size, int max_blocks_per_seq) {
  using namespace mskv;
  if (batch <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads != 0 ||
      block_size <= 0 || max_blocks_per_seq <= 0)
    return 0;
  const int splits = mskv_decode_num_splits(batch, num_q_heads, num_kv_heads, max_blocks_per_seq,
                                            block_size);
  if (track_scores(batch, num_q_heads, max_blocks_per_seq, block_size))
    return track_scores_at(batch, num_q_heads, num_kv_heads, splits) +
           track_scores_bytes(batch, num_q_heads, max_blocks_per_seq, block_size);
  // the decode's own workspace, then the window kernels' one
  return std::max(mskv_decode_workspace_bytes(batch, num_q_heads, num_kv_heads, kHeadDim, splits),
                  mskv_window_weights_bounded_workspace_bytes(batch, 1, 0, num_q_heads,
                                                              num_kv_heads, block_size,
                                                              max_blocks_per_seq));
}

extern "C" int mskv_fp8_decode_attention_weights(
    const void* query, const void* k_cache, const void* v_cache, const float* k_scale_cache,
    const float* v_scale_cache, const int32_t* cache_seqlens, const int32_t* block_tables,
    float* weights, const int32_t* starts, int start, void* out, int batch, int num_q_heads,
    int num_kv_heads, int head_dim, int block_size, int64_t num_blocks, int max_blocks_per_seq,
    float softmax_scale, int act_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace mskv;
  if (batch < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || block_size <= 0 ||
      max_blocks_per_seq <= 0 || start < 0 || num_q_heads % num_kv_heads != 0)
    return MSKV_EINVAL;
  if (batch > 65535 || num_q_heads / num_kv_heads > 8192 ||
      (int64_t)batch * num_q_heads > 0x3FFFFFFF / kTrackThreads)
    return MSKV_EUNSUPPORTED;
  if (batch > 0 && (!weights || misaligned({weights}))) return MSKV_EINVAL;
  if (batch > 0 && (!workspace || workspace_bytes < mskv_decode_weights_workspace_bytes(
                                                        batch, num_q_heads, num_kv_heads,
                                                        block_size, max_blocks_per_seq)))
    return MSKV_EWORKSPACE;
  const int splits = mskv_decode_num_splits(batch, num_q_heads, num_kv_heads, max_blocks_per_seq,
                                            block_size);
  if (!track_scores(batch, num_q_heads, max_blocks_per_seq, block_size)) {
    // (before the decode is launched)
    if (block_size % 128 != 0 || !window_fits(batch, batch, num_q_heads / num_kv_heads,
                                              num_kv_heads, block_size, max_blocks_per_seq))
      return MSKV_EUNSUPPORTED;
    const int status = decode_checked<Fp8Cache>(
        query, k_cache, v_cache, k_scale_cache, v_scale_cache, cache_seqlens, block_tables, out,
        batch, num_q_heads, num_kv_heads, head_dim, block_size, num_blocks, max_blocks_per_seq,
        softmax_scale, act_dtype, splits, workspace, workspace_bytes, stream);
    if (status != MSKV_OK || batch == 0) return status;
    return window_checked(query, k_cache, k_scale_cache, block_tables, nullptr, cache_seqlens,
                          weights, starts, start, true, batch, batch, 1, 0, num_q_heads,
                          num_kv_heads, head_dim, block_size, num_blocks, max_blocks_per_seq,
                          softmax_scale, act_dtype, workspace, workspace_bytes, stream);
  }
  auto track = [&](const DecodeArgs& d, hipStream_t s) -> int {
    // (a table's width says little of the lengths: workgroups walk the turns
    // past a grid of 4096)
    const int64_t turns = ((int64_t)d.w * d.bs + kTrackTokens - 1) / kTrackTokens;
    const int64_t most = std::max<int64_t>(1, 4096 / ((int64_t)d.batch * d.hk));
    const bool merge = d.splits > 1 && d.splits <= kWideThreshold;
    const int per = kTrackThreads / 64;
    const TrackArgs t = {d, weights, starts, start,
                         merge ? (int)(((int64_t)d.batch * d.hq + per - 1) / per) : 0,
                         (int)std::min(turns, most)};
    const dim3 grid((unsigned)(t.merge_blocks + (int64_t)t.turns * d.batch * d.hk));
    const unsigned lds = (unsigned)(d.group * sizeof(float));
    auto run = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, grid, dim3(kTrackThreads), lds, s, t);
      return (int)hipGetLastError();
    };
    const bool bf16 = act_dtype == MSKV_BFLOAT16;
    if (d.rule.adapt || d.rule.info)
      return bf16 ? run(track_weights_kernel<__bf16, true>)
                  : run(track_weights_kernel<_Float16, true>);
    return bf16 ? run(track_weights_kernel<__bf16, false>)
                : run(track_weights_kernel<_Float16, false>);
  };
  return decode_checked<TrackedFp8Cache>(
      query, k_cache, v_cache, k_scale_cache, v_scale_cache, cache_seqlens, block_tables, out,
      batch, num_q_heads, num_kv_heads, head_dim, block_size, num_blocks, max_blocks_per_seq,
      softmax_scale, act_dtype, splits, workspace, workspace_bytes, stream, track);
}
