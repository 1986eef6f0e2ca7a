// Eviction from the FP8 paged cache: the tokens of every (sequence, kv head)
// that stay, and the moving of their rows to the front of the sequence's pages.
//
//  * select_kv_tokens_kernel: of L tokens n = min(L, budget) stay: the first
//    `start`, the last `recent`, and the heaviest of those between.  The
//    threshold weight is found by its digits, from the highest (11, 11 and 10
//    bits of an order-preserving integer form of the weight), each by a
//    histogram in LDS; one more pass writes the kept positions in ascending
//    order, of the tokens at the threshold the earliest.  One workgroup a
//    (sequence, kv head), which holds the keys in registers, up to 32 a thread.
//    Latency-bound: three rounds of counts and scans; 64 pairs of 32768 tokens
//    take 21 us (42 by single tokens and one copy of the counts), 512 of 4352 20.
//  * evict_kv_tokens_kernel: place i of a (sequence, kv head) gets the row of
//    position kept[i].  The positions ascend, so kept[i] >= i, and a workgroup
//    that walks the places in order may overwrite what it has read: a run of
//    places is loaded whole, then stored, and no later run reads below its own
//    first place.  HBM-bound, two bytes moved per byte that changes its place: 64
//    sequences of 4096 kept tokens at eight heads, 0.9 GB, take 219 us (4.1 TB/s),
//    8 of them 33.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "mskv_device.h"
#include "../../include/mskv.h"

namespace mskv {

constexpr int kSelectBins = 2048;

struct SelectArgs {
  const float* weights;
  const int32_t *seqlens, *bt, *starts;
  int32_t *kept, *new_lens;
  int64_t num_blocks;
  int hk, bs, w, start, recent, budget;
  Divider by_block;
};

// An integer that orders as the weight does: NaN lowest, -0 as 0.
__device__ __forceinline__ uint32_t weight_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);  // (-0 + 0 is 0)
  const uint32_t key = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
  return x != x ? 0u : key;
}

__device__ __forceinline__ int lanes_below(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                   __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// The sum of v over the threads before this one, and over all.
template <int kWaves>
__device__ __forceinline__ uint32_t scan_before(uint32_t v, uint32_t* s_wave, uint32_t& all) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t x = (uint32_t)wave_scan_i32((int)v);
  if ((threadIdx.x & 63) == 63) s_wave[wave] = x;
  __syncthreads();
  uint32_t before = x - v;
  all = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    const uint32_t t = s_wave[i];
    if (i < wave) before += t;
    all += t;
  }
  __syncthreads();
  return before;
}

// kQuads: runs of four tokens that a thread holds the keys of, thread t's j-th
// run that number j * kThreads + t of the range; kReread: as many at a time, read
// again on every pass.
template <int kThreads, int kQuads, bool kReread>
__global__ __launch_bounds__(kThreads) void select_kv_tokens_kernel(SelectArgs a) {
  constexpr int kWaves = kThreads / 64;
  constexpr int kEntries = kQuads * kWaves;  // waves' counts of a turn
  static_assert(kEntries <= kThreads, "a thread takes one of the counts");
  constexpr int kBinsEach = kSelectBins / kThreads;
  // four copies of the counts, for lanes side by side: weights lie in few bins
  __shared__ __attribute__((aligned(16))) uint32_t s_hist[kSelectBins][4];
  __shared__ uint32_t s_wave[kWaves];
  __shared__ uint32_t s_found[3];
  __shared__ uint32_t s_count[kEntries];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = blockIdx.x / a.hk, h = blockIdx.x - b * a.hk;
  const int L = max(0, min(__builtin_amdgcn_readfirstlane(a.seqlens[b]), a.w * a.bs));
  const int n = min(L, a.budget);
  int32_t* kept = a.kept + (int64_t)blockIdx.x * a.budget;
  if (h == 0 && tid == 0) a.new_lens[b] = n;
  const int first =
      min(max(a.starts ? __builtin_amdgcn_readfirstlane(a.starts[b]) : a.start, 0), n);
  const int last = min(a.recent, n - first);
  // what stays whatever it weighs
  const int fixed_front = n == L ? n : first;
  for (int i = tid; i < fixed_front; i += kThreads) kept[i] = i;
  // (unsigned: a budget may lie within kThreads of 2^31)
  for (uint32_t i = n + tid; i < (uint32_t)a.budget; i += kThreads) kept[i] = -1;
  if (n == L) return;
  for (int i = tid; i < last; i += kThreads) kept[n - last + i] = L - last + i;
  const int quota = n - first - last;
  if (quota == 0) return;
  // the tokens that compete, more than quota: [first, end); runs of four of them
  // start at multiples of four and lie in one page
  const int end = L - last, base = first & ~3;
  const int quads = (end - base + 3) / 4;

  const int32_t* table = a.bt + (int64_t)b * a.w;
  uint32_t own[kQuads][4];
  // The keys of a turn's runs.  Without branches, so that all of a thread's reads
  // are in flight at once: a run past the end stands for the last one, an invalid
  // block for the first.  A token that does not compete has key 0, with the
  // lightest.
  auto fill = [&](int at) {
#pragma unroll
    for (int j = 0; j < kQuads; ++j) {
      const int t = base + 4 * min(at + j * kThreads + tid, quads - 1), page = a.by_block(t);
      const int blk = table[page];
      const bool ok = (uint32_t)blk < (uint32_t)a.num_blocks;
      const f32x4 x = *reinterpret_cast<const f32x4*>(
          a.weights + ((int64_t)(ok ? blk : 0) * a.hk + h) * a.bs + (t - page * a.bs));
#pragma unroll
      for (int q = 0; q < 4; ++q)
        own[j][q] = ok && t + q >= first && t + q < end ? weight_key(x[q]) : 0u;
    }
  };
  constexpr int kTurn = kQuads * kThreads;
  if (!kReread) fill(0);
  // keys that live past a barrier, seen anew: the compiler would keep masks of
  // what it knows of each key from pass to pass, and spill them
  auto anew = [&] {
#pragma unroll
    for (int j = 0; j < kQuads; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) asm volatile("" : "+v"(own[j][q]));
  };

  // The threshold: the quota-th largest key, digit by digit; `need` of the
  // tokens whose digits so far are the threshold's are still to be found.
  uint32_t need = quota, digits = 0;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t mask = pass == 2 ? 1023u : 2047u;
#pragma unroll
    for (int i = 0; i < kBinsEach; ++i)
      *reinterpret_cast<u32x4*>(s_hist[i * kThreads + tid]) = u32x4{0u, 0u, 0u, 0u};
    __syncthreads();
    for (int at = 0; at < quads; at += kTurn) {
      if (kReread) fill(at);
#pragma unroll
      for (int j = 0; j < kQuads; ++j) {
        if (at + j * kThreads + tid < quads) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            // (the digits above: all 32 bits on the first pass have none)
            if (pass == 0 || (own[j][q] >> (pass == 1 ? 21 : 10)) == digits)
              atomicAdd(&s_hist[(own[j][q] >> shift) & mask][lane & 3], 1u);
        }
      }
    }
    __syncthreads();
    // this thread's bins, from the highest down
    uint32_t bins[kBinsEach], sum = 0, all;
#pragma unroll
    for (int i = 0; i < kBinsEach; ++i) {
      const u32x4 c =
          *reinterpret_cast<const u32x4*>(s_hist[kSelectBins - 1 - (kBinsEach * tid + i)]);
      bins[i] = (c[0] + c[1]) + (c[2] + c[3]);
      sum += bins[i];
    }
    uint32_t before = scan_before<kWaves>(sum, s_wave, all);
    if (before < need && before + sum >= need) {
#pragma unroll
      for (int i = 0; i < kBinsEach; ++i) {
        if (before < need && before + bins[i] >= need) {
          s_found[0] = kSelectBins - 1 - (kBinsEach * tid + i);
          s_found[1] = need - before;
          s_found[2] = bins[i];
        }
        before += bins[i];
      }
    }
    __syncthreads();
    digits = pass == 0 ? s_found[0] : digits << (pass == 1 ? 11 : 10) | s_found[0];
    need = s_found[1];
    if (!kReread) anew();
  }
  const uint32_t threshold = digits;

  // The kept positions in order: a wave's counts of 64 runs, their running sums
  // over the workgroup, then each token's place.  Where every token at the
  // threshold stays, one comparison decides; else those above it stay and the
  // first `need` at it, whose counts travel in the upper halves of the words (at
  // most 2^15 tokens a turn).
  static_assert(4 * kTurn <= 1 << 15, "two counts fit a word");
  int32_t* to = kept + first;
  auto write = [&](auto ties) {
    constexpr bool kTies = decltype(ties)::value;
    uint32_t above0 = 0, equal0 = 0;  // before this turn
    for (int at = 0; at < quads; at += kTurn) {
      if (kReread) fill(at);
      auto is_above = [&](int j, int q) {
        return kTies ? own[j][q] > threshold : own[j][q] >= threshold;
      };
      auto is_equal = [&](int j, int q) {  // (a token that does not compete is none)
        const int t = base + 4 * (at + j * kThreads + tid) + q;
        return own[j][q] == threshold && t >= first && t < end;
      };
      auto live = [&](int j) { return at + j * kThreads + tid < quads; };
#pragma unroll
      for (int j = 0; j < kQuads; ++j) {
        uint32_t above = 0, equal = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          above += __popcll(__ballot(live(j) && is_above(j, q)));
          if (kTies) equal += __popcll(__ballot(live(j) && is_equal(j, q)));
        }
        if (lane == 0) s_count[j * kWaves + wave] = above | equal << 16;
        __builtin_amdgcn_sched_barrier(0);  // (masks of many keys at once would spill)
      }
      anew();
      __syncthreads();
      uint32_t all;
      const uint32_t before =
          scan_before<kWaves>(tid < kEntries ? s_count[tid] : 0u, s_wave, all);
      if (tid < kEntries) s_count[tid] = before;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kQuads; ++j) {
        const uint32_t counts = s_count[j * kWaves + wave];
        uint32_t above = above0 + (counts & 0xFFFFu), equal = equal0 + (counts >> 16);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          above += lanes_below(__ballot(live(j) && is_above(j, q)));
          if (kTies) equal += lanes_below(__ballot(live(j) && is_equal(j, q)));
        }
        const int t = base + 4 * (at + j * kThreads + tid);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const bool up = live(j) && is_above(j, q);
          const bool tie = kTies && live(j) && is_equal(j, q);
          if (up || (tie && equal < need)) to[above + (kTies ? min(equal, need) : 0u)] = t + q;
          above += up;
          equal += tie;
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      above0 += all & 0xFFFFu;
      equal0 += all >> 16;
      if (kReread) __syncthreads();  // (the counts are read before the next turn's)
    }
  };
  if (s_found[2] == need)
    write(std::false_type());
  else
    write(std::true_type());
}

constexpr int kEvictLoads = 4;  // 16-byte pieces of a lane and run

struct EvictArgs {
  uint8_t *kc, *vc;
  float *ks, *vs, *weights;
  const int32_t *kept, *lens, *bt;
  int64_t num_blocks;
  int hk, bs, w, budget, scale_heads, scale_units, row_heads, row_units;
  Divider by_block, by_heads, by_row_heads;
};

// A token's slot (its row among all pages' rows), -1 if it has none.
// (No branches: a lane's table entries are read all at once.)
__device__ __forceinline__ int64_t slot_of(const EvictArgs& a, const int32_t* table, int t) {
  const int in = min(max(t, 0), a.w * a.bs - 1);
  const int page = a.by_block(in);
  const int blk = table[page];
  return t != in || blk < 0 || (int64_t)blk >= a.num_blocks
             ? -1
             : (int64_t)blk * a.bs + (in - page * a.bs);
}

// A run of places: this lane's pieces of rows, and where they go (-1: nowhere).
struct EvictRun {
  u32x4 v[kEvictLoads];
  int64_t dst[kEvictLoads];
};

// What a workgroup of a sequence moves: rows of K or of V, scales of either (both
// of so many heads of a token at a time), or a head's weights.
//
// The rows of the next run are asked for before those of this one are stored,
// and what they are is known a run earlier still.  Between two runs there is
// one barrier, behind the arrival of the first one's rows: nobody stores to a
// run's places before all have read it.
//
// A token's scales of all heads are one piece of memory (32 bytes at eight
// heads): moved head by head, by workgroups on other XCDs, each line is written
// in parts that memory has to read first (64 x 4096 rows of eight heads: 273 us
// for the whole call).
template <int kThreads>
__global__ __launch_bounds__(kThreads) void evict_kv_tokens_kernel(EvictArgs a) {
  const int tid = threadIdx.x;
  const int b = blockIdx.y;
  const int32_t* table = a.bt + (int64_t)b * a.w;
  const int32_t* kept = a.kept + (int64_t)b * a.hk * a.budget;
  // (places past the table have no slots)
  const int n = min(min(__builtin_amdgcn_readfirstlane(a.lens[b]), a.budget), a.w * a.bs);
  if (n <= 0) return;
  int unit = blockIdx.x;

  // Runs of single floats: `of(e)` is element e's (position it comes from,
  // place, offset of a slot); `count` elements, whose places ascend.
  auto floats = [&](float* x, int count, auto&& of) {
    constexpr int kFloats = 8;
    for (int at = 0; at < count; at += kThreads * kFloats) {
      float v[kFloats];
      int64_t dst[kFloats];
#pragma unroll
      for (int k = 0; k < kFloats; ++k) {
        const int e = at + k * kThreads + tid;
        int64_t src, to;
        of(min(e, count - 1), src, to);
        dst[k] = e < count && src != to && src >= 0 ? to : -1;
        v[k] = x[max(src, (int64_t)0)];
      }
#pragma unroll
      for (int k = 0; k < kFloats; ++k) asm volatile("" ::"v"(v[k]));  // they are here
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
#pragma unroll
      for (int k = 0; k < kFloats; ++k)
        if (dst[k] >= 0) x[dst[k]] = v[k];
    }
  };
  if (unit < 2 * a.scale_units) {  // `scale_heads` heads of K's or V's scales
    const int h0 = unit % a.scale_units * a.scale_heads;
    floats(unit < a.scale_units ? a.ks : a.vs, n * a.scale_heads,
           [&](int e, int64_t& src, int64_t& to) {
             const int i = a.by_heads(e), h = h0 + e - i * a.scale_heads;
             const int64_t s = slot_of(a, table, kept[(int64_t)h * a.budget + i]);
             const int64_t d = slot_of(a, table, i);
             src = s < 0 ? -1 : s * a.hk + h;
             to = d < 0 ? -1 : d * a.hk + h;
           });
    return;
  }
  unit -= 2 * a.scale_units;
  if (a.weights) {
    if (unit < a.hk) {
      floats(a.weights, n, [&](int e, int64_t& src, int64_t& to) {
        // a head's weights of a page are one piece
        auto place = [&](int64_t slot) {
          const int64_t page = slot / a.bs;
          return slot < 0 ? -1 : (page * a.hk + unit) * a.bs + (slot - page * a.bs);
        };
        src = place(slot_of(a, table, kept[(int64_t)unit * a.budget + e]));
        to = place(slot_of(a, table, e));
      });
      return;
    }
    unit -= a.hk;
  }
  constexpr int kLanes = kHeadDim / 16;  // of a row
  constexpr int kRows = kThreads / kLanes;
  constexpr int kRun = kRows * kEvictLoads;
  // row r is place r / row_heads of head h0 + r % row_heads
  const int h0 = unit % a.row_units * a.row_heads;
  const int count = n * a.row_heads;
  kept += (int64_t)h0 * a.budget;
  uint8_t* rows = (unit < a.row_units ? a.kc : a.vc) + h0 * kHeadDim + 16 * (tid % kLanes);
  const int64_t stride = (int64_t)a.hk * kHeadDim;
  const int own = tid / kLanes;
  // A run's rows are known in three steps, each a run ahead of the next: the
  // positions (kept), their blocks (the table), the rows.  A wave's loads come
  // back in order, so whatever a later run needs first is asked for before the
  // rows of an earlier one: waiting for it is then no wait for those.
  int from[kEvictLoads];  // positions
  int from_blk[kEvictLoads], to_blk[kEvictLoads], from_off[kEvictLoads], to_off[kEvictLoads];
  auto look = [&](int at) {
#pragma unroll
    for (int k = 0; k < kEvictLoads; ++k) {
      const int r = min(at + k * kRows + own, count - 1);
      const int i = a.by_row_heads(r);
      from[k] = kept[(int64_t)(r - i * a.row_heads) * a.budget + i];
    }
  };
  auto find = [&](int at) {
#pragma unroll
    for (int k = 0; k < kEvictLoads; ++k) {
      const int i = a.by_row_heads(min(at + k * kRows + own, count - 1));
      const int t = min(max(from[k], 0), a.w * a.bs - 1);
      const int page = a.by_block(t), to_page = a.by_block(i);
      // (a row that stays, or whose position is none, goes nowhere: block -1)
      from_off[k] = at + k * kRows + own < count && t == from[k] && t != i ? t - page * a.bs : -1;
      to_off[k] = i - to_page * a.bs;
      from_blk[k] = table[page];
      to_blk[k] = table[to_page];
    }
  };
  int64_t src[kEvictLoads];
  auto place = [&](int at, EvictRun& run) {
#pragma unroll
    for (int k = 0; k < kEvictLoads; ++k) {
      const int r = min(at + k * kRows + own, count - 1);
      const int64_t head = (r - a.by_row_heads(r) * a.row_heads) * kHeadDim;
      const bool moves = from_off[k] >= 0 && from_blk[k] >= 0 && from_blk[k] < a.num_blocks &&
                         to_blk[k] >= 0 && to_blk[k] < a.num_blocks;
      src[k] = (moves ? (int64_t)from_blk[k] * a.bs + from_off[k] : 0) * stride + head;
      run.dst[k] = moves ? ((int64_t)to_blk[k] * a.bs + to_off[k]) * stride + head : -1;
    }
  };
  auto ask = [&](EvictRun& run) {
#pragma unroll
    for (int k = 0; k < kEvictLoads; ++k)
      run.v[k] = *reinterpret_cast<const u32x4*>(rows + src[k]);
  };
  auto store = [&](const EvictRun& r) {
#pragma unroll
    for (int k = 0; k < kEvictLoads; ++k) asm volatile("" ::"v"(r.v[k]));  // they are here
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int k = 0; k < kEvictLoads; ++k)
      if (r.dst[k] >= 0)
        __builtin_nontemporal_store(r.v[k], reinterpret_cast<u32x4*>(rows + r.dst[k]));
  };
  // the run at `at` is on its way in `now`; `next` takes the one after it, whose
  // blocks are known, as are the positions of the one after that
  auto turn = [&](int at, EvictRun& now, EvictRun& next) {
    place(at + kRun, next);
    find(at + 2 * kRun);
    look(at + 3 * kRun);
    __builtin_amdgcn_sched_barrier(0);
    ask(next);
    __builtin_amdgcn_sched_barrier(0);
    store(now);
    __builtin_amdgcn_sched_barrier(0);
  };
  EvictRun even, odd;
  look(0);
  find(0);
  look(kRun);
  place(0, even);
  find(kRun);
  look(2 * kRun);
  __builtin_amdgcn_sched_barrier(0);
  ask(even);
  for (int at = 0; at < count; at += 2 * kRun) {
    turn(at, even, odd);
    if (at + kRun >= count) break;
    turn(at + kRun, odd, even);
  }
}

static int evict_shape(int batch, int num_kv_heads, int block_size, int64_t num_blocks,
                       int max_blocks_per_seq, int budget) {
  if (batch < 0 || num_kv_heads <= 0 || block_size <= 0 || num_blocks < 0 ||
      max_blocks_per_seq <= 0 || budget <= 0)
    return MSKV_EINVAL;
  if ((int64_t)max_blocks_per_seq * block_size >= 1LL << 30 || batch > 65535 ||
      num_kv_heads > 65535)
    return MSKV_EUNSUPPORTED;
  return MSKV_OK;
}

}  // namespace mskv

extern "C" int mskv_select_kv_tokens(const float* weights, const int32_t* cache_seqlens,
                                     const int32_t* block_tables, const int32_t* starts, int start,
                                     int recent, int budget, int32_t* kept, int32_t* new_seqlens,
                                     int batch, int num_kv_heads, int block_size,
                                     int64_t num_blocks, int max_blocks_per_seq, void* stream) {
  using namespace mskv;
  const int status = evict_shape(batch, num_kv_heads, block_size, num_blocks, max_blocks_per_seq,
                                 budget);
  if (status != MSKV_OK) return status;
  if (start < 0 || recent < 0) return MSKV_EINVAL;
  if (batch == 0) return MSKV_OK;
  if (num_blocks == 0) return MSKV_EINVAL;  // (there are no weights to read)
  if (block_size % 4 != 0 || num_blocks > 0x7FFFFFFFLL) return MSKV_EUNSUPPORTED;
  // (a grid's threads fit 32 bits)
  if ((int64_t)batch * num_kv_heads > 0x3FFFFF) return MSKV_EUNSUPPORTED;
  if (!weights || !cache_seqlens || !block_tables || !kept || !new_seqlens ||
      misaligned({weights}))
    return MSKV_EINVAL;
  const SelectArgs a = {weights, cache_seqlens, block_tables,       starts, kept,   new_seqlens,
                        num_blocks, num_kv_heads, block_size, max_blocks_per_seq, start, recent,
                        budget, divider_of(block_size)};
  const dim3 grid((unsigned)(batch * num_kv_heads));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  // (by the most tokens that can compete)
  const int64_t tokens = (int64_t)max_blocks_per_seq * block_size;
  auto run = [&](auto kernel, int threads) {
    hipLaunchKernelGGL(kernel, grid, dim3((unsigned)threads), 0, s, a);
    return (int)hipGetLastError();
  };
  if (tokens <= 2048) return run(select_kv_tokens_kernel<512, 1, false>, 512);
  if (tokens <= 8192) return run(select_kv_tokens_kernel<1024, 2, false>, 1024);
  if (tokens <= 32768) return run(select_kv_tokens_kernel<1024, 8, false>, 1024);
  return run(select_kv_tokens_kernel<1024, 4, true>, 1024);
}

extern "C" int mskv_evict_kv_tokens(void* k_cache, void* v_cache, float* k_scale_cache,
                                    float* v_scale_cache, float* weights, const int32_t* kept,
                                    const int32_t* new_seqlens, const int32_t* block_tables,
                                    int batch, int num_kv_heads, int head_dim, int block_size,
                                    int64_t num_blocks, int max_blocks_per_seq, int budget,
                                    void* stream) {
  using namespace mskv;
  const int status = evict_shape(batch, num_kv_heads, block_size, num_blocks, max_blocks_per_seq,
                                 budget);
  if (status != MSKV_OK) return status;
  if (head_dim != kHeadDim) return MSKV_EUNSUPPORTED;
  // (a run of one plus a sequence's rows of all heads)
  if ((int64_t)max_blocks_per_seq * block_size * num_kv_heads > 0x7FFFFFFFLL - (1 << 14))
    return MSKV_EUNSUPPORTED;
  if (batch == 0 || num_blocks == 0) return MSKV_OK;
  if (!k_cache || !v_cache || !k_scale_cache || !v_scale_cache || !kept || !new_seqlens ||
      !block_tables || misaligned({k_cache, v_cache}))
    return MSKV_EINVAL;
  // The heads of a token that one workgroup moves, all of them where the
  // sequences alone are workgroups enough.
  auto heads_of = [&](int64_t units) {
    int heads = (int)std::max<int64_t>(1, std::min<int64_t>(num_kv_heads, units));
    while (num_kv_heads % heads != 0) --heads;
    return heads;
  };
  const int scale_heads = heads_of((int64_t)batch * num_kv_heads / 32);
  const int row_heads = heads_of((int64_t)batch * 2 * num_kv_heads / 512);
  const int scale_units = num_kv_heads / scale_heads, row_units = num_kv_heads / row_heads;
  const EvictArgs a = {(uint8_t*)k_cache, (uint8_t*)v_cache, k_scale_cache, v_scale_cache, weights,
                       kept, new_seqlens, block_tables, num_blocks, num_kv_heads, block_size,
                       max_blocks_per_seq, budget, scale_heads, scale_units, row_heads, row_units,
                       divider_of(block_size), divider_of(scale_heads), divider_of(row_heads)};
  const dim3 grid((unsigned)(2 * scale_units + (weights ? num_kv_heads : 0) + 2 * row_units),
                  (unsigned)batch);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  // Longer runs where the workgroups are too few to fill the chip and the places
  // are more than four short ones (one to eight sequences at eight heads, 512 / 1024
  // threads: 256 places 6 / 7.5 us, 1024 9.3 to 10.6 / 9.4 to 10.7, 4096 27 to 37 / 24
  // to 30).
  const int64_t places = std::min<int64_t>(budget, (int64_t)max_blocks_per_seq * block_size);
  if ((int64_t)grid.x * batch > 256 || places <= 1024)
    hipLaunchKernelGGL(evict_kv_tokens_kernel<512>, grid, dim3(512), 0, s, a);
  else
    hipLaunchKernelGGL(evict_kv_tokens_kernel<1024>, grid, dim3(1024), 0, s, a);
  return (int)hipGetLastError();
}
