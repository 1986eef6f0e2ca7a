// Moving whole pages of a paged KV pool: copies (a forked sequence's last
// page) and compaction (the live pages to the lowest places).
//
// A pool is up to kMaxPools tensors whose pages are numbered alike (codes and
// scales, FP8 or 4-bit, one layer's or all layers'): `planes` stacks of pages
// `plane_stride` bytes apart, pages of `page_bytes` back to back.  All of a
// call's bytes move in one launch: workgroups take segments of a page, 16
// bytes a lane and load, copied through registers.  HBM-bound, 2 bytes moved
// per byte of the pages.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <vector>

#include "mskv_device.h"
#include "../../include/mskv.h"

namespace mskv {

constexpr int kMaxPools = MSKV_MAX_POOLS;
constexpr int kMoveThreads = 256;
// 16-byte pieces of a lane's turn.  A copy's workgroups come and go with one
// each: 1.2 GB in 206 us (226 with two, 236 with four).  A compaction's walk the
// moves, two pieces at a time: 122 of 512 pages in 212 us (265 with one, 214
// with four; the same pages as a copy 174).  Asking for a workgroup's next
// segment before it stores one gained nothing (216 to 227).
constexpr int kCopyLoads = 1, kCompactLoads = 2;
constexpr int seg_bytes(int loads) { return kMoveThreads * loads * 16; }
// pairs that travel as arguments of one launch
constexpr int kMaxPairs = 256;

struct Pools {
  uint8_t* base[kMaxPools];
  int64_t plane_stride[kMaxPools], page_bytes[kMaxPools];
  int segs[kMaxPools];       // segments per page
  int first[kMaxPools + 1];  // of a pool's planes, among a page's segments
  int count;
};

struct PagePairs {
  int32_t src[kMaxPairs], dst[kMaxPairs];
};

// Copies segment `seg` (of all the pools' planes) of page src to page dst.
template <int kLoads>
__device__ __forceinline__ void copy_segment(const Pools& p, int seg, int64_t src, int64_t dst) {
  int t = 0;
  while (t + 1 < p.count && seg >= p.first[t + 1]) ++t;
  const int s = seg - p.first[t];
  const int plane = s / p.segs[t], part = s - plane * p.segs[t];
  const int64_t page = p.page_bytes[t], begin = (int64_t)part * seg_bytes(kLoads);
  uint8_t* stack = p.base[t] + plane * p.plane_stride[t] + begin;
  const u32x4* from = reinterpret_cast<const u32x4*>(stack + src * page);
  u32x4* to = reinterpret_cast<u32x4*>(stack + dst * page);
  const int n = (int)min((int64_t)seg_bytes(kLoads), page - begin) / 16;
  u32x4 v[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int at = i * kMoveThreads + threadIdx.x;
    if (at < n) v[i] = __builtin_nontemporal_load(from + at);
  }
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int at = i * kMoveThreads + threadIdx.x;
    if (at < n) __builtin_nontemporal_store(v[i], to + at);
  }
}

// grid (segments of a page in all pools, pairs)
__global__ __launch_bounds__(kMoveThreads) void copy_kv_blocks_kernel(Pools p, PagePairs pairs) {
  copy_segment<kCopyLoads>(p, blockIdx.x, pairs.src[blockIdx.y], pairs.dst[blockIdx.y]);
}

// A compaction: n pages are named by the tables; the i-th named page at or
// above n (ascending) goes to the i-th free page below n, so no page is both
// read and written.  Every workgroup makes the plan for itself, from the
// tables: the pages' flags are a bitmap in LDS with running counts per word,
// in which a move's source and destination are found by bisection.  A kernel
// of its own for the plan costs a launch, and its one workgroup 7 us (20 of 32
// pages: 12.2 us with it).
constexpr int kPlanMaxBlocks = 1 << 18;  // 32 KB of flags, 64 KB of counts

struct CompactArgs {
  const int32_t* tables;
  int32_t *new_tables, *remap, *num_live;
  int64_t entries;
  int num_blocks, segs;
};

// (sum over the threads before this one, sum over all) of two counts
struct Scan2 {
  int before_a, before_b, all_a, all_b;
};
__device__ __forceinline__ Scan2 block_scan(int a, int b, int2* s_wave) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = a, y = b;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int u = __shfl_up(x, d), v = __shfl_up(y, d);
    if (lane >= d) x += u, y += v;
  }
  if (lane == 63) s_wave[wave] = int2{x, y};
  __syncthreads();
  Scan2 r = {x - a, y - b, 0, 0};
#pragma unroll
  for (int w = 0; w < kMoveThreads / 64; ++w) {
    const int2 t = s_wave[w];
    if (w < wave) r.before_a += t.x, r.before_b += t.y;
    r.all_a += t.x, r.all_b += t.y;
  }
  __syncthreads();
  return r;
}

// The page of the i-th set bit of words f(w), whose running counts are c.
template <typename F>
__device__ __forceinline__ int find_bit(const int* c, int words, int i, F f) {
  int lo = 0, hi = words;  // the last word with c <= i
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (c[mid] <= i)
      lo = mid;
    else
      hi = mid;
  }
  uint32_t w = f(lo);
  for (int k = i - c[lo]; k > 0; --k) w &= w - 1;  // drops the bits before it
  return 32 * lo + __ffs(w) - 1;
}

__global__ __launch_bounds__(kMoveThreads) void compact_kv_blocks_kernel(Pools p, CompactArgs a) {
  // flags[words], then per word: the free pages below n and the named ones
  // from n up, in the words before it
  extern __shared__ uint32_t flags[];
  __shared__ int2 s_wave[kMoveThreads / 64];
  const int tid = threadIdx.x;
  const int words = (a.num_blocks + 31) / 32;
  int* holes_at = (int*)flags + words;
  int* movers_at = holes_at + words;
  for (int w = tid; w < words; w += kMoveThreads) flags[w] = 0;
  __syncthreads();
  for (int64_t i = tid; i < a.entries; i += kMoveThreads) {
    const int32_t page = a.tables[i];
    if (page >= 0 && page < a.num_blocks) atomicOr(&flags[page >> 5], 1u << (page & 31));
  }
  __syncthreads();
  const int per = (words + kMoveThreads - 1) / kMoveThreads;
  const int w0 = min(tid * per, words), w1 = min(w0 + per, words);
  int own = 0;
  for (int w = w0; w < w1; ++w) own += __popc(flags[w]);
  const int n = block_scan(own, 0, s_wave).all_a;
  // the pages of word w that are free and below n / named and at least n
  auto low = [&](int w) {
    const int below = min(max(n - 32 * w, 0), 32);
    return below == 32 ? ~0u : (1u << below) - 1u;
  };
  auto holes = [&](int w) { return ~flags[w] & low(w); };
  auto movers = [&](int w) { return flags[w] & ~low(w); };
  int h = 0, m = 0;
  for (int w = w0; w < w1; ++w) h += __popc(holes(w)), m += __popc(movers(w));
  const Scan2 sums = block_scan(h, m, s_wave);
  h = sums.before_a, m = sums.before_b;
  for (int w = w0; w < w1; ++w) {
    holes_at[w] = h, movers_at[w] = m;
    h += __popc(holes(w)), m += __popc(movers(w));
  }
  __syncthreads();
  const int moves = sums.all_a;
  auto place = [&](int page) {  // -1 for a free page
    const int w = page >> 5;
    const uint32_t bit = 1u << (page & 31);
    if (!(flags[w] & bit)) return -1;
    if (page < n) return page;
    return find_bit(holes_at, words, movers_at[w] + __popc(movers(w) & (bit - 1)), holes);
  };
  const int64_t first = (int64_t)blockIdx.x * kMoveThreads + tid;
  const int64_t step = (int64_t)gridDim.x * kMoveThreads;
  if (first == 0) *a.num_live = n;
  for (int64_t i = first; i < a.num_blocks; i += step) a.remap[i] = place((int)i);
  const int64_t total = (int64_t)moves * a.segs;
  for (int64_t i = blockIdx.x; i < total; i += gridDim.x) {
    const int pair = (int)(i / a.segs);
    copy_segment<kCompactLoads>(
        p, (int)(i - (int64_t)pair * a.segs),
        __builtin_amdgcn_readfirstlane(find_bit(movers_at, words, pair, movers)),
        __builtin_amdgcn_readfirstlane(find_bit(holes_at, words, pair, holes)));
  }
  for (int64_t i = first; i < a.entries; i += step) {
    const int32_t page = a.tables[i];
    a.new_tables[i] = page >= 0 && page < a.num_blocks ? place(page) : page;
  }
}

// Checks a call's pools and lays their segments out.
static int pools_of(Pools& p, int count, void* const* bases, const int64_t* planes,
                    const int64_t* plane_strides, const int64_t* page_bytes, int64_t num_blocks,
                    int loads) {
  if (count <= 0 || count > kMaxPools || !bases || !planes || !plane_strides || !page_bytes)
    return MSKV_EINVAL;
  if (num_blocks < 0 || num_blocks > 0x7FFFFFFFLL) return MSKV_EINVAL;
  int64_t first = 0;
  p.count = count;
  for (int t = 0; t < count; ++t) {
    if (!bases[t] || planes[t] <= 0 || page_bytes[t] <= 0 || plane_strides[t] < 0)
      return MSKV_EINVAL;
    if (misaligned({bases[t]}) || page_bytes[t] % 16 != 0 || plane_strides[t] % 16 != 0)
      return MSKV_EUNSUPPORTED;
    // every byte offset fits an int64, and the planes do not overlap
    if (num_blocks > 0 && page_bytes[t] > (INT64_MAX >> 1) / num_blocks) return MSKV_EINVAL;
    if (planes[t] > 1 && plane_strides[t] < page_bytes[t] * num_blocks) return MSKV_EINVAL;
    if (planes[t] > 1 && plane_strides[t] > (INT64_MAX >> 1) / planes[t]) return MSKV_EINVAL;
    const int64_t segs = (page_bytes[t] + seg_bytes(loads) - 1) / seg_bytes(loads);
    if (segs > 0x3FFFFFFF || planes[t] > 0x3FFFFFFF / segs) return MSKV_EUNSUPPORTED;
    p.base[t] = (uint8_t*)bases[t];
    p.plane_stride[t] = plane_strides[t];
    p.page_bytes[t] = page_bytes[t];
    p.segs[t] = (int)segs;
    p.first[t] = (int)first;
    first += segs * planes[t];
    if (first > 0xFFFFFF) return MSKV_EUNSUPPORTED;  // a grid's threads fit 32 bits
  }
  p.first[count] = (int)first;
  return MSKV_OK;
}

// The same for a compaction, which numbers its pages in LDS.
static int compact_pools_of(Pools& p, int count, void* const* bases, const int64_t* planes,
                            const int64_t* plane_strides, const int64_t* page_bytes,
                            int64_t num_blocks) {
  const int status = pools_of(p, count, bases, planes, plane_strides, page_bytes, num_blocks,
                              kCompactLoads);
  if (status != MSKV_OK) return status;
  if (num_blocks <= 0) return MSKV_EINVAL;
  return num_blocks > kPlanMaxBlocks ? MSKV_EUNSUPPORTED : MSKV_OK;
}

}  // namespace mskv

extern "C" int mskv_check_kv_blocks(int num_pools, void* const* bases, const int64_t* planes,
                                    const int64_t* plane_strides, const int64_t* page_bytes,
                                    int64_t num_blocks, int compact) {
  using namespace mskv;
  Pools p;
  return compact ? compact_pools_of(p, num_pools, bases, planes, plane_strides, page_bytes,
                                    num_blocks)
                 : pools_of(p, num_pools, bases, planes, plane_strides, page_bytes, num_blocks,
                            kCopyLoads);
}

extern "C" int mskv_copy_kv_blocks(int num_pools, void* const* bases, const int64_t* planes,
                                   const int64_t* plane_strides, const int64_t* page_bytes,
                                   int64_t num_blocks, const int32_t* src_blocks,
                                   const int32_t* dst_blocks, int64_t num_pairs, void* stream) {
  using namespace mskv;
  Pools p;
  const int status = pools_of(p, num_pools, bases, planes, plane_strides, page_bytes, num_blocks,
                              kCopyLoads);
  if (status != MSKV_OK) return status;
  if (num_pairs < 0) return MSKV_EINVAL;
  if (num_pairs == 0) return MSKV_OK;
  if (!src_blocks || !dst_blocks || num_pairs > num_blocks) return MSKV_EINVAL;
  // Pages are read and written side by side: each is written once, and none
  // that is written is read.
  try {
    std::vector<int32_t> from(src_blocks, src_blocks + num_pairs),
        to(dst_blocks, dst_blocks + num_pairs);
    std::sort(from.begin(), from.end());
    std::sort(to.begin(), to.end());
    if (from.front() < 0 || to.front() < 0 || from.back() >= num_blocks ||
        to.back() >= num_blocks)
      return MSKV_EINVAL;
    if (std::adjacent_find(to.begin(), to.end()) != to.end()) return MSKV_EINVAL;
    for (int32_t d : to)
      if (std::binary_search(from.begin(), from.end(), d)) return MSKV_EINVAL;
  } catch (...) {
    return MSKV_EINVAL;
  }
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  for (int64_t at = 0; at < num_pairs; at += kMaxPairs) {
    const int n = (int)std::min<int64_t>(kMaxPairs, num_pairs - at);
    PagePairs pairs = {};
    std::copy_n(src_blocks + at, n, pairs.src);
    std::copy_n(dst_blocks + at, n, pairs.dst);
    hipLaunchKernelGGL(copy_kv_blocks_kernel, dim3((unsigned)p.first[p.count], (unsigned)n),
                       dim3(kMoveThreads), 0, s, p, pairs);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  return MSKV_OK;
}

extern "C" int mskv_compact_kv_blocks(int num_pools, void* const* bases, const int64_t* planes,
                                      const int64_t* plane_strides, const int64_t* page_bytes,
                                      int64_t num_blocks, const int32_t* block_tables,
                                      int64_t num_entries, int32_t* new_tables, int32_t* remap,
                                      int32_t* num_live, void* stream) {
  using namespace mskv;
  Pools p;
  const int status = compact_pools_of(p, num_pools, bases, planes, plane_strides, page_bytes,
                                      num_blocks);
  if (status != MSKV_OK) return status;
  if (num_entries < 0) return MSKV_EINVAL;
  if (num_entries > (int64_t)1 << 40) return MSKV_EUNSUPPORTED;
  if (!remap || !num_live || (num_entries > 0 && (!block_tables || !new_tables)))
    return MSKV_EINVAL;
  // every workgroup reads the tables while others write the renamed ones
  const uintptr_t from = (uintptr_t)block_tables, end = from + (uintptr_t)num_entries * 4;
  auto overlaps = [&](const int32_t* to, int64_t n) {
    return from < (uintptr_t)to + (uintptr_t)n * 4 && (uintptr_t)to < end;
  };
  if (overlaps(new_tables, num_entries) || overlaps(remap, num_blocks) || overlaps(num_live, 1))
    return MSKV_EINVAL;
  CompactArgs a;
  a.tables = block_tables;
  a.new_tables = new_tables;
  a.remap = remap;
  a.num_live = num_live;
  a.entries = num_entries;
  a.num_blocks = (int)num_blocks;
  a.segs = p.first[p.count];
  // A grid that fills the chip walks the moves, whose number only the device
  // knows; every workgroup reads the tables, so fewer where these are long.
  const int64_t most =
      std::max<int64_t>(num_blocks / 2 * a.segs,
                        (std::max(num_entries, num_blocks) + kMoveThreads - 1) / kMoveThreads);
  const int64_t cap = num_entries > 1 << 16 ? 512 : 2048;
  const unsigned grid = (unsigned)std::min<int64_t>(std::max<int64_t>(most, 1), cap);
  const unsigned lds = (unsigned)((num_blocks + 31) / 32 * 12);
  hipLaunchKernelGGL(compact_kv_blocks_kernel, dim3(grid), dim3(kMoveThreads), lds,
                     reinterpret_cast<hipStream_t>(stream), p, a);
  return (int)hipGetLastError();
}
