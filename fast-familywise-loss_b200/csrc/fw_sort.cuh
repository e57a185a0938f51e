// Stable radix sort of int64 ids in [0, V): the parts shared by the embedding's
// gradient and the packing of rows by label.  Two launches per digit; the
// embedding sorts what fits one cluster in one (fw_embed.cu).
#pragma once

#include "fw_host.cuh"

namespace fwb200 {
namespace {

constexpr int kSortThreads = 256;
constexpr int kSortItems = 8;
constexpr int kSortTile = kSortThreads * kSortItems;
constexpr int kMaxDigitBits = 9;
constexpr int kMaxBins = 1 << kMaxDigitBits;

// Entries are (key, position); key V marks ids out of range, key V + tail the
// ones equal to `padding`; both sort behind every row.
struct SortArgs {
  const int64_t* ids;   // first pass: keys come from here
  const uint2* src;     // later passes
  uint2* dst;
  uint32_t* hist;       // [tiles, bins]
  int64_t T, V, padding;
  uint32_t tail;
  int shift, bits;
  int tiles;
  int32_t* status;
};

__device__ __forceinline__ uint2 sort_entry(const SortArgs& a, int64_t i, bool report) {
  if (a.src) return a.src[i];
  const int64_t id = a.ids[i];
  const bool ok = id >= 0 && id < a.V;
  if (!ok && report) raise_status(a.status, FWB_STATUS_LABEL_RANGE);
  return make_uint2(id == a.padding ? (uint32_t)a.V + a.tail : ok ? (uint32_t)id : (uint32_t)a.V, (uint32_t)i);
}

// Ranks the tile's entries by digit, stably: after the call, entry i of this
// thread goes to (place of its digit) + cnt[warp][digit] + rank[i], and
// total[digit] is the tile's count.  Entry i of lane l of warp w is number
// w * 32 * kSortItems + 32 * i + l of the tile.
template <int THREADS>
__device__ __forceinline__ void tile_rank(const uint32_t (&digit)[kSortItems], uint32_t (&rank)[kSortItems],
                                          uint16_t (*cnt)[kMaxBins + 2], uint32_t* total, int bins) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  uint32_t* words = reinterpret_cast<uint32_t*>(&cnt[0][0]);
  for (int i = threadIdx.x; i < THREADS / 32 * (kMaxBins + 2) / 2; i += THREADS) words[i] = 0u;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSortItems; ++i) {
    const uint32_t d = digit[i];  // `bins` for entries past the end
    const uint32_t same = __match_any_sync(kFull, d);
    const uint32_t before = cnt[w][d];
    __syncwarp();
    if (lane == __ffs(same) - 1) cnt[w][d] = (uint16_t)(before + __popc(same));
    __syncwarp();
    rank[i] = before + __popc(same & ((1u << lane) - 1u));
  }
  __syncthreads();
  for (int d = threadIdx.x; d < bins; d += THREADS) {
    uint32_t run = 0u;
#pragma unroll
    for (int q = 0; q < THREADS / 32; ++q) {
      const uint32_t c = cnt[q][d];
      cnt[q][d] = (uint16_t)run;
      run += c;
    }
    total[d] = run;
  }
  __syncthreads();
}

// Exclusive scan of total[0 .. bins) in place by the whole CTA.
template <int THREADS>
__device__ __forceinline__ void scan_bins(uint32_t* total, uint32_t* warp_sum, int bins) {
  constexpr int kPer = kMaxBins / THREADS;
  static_assert(kPer * THREADS == kMaxBins, "whole bins per thread");
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  uint32_t v[kPer], s = 0u;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int d = threadIdx.x * kPer + k;
    v[k] = d < bins ? total[d] : 0u;
    s += v[k];
  }
  uint32_t inc = s;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(kFull, inc, o);
    if (lane >= o) inc += u;
  }
  if (lane == 31) warp_sum[w] = inc;
  __syncthreads();
  uint32_t base = inc - s;
  for (int q = 0; q < w; ++q) base += warp_sum[q];
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int d = threadIdx.x * kPer + k;
    if (d < bins) total[d] = base;
    base += v[k];
  }
  __syncthreads();
}

__global__ void __launch_bounds__(kSortThreads) fw_sort_hist_kernel(SortArgs a) {
  __shared__ uint32_t h[kMaxBins];
  const int bins = 1 << a.bits;
  for (int d = threadIdx.x; d < bins; d += kSortThreads) h[d] = 0u;
  __syncthreads();
  const int64_t t0 = (int64_t)blockIdx.x * kSortTile;
#pragma unroll
  for (int i = 0; i < kSortItems; ++i) {
    const int64_t e = t0 + i * kSortThreads + threadIdx.x;
    if (e < a.T) atomicAdd(&h[(sort_entry(a, e, true).x >> a.shift) & (bins - 1)], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < bins; d += kSortThreads) a.hist[(int64_t)blockIdx.x * bins + d] = h[d];
}

// One pass: every tile adds up the histograms itself (all digits' totals, and
// its own digit counts in the tiles before it), so no scan kernel runs
// between the histograms and the scatter.
__global__ void __launch_bounds__(kSortThreads) fw_sort_scatter_kernel(SortArgs a) {
  __shared__ __align__(4) uint16_t cnt[kSortThreads / 32][kMaxBins + 2];
  __shared__ uint32_t total[kMaxBins], place[kMaxBins], warp_sum[kSortThreads / 32];
  const int bins = 1 << a.bits;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t t0 = (int64_t)blockIdx.x * kSortTile;
  uint2 ent[kSortItems];
  uint32_t digit[kSortItems], rank[kSortItems];
#pragma unroll
  for (int i = 0; i < kSortItems; ++i) {
    const int64_t e = t0 + w * 32 * kSortItems + 32 * i + lane;
    ent[i] = e < a.T ? sort_entry(a, e, false) : make_uint2(0u, 0u);
    digit[i] = e < a.T ? (ent[i].x >> a.shift) & (bins - 1) : (uint32_t)bins;
  }
  tile_rank<kSortThreads>(digit, rank, cnt, total, bins);
  for (int d = threadIdx.x; d < bins; d += kSortThreads) {
    uint32_t before = 0u, all = 0u;
#pragma unroll 4
    for (int q = 0; q < a.tiles; ++q) {
      const uint32_t c = a.hist[(int64_t)q * bins + d];
      before += q < (int)blockIdx.x ? c : 0u;
      all += c;
    }
    place[d] = before;
    total[d] = all;
  }
  __syncthreads();
  scan_bins<kSortThreads>(total, warp_sum, bins);
#pragma unroll
  for (int i = 0; i < kSortItems; ++i)
    if (digit[i] < (uint32_t)bins) a.dst[total[digit[i]] + place[digit[i]] + cnt[w][digit[i]] + rank[i]] = ent[i];
}

// Digits of keys 0 .. most.
inline void sort_digits(int64_t most, int* passes, int* bits) {
  int total = 1;
  while (((int64_t)1 << total) <= most) ++total;
  *passes = (total + kMaxDigitBits - 1) / kMaxDigitBits;
  *bits = (total + *passes - 1) / *passes;
}

// All passes, two launches each; the sorted entries are where it says.
inline const uint2* sort_launch(SortArgs s, uint2* first, uint2* second, int passes, cudaStream_t st) {
  uint2* ent[2] = {first, second};
  for (int i = 0; i < passes; ++i) {
    s.src = i == 0 ? nullptr : ent[(i - 1) & 1];
    s.dst = ent[i & 1];
    s.shift = i * s.bits;
    fw_sort_hist_kernel<<<(unsigned)s.tiles, kSortThreads, 0, st>>>(s);
    fw_sort_scatter_kernel<<<(unsigned)s.tiles, kSortThreads, 0, st>>>(s);
  }
  return ent[(passes - 1) & 1];
}

}  // namespace
}  // namespace fwb200
