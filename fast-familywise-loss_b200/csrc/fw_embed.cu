// Rows of an embedding table, scaled, and the table's gradient.
//
//   out[t] = scale * W[ids[t]]
//   dW[v]  = scale * sum over {t : ids[t] = v} of g[t]
//
// Bound by HBM: the lookup reads and writes T rows; the gradient reads g once
// and writes every row of dW once (zeros where no token points), which for a
// large vocabulary is most of the bytes.  Nothing is added with atomics: the
// tokens are sorted by id (a stable radix sort), and a row's contributions
// are added in position order, in fp32, so the result does not vary.
//
// Skewed ids (the commonest token may take a tenth of the positions) are cut
// at fixed chunks of kChunk sorted entries: a run of equal ids inside one
// chunk is summed by the warp that owns the table row; a run that crosses a
// chunk boundary is first summed chunk by chunk into fp32 partial rows by
// other warps.  The longest serial sum is then kChunk rows plus one partial
// per chunk.
//
// Rows are read and written in 16-byte slots of the destination row, whatever
// the alignment of either (fw_rowslots.cuh).
#include <cuda_runtime.h>

#include <climits>

#include "fw_host.cuh"
#include "fw_rowslots.cuh"

namespace fwb200 {
namespace {

constexpr int kSlab = 4;         // slots per lane and step: 2 KB of a row per warp
constexpr int kChunk = 32;       // sorted entries per partial sum
constexpr int kSortThreads = 256;
constexpr int kSortItems = 8;
constexpr int kSortTile = kSortThreads * kSortItems;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxDigitBits = 9;
constexpr int kMaxBins = 1 << kMaxDigitBits;

__host__ __device__ constexpr int slots_of(int64_t D, int esize) {  // at any alignment
  return (int)((D * esize + 15) / 16 + 1);
}

template <class T>
__device__ __forceinline__ int dst_off(const T* row) {
  return (int)(reinterpret_cast<uintptr_t>(row) & 15u) / (int)sizeof(T);
}

struct EmbedArgs {
  const int64_t* ids;
  const void* w;
  void* out;
  int64_t T, V, D, ldw, ldo;
  float scale;
  int32_t* status;
  int nslabs;
};

template <class T>
__global__ void __launch_bounds__(256) fw_embed_rows_kernel(EmbedArgs a) {
  constexpr int V = 16 / sizeof(T);
  const int lane = threadIdx.x & 31;
  const int64_t nw = (int64_t)gridDim.x * (blockDim.x / 32);
  const int64_t work = a.T * a.nslabs;
  for (int64_t i = (int64_t)blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5); i < work; i += nw) {
    const int64_t t = i / a.nslabs;
    const int slab = (int)(i - t * a.nslabs);
    const int64_t id = a.ids[t];
    const bool ok = id >= 0 && id < a.V;
    if (!ok && lane == 0) raise_status(a.status, FWB_STATUS_LABEL_RANGE);
    const T* src = static_cast<const T*>(a.w) + (ok ? id : 0) * a.ldw;
    T* dst = static_cast<T*>(a.out) + t * a.ldo;
    const int off = dst_off(dst);
    uint4 u[kSlab];
#pragma unroll
    for (int k = 0; k < kSlab; ++k) {
      const int64_t e0 = (int64_t)((slab * kSlab + k) * 32 + lane) * V - off;
      u[k] = e0 < a.D ? load_slot_shifted(src, e0, a.D) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int k = 0; k < kSlab; ++k) {
      const int64_t e0 = (int64_t)((slab * kSlab + k) * 32 + lane) * V - off;
      if (a.scale != 1.0f || !ok) {
        float v[V];
        unpack16<T>(u[k], v);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = ok ? v[j] * a.scale : CUDART_NAN_F;
        u[k] = pack16<T>(v);
      }
      if (e0 < a.D) store_slot(dst, e0, a.D, true, u[k]);
    }
  }
}

// ------------------------------------------------------------ stable sort
// Entries are (key, position); key V marks tokens that give nothing (padding
// or out of range) and sorts behind every row.
struct SortArgs {
  const int64_t* ids;   // first pass: keys come from here
  const uint2* src;     // later passes
  uint2* dst;
  uint32_t* hist;       // [tiles, bins]
  int64_t T, V, padding;
  int shift, bits;
  int tiles;
  int32_t* status;
};

__device__ __forceinline__ uint2 sort_entry(const SortArgs& a, int64_t i, bool report) {
  if (a.src) return a.src[i];
  const int64_t id = a.ids[i];
  const bool ok = id >= 0 && id < a.V;
  if (!ok && report) raise_status(a.status, FWB_STATUS_LABEL_RANGE);
  return make_uint2(ok && id != a.padding ? (uint32_t)id : (uint32_t)a.V, (uint32_t)i);
}

// Ranks the tile's entries by digit, stably: after the call, entry i of this
// thread goes to (place of its digit) + cnt[warp][digit] + rank[i], and
// total[digit] is the tile's count.  Entry i of lane l of warp w is number
// w * 32 * kSortItems + 32 * i + l of the tile.
__device__ __forceinline__ void tile_rank(const uint32_t (&digit)[kSortItems], uint32_t (&rank)[kSortItems],
                                          uint32_t (*cnt)[kMaxBins + 1], uint32_t* total, int bins) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < kSortWarps * (kMaxBins + 1); i += kSortThreads) (&cnt[0][0])[i] = 0u;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSortItems; ++i) {
    const uint32_t d = digit[i];  // `bins` for entries past the end
    const uint32_t same = __match_any_sync(kFull, d);
    const uint32_t before = cnt[w][d];
    __syncwarp();
    if (lane == __ffs(same) - 1) cnt[w][d] = before + __popc(same);
    __syncwarp();
    rank[i] = before + __popc(same & ((1u << lane) - 1u));
  }
  __syncthreads();
  for (int d = threadIdx.x; d < bins; d += kSortThreads) {
    uint32_t run = 0u;
#pragma unroll
    for (int q = 0; q < kSortWarps; ++q) {
      const uint32_t c = cnt[q][d];
      cnt[q][d] = run;
      run += c;
    }
    total[d] = run;
  }
  __syncthreads();
}

// Exclusive scan of total[0 .. bins) in place by the whole CTA.
__device__ __forceinline__ void scan_bins(uint32_t* total, uint32_t* warp_sum, int bins) {
  constexpr int kPer = kMaxBins / kSortThreads;
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
  __shared__ uint32_t cnt[kSortWarps][kMaxBins + 1];
  __shared__ uint32_t total[kMaxBins], place[kMaxBins], warp_sum[kSortWarps];
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
  tile_rank(digit, rank, cnt, total, bins);
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
  scan_bins(total, warp_sum, bins);
#pragma unroll
  for (int i = 0; i < kSortItems; ++i)
    if (digit[i] < (uint32_t)bins) a.dst[total[digit[i]] + place[digit[i]] + cnt[w][digit[i]] + rank[i]] = ent[i];
}

// Up to one tile of tokens: all passes in one CTA, entries in shared memory.
__global__ void __launch_bounds__(kSortThreads) fw_sort_small_kernel(SortArgs a, int passes, int total_bits) {
  __shared__ uint32_t cnt[kSortWarps][kMaxBins + 1];
  __shared__ uint32_t total[kMaxBins], warp_sum[kSortWarps];
  __shared__ uint2 buf[kSortTile];
  const int bins = 1 << a.bits;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  uint2 ent[kSortItems];
  uint32_t digit[kSortItems], rank[kSortItems];
#pragma unroll
  for (int i = 0; i < kSortItems; ++i) {
    const int e = w * 32 * kSortItems + 32 * i + lane;
    ent[i] = e < a.T ? sort_entry(a, e, true) : make_uint2(0u, 0u);
  }
  for (int p = 0; p < passes; ++p) {
#pragma unroll
    for (int i = 0; i < kSortItems; ++i) {
      const int e = w * 32 * kSortItems + 32 * i + lane;
      if (p > 0 && e < a.T) ent[i] = buf[e];
      digit[i] = e < a.T ? (ent[i].x >> (p * a.bits)) & (bins - 1) : (uint32_t)bins;
    }
    tile_rank(digit, rank, cnt, total, bins);  // its barriers also end the reads of buf
    scan_bins(total, warp_sum, bins);
#pragma unroll
    for (int i = 0; i < kSortItems; ++i)
      if (digit[i] < (uint32_t)bins) buf[total[digit[i]] + cnt[w][digit[i]] + rank[i]] = ent[i];
    __syncthreads();
  }
  for (int e = threadIdx.x; e < a.T; e += kSortThreads) a.dst[e] = buf[e];
}

// ------------------------------------------------------------ row sums
struct EmbedGradArgs {
  const uint2* sorted;
  const void* g;
  void* dw;
  float* part;  // [2 * chunks, pitch]
  int64_t T, V, D, ldg, pitch;
  float scale;
  int nslabs;
};

// First sorted entry in [lo, hi) whose key is at least v; the whole warp.
__device__ __forceinline__ int64_t lower_bound_warp(const uint2* s, int64_t lo, int64_t hi, uint32_t v, int lane) {
  while (lo < hi) {
    const int64_t step = (hi - lo + 31) / 32;
    const int64_t at = lo + lane * step;
    const bool less = at < hi && s[at].x < v;
    const int c = __popc(__ballot_sync(kFull, less));
    const int64_t nhi = lo + c * step;
    if (c > 0) lo += (c - 1) * step + 1;
    hi = nhi < hi ? nhi : hi;
  }
  return lo;
}

// Adds rows sorted[i0 .. i1) of g, in that order, to the slots of this lane.
template <class T>
__device__ __forceinline__ void add_rows(const EmbedGradArgs& a, int64_t i0, int64_t i1, int64_t e0, float* acc) {
  constexpr int V = 16 / sizeof(T);
#pragma unroll 2
  for (int64_t i = i0; i < i1; ++i) {
    const T* row = static_cast<const T*>(a.g) + (int64_t)a.sorted[i].y * a.ldg;
    uint4 u[kSlab];
#pragma unroll
    for (int k = 0; k < kSlab; ++k) {
      const int64_t e = e0 + (int64_t)k * 32 * V;
      u[k] = e < a.D ? load_slot_shifted(row, e, a.D) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int k = 0; k < kSlab; ++k) {
      float v[V];
      unpack16<T>(u[k], v);
#pragma unroll
      for (int j = 0; j < V; ++j) acc[k * V + j] += v[j];
    }
  }
}

// Partial rows of the runs that cross a chunk boundary: row 2c is the part in
// chunk c of a run that began before it, row 2c + 1 the part of a run that
// begins in it and goes on.
template <class T>
__global__ void __launch_bounds__(256) fw_embed_part_kernel(EmbedGradArgs a) {
  constexpr int V = 16 / sizeof(T);
  const int lane = threadIdx.x & 31;
  const int64_t chunks = (a.T + kChunk - 1) / kChunk;
  const int64_t work = chunks * a.nslabs;
  const int64_t nw = (int64_t)gridDim.x * (blockDim.x / 32);
  for (int64_t i = (int64_t)blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5); i < work; i += nw) {
    const int64_t c = i / a.nslabs;
    const int slab = (int)(i - c * a.nslabs);
    const int64_t b = c * kChunk, n = min((int64_t)kChunk, a.T - b);
    const uint32_t key = lane < n ? a.sorted[b + lane].x : 0xffffffffu;
    const uint32_t first = __shfl_sync(kFull, key, 0), last = __shfl_sync(kFull, key, (int)n - 1);
    const bool from = b > 0 && a.sorted[b - 1].x == first;
    const bool on = b + n < a.T && a.sorted[b + n].x == last;
    for (int half = 0; half < 2; ++half) {
      int64_t i0 = b, i1 = b + n;
      if (half == 0) {
        if (!from || first >= (uint32_t)a.V) continue;
        i1 = b + __popc(__ballot_sync(kFull, lane < n && key == first));
      } else {
        if (!on || last >= (uint32_t)a.V || (from && first == last)) continue;
        i0 = b + n - __popc(__ballot_sync(kFull, lane < n && key == last));
      }
      float acc[kSlab * V];
#pragma unroll
      for (int j = 0; j < kSlab * V; ++j) acc[j] = 0.0f;
      const int64_t e0 = (int64_t)(slab * kSlab * 32 + lane) * V;
      add_rows<T>(a, i0, i1, e0, acc);
      float* out = a.part + (2 * c + half) * a.pitch;
#pragma unroll
      for (int k = 0; k < kSlab; ++k) {
        const int64_t e = e0 + (int64_t)k * 32 * V;
        if (e < a.D) {
#pragma unroll
          for (int j = 0; j < V; j += 4)  // pitch is a multiple of V
            *reinterpret_cast<float4*>(out + e + j) =
                make_float4(acc[k * V + j], acc[k * V + j + 1], acc[k * V + j + 2], acc[k * V + j + 3]);
        }
      }
    }
  }
}

// One warp per table row.
template <class T>
__global__ void __launch_bounds__(256) fw_embed_grad_kernel(EmbedGradArgs a) {
  constexpr int V = 16 / sizeof(T);
  const int lane = threadIdx.x & 31;
  const int64_t nw = (int64_t)gridDim.x * (blockDim.x / 32);
  for (int64_t v = (int64_t)blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5); v < a.V; v += nw) {
    const int64_t i0 = lower_bound_warp(a.sorted, 0, a.T, (uint32_t)v, lane);
    const uint32_t hit = __ballot_sync(kFull, i0 + lane < a.T && a.sorted[i0 + lane].x == (uint32_t)v);
    int64_t i1 = i0 + __popc(hit);
    if (hit == kFull) i1 = lower_bound_warp(a.sorted, i1, a.T, (uint32_t)v + 1u, lane);
    const int64_t c0 = i0 / kChunk, c1 = i1 > i0 ? (i1 - 1) / kChunk : c0;
    T* dst = static_cast<T*>(a.dw) + v * a.D;
    const int off = dst_off(dst);
    for (int slab = 0; slab < a.nslabs; ++slab) {
      float acc[kSlab * V];
#pragma unroll
      for (int j = 0; j < kSlab * V; ++j) acc[j] = 0.0f;
      const int64_t e0 = (int64_t)(slab * kSlab * 32 + lane) * V - off;
      if (c0 == c1) {
        add_rows<T>(a, i0, i1, e0, acc);
      } else {
        for (int64_t c = c0; c <= c1; ++c) {
          const float* p = a.part + (2 * c + (c == c0 ? 1 : 0)) * a.pitch;
#pragma unroll
          for (int j = 0; j < kSlab * V; ++j) {
            const int64_t e = e0 + (int64_t)(j / V) * 32 * V + j % V;
            if (e >= 0 && e < a.D) acc[j] += p[e];
          }
        }
      }
#pragma unroll
      for (int k = 0; k < kSlab; ++k) {
        const int64_t e = e0 + (int64_t)k * 32 * V;
        if (e >= a.D) continue;
        float s[V];
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] = acc[k * V + j] * a.scale;
        store_slot(dst, e, a.D, true, pack16<T>(s));
      }
    }
  }
}

struct EmbedPlan {
  int passes, bits;
  int64_t tiles, chunks, pitch;
  int64_t hist_at, part_at, bytes;  // workspace: two entry arrays, histograms, partial rows
};

EmbedPlan embed_plan(int64_t T, int64_t V, int64_t D) {
  EmbedPlan p = {};
  int total = 1;
  while (((int64_t)1 << total) <= V) ++total;  // keys 0 .. V
  p.passes = (total + kMaxDigitBits - 1) / kMaxDigitBits;
  p.bits = (total + p.passes - 1) / p.passes;
  p.tiles = (T + kSortTile - 1) / kSortTile;
  p.chunks = (T + kChunk - 1) / kChunk;
  p.pitch = (D + 7) / 8 * 8;
  p.hist_at = (2 * T * (int64_t)sizeof(uint2) + 255) / 256 * 256;
  p.part_at = (p.hist_at + p.tiles * ((int64_t)4 << p.bits) + 255) / 256 * 256;
  p.bytes = p.part_at + (p.chunks > 1 ? 2 * p.chunks * p.pitch * 4 : 0);
  return p;
}

bool embed_sizes_ok(int64_t T, int64_t V, int64_t D) {
  return T >= 0 && V >= 1 && D >= 1 && T <= (int64_t)INT_MAX - kSortTile && V <= (int64_t)INT_MAX - 1 &&
         D <= (int64_t)1 << 24;
}

template <class T>
cudaError_t launch_embed_grad(const EmbedGradArgs& a, int64_t chunks, cudaStream_t st) {
  if (chunks > 1) {
    const int64_t warps = chunks * a.nslabs;
    const int64_t g = (warps + 7) / 8, cap = (int64_t)sm_count() * 64;
    fw_embed_part_kernel<T><<<(unsigned)(g < cap ? g : cap), 256, 0, st>>>(a);
  }
  const int64_t g = (a.V + 7) / 8, cap = (int64_t)sm_count() * 64;
  fw_embed_grad_kernel<T><<<(unsigned)(g < cap ? g : cap), 256, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace
}  // namespace fwb200

using namespace fwb200;

extern "C" {

int fw_embed_rows(int dtype, const int64_t* ids, int64_t T, const void* weight, int64_t ldw, int64_t V, int64_t D,
                  float scale, void* out, int64_t ldo, int32_t* status, void* stream) {
  if (dtype != FWB_DTYPE_F32 && dtype != FWB_DTYPE_BF16 && dtype != FWB_DTYPE_F16) return FWB_E_DTYPE;
  if (!embed_sizes_ok(T, V, D) || ldw < D || ldo < D || ldw > ((int64_t)1 << 60) / V) return FWB_E_SHAPE;
  if (T == 0) return FWB_OK;
  if (ldo > ((int64_t)1 << 60) / T) return FWB_E_SHAPE;
  if (!ids || !weight || !out) return FWB_E_POINTER;
  const int es = dtype == FWB_DTYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(weight) % es || reinterpret_cast<uintptr_t>(out) % es) return FWB_E_POINTER;
  EmbedArgs a = {ids, weight, out, T, V, D, ldw, ldo, scale, status, 0};
  a.nslabs = (slots_of(D, es) + 32 * kSlab - 1) / (32 * kSlab);
  const int64_t need = (T * a.nslabs + 7) / 8, cap = (int64_t)sm_count() * 64;
  const unsigned grid = (unsigned)(need < cap ? need : cap);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == FWB_DTYPE_BF16) fw_embed_rows_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a);
  else if (dtype == FWB_DTYPE_F16) fw_embed_rows_kernel<__half><<<grid, 256, 0, st>>>(a);
  else fw_embed_rows_kernel<float><<<grid, 256, 0, st>>>(a);
  return launch_status(cudaGetLastError());
}

int64_t fw_embed_grad_workspace(int64_t T, int64_t V, int64_t D) {
  return embed_sizes_ok(T, V, D) ? embed_plan(T, V, D).bytes : 0;
}

int fw_embed_grad(int dtype, const int64_t* ids, int64_t T, const void* grad, int64_t ldg, int64_t V, int64_t D,
                  float scale, int64_t padding, void* dweight, void* workspace, int64_t workspace_bytes,
                  int32_t* status, void* stream) {
  if (dtype != FWB_DTYPE_F32 && dtype != FWB_DTYPE_BF16 && dtype != FWB_DTYPE_F16) return FWB_E_DTYPE;
  if (!embed_sizes_ok(T, V, D) || ldg < D || (T > 0 && ldg > ((int64_t)1 << 60) / T)) return FWB_E_SHAPE;
  if (!dweight) return FWB_E_POINTER;
  const int es = dtype == FWB_DTYPE_F32 ? 4 : 2;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (T == 0) return cudaMemsetAsync(dweight, 0, (size_t)(V * D * es), st) == cudaSuccess ? FWB_OK : FWB_E_LAUNCH;
  if (!ids || !grad || !workspace) return FWB_E_POINTER;
  if (reinterpret_cast<uintptr_t>(grad) % es || reinterpret_cast<uintptr_t>(dweight) % es || !aligned16(workspace))
    return FWB_E_POINTER;
  const EmbedPlan p = embed_plan(T, V, D);
  if (workspace_bytes < p.bytes) return FWB_E_CAPACITY;
  char* ws = static_cast<char*>(workspace);
  uint2* ent[2] = {reinterpret_cast<uint2*>(ws), reinterpret_cast<uint2*>(ws) + T};
  SortArgs s = {};
  s.ids = ids;
  s.hist = reinterpret_cast<uint32_t*>(ws + p.hist_at);
  s.T = T;
  s.V = V;
  s.padding = padding;
  s.bits = p.bits;
  s.tiles = (int)p.tiles;
  s.status = status;
  const uint2* sorted;
  if (p.tiles == 1) {
    s.dst = ent[0];
    fw_sort_small_kernel<<<1, kSortThreads, 0, st>>>(s, p.passes, p.bits * p.passes);
    sorted = ent[0];
  } else {
    for (int i = 0; i < p.passes; ++i) {
      s.src = i == 0 ? nullptr : ent[(i - 1) & 1];
      s.dst = ent[i & 1];
      s.shift = i * p.bits;
      fw_sort_hist_kernel<<<(unsigned)p.tiles, kSortThreads, 0, st>>>(s);
      fw_sort_scatter_kernel<<<(unsigned)p.tiles, kSortThreads, 0, st>>>(s);
    }
    sorted = ent[(p.passes - 1) & 1];
  }
  if (cudaGetLastError() != cudaSuccess) return FWB_E_LAUNCH;
  EmbedGradArgs a = {};
  a.sorted = sorted;
  a.g = grad;
  a.dw = dweight;
  a.part = reinterpret_cast<float*>(ws + p.part_at);
  a.T = T;
  a.V = V;
  a.D = D;
  a.ldg = ldg;
  a.pitch = p.pitch;
  a.scale = scale;
  a.nslabs = (slots_of(D, es) + 32 * kSlab - 1) / (32 * kSlab);
  return launch_status(dtype == FWB_DTYPE_BF16  ? launch_embed_grad<__nv_bfloat16>(a, p.chunks, st)
                       : dtype == FWB_DTYPE_F16 ? launch_embed_grad<__half>(a, p.chunks, st)
                                                : launch_embed_grad<float>(a, p.chunks, st));
}

}  // extern "C"
