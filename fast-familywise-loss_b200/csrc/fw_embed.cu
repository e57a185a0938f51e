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
// The sort is one launch, a cluster of 8 CTAs that exchange digit counts and
// entries through distributed shared memory, up to kClusterTokens tokens, and
// two launches per digit beyond.  For few tokens and a small table nothing is
// sorted: every warp finds its row's positions in the list itself.
//
// Skewed ids (the commonest token may take a tenth of the positions) do not
// unbalance the sums: a warp takes kChunk sorted entries and 512 bytes of
// their rows, whoever they belong to, with kAhead rows in flight.  A run of
// equal ids that ends inside its chunk is finished there and its table row
// written; the parts of a run that crosses chunks go to fp32 partial rows,
// which a last small launch adds up in order.
//
// The rows of dW without a token, most of the bytes for a large vocabulary,
// are zeroed by CTAs that run beside the sort (each marks its rows' tokens in
// a bitmap, from the unsorted list), or beside the sums for more tokens than
// one cluster sorts.
//
// Rows are read and written in 16-byte slots of the destination row, whatever
// the alignment of either (fw_rowslots.cuh).
//
// bfloat16, 32768 tokens (11998 different ones), 128256 x 4096: lookup and
// gradient 307 us for 1.69 GB, 5.5 TB/s, of which the lookup 65, sort and
// zeroing 160, the sums 59, the join 20.  8191 tokens, 32000 x 2048: 60 us.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <climits>

#include "fw_host.cuh"
#include "fw_rowslots.cuh"

namespace fwb200 {
namespace {

constexpr int kSlab = 4;         // slots per lane and step: 2 KB of a row per warp
constexpr int kChunk = 32;       // sorted entries per warp
constexpr int kAhead = 8;        // rows of g in flight per warp
constexpr int kSortThreads = 256;
constexpr int kSortItems = 8;
constexpr int kSortTile = kSortThreads * kSortItems;
constexpr int kClusterCtas = 8;
constexpr int kClusterThreads = 512;
constexpr int kClusterTile = kClusterThreads * kSortItems;
// Sorted by one cluster; 32768 tokens, 128256 x 4096: 307 us in all, 336 with
// two launches per digit; 8191 tokens, 32000 x 2048: 71 and 86.
constexpr int kClusterTokens = kClusterCtas * kClusterTile;
constexpr int kMaxDigitBits = 9;
constexpr int kMaxBins = 1 << kMaxDigitBits;

// Few tokens and a small table: no sort.  64 tokens, 1000 x 1024 bfloat16: 3.9
// us against 18 sorted; 250 tokens, 8000 x 1024: 13 against 21; 16000 x 1024:
// 23 against 20 (every part of a row searches the list of ids again).
constexpr int kDirectTokens = 256;
constexpr int64_t kDirectElems = (int64_t)1 << 23;  // of the table

// Slots that a row of the matrix covers at most: one more than its elements
// fill where a row may start inside a slot.
int slots_of(const void* base, int64_t ld, int64_t D, int esize) {
  const bool inside = !aligned16(base) || ld * esize % 16 != 0;
  return (int)((D * esize + 15) / 16 + (inside ? 1 : 0));
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
  int nsteps, nslabs;  // 32 slots each; parts of at most kSlab of them
};

template <class T>
__global__ void __launch_bounds__(256) fw_embed_rows_kernel(EmbedArgs a) {
  constexpr int V = 16 / sizeof(T);
  wait_prior_kernel();
  allow_dependent_launch();
  const int lane = threadIdx.x & 31;
  const int64_t nw = (int64_t)gridDim.x * (blockDim.x / 32);
  const int64_t work = a.T * a.nslabs;
  const int D = (int)a.D, steps = (a.nsteps + a.nslabs - 1) / a.nslabs;  // of 32 slots, per slab
  const Span<T> table(a.w, a.V, a.ldw, a.D);
  for (int64_t i = (int64_t)blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5); i < work; i += nw) {
    const int64_t t = i / a.nslabs;
    const int slab = (int)(i - t * a.nslabs);
    const int64_t id = a.ids[t];
    const bool ok = id >= 0 && id < a.V;
    if (!ok && lane == 0) raise_status(a.status, FWB_STATUS_LABEL_RANGE);
    const T* src = static_cast<const T*>(a.w) + (ok ? id : 0) * a.ldw;
    T* dst = static_cast<T*>(a.out) + t * a.ldo;
    const int off = dst_off(dst), first = slab * steps;
    uint4 u[kSlab];
#pragma unroll
    for (int k = 0; k < kSlab; ++k) {
      const int e0 = ((first + k) * 32 + lane) * V - off;
      u[k] = k < steps && e0 < D ? load_slot_shifted(src, e0, table) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int k = 0; k < kSlab; ++k) {
      const int e0 = ((first + k) * 32 + lane) * V - off;
      if (a.scale != 1.0f || !ok) {
        float v[V];
        unpack16<T>(u[k], v);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = ok ? v[j] * a.scale : CUDART_NAN_F;
        u[k] = pack_slot<T>(v);
      }
      if (k < steps && e0 < D) store_slot(dst, e0, D, true, u[k]);
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

// Zeroes row v of dw: the lanes of a warp over its slots.
template <class T, bool ALIGNED>
__device__ __forceinline__ void zero_row(T* dst, int64_t D, int nslots, int lane) {
  constexpr int V = 16 / sizeof(T);
  const int64_t off = ALIGNED ? 0 : dst_off(dst);
#pragma unroll 4
  for (int64_t slot = lane; slot < nslots; slot += 32) {
    const int64_t e0 = slot * V - off;
    if (e0 >= D) continue;
    if (ALIGNED)
      *reinterpret_cast<uint4*>(dst + e0) = make_uint4(0u, 0u, 0u, 0u);
    else
      store_slot(dst, e0, D, true, make_uint4(0u, 0u, 0u, 0u));
  }
}

struct ZeroArgs {
  void* dw;
  int64_t D;
  int nslots;
  int rows;  // rows per CTA, at most kZeroRows
};

constexpr int kZeroRows = 1024;

// Rows first .. first + a.rows of dw that no entry names, by a whole CTA.
template <class T, bool ALIGNED>
__device__ __forceinline__ void zero_unnamed(const SortArgs& s, const ZeroArgs& z, int64_t first, uint32_t* named) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < kZeroRows / 32; i += kClusterThreads) named[i] = 0u;
  __syncthreads();
#pragma unroll 4
  for (int64_t t = threadIdx.x; t < s.T; t += kClusterThreads) {
    const int64_t r = s.ids[t] - first;
    if (r >= 0 && r < z.rows && r + first != s.padding) atomicOr(&named[r >> 5], 1u << (r & 31));
  }
  __syncthreads();
  const int n = (int)min((int64_t)z.rows, s.V - first);
  for (int r = w; r < n; r += kClusterThreads / 32)
    if (!(named[r >> 5] >> (r & 31) & 1u))
      zero_row<T, ALIGNED>(static_cast<T*>(z.dw) + (first + r) * z.D, z.D, z.nslots, lane);
}

// All passes in one launch: a cluster holds the entries in shared memory, CTA
// c the entries c * per .. of the current order.  Per pass the CTAs rank their
// own entries, read each other's digit counts, and store every entry where it
// belongs in the cluster.  The grid's other clusters zero.
template <class TW, bool ALIGNED>
__global__ void __launch_bounds__(kClusterThreads, 2) fw_sort_cluster_kernel(SortArgs a, int passes, ZeroArgs z) {
  wait_prior_kernel();
  allow_dependent_launch();
  namespace cg = cooperative_groups;
  cg::cluster_group cl = cg::this_cluster();
  extern __shared__ __align__(16) unsigned char sort_smem[];
  uint2* buf = reinterpret_cast<uint2*>(sort_smem);  // two halves of kClusterTile entries
  uint16_t(*cnt)[kMaxBins + 2] = reinterpret_cast<uint16_t(*)[kMaxBins + 2]>(sort_smem + 2 * kClusterTile * sizeof(uint2));
  __shared__ uint32_t total[kMaxBins], base[kMaxBins], warp_sum[kClusterThreads / 32];
  const int bins = 1 << a.bits;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int nc = (int)cl.num_blocks(), me = (int)cl.block_rank();
  if ((int)blockIdx.x >= nc) {
    for (int64_t v = (int64_t)(blockIdx.x - nc) * z.rows; v < a.V; v += (int64_t)(gridDim.x - nc) * z.rows) {
      zero_unnamed<TW, ALIGNED>(a, z, v, total);
      __syncthreads();
    }
    return;
  }
  const int T = (int)a.T;
  const int per = (T + nc - 1) / nc;
  const int first = me * per, mine = max(0, min(per, T - first));
  uint2 ent[kSortItems];
  uint32_t digit[kSortItems], rank[kSortItems];
#pragma unroll
  for (int i = 0; i < kSortItems; ++i) {
    const int e = w * 32 * kSortItems + 32 * i + lane;
    ent[i] = e < mine ? sort_entry(a, first + e, true) : make_uint2(0u, 0u);
  }
  for (int p = 0; p < passes; ++p) {
#pragma unroll
    for (int i = 0; i < kSortItems; ++i) {
      const int e = w * 32 * kSortItems + 32 * i + lane;
      if (p > 0 && e < mine) ent[i] = buf[(p & 1) * kClusterTile + e];
      digit[i] = e < mine ? (ent[i].x >> (p * a.bits)) & (bins - 1) : (uint32_t)bins;
    }
    tile_rank<kClusterThreads>(digit, rank, cnt, total, bins);
    cl.sync();  // the counts of every CTA are in place
    uint32_t before[kMaxBins / kClusterThreads], all[kMaxBins / kClusterThreads];
#pragma unroll
    for (int k = 0; k < kMaxBins / kClusterThreads; ++k) {
      const int d = k * kClusterThreads + threadIdx.x;
      before[k] = all[k] = 0u;
      if (d < bins)
        for (int q = 0; q < nc; ++q) {
          const uint32_t c = cl.map_shared_rank(total, q)[d];
          before[k] += q < me ? c : 0u;
          all[k] += c;
        }
    }
#pragma unroll
    for (int k = 0; k < kMaxBins / kClusterThreads; ++k) {
      const int d = k * kClusterThreads + threadIdx.x;
      if (d < bins) base[d] = all[k];
    }
    __syncthreads();
    scan_bins<kClusterThreads>(base, warp_sum, bins);
#pragma unroll
    for (int k = 0; k < kMaxBins / kClusterThreads; ++k) {
      const int d = k * kClusterThreads + threadIdx.x;
      if (d < bins) base[d] += before[k];
    }
    __syncthreads();
    const bool end = p == passes - 1;
    uint2* next = buf + ((p + 1) & 1) * kClusterTile;
#pragma unroll
    for (int i = 0; i < kSortItems; ++i) {
      if (digit[i] >= (uint32_t)bins) continue;
      const int to = (int)(base[digit[i]] + cnt[w][digit[i]] + rank[i]);
      if (end)
        a.dst[to] = ent[i];
      else
        cl.map_shared_rank(next, to / per)[to % per] = ent[i];
    }
    cl.sync();  // entries in place; nobody reads these counts any more
  }
}

// ------------------------------------------------------------ row sums
struct EmbedGradArgs {
  const uint2* sorted;
  const int64_t* ids;  // direct form
  const void* g;
  void* dw;
  float* part;  // [2 * chunks, pitch]
  int64_t T, V, D, ldg, pitch, padding;
  float scale;
  int nslots;       // slots of a row, at any alignment
  int sum_blocks;   // CTAs that add rows; the others zero
  int32_t* status;
};

template <class T, bool ALIGNED>
__device__ __forceinline__ void store_sum(const EmbedGradArgs& a, T* dst, int e0, const float* acc) {
  constexpr int V = 16 / sizeof(T);
  if (e0 >= a.D) return;
  float s[V];
#pragma unroll
  for (int j = 0; j < V; ++j) s[j] = acc[j] * a.scale;
  if (ALIGNED)
    *reinterpret_cast<uint4*>(dst + e0) = pack_slot<T>(s);
  else
    store_slot(dst, e0, a.D, true, pack_slot<T>(s));
}

// Start of slot `slot` in the row at dst: every row's own slots, so that a
// run's partial rows (kept by slot) and its table row agree.
template <class T, bool ALIGNED>
__device__ __forceinline__ int slot_elem(const T* dst, int slot) {
  constexpr int V = 16 / sizeof(T);
  return slot * V - (ALIGNED ? 0 : dst_off(dst));
}

// Adds the rows of chunk c, slots slot .. of which this lane has one, in
// order.  Partial row 2c is the part of a run that began in an earlier chunk,
// 2c + 1 the part of a run that begins here and goes on.
template <class T, bool ALIGNED>
__device__ __forceinline__ void sum_chunk(const EmbedGradArgs& a, const Span<T>& span, int64_t c, int slot, int lane) {
  constexpr int V = 16 / sizeof(T);
  const int64_t b = c * kChunk;
  const int n = (int)min((int64_t)kChunk, a.T - b);
  const uint2 ent = lane < n ? a.sorted[b + lane] : make_uint2((uint32_t)a.V, 0u);
  const uint32_t first = __shfl_sync(kFull, ent.x, 0), last = __shfl_sync(kFull, ent.x, n - 1);
  const bool from = b > 0 && a.sorted[b - 1].x == first;
  const bool on = b + n < a.T && a.sorted[b + n].x == last;
  // per entry, as bits: its run begins here / ends here, and where the sum goes
  const uint32_t up = __shfl_up_sync(kFull, ent.x, 1), down = __shfl_down_sync(kFull, ent.x, 1);
  const uint32_t begins = __ballot_sync(kFull, lane == 0 || up != ent.x);
  const uint32_t ends = __ballot_sync(kFull, lane == n - 1 || down != ent.x);
  const uint32_t to0 = __ballot_sync(kFull, from && ent.x == first);
  const uint32_t to1 = __ballot_sync(kFull, on && ent.x == last) & ~to0;
  const int live = __popc(__ballot_sync(kFull, ent.x < (uint32_t)a.V));  // the others sort behind
  float acc[V];
  for (int i0 = 0; i0 < live; i0 += kAhead) {
    uint4 u[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const T* row = static_cast<const T*>(a.g) + (int64_t)__shfl_sync(kFull, ent.y, (i0 + i) & 31) * a.ldg;
      int e0 = slot * V;
      if (!ALIGNED)
        e0 -= dst_off(static_cast<const T*>(a.dw) + (int64_t)__shfl_sync(kFull, ent.x, (i0 + i) & 31) * a.D);
      u[i] = i0 + i >= live || e0 >= a.D ? make_uint4(0u, 0u, 0u, 0u)
             : ALIGNED                   ? ld_global16_once(row + e0)
                                         : load_slot_shifted(row, e0, span);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int at = i0 + i;
      if (at >= live) break;
      float v[V];
      unpack16<T>(u[i], v);
      const bool begin = begins >> at & 1u;
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] = begin ? v[j] : acc[j] + v[j];
      if (!(ends >> at & 1u)) continue;
      if (!((to0 | to1) >> at & 1u)) {
        T* dst = static_cast<T*>(a.dw) + (int64_t)__shfl_sync(kFull, ent.x, at) * a.D;
        store_sum<T, ALIGNED>(a, dst, slot_elem<T, ALIGNED>(dst, slot), acc);
      } else if (slot < a.nslots) {
        float* out = a.part + (2 * c + (to1 >> at & 1u)) * a.pitch + slot * V;
#pragma unroll
        for (int j = 0; j < V; j += 4)
          *reinterpret_cast<float4*>(out + j) = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
      }
    }
  }
}

// sum_blocks of the CTAs add; the others, spread among them (more tokens than
// one cluster sorts), look for the rows without a token and zero them: 8 rows
// per warp, one binary search per lane.
template <class T, bool ALIGNED>
__global__ void __launch_bounds__(256, ALIGNED ? 4 : 2) fw_embed_sum_kernel(EmbedGradArgs a) {
  wait_prior_kernel();
  allow_dependent_launch();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const Span<T> span(a.g, a.T, a.ldg, a.D);
  const int64_t total = gridDim.x, adding = a.sum_blocks;
  const int64_t before = blockIdx.x * adding / total;  // adding CTAs ahead of this one
  if ((blockIdx.x + 1) * adding / total != before) {
    const int64_t slabs = (a.nslots + 31) / 32;
    const int64_t work = (a.T + kChunk - 1) / kChunk * slabs;
    for (int64_t i = before * 8 + w; i < work; i += adding * 8)
      sum_chunk<T, ALIGNED>(a, span, i / slabs, (int)(i % slabs) * 32 + lane, lane);
    return;
  }
  for (int64_t v0 = ((blockIdx.x - before) * 8 + w) * 8; v0 < a.V; v0 += (total - adding) * 64) {
    const int64_t v = v0 + (lane & 7);
    int64_t lo = 0, hi = a.T;  // first entry whose key is at least v
    while (lo < hi) {
      const int64_t mid = (lo + hi) / 2;
      if (a.sorted[mid].x < (uint32_t)v)
        lo = mid + 1;
      else
        hi = mid;
    }
    const bool none = v < a.V && !(lo < a.T && a.sorted[lo].x == (uint32_t)v);
    for (uint32_t empty = __ballot_sync(kFull, none) & 0xffu; empty != 0u; empty &= empty - 1u)
      zero_row<T, ALIGNED>(static_cast<T*>(a.dw) + (v0 + __ffs(empty) - 1) * a.D, a.D, a.nslots, lane);
  }
}

// Runs that cross chunks: one warp per chunk that such a run begins in and
// slab of its row; runs of more than kJoinAlone parts by the eight warps of
// the CTA, a stretch of parts each (its items are eight chunks of one slab, so
// that one long run asks for one CTA per slab).
constexpr int kJoinAlone = 16;

template <class T, bool ALIGNED>
__global__ void __launch_bounds__(256) fw_embed_join_kernel(EmbedGradArgs a) {
  constexpr int V = 16 / sizeof(T);
  __shared__ int64_t count[8];  // parts of the run of each warp's item, 0 for none
  __shared__ float4 stretch[8][V / 4][32];
  wait_prior_kernel();
  allow_dependent_launch();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t slabs = (a.nslots + 31) / 32, chunks = (a.T + kChunk - 1) / kChunk;
  const int64_t groups = (chunks + 7) / 8, work = groups * slabs;
  for (int64_t i = blockIdx.x; i < work; i += gridDim.x) {
    const int64_t c0 = i % groups * 8, c = c0 + w, b = c * kChunk;
    const int slot = (int)(i / groups) * 32 + lane;
    int64_t n = 0;
    if (b + kChunk < a.T) {
      const uint32_t key = a.sorted[b + kChunk - 1].x;
      const bool on = key < (uint32_t)a.V && a.sorted[b + kChunk].x == key;
      const bool earlier = a.sorted[b].x == key && b > 0 && a.sorted[b - 1].x == key;
      if (on && !earlier) {
        n = 2;  // its parts, found 32 chunks at a time
        for (;;) {
          const int64_t next = c + n + lane;  // does chunk `next` begin with the key?
          const uint32_t more = __ballot_sync(kFull, next < chunks && a.sorted[next * kChunk].x == key);
          n += more == kFull ? 32 : __ffs(~more) - 1;
          if (more != kFull) break;
        }
      }
    }
    // parts from .. to of the run that begins in chunk c, in order
    auto add = [&](int64_t c, int64_t from, int64_t to, float* acc) {
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] = 0.0f;
      if (slot >= a.nslots) return;
#pragma unroll 8
      for (int64_t q = from; q < to; ++q) {
        const float4* p = reinterpret_cast<const float4*>(a.part + (2 * (c + q) + (q == 0 ? 1 : 0)) * a.pitch + slot * V);
#pragma unroll
        for (int j = 0; j < V / 4; ++j) {
          const float4 x = p[j];
          acc[4 * j] += x.x, acc[4 * j + 1] += x.y, acc[4 * j + 2] += x.z, acc[4 * j + 3] += x.w;
        }
      }
    };
    auto store = [&](int64_t c, const float* acc) {
      T* dst = static_cast<T*>(a.dw) + (int64_t)a.sorted[c * kChunk + kChunk - 1].x * a.D;
      if (slot < a.nslots) store_sum<T, ALIGNED>(a, dst, slot_elem<T, ALIGNED>(dst, slot), acc);
    };
    float acc[V];
    if (n > 0 && n <= kJoinAlone) {
      add(c, 0, n, acc);
      store(c, acc);
    }
    if (lane == 0) count[w] = n;
    __syncthreads();
    for (int k = 0; k < 8; ++k) {
      const int64_t parts = count[k];
      if (parts <= kJoinAlone) continue;
      add(c0 + k, parts * w / 8, parts * (w + 1) / 8, acc);
#pragma unroll
      for (int j = 0; j < V / 4; ++j)
        stretch[w][j][lane] = make_float4(acc[4 * j], acc[4 * j + 1], acc[4 * j + 2], acc[4 * j + 3]);
      __syncthreads();
      if (w == 0) {
        for (int q = 1; q < 8; ++q)
#pragma unroll
          for (int j = 0; j < V / 4; ++j) {
            const float4 x = stretch[q][j][lane];
            acc[4 * j] += x.x, acc[4 * j + 1] += x.y, acc[4 * j + 2] += x.z, acc[4 * j + 3] += x.w;
          }
        store(c0 + k, acc);
      }
      __syncthreads();
    }
    __syncthreads();
  }
}

// Few tokens: every warp looks for its row in the list of ids.
template <class T, bool ALIGNED>
__global__ void __launch_bounds__(256) fw_embed_direct_kernel(EmbedGradArgs a) {
  constexpr int V = 16 / sizeof(T);
  wait_prior_kernel();
  allow_dependent_launch();
  __shared__ int32_t key[kDirectTokens];
  const int n = (int)a.T;
  const Span<T> span(a.g, a.T, a.ldg, a.D);
  for (int i = threadIdx.x; i < kDirectTokens; i += 256) {
    const int64_t id = i < n ? a.ids[i] : -1;
    const bool ok = id >= 0 && id < a.V;
    if (i < n && !ok && blockIdx.x == 0) raise_status(a.status, FWB_STATUS_LABEL_RANGE);
    key[i] = ok && id != a.padding ? (int32_t)id : -1;
  }
  __syncthreads();
  const int lane = threadIdx.x & 31;
  const int64_t slabs = (a.nslots + 31) / 32;
  const int64_t nw = (int64_t)gridDim.x * (blockDim.x / 32), work = a.V * slabs;
  for (int64_t w = (int64_t)blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5); w < work; w += nw) {
    const int64_t v = w / slabs;
    T* dst = static_cast<T*>(a.dw) + v * a.D;
    const int e0 = slot_elem<T, ALIGNED>(dst, (int)(w % slabs) * 32 + lane);
    float acc[V];
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = 0.0f;
    for (int t0 = 0; t0 < n; t0 += 32) {
      uint32_t hit = __ballot_sync(kFull, key[t0 + lane] == (int32_t)v);
      if (e0 >= a.D) continue;
#pragma unroll 4
      for (; hit != 0u; hit &= hit - 1u) {
        const T* row = static_cast<const T*>(a.g) + (int64_t)(t0 + __ffs(hit) - 1) * a.ldg;
        float x[V];
        unpack16<T>(ALIGNED ? ld_global16_once(row + e0) : load_slot_shifted(row, e0, span), x);
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] += x[j];
      }
    }
    store_sum<T, ALIGNED>(a, dst, e0, acc);
  }
}

struct EmbedPlan {
  int passes, bits;
  int64_t tiles, chunks, pitch;
  int64_t hist_at, part_at, bytes;  // workspace: entries, histograms, partial rows
};

bool direct_form(int64_t T, int64_t V, int64_t D) { return T <= kDirectTokens && V * D <= kDirectElems; }

EmbedPlan embed_plan(int64_t T, int64_t V, int64_t D) {
  EmbedPlan p = {};
  int total = 1;
  while (((int64_t)1 << total) <= V) ++total;  // keys 0 .. V
  p.passes = (total + kMaxDigitBits - 1) / kMaxDigitBits;
  p.bits = (total + p.passes - 1) / p.passes;
  p.tiles = (T + kSortTile - 1) / kSortTile;
  p.chunks = (T + kChunk - 1) / kChunk;
  p.pitch = (D + 7) / 8 * 8 + 8;  // whole slots at any alignment
  const bool one = T <= kClusterTokens;
  p.hist_at = ((one ? 1 : 2) * T * (int64_t)sizeof(uint2) + 255) / 256 * 256;
  p.part_at = (p.hist_at + (one ? 0 : p.tiles * ((int64_t)4 << p.bits)) + 255) / 256 * 256;
  p.bytes = p.part_at + 2 * p.chunks * p.pitch * 4;
  return p;
}

bool embed_sizes_ok(int64_t T, int64_t V, int64_t D) {
  return T >= 0 && V >= 1 && D >= 1 && T <= (int64_t)INT_MAX - kSortTile && V <= (int64_t)INT_MAX - 1 &&
         D <= (int64_t)1 << 24;
}

unsigned warps_grid(int64_t warps) {
  const int64_t need = (warps + 7) / 8, cap = (int64_t)sm_count() * 64;
  return (unsigned)(need < cap ? need : cap);
}

template <class T, bool ALIGNED>
cudaError_t sort_cluster(const SortArgs& s, int passes, const EmbedGradArgs& g, cudaStream_t st) {
  constexpr int kSmem = 2 * kClusterTile * (int)sizeof(uint2) + kClusterThreads / 32 * (kMaxBins + 2) * 2;
  auto kernel = fw_sort_cluster_kernel<T, ALIGNED>;
  static std::atomic<bool> attr_set[kMaxDevices] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= kMaxDevices || !attr_set[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    if (dev < kMaxDevices) attr_set[dev].store(true, std::memory_order_release);
  }
  // as many sorting CTAs as the tokens ask for, so that few do not exchange with idle ones
  int ctas = 1;
  while (ctas < kClusterCtas && (int64_t)ctas * (kClusterTile / 4) < s.T) ctas *= 2;
  // zeroing: about 1 MB of rows per CTA, fewer where that leaves SMs without any
  const int64_t row = g.D * (int64_t)sizeof(T), two = 2 * (int64_t)sm_count() - ctas;
  int64_t rows = ((int64_t)1 << 20) / row;
  if (rows > (s.V + two - 1) / two) rows = (s.V + two - 1) / two;
  rows = rows < 1 ? 1 : rows > kZeroRows ? kZeroRows : rows;
  int64_t zero = (s.V + rows - 1) / rows;
  if (zero > 65536) zero = 65536;
  const ZeroArgs z = {g.dw, g.D, g.nslots, (int)rows};
  return launch_dependent(kernel, ctas + (zero + ctas - 1) / ctas * ctas, kClusterThreads, kSmem, ctas, st, s, passes, z);
}

template <class T, bool ALIGNED>
cudaError_t launch_embed_grad(EmbedGradArgs a, SortArgs s, const EmbedPlan& p, uint2* other, cudaStream_t st) {
  const int64_t slabs = (a.nslots + 31) / 32;
  if (direct_form(a.T, a.V, a.D)) {
    return launch_dependent(fw_embed_direct_kernel<T, ALIGNED>, warps_grid(a.V * slabs), 256, 0, 1, st, a);
  }
  a.sorted = s.dst;
  unsigned zero = 0;
  cudaError_t e = cudaSuccess;
  if (a.T <= kClusterTokens) {
    e = sort_cluster<T, ALIGNED>(s, p.passes, a, st);
  } else {
    uint2* ent[2] = {s.dst, other};
    for (int i = 0; i < p.passes; ++i) {
      s.src = i == 0 ? nullptr : ent[(i - 1) & 1];
      s.dst = ent[i & 1];
      s.shift = i * p.bits;
      fw_sort_hist_kernel<<<(unsigned)p.tiles, kSortThreads, 0, st>>>(s);
      fw_sort_scatter_kernel<<<(unsigned)p.tiles, kSortThreads, 0, st>>>(s);
    }
    a.sorted = ent[(p.passes - 1) & 1];
    zero = warps_grid((a.V + 7) / 8);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) return e;
  a.sum_blocks = (int)warps_grid(p.chunks * slabs);
  e = launch_dependent(fw_embed_sum_kernel<T, ALIGNED>, a.sum_blocks + zero, 256, 0, 1, st, a);
  if (e != cudaSuccess) return e;
  return launch_dependent(fw_embed_join_kernel<T, ALIGNED>, warps_grid((p.chunks + 7) / 8 * 8 * slabs), 256, 0, 1, st, a);
}

template <class T>
cudaError_t launch_embed_grad(const EmbedGradArgs& a, const SortArgs& s, const EmbedPlan& p, uint2* other,
                              cudaStream_t st) {
  const int64_t es = sizeof(T);
  const bool aligned = aligned16(a.g) && aligned16(a.dw) && a.ldg * es % 16 == 0 && a.D * es % 16 == 0;
  return aligned ? launch_embed_grad<T, true>(a, s, p, other, st) : launch_embed_grad<T, false>(a, s, p, other, st);
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
  EmbedArgs a = {ids, weight, out, T, V, D, ldw, ldo, scale, status, 0, 0};
  a.nsteps = (slots_of(out, ldo, D, es) + 31) / 32;
  a.nslabs = (a.nsteps + kSlab - 1) / kSlab;
  const int64_t need = (T * a.nslabs + 7) / 8, cap = (int64_t)sm_count() * 64;
  const int64_t grid = need < cap ? need : cap;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return launch_status(
      dtype == FWB_DTYPE_BF16  ? launch_dependent(fw_embed_rows_kernel<__nv_bfloat16>, grid, 256, 0, 1, st, a)
      : dtype == FWB_DTYPE_F16 ? launch_dependent(fw_embed_rows_kernel<__half>, grid, 256, 0, 1, st, a)
                               : launch_dependent(fw_embed_rows_kernel<float>, grid, 256, 0, 1, st, a));
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
  const EmbedPlan p = embed_plan(T, V, D);
  if (!ids || !grad || (p.bytes > 0 && !workspace)) return FWB_E_POINTER;
  if (reinterpret_cast<uintptr_t>(grad) % es || reinterpret_cast<uintptr_t>(dweight) % es || !aligned16(workspace))
    return FWB_E_POINTER;
  if (workspace_bytes < p.bytes) return FWB_E_CAPACITY;
  char* ws = static_cast<char*>(workspace);
  SortArgs s = {};
  s.ids = ids;
  s.dst = reinterpret_cast<uint2*>(ws);
  s.hist = reinterpret_cast<uint32_t*>(ws + p.hist_at);
  s.T = T;
  s.V = V;
  s.padding = padding;
  s.bits = p.bits;
  s.tiles = (int)p.tiles;
  s.status = status;
  EmbedGradArgs a = {};
  a.ids = ids;
  a.g = grad;
  a.dw = dweight;
  a.part = reinterpret_cast<float*>(ws + p.part_at);
  a.T = T;
  a.V = V;
  a.D = D;
  a.ldg = ldg;
  a.pitch = p.pitch;
  a.padding = padding;
  a.scale = scale;
  a.nslots = slots_of(dweight, D, D, es);
  a.status = status;
  uint2* other = reinterpret_cast<uint2*>(ws) + T;  // second array of entries, more than kClusterTokens only
  return launch_status(dtype == FWB_DTYPE_BF16  ? launch_embed_grad<__nv_bfloat16>(a, s, p, other, st)
                       : dtype == FWB_DTYPE_F16 ? launch_embed_grad<__half>(a, s, p, other, st)
                                                : launch_embed_grad<float>(a, s, p, other, st));
}

}  // extern "C"
