// Log probabilities of given tokens, with the entropy of each row and its
// likeliest alternatives, from logits; and their gradient.  For a row z of V
// logits and a temperature T,
//   m = max z,  t_j = (z_j - m) / T,  S = sum exp t_j,  l_j = t_j - log S,
//   logp = l_y,  H = log S - (sum exp(t_j) t_j) / S,
//   dz_j = ((1[j = y] - p_j) g - p_j (l_j + H) h) / T,  p_j = exp l_j,
// with upstream factors g of logp and h of H.  Both terms of H are positive, so
// nothing cancels; exp(t) t is 0 where exp(t) is (masked columns are -inf).
//
// One pass over the row: every thread keeps its maximum, and both sums relative
// to a reference near it, which moves in few batches of slots.  Bound by HBM: the forward reads the logits once, the gradient reads them again and
// writes theirs.  4096 x 32000: forward float32 77 us (6.8 TB/s), bfloat16 48
// (5.5: the exponentials beside it), with 5 alternatives 88 and 60, gradient 167
// and 86 (6.1 to 6.3 TB/s).  Few rows are bound by latency: 48 x 128256 bfloat16
// 6.3 to 6.8 us (8 CTAs a row), with 20 alternatives 10.7 to 11.3 (4 CTAs a row).
//
// The k likeliest columns come without a second pass over the row.  Every
// thread also knows its largest element; the k-th largest of these (taken over
// up to 64 groups of threads) is a bound that k different elements reach, so
// whatever is among the row's k largest reaches it too, and lies with the few
// threads (k and some) whose largest element does.  Their slots are read again,
// from L2, by whole warps, and the elements that reach the bound are ranked by
// 64-bit keys (value, then lowest column first), all different.  Where that
// would be very many, because the bound's value is a mask's, those above it and
// the first k of that value are enough.
#include <cooperative_groups.h>

#include <cmath>

#include "fw_host.cuh"
#include "fw_rowslots.cuh"

namespace cg = cooperative_groups;

namespace fwb200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kFloor = -200.0f;  // 2^kFloor is 0 in fp32; keeps 0 * t finite
// Slots in flight per thread, and CTAs of 256 threads per SM.  4096 x 32000
// without and with 5 alternatives, float32: 4 slots and 4 CTAs 82 and 97 us, 4
// and 5 80 and 93, 8 and 4 77 and 88; bfloat16: 52 and 66, 48 and 60, 48 and 68.
// Rows split over CTAs, 48 x 128256 bfloat16 without (8 CTAs a row) and with 20
// alternatives (4): 4 and 4 7.4 and 11.8, 8 and 4 7.5 and 11.4, 8 and 3 6.7 and
// 11.2.
template <class T, int CL>
constexpr int kBatch = sizeof(T) == 4 || CL > 1 ? 8 : 4;
constexpr int kSplitCtas = 3;
template <class T, int CL>
constexpr int kCtas = CL > 1 ? kSplitCtas : sizeof(T) == 2 ? 5 : 4;
constexpr int kAgain = 4;  // slots in flight per thread where they are read again

struct ScoreArgs {
  const void* z;
  const int64_t* y;
  int64_t B, ld, ignore;
  int V, k;
  float inv_t;
  float *logp, *entropy, *top_logp;
  int64_t* top_ids;
  float4* state;  // maximum, log S, H, the token's bits (-2: ignored); may be NULL
  int32_t* status;
};

__device__ __forceinline__ float exp2_ftz(float x) {  // relative error 2^-22; 0 under 2^-126
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Maximum of some elements, and the sums over them of 2^t and 2^t t with
// t = (z - maximum) * c.  No elements: maximum -inf, sums 0.
struct Sums {
  float m, s, u;
  __device__ __forceinline__ void raise(float to, float c) {  // to >= m, or NaN
    if (m != -CUDART_INF_F) {
      const float d = fmaxf((m - to) * c, kFloor), f = exp2_ftz(d);
      u = f * fmaf(d, s, u);
      s *= f;
    }
    m = to;
  }
  // Of every N neighbouring lanes, in all of them.
  template <int N>
  __device__ __forceinline__ void join_lanes(float c) {
    float to = m;
#pragma unroll
    for (int o = N / 2; o > 0; o >>= 1) to = max_nan(to, __shfl_xor_sync(kFull, to, o));
    raise(to, c);
#pragma unroll
    for (int o = N / 2; o > 0; o >>= 1) {
      s += __shfl_xor_sync(kFull, s, o);
      u += __shfl_xor_sync(kFull, u, o);
    }
  }
};

// Order of (value, column): larger values first, among equal ones the lower column.
__device__ __forceinline__ uint64_t rank_key(float v, int e) {
  return ((uint64_t)sort_key(v) << 32) | (uint32_t)~e;
}

// A slot of the row, elements outside it as -inf.
template <class T>
__device__ __forceinline__ uint4 load_slot_row(const T* row, int e0, int V) {
  constexpr int VN = 16 / sizeof(T);
  if (e0 >= 0 && e0 + VN <= V) return ld_global16_once(row + e0);
  const uint4 none = neg_inf_slot<T>();
  uint32_t w[4] = {none.x, none.y, none.z, none.w};
#pragma unroll
  for (int j = 0; j < VN; ++j) {
    if (e0 + j < 0 || e0 + j >= V) continue;
    if constexpr (sizeof(T) == 4) {
      w[j] = __float_as_uint(row[e0 + j]);
    } else {
      const uint32_t b = *reinterpret_cast<const unsigned short*>(row + e0 + j), at = 16 * (j & 1);
      w[j >> 1] = (w[j >> 1] & ~(0xffffu << at)) | (b << at);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Two floats in one register pair, for the packed fp32 instructions.
struct Pair {
  uint64_t v;
  __device__ __forceinline__ static Pair of(float lo, float hi) {
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(lo), "f"(hi));
    return p;
  }
  __device__ __forceinline__ float2 get() const {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
  }
};
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return d;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}

// Both halves raised to `floor`, a pair of finite values.
template <class T>
__device__ __forceinline__ uint32_t floor2(uint32_t x, uint32_t floor) {
  uint32_t r;
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(floor));
  else
    asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(floor));
  return r;
}
// -2^100 in bfloat16; the lowest finite float16
template <class T>
constexpr uint32_t kFloor2 = std::is_same<T, __nv_bfloat16>::value ? 0xf180f180u : 0xfbfffbffu;
template <class T>
constexpr float kFloor16 = std::is_same<T, __nv_bfloat16>::value ? -1.2676506e30f : -65504.0f;

// A thread's maximum, and its sums of 2^t and 2^t t relative to a reference,
// which is not moved before the maximum has passed it by 8 powers of two (a
// maximum of a few elements is passed all the time, and moving costs as much
// as three elements).  With r2 = fl(ref c), t = fma(z, c, -r2) is rounded once,
// and off = r2 - ref c is what t is away from (z - ref) c.  Where r2 is large,
// off could be, too, and t is (z - ref) c.
// Elements that are -inf or far down are raised so that 0 * t is finite: t
// itself, or in pairs the 16-bit elements, if their floor is 200 powers of two
// under the reference.  Pairs take 4.5 instructions an element with the
// maximum, single ones 8 (4096 x 32000 bfloat16: 51 and 55 us).
template <class T>
struct Running {
  float m, ref, r2, off, lim;
  bool pairs;
  Pair s, u;
  __device__ __forceinline__ Running() {
    m = ref = lim = -CUDART_INF_F;
    r2 = off = 0.0f;
    pairs = false;
    s = u = Pair::of(0.0f, 0.0f);
  }
  __device__ __forceinline__ void move(float to, float c) {  // to >= ref, or NaN
    const float n2 = to * c;
    bool fits = fabsf(n2) < 1048576.0f;  // |off| < 2^-4
    if constexpr (sizeof(T) == 2) fits = fits && n2 - kFloor16<T> * c >= 200.0f && kFloor16<T> * c > -1e38f;
    const float n_off = fits ? fmaf(-to, c, n2) : 0.0f;
    if (ref != -CUDART_INF_F) {
      const float d = fmaxf((ref - to) * c + (off - n_off), kFloor), f = exp2_ftz(d);
      const float2 a = s.get(), b = u.get();
      u = Pair::of(f * fmaf(d, a.x, b.x), f * fmaf(d, a.y, b.y));
      s = Pair::of(f * a.x, f * a.y);
    }
    ref = to, r2 = n2, off = n_off, pairs = fits;
    lim = fits ? to + 8.0f / c : to;
  }
  template <int N>
  __device__ __forceinline__ void add(const uint4 (&x)[N], float c) {
    constexpr int VN = 16 / sizeof(T);
    if (pairs) {
      const Pair c2 = Pair::of(c, c), back = Pair::of(-r2, -r2);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        uint4 v = x[i];
        if constexpr (sizeof(T) == 2)
          v = make_uint4(floor2<T>(v.x, kFloor2<T>), floor2<T>(v.y, kFloor2<T>), floor2<T>(v.z, kFloor2<T>),
                         floor2<T>(v.w, kFloor2<T>));
        float z[VN];
        unpack16<T>(v, z);
#pragma unroll
        for (int j = 0; j < VN; j += 2) {
          Pair t = fma2(Pair::of(z[j], z[j + 1]), c2, back);
          float2 f = t.get();
          if constexpr (sizeof(T) == 4) {
            f = make_float2(fmaxf(f.x, kFloor), fmaxf(f.y, kFloor));
            t = Pair::of(f.x, f.y);
          }
          const Pair e = Pair::of(exp2_ftz(f.x), exp2_ftz(f.y));
          s = add2(s, e);
          u = fma2(e, t, u);
        }
      }
    } else {
      float2 a = s.get(), b = u.get();
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float z[VN];
        unpack16<T>(x[i], z);
#pragma unroll
        for (int j = 0; j < VN; ++j) {
          const float t = fmaxf((z[j] - ref) * c, kFloor), e = exp2_ftz(t);
          (j & 1 ? a.y : a.x) += e;
          (j & 1 ? b.y : b.x) = fmaf(e, t, j & 1 ? b.y : b.x);
        }
      }
      s = Pair::of(a.x, a.y);
      u = Pair::of(b.x, b.y);
    }
  }
  __device__ __forceinline__ Sums result(float c) const {  // relative to the maximum
    const float2 a = s.get(), b = u.get();
    Sums q = {m, a.x + a.y, b.x + b.y};
    if (ref != -CUDART_INF_F) {
      const float d = fmaxf((ref - m) * c + off, kFloor), f = exp2_ftz(d);
      q.u = f * fmaf(d, q.s, q.u);
      q.s *= f;
    }
    return q;
  }
};

// Descending over the lanes.
__device__ __forceinline__ uint64_t warp_sort(uint64_t x, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int step = size >> 1; step > 0; step >>= 1) {
      const uint64_t o = __shfl_xor_sync(kFull, x, step);
      const bool larger = ((lane & step) == 0) == ((lane & size) == 0);  // this lane keeps the larger
      x = (x > o) == larger ? x : o;
    }
  return x;
}

// The 32 largest of two descending lists, descending.
__device__ __forceinline__ uint64_t warp_merge(uint64_t a, uint64_t b, int lane) {
  const uint64_t r = __shfl_sync(kFull, b, 31 - lane);
  uint64_t x = a > r ? a : r;
#pragma unroll
  for (int step = 16; step > 0; step >>= 1) {
    const uint64_t o = __shfl_xor_sync(kFull, x, step);
    x = (x > o) == ((lane & step) == 0) ? x : o;
  }
  return x;
}

// The threads of a row's group: a CTA, or one of its warps.
template <int NW>
__device__ __forceinline__ void group_sync() {
  if constexpr (NW == 1)
    __syncwarp();
  else
    __syncthreads();
}
constexpr int kWarpRows = 8;  // rows per CTA, a warp each, of the short ones

constexpr int kFound = 256;  // keys that reach the bound, before the slower way is taken

template <int NW>
struct TopShared {
  static constexpr int NT = NW * 32, NG = NT < 64 ? NT : 64;  // threads; groups of NT / NG neighbours
  float group[NG];        // the largest element of each group
  uint64_t found[kFound];
  uint64_t held[NW][64];  // the slower way: keys that reach the bound, per warp
  uint64_t best[32];      // the CTA's k largest, descending, 0 where there are fewer
  float bound;
  int n, n_who, count[NW];
  uint16_t who[NT];       // threads whose largest element reaches the bound
};

// A CTA's part of a row: slots [k0, k1), of which [lo, hi) are whole.
template <class T>
struct Segment {
  const T* row;
  int off, V, k0, k1, lo, hi;
  __device__ __forceinline__ int element(int k) const { return k * (16 / (int)sizeof(T)) - off; }
  __device__ __forceinline__ uint4 load(int k) const {
    return k >= lo && k < hi ? ld_global16_once(row + element(k)) : load_slot_row(row, element(k), V);
  }
};

// The bound: the k-th largest of the groups' largest elements, which k
// different elements reach.  top.bound is -inf before.
template <int NW>
__device__ __forceinline__ void top_bound(TopShared<NW>& top, int k) {
  using S = TopShared<NW>;
  constexpr int P = S::NT / S::NG, M = S::NG / P;  // threads per group, groups each compares with
  const int tid = threadIdx.x % S::NT;
  const float own = top.group[tid / P];
  int above = 0, reach = 0;  // groups above this one; not under it
#pragma unroll
  for (int i = 0; i < M; ++i) {
    const float o = top.group[(tid % P) + i * P];
    above += o > own;
    reach += o >= own;
  }
#pragma unroll
  for (int o = 1; o < P; o <<= 1) {
    above += __shfl_xor_sync(kFull, above, o);
    reach += __shfl_xor_sync(kFull, reach, o);
  }
  if (above < k && reach >= k) top.bound = own;  // equal ones all write it
}

// How many of n keys are above `own`.
__device__ __forceinline__ int keys_above(const uint64_t* keys, int n, uint64_t own) {
  int above = 0, i = 0;
  for (; i + 8 <= n; i += 8)
#pragma unroll
    for (int j = 0; j < 8; ++j) above += keys[i + j] > own;
  for (; i < n; ++i) above += keys[i] > own;
  return above;
}

// Leaves the k largest keys of the segment in top.best.  `largest` is this
// thread's largest element, the bound is there, top.n and top.n_who are 0.
template <class T, int NW>
__device__ __forceinline__ void top_of(TopShared<NW>& top, const Segment<T>& seg, float largest, int k) {
  constexpr int VN = 16 / sizeof(T), NT = NW * 32;
  const int tid = threadIdx.x % NT, lane = tid & 31, w = tid >> 5;
  const float least = top.bound;
  const uint64_t bound = (uint64_t)sort_key(least) << 32;
  const bool in = seg.k0 + tid < seg.k1 && largest >= least;
  const auto look = [&](const uint4& x, int kk, bool above) {
    if (!(slot_max_nan<T>(x) >= least)) return;
    if (*const_cast<volatile int*>(&top.n) > kFound) return;  // the list has overflowed already
    float z[VN];
    unpack16<T>(x, z);
#pragma unroll
    for (int j = 0; j < VN; ++j) {
      const int e = seg.element(kk) + j;
      if ((above ? z[j] > least : z[j] >= least) && e >= 0 && e < seg.V) {
        const int at = atomicAdd(&top.n, 1);
        if (at < kFound) top.found[at] = rank_key(z[j], e);
      }
    }
  };
  const uint32_t all = __ballot_sync(kFull, in);
  int base = 0;
  if (lane == 0 && all) base = atomicAdd(&top.n_who, __popc(all));
  base = __shfl_sync(kFull, base, 0);
  if (in) top.who[base + __popc(all & ((1u << lane) - 1u))] = (uint16_t)tid;
  if (tid < 32) top.best[tid] = 0;
  group_sync<NW>();
  const auto overflow = [&] { return *const_cast<volatile int*>(&top.n) > kFound; };
  const auto rank_found = [&](int n) {
    for (int i = tid; i < n; i += NT) {
      const uint64_t own = top.found[i];
      const int rank = keys_above(top.found, n, own);
      if (rank < k) top.best[rank] = own;
    }
    group_sync<NW>();
  };
  const int n_who = top.n_who;
  // More than half of the threads reach the bound where the elements at it are many of one value: a mask's, say.
  bool many = NW > 1 && n_who > NT / 2;
  if (!many) {
    if (seg.k1 - seg.k0 <= kAgain * NT) {  // few slots each: every thread its own
      if (in) {
        uint4 x[kAgain];
#pragma unroll
        for (int b = 0; b < kAgain; ++b)
          if (seg.k0 + tid + b * NT < seg.k1) x[b] = seg.load(seg.k0 + tid + b * NT);
#pragma unroll
        for (int b = 0; b < kAgain; ++b)
          if (seg.k0 + tid + b * NT < seg.k1) look(x[b], seg.k0 + tid + b * NT, false);
      }
    } else {  // a warp per thread of the list, its slots over the lanes, kAgain such loads in flight
      for (int t0 = w; t0 < n_who && !overflow(); t0 += kAgain * NW) {
        for (int s0 = lane * NT; s0 < seg.k1 - seg.k0; s0 += 32 * NT) {
          uint4 x[kAgain];
          int kk[kAgain];
#pragma unroll
          for (int b = 0; b < kAgain; ++b) {
            kk[b] = t0 + b * NW < n_who ? seg.k0 + top.who[t0 + b * NW] + s0 : seg.k1;
            if (kk[b] < seg.k1) x[b] = seg.load(kk[b]);
          }
#pragma unroll
          for (int b = 0; b < kAgain; ++b)
            if (kk[b] < seg.k1) look(x[b], kk[b], false);
        }
      }
    }
    group_sync<NW>();
    const int n = top.n;
    if (n <= kFound) {
      rank_found(n);
      return;
    }
    group_sync<NW>();
    if (tid == 0) top.n = 0;
    group_sync<NW>();
  }
  // Many elements reach the bound.  If few are above it, those and the first k at it will do, which are looked for
  // from the start of the segment.
  if (largest > least) {
    for (int kk = seg.k0 + tid; kk < seg.k1 && !overflow(); kk += NT) look(seg.load(kk), kk, true);
  }
  group_sync<NW>();
  const int above = top.n;
  if (above <= kFound - 32) {
    int at = 0;  // elements at the bound so far
    for (int base = seg.k0; base < seg.k1 && at < k; base += NT) {
      const int kk = base + tid;
      float z[VN];
      unpack16<T>(kk < seg.k1 ? seg.load(kk) : neg_inf_slot<T>(), z);
      uint32_t here = 0u;
#pragma unroll
      for (int j = 0; j < VN; ++j) {
        const int e = seg.element(kk) + j;
        here |= (z[j] == least && kk < seg.k1 && e >= 0 && e < seg.V ? 1u : 0u) << j;
      }
      int before = __popc(here);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(kFull, before, o);
        if (lane >= o) before += u;
      }
      if (lane == 31) top.count[w] = before;
      group_sync<NW>();
      before += at - __popc(here);
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        before += i < w ? top.count[i] : 0;
        at += top.count[i];
      }
      for (; here && before < k; here &= here - 1u, ++before)
        top.found[above + before] = rank_key(least, seg.element(kk) + __ffs(here) - 1);
      group_sync<NW>();
    }
    rank_found(above + min(at, k));
    return;
  }
  // The slower way, for rows whose largest elements lie with few threads (4096 x 32000 rising float32: 249 us, 98
  // for rows without an order): each warp keeps the 32 largest of what it
  // has seen in order, one per lane, and raises its own bound by them.
  uint64_t mine = bound, list = 0;
  uint64_t* held = top.held[w];
  int have = 0;  // keys in the buffer
  const auto drain = [&] {
    __syncwarp();
    uint64_t x = lane < have ? held[lane] : 0;
    list = warp_merge(list, warp_sort(x, lane), lane);
    if (lane + 32 < have) x = held[lane + 32];
    __syncwarp();
    if (lane + 32 < have) held[lane] = x;
    have = max(have - 32, 0);
    const uint64_t kth = __shfl_sync(kFull, list, k - 1);
    mine = kth > mine ? kth : mine;
    __syncwarp();
  };
  for (int t = w; t < top.n_who; t += NW) {
    for (int k0 = seg.k0 + top.who[t]; k0 < seg.k1; k0 += NT * 32) {
      const int kk = k0 + lane * NT;
      float z[VN];
      unpack16<T>(kk < seg.k1 ? seg.load(kk) : neg_inf_slot<T>(), z);
#pragma unroll
      for (int j = 0; j < VN; ++j) {
        const int e = seg.element(kk) + j;
        const uint64_t key = rank_key(z[j], e);
        const bool reaches = kk < seg.k1 && e >= 0 && e < seg.V && key >= mine;
        const uint32_t who = __ballot_sync(kFull, reaches);
        if (!who) continue;
        if (reaches) held[have + __popc(who & ((1u << lane) - 1u))] = key;
        have += __popc(who);
        if (have > 32) drain();
      }
    }
  }
  drain();
  held[lane] = list;
  group_sync<NW>();
  const uint64_t own = held[lane];
  int rank = 0;
  for (int g = 0; g < NW; ++g) rank += keys_above(top.held[g], 32, own);
  if (own != 0 && rank < k) top.best[rank] = own;
  group_sync<NW>();
}

// One row per cluster of CL CTAs of NW warps, each taking an equal part of it;
// or, for NW = 1, one row per warp of a CTA.
template <class T, int NW, bool TOP, int CL>
__global__ void __launch_bounds__(NW == 1 ? kWarpRows * 32 : NW * 32, NW == 8 ? kCtas<T, CL> : NW == 4 ? 8 : 3) fw_logprob_kernel(ScoreArgs a) {
  constexpr int VN = 16 / sizeof(T), NT = NW * 32, N = kBatch<T, CL>;
  constexpr int R = NW == 1 ? kWarpRows : 1;
  __shared__ Sums parts[R][NW];
  __shared__ Sums whole;  // of this CTA, for its cluster
  __shared__ TopShared<TOP ? NW : 1> tops[TOP ? R : 1];
  wait_prior_kernel();
  allow_dependent_launch();
  const int group = R > 1 ? threadIdx.x / NT : 0;
  const int tid = threadIdx.x % NT, lane = tid & 31, w = tid >> 5;
  const int64_t r = (int64_t)blockIdx.x * R / CL + group;
  if (r >= a.B) return;
  Sums(&part)[NW] = parts[group];
  TopShared<TOP ? NW : 1>& top = tops[TOP ? group : 0];
  const int rank = CL > 1 ? (int)(blockIdx.x % CL) : 0;
  const int64_t y = a.y[r];
  if (y == a.ignore) {
    if (rank != 0) return;
    if (tid == 0) {
      a.logp[r] = 0.0f;
      a.entropy[r] = 0.0f;
      if (a.state) a.state[r] = make_float4(0.0f, 0.0f, 0.0f, __int_as_float(-2));
    }
    if (TOP && tid < a.k) {
      a.top_logp[r * a.k + tid] = 0.0f;
      a.top_ids[r * a.k + tid] = -1;
    }
    return;
  }
  const T* row = static_cast<const T*>(a.z) + r * a.ld;
  const bool label = y >= 0 && y < a.V;
  const float zy = tid == 0 && label ? Elem<T>::to_f(row[y]) : 0.0f;
  Segment<T> seg;
  seg.row = row;
  seg.V = a.V;
  seg.off = (int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
  const int slots = (int)(((int64_t)seg.off + a.V + VN - 1) / VN);
  seg.k0 = (int)((int64_t)slots * rank / CL);
  seg.k1 = (int)((int64_t)slots * (rank + 1) / CL);
  seg.lo = seg.off ? 1 : 0;
  seg.hi = (int)(((int64_t)seg.off + a.V) / VN);
  const float c = a.inv_t * kLog2e;
  Running<T> run;
  for (int k0 = seg.k0 + tid; k0 < seg.k1; k0 += NT * N) {
    uint4 x[N];
    if (k0 >= seg.lo && k0 + (N - 1) * NT < min(seg.hi, seg.k1)) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = ld_global16_once(row + seg.element(k0 + i * NT));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = k0 + i * NT < seg.k1 ? seg.load(k0 + i * NT) : neg_inf_slot<T>();
    }
    float bm = -CUDART_INF_F;
#pragma unroll
    for (int i = 0; i < N; ++i) bm = max_nan(bm, slot_max_nan<T>(x[i]));
    run.m = max_nan(run.m, bm);
    if (!(bm <= run.lim)) run.move(run.m, c);
    if (run.ref != -CUDART_INF_F) run.add(x, c);
  }
  Sums q = run.result(c);
  const float m_thread = q.m;
  q.join_lanes<32>(c);
  if (lane == 0) part[w] = q;
  if constexpr (TOP) {
    float g = m_thread;
#pragma unroll
    for (int o = 1; o < NT / TopShared<NW>::NG; o <<= 1) g = fmaxf(g, __shfl_xor_sync(kFull, g, o));
    top.group[tid / (NT / TopShared<NW>::NG)] = g;
    if (tid == 0) {
      top.bound = -CUDART_INF_F;
      top.n = 0;
      top.n_who = 0;
    }
  }
  group_sync<NW>();
  if (w == 0) {
    q = lane < NW ? part[lane] : Sums{-CUDART_INF_F, 0.0f, 0.0f};
    q.join_lanes<NW>(c);
    if (CL > 1 && lane == 0) whole = q;
  }
  if constexpr (TOP) {
    top_bound(top, a.k);
    group_sync<NW>();
    top_of<T, NW>(top, seg, m_thread, a.k);
  }
  float m = CUDART_NAN_F, logs = CUDART_NAN_F, h = CUDART_NAN_F, logp = CUDART_NAN_F;
  const auto finish = [&] {  // of the row, from q; one thread or several
    if (!label || !(fabsf(q.m) < CUDART_INF_F)) return;
    m = q.m;
    logs = logf(q.s);
    h = logs - q.u * kLn2 / q.s;
    logp = (zy - m) * a.inv_t - logs;
  };
  const auto give = [&] {
    if (!label) raise_status(a.status, FWB_STATUS_LABEL_RANGE);
    if (!(fabsf(q.m) < CUDART_INF_F)) raise_status(a.status, FWB_STATUS_NONFINITE);
    a.logp[r] = logp;
    a.entropy[r] = h;
    if (a.state) a.state[r] = make_float4(m, logs, h, __int_as_float(label ? (int)y : -1));
  };
  const auto give_top = [&](uint64_t key, int i) {
    const bool bad = isnan(m);
    a.top_logp[r * a.k + i] = bad ? CUDART_NAN_F : (key_value((uint32_t)(key >> 32)) - m) * a.inv_t - logs;
    a.top_ids[r * a.k + i] = bad ? -1 : (int64_t)(uint32_t)~(uint32_t)key;
  };
  if constexpr (CL == 1) {
    if (w == 0) {
      q = {__shfl_sync(kFull, q.m, 0), __shfl_sync(kFull, q.s, 0), __shfl_sync(kFull, q.u, 0)};
      finish();
      if (tid == 0) give();
      if (TOP && lane < a.k) give_top(top.best[lane], lane);
    }
  } else {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (rank == 0) {
      if (w == 0) {
        q = *cluster.map_shared_rank(&whole, lane % CL);
        q.join_lanes<CL>(c);
        finish();
        if (tid == 0) {
          give();
          part[0] = {m, logs, 0.0f};
        }
      }
      if constexpr (TOP) {
        static_assert(CL * 32 <= NT && CL * 32 <= kFound, "a key per thread");
        uint64_t own = 0;
        if (w < CL && lane < a.k) {
          own = cluster.map_shared_rank(&top, w)->best[lane];
          top.found[w * a.k + lane] = own;
        }
        group_sync<NW>();
        m = part[0].m;
        logs = part[0].s;
        if (isnan(m)) {  // a bad row need not have given k keys
          if (tid < a.k) give_top(0, tid);
        } else if (own != 0) {
          const int i = keys_above(top.found, CL * a.k, own);
          if (i < a.k) give_top(own, i);
        }
      }
    }
    cluster.sync();  // rank 0 has read the others' shared memory
  }
}

// ------------------------------------------------------------ gradient
struct ScoreGradArgs {
  const void* z;
  int64_t B, ld, ldg;
  int V, parts;  // CTAs per row
  float inv_t;
  const float4* state;
  const float *dlogp, *dentropy;  // either may be NULL: zero
  void* grad;
};

// 16-byte slots in flight per thread, and CTAs of 256 threads per SM.  4096 x
// 32000, float32 and bfloat16, with 2 and 8: 171 and 88 us; 4 and 4: 167 and
// 90; 4 and 5: 167 and 86; 8 and 3: 163 and 91.
constexpr int kGradBatch = 4, kGradCtas = 5;

// What a row's elements are worked out from, in powers of two:
//   l = log2 p = fma(z, c, -r2) + shift, or (z - m) c + shift where r2 is large
//   d = -2^l (h l + g)
struct RowGrad {
  float m, c, r2, shift, g, h;
  bool live, fits;
};

// Rows in `parts` parts, a CTA each, or (NW = 1) a row per warp.
template <class T, int NW>
__global__ void __launch_bounds__(256, kGradCtas) fw_logprob_grad_kernel(ScoreGradArgs a) {
  constexpr int VN = 16 / sizeof(T), NT = NW * 32, N = kGradBatch;
  wait_prior_kernel();
  allow_dependent_launch();
  const int tid = threadIdx.x % NT;
  const int64_t r = NW == 1 ? (int64_t)blockIdx.x * 8 + threadIdx.x / 32 : blockIdx.x / a.parts;
  if (r >= a.B) return;
  const int part = NW == 1 ? 0 : (int)(blockIdx.x - r * a.parts);
  const T* row = static_cast<const T*>(a.z) + r * a.ld;
  T* out = static_cast<T*>(a.grad) + r * a.ldg;
  const int V = a.V;
  const int off = (int)((reinterpret_cast<uintptr_t>(out) & 15u) / sizeof(T));
  const int slots = (int)(((int64_t)off + V + VN - 1) / VN);
  const int k1 = (int)((int64_t)slots * (part + 1) / a.parts);
  // where the gradient's whole slots are whole slots of the logits
  const bool same = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
  const int lo = same ? (off ? 1 : 0) : k1, hi = min(k1, (int)(((int64_t)off + V) / VN));
  const Span<T> span(a.z, a.B, a.ld, V);

  const float4 st = a.state[r];
  const int y = __float_as_int(st.w);
  RowGrad q;
  q.live = y != -2;
  q.m = st.x;
  q.c = a.inv_t * kLog2e;
  q.r2 = q.m * q.c;
  q.fits = fabsf(q.r2) < 1048576.0f;
  q.shift = -st.y * kLog2e + (q.fits ? fmaf(-q.m, q.c, q.r2) : 0.0f);
  const float g = a.dlogp ? a.dlogp[r] * a.inv_t : 0.0f, h = a.dentropy ? a.dentropy[r] * a.inv_t : 0.0f;
  q.h = -h * kLn2;
  q.g = a.dentropy ? -fmaf(h, st.z, g) : -g;
  if (isnan(st.x)) q.g = CUDART_NAN_F;

  for (int k0 = (int)((int64_t)slots * part / a.parts) + tid; k0 < k1; k0 += NT * N) {
    uint4 x[N];
    if (!q.live) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (k0 + i * NT < k1) store_slot(out, (int64_t)(k0 + i * NT) * VN - off, (int64_t)V, true, make_uint4(0u, 0u, 0u, 0u));
      continue;
    }
    const bool whole = k0 >= lo && k0 + (N - 1) * NT < hi;
    if (whole) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = ld_global16_once(row + ((k0 + i * NT) * VN - off));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        x[i] = k0 + i * NT < k1 ? load_slot_shifted(row, (k0 + i * NT) * VN - off, span) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = (k0 + i * NT) * VN - off;
      float z[VN];
      unpack16<T>(x[i], z);
#pragma unroll
      for (int j = 0; j < VN; ++j) {
        // an element outside the row may be anything; it is not stored
        float l = q.fits ? fmaf(z[j], q.c, -q.r2) : (z[j] - q.m) * q.c;
        l = fmaxf(l + q.shift, kFloor);
        z[j] = exp2_ftz(l) * fmaf(q.h, l, q.g);
      }
      if ((unsigned)(y - e) < (unsigned)VN) {
#pragma unroll
        for (int j = 0; j < VN; ++j)
          if (e + j == y) z[j] += g;
      }
      x[i] = pack_slot<T>(z);
    }
    if (whole) {
#pragma unroll
      for (int i = 0; i < N; ++i) *reinterpret_cast<uint4*>(out + ((k0 + i * NT) * VN - off)) = x[i];
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (k0 + i * NT < k1) store_slot(out, (int64_t)(k0 + i * NT) * VN - off, (int64_t)V, true, x[i]);
    }
  }
}

// ------------------------------------------------------------ host
int score_check(int dtype, int64_t B, int64_t V, int64_t ld, float inv_t) {
  if (dtype != FWB_DTYPE_F32 && dtype != FWB_DTYPE_BF16 && dtype != FWB_DTYPE_F16) return FWB_E_DTYPE;
  if (B < 0 || V < 1 || ld < V || B > (1 << 28) || V > (1 << 28) || ld > ((int64_t)1 << 32)) return FWB_E_SHAPE;
  if (!(inv_t > 0.0f) || !std::isfinite(inv_t * kLog2e)) return FWB_E_SHAPE;
  return FWB_OK;
}

bool misaligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }

template <class T, int NW, int CL>
int launch_score(const ScoreArgs& a, cudaStream_t st) {
  const int64_t grid = NW == 1 ? (a.B + kWarpRows - 1) / kWarpRows : a.B * CL;
  const int threads = NW == 1 ? kWarpRows * 32 : NW * 32;
  return launch_status(a.k > 0 ? launch_dependent(fw_logprob_kernel<T, NW, true, CL>, grid, threads, 0, CL, st, a)
                               : launch_dependent(fw_logprob_kernel<T, NW, false, CL>, grid, threads, 0, CL, st, a));
}

// Rows of one warp each: up to 256 slots, or 512 where there are warps' worth
// of rows on every SM.  4096 x 4000 bfloat16 (500 slots) by warps and by CTAs:
// gradient 16.8 and 25.0 us, 5 alternatives 20.4 and 23.6; 512 such rows: 7.8
// and 6.3, 10.1 and 6.6; 4096 x 8000: 29 and 26, 29 and 29.
bool by_warps(int64_t slots, int64_t B) { return slots <= (B >= (int64_t)sm_count() * 16 ? 512 : 256); }

template <class T>
int run_score(const ScoreArgs& a, cudaStream_t st) {
  const int64_t slots = a.V / (16 / (int)sizeof(T)), ctas = (int64_t)sm_count() * kSplitCtas;
  if (by_warps(slots, a.B)) return launch_score<T, 1, 1>(a, st);
  // Few long rows: split until a CTA has one round of loads (2048 slots), as long as all parts run at once; for more
  // than 8 alternatives over 4 CTAs at most, since each gives its k to be ranked again.  128256 bfloat16 in 1, 2, 4, 8
  // parts, 16 rows without and with 20 alternatives: 11.2, 6.7, 4.7, 4.3 and 14.5, 10.7, 8.6, 9.2 us; 48 rows 17.7, 8.6,
  // 6.8, 6.3 and 21.1, 12.4, 10.6, 12.6; 128 rows 19.0, 13.6, 14.5, 16.3 and 23.5, 18.6, 22.4, 31.8; 32000 float32 (8000
  // slots), 1 row: 4.5, 4.0, 3.2, 3.0 and (5 alternatives) 6.2, 6.1, 5.3, 5.7.
  int parts = 1;
  while (parts < (a.k > 8 ? 4 : 8) && slots > parts * 2048 && a.B * parts * 2 <= ctas) parts *= 2;
  if (parts == 8) return launch_score<T, 8, 8>(a, st);
  if (parts == 4) return launch_score<T, 8, 4>(a, st);
  if (parts == 2) return launch_score<T, 8, 2>(a, st);
  if (slots <= 2048) return launch_score<T, 4, 1>(a, st);
  return launch_score<T, 8, 1>(a, st);
}

template <class T>
int run_score_grad(ScoreGradArgs a, cudaStream_t st) {
  const int64_t slots = a.V / (16 / (int)sizeof(T)) + 2;  // whatever the row's start
  a.parts = 1;
  if (by_warps(slots, a.B))
    return launch_status(launch_dependent(fw_logprob_grad_kernel<T, 1>, (a.B + 7) / 8, 256, 0, 1, st, a));
  // parts of no less than one step of a CTA, as many as run at once
  const int64_t most = (slots + 256 * kGradBatch - 1) / (256 * kGradBatch), want = (int64_t)sm_count() * kGradCtas / a.B;
  a.parts = (int)(want < 1 ? 1 : want < most ? want : most);
  return launch_status(launch_dependent(fw_logprob_grad_kernel<T, 8>, a.B * a.parts, 256, 0, 1, st, a));
}

}  // namespace
}  // namespace fwb200

using namespace fwb200;

extern "C" {

int fw_token_log_probs(int dtype, const void* logits, int64_t ld, const int64_t* y, int64_t B, int64_t V, float inv_t,
                       int64_t ignore_index, int k, float* logp, float* entropy, float* top_logp, int64_t* top_ids,
                       float* state, int32_t* status, void* stream) {
  if (int rc = score_check(dtype, B, V, ld, inv_t)) return rc;
  if (k < 0 || k > V) return FWB_E_SHAPE;
  if (k > FWB_TOP_MAX) return FWB_E_CAPACITY;
  if (B == 0) return FWB_OK;
  if (!logits || !y || !logp || !entropy || (k > 0 && (!top_logp || !top_ids))) return FWB_E_POINTER;
  if (misaligned(logits, dtype == FWB_DTYPE_F32 ? 4 : 2) || (state && !aligned16(state))) return FWB_E_POINTER;
  const ScoreArgs a = {logits, y,    B,       ld,       ignore_index, (int)V, k, inv_t,
                       logp,   entropy, top_logp, top_ids, reinterpret_cast<float4*>(state), status};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == FWB_DTYPE_F32    ? run_score<float>(a, st)
         : dtype == FWB_DTYPE_BF16 ? run_score<__nv_bfloat16>(a, st)
                                   : run_score<__half>(a, st);
}

int fw_token_log_probs_grad(int dtype, const void* logits, int64_t ld, int64_t B, int64_t V, float inv_t,
                            const float* state, const float* dlogp, const float* dentropy, void* grad, int64_t ldg,
                            void* stream) {
  if (int rc = score_check(dtype, B, V, ld, inv_t)) return rc;
  if (ldg < V || ldg > ((int64_t)1 << 32)) return FWB_E_SHAPE;
  if (B == 0) return FWB_OK;
  if (!logits || !state || !grad) return FWB_E_POINTER;
  const size_t es = dtype == FWB_DTYPE_F32 ? 4 : 2;
  if (misaligned(logits, es) || misaligned(grad, es) || !aligned16(state)) return FWB_E_POINTER;
  const ScoreGradArgs a = {logits, B, ld, ldg, (int)V, 0, inv_t, reinterpret_cast<const float4*>(state), dlogp, dentropy, grad};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == FWB_DTYPE_F32    ? run_score_grad<float>(a, st)
         : dtype == FWB_DTYPE_BF16 ? run_score_grad<__nv_bfloat16>(a, st)
                                   : run_score_grad<__half>(a, st);
}

}  // extern "C"
