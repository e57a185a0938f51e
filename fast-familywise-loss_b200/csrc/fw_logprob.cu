// Log probabilities of given tokens, with the entropy of each row and its
// likeliest alternatives, from logits; and their gradient.  For a row z of V
// logits and a temperature T,
//   m = max z,  t_j = (z_j - m) / T,  S = sum exp t_j,  l_j = t_j - log S,
//   logp = l_y,  H = log S - (sum exp(t_j) t_j) / S,
//   dz_j = ((1[j = y] - p_j) g - p_j (l_j + H) h) / T,  p_j = exp l_j,
// with upstream factors g of logp and h of H.  Both terms of H are positive, so
// nothing cancels; exp(t) t is 0 where exp(t) is (masked columns are -inf).
//
// One pass over the row: every thread keeps a maximum and both sums relative
// to it, and rescales them in the rare batch of slots that raises it.  Bound by
// HBM: the forward reads the logits once, the gradient reads them again and
// writes theirs.
//
// The k likeliest columns come without a second pass over the row.  Every
// thread also knows where its maximum first stood; the k-th largest of these
// maxima is a bound that k different elements reach, so whatever is among the
// row's k largest is not under it, and lies with the few threads (about k)
// whose maximum is not under it.  Their slots are read again, from L2, by
// whole warps, and the elements that reach the bound are ranked.  Elements are
// ordered by 64-bit keys (value, then lowest column first), all different, so
// ties need no case of their own.
#include <cmath>

#include "fw_host.cuh"
#include "fw_rowslots.cuh"

namespace fwb200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kFloor = -200.0f;  // 2^kFloor is 0 in fp32; keeps 0 * t finite
constexpr int kBatch = 4;          // slots in flight per thread

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
  __device__ __forceinline__ void join(Sums o, float c) {
    const float to = max_nan(m, o.m);
    raise(to, c);
    o.raise(to, c);
    s += o.s;
    u += o.u;
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

template <int NW>
struct TopShared {
  uint64_t first[NW * 32];  // each thread's largest key
  uint64_t held[NW][64];    // keys that reach the bound, per warp
  uint64_t best[32];        // the CTA's largest, descending
  uint64_t bound;
  int count[NW];
};

// Largest bound that at least k of the keys reach, to the point where no more
// than 2 k do; 0 if there are fewer than k.  One warp.
template <int NT>
__device__ __forceinline__ uint64_t top_bound(const uint64_t* keys, int k, int lane) {
  uint64_t mine[NT / 32], t = 0;
#pragma unroll
  for (int i = 0; i < NT / 32; ++i) mine[i] = keys[i * 32 + lane];
  for (int bit = 63; bit >= 0; --bit) {
    const uint64_t up = t | (1ull << bit);
    int n = 0;
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) n += mine[i] >= up;
    n = __reduce_add_sync(kFull, n);
    if (n < k) continue;
    t = up;
    if (n <= 2 * k) break;
  }
  return t;
}

// One row per CTA of NW warps.
template <class T, int NW, bool TOP>
__global__ void __launch_bounds__(NW * 32, NW == 8 ? 4 : NW == 4 ? 8 : 16) fw_logprob_kernel(ScoreArgs a) {
  constexpr int VN = 16 / sizeof(T), NT = NW * 32;
  __shared__ Sums part[NW];
  __shared__ float2 row_stat;
  __shared__ TopShared<TOP ? NW : 1> top;
  wait_prior_kernel();
  allow_dependent_launch();
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int64_t r = blockIdx.x;
  const int64_t y = a.y[r];
  if (y == a.ignore) {
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
  const int V = a.V;
  const int off = (int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
  const int slots = (int)(((int64_t)off + V + VN - 1) / VN);
  const int lo = off ? 1 : 0, hi = (int)(((int64_t)off + V) / VN);  // whole slots
  const float c = a.inv_t * kLog2e;
  Sums q = {-CUDART_INF_F, 0.0f, 0.0f};
  int at = tid;  // slot where the maximum first stood
  for (int k0 = tid; k0 < slots; k0 += NT * kBatch) {
    uint4 x[kBatch];
    if (k0 >= lo && k0 + (kBatch - 1) * NT < hi) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) x[i] = ld_global16_once(row + ((k0 + i * NT) * VN - off));
    } else {
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        x[i] = k0 + i * NT < slots ? load_slot_row(row, (k0 + i * NT) * VN - off, V) : neg_inf_slot<T>();
    }
    float sm[kBatch], bm = -CUDART_INF_F;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      sm[i] = slot_max_nan<T>(x[i]);
      bm = max_nan(bm, sm[i]);
    }
    if (!(bm <= q.m)) {
      const float to = max_nan(q.m, bm);
      q.raise(to, c);
      if (TOP) {
#pragma unroll
        for (int i = kBatch - 1; i >= 0; --i)
          if (sm[i] == to) at = k0 + i * NT;
      }
    }
    if (q.m == -CUDART_INF_F) continue;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      float z[VN];
      unpack16<T>(x[i], z);
#pragma unroll
      for (int j = 0; j < VN; ++j) {
        const float t = fmaxf((z[j] - q.m) * c, kFloor), e = exp2_ftz(t);
        q.s += e;
        q.u = fmaf(e, t, q.u);
      }
    }
  }
  if constexpr (TOP) {
    uint64_t first = 0;  // a thread without elements
    if (tid < slots) {
      float z[VN];
      const int e0 = at * VN - off;
      unpack16<T>(load_slot_row(row, e0, V), z);
#pragma unroll
      for (int j = VN - 1; j >= 0; --j)
        if (z[j] == q.m && e0 + j >= 0 && e0 + j < V) first = rank_key(z[j], e0 + j);
    }
    top.first[tid] = first;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Sums p = {__shfl_xor_sync(kFull, q.m, o), __shfl_xor_sync(kFull, q.s, o), __shfl_xor_sync(kFull, q.u, o)};
    q.join(p, c);
  }
  if (lane == 0) part[w] = q;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < NW; ++i) q.join(part[i], c);
    const bool label = y >= 0 && y < V, finite = fabsf(q.m) < CUDART_INF_F;
    const float nan = CUDART_NAN_F;
    float m = nan, logs = nan, h = nan, logp = nan;
    if (label && finite) {
      m = q.m;
      logs = logf(q.s);
      h = logs - q.u * kLn2 / q.s;
      logp = (Elem<T>::to_f(row[y]) - m) * a.inv_t - logs;
    }
    if (!label) raise_status(a.status, FWB_STATUS_LABEL_RANGE);
    if (!finite) raise_status(a.status, FWB_STATUS_NONFINITE);
    a.logp[r] = logp;
    a.entropy[r] = h;
    if (a.state) a.state[r] = make_float4(m, logs, h, __int_as_float(label ? (int)y : -1));
    row_stat = make_float2(m, logs);
  }
  if constexpr (TOP) {
    if (w == NW - 1) {
      const uint64_t b = top_bound<NT>(top.first, a.k, lane);
      if (lane == 0) top.bound = b;
    }
    __syncthreads();
    // `list`: the warp's 32 largest so far, once its buffer has overflowed; they raise its own bound, not the
    // one by which all warps share out the threads
    const uint64_t common = top.bound;
    uint64_t bound = common, list = 0;
    uint64_t* held = top.held[w];
    int n = 0;  // keys in the buffer
    bool full = false;
    const auto drain = [&] {
      __syncwarp();
      uint64_t x = lane < n ? held[lane] : 0;
      list = warp_merge(list, warp_sort(x, lane), lane);
      if (lane + 32 < n) x = held[lane + 32];
      __syncwarp();
      if (lane + 32 < n) held[lane] = x;
      n = max(n - 32, 0);
      full = true;
      __syncwarp();
    };
    int turn = 0;
    for (int g = 0; g < NW; ++g) {
      const uint64_t f = top.first[g * 32 + lane];
      // a bound of 0 stands for all of the row: threads without elements have none
      uint32_t who = __ballot_sync(kFull, f >= common && f != 0);
      for (; who; who &= who - 1) {
        if (turn++ % NW != w) continue;
        const int t = g * 32 + __ffs(who) - 1;
        for (int k0 = t; k0 < slots; k0 += NT * 32) {
          const int k = k0 + lane * NT;
          float z[VN];
          unpack16<T>(k < slots ? load_slot_row(row, k * VN - off, V) : neg_inf_slot<T>(), z);
#pragma unroll
          for (int j = 0; j < VN; ++j) {
            const int e = k * VN - off + j;
            const uint64_t key = k < slots && e >= 0 && e < V ? rank_key(z[j], e) : 0;
            const bool in = key != 0 && key >= bound;
            const uint32_t all = __ballot_sync(kFull, in);
            if (!all) continue;
            if (in) held[n + __popc(all & ((1u << lane) - 1u))] = key;
            n += __popc(all);
            if (n > 32) {
              drain();
              const uint64_t kth = __shfl_sync(kFull, list, a.k - 1);
              bound = kth > bound ? kth : bound;
            }
          }
        }
      }
    }
    if (full) {
      drain();
      held[lane] = list;
      n = __popc(__ballot_sync(kFull, list != 0));
    }
    if (lane == 0) top.count[w] = n;
    __syncthreads();
    const bool mine = lane < top.count[w];
    const uint64_t own = mine ? held[lane] : 0;
    int rank = 0;
    for (int g = 0; g < NW; ++g)
      for (int i = 0, ng = top.count[g]; i < ng; ++i) rank += top.held[g][i] > own;
    if (mine && rank < a.k) {
      const float2 st = row_stat;
      const bool bad = isnan(st.x);
      a.top_logp[r * a.k + rank] = bad ? CUDART_NAN_F : (key_value((uint32_t)(own >> 32)) - st.x) * a.inv_t - st.y;
      a.top_ids[r * a.k + rank] = bad ? -1 : (int64_t)(uint32_t)~(uint32_t)own;
    }
  }
}

// ------------------------------------------------------------ gradient
struct ScoreGradArgs {
  const void* z;
  int64_t B, ld, ldg;
  int V, units;  // units of kGradSlots slots per row
  float inv_t;
  const float4* state;
  const float *dlogp, *dentropy;  // either may be NULL: zero
  void* grad;
};

constexpr int kGradSlots = 32 * kBatch;  // a warp's step

// One warp per kGradSlots slots of the gradient's rows.
template <class T>
__global__ void __launch_bounds__(256, 4) fw_logprob_grad_kernel(ScoreGradArgs a) {
  constexpr int VN = 16 / sizeof(T);
  wait_prior_kernel();
  allow_dependent_launch();
  const int lane = threadIdx.x & 31;
  const int64_t work = a.B * a.units, step = (int64_t)gridDim.x * 8;
  const Span<T> span(a.z, a.B, a.ld, a.V);
  for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < work; i += step) {
    const int64_t r = i / a.units;
    const T* row = static_cast<const T*>(a.z) + r * a.ld;
    T* out = static_cast<T*>(a.grad) + r * a.ldg;
    const int off = (int)((reinterpret_cast<uintptr_t>(out) & 15u) / sizeof(T));
    const int e0 = (int)((i - r * a.units) * kGradSlots + lane) * VN - off;
    const float4 st = a.state[r];
    const int y = __float_as_int(st.w);
    const bool live = y != -2;
    uint4 x[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int e = e0 + b * 32 * VN;
      x[b] = make_uint4(0u, 0u, 0u, 0u);
      if (live && e < a.V) x[b] = load_slot_shifted(row, e, span);
    }
    const float g = a.dlogp ? a.dlogp[r] * a.inv_t : 0.0f, h = a.dentropy ? a.dentropy[r] * a.inv_t : 0.0f;
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int e = e0 + b * 32 * VN;
      if (e >= a.V) continue;
      float z[VN];
      unpack16<T>(x[b], z);
#pragma unroll
      for (int j = 0; j < VN; ++j) {
        // an element outside the row may be anything; it is not stored
        const float l = fmaxf((z[j] - st.x) * a.inv_t - st.y, kFloor);
        float d = -exp2_ftz(l * kLog2e) * (a.dentropy ? fmaf(h, l + st.z, g) : g);
        if (e + j == y) d += g;
        z[j] = live ? (isnan(st.x) ? CUDART_NAN_F : d) : 0.0f;
      }
      store_slot(out, (int64_t)e, (int64_t)a.V, true, pack_slot<T>(z));
    }
  }
}

// ------------------------------------------------------------ host
int score_check(int dtype, int64_t B, int64_t V, int64_t ld, float inv_t) {
  if (dtype != FWB_DTYPE_F32 && dtype != FWB_DTYPE_BF16 && dtype != FWB_DTYPE_F16) return FWB_E_DTYPE;
  if (B < 0 || V < 1 || ld < V || B > (1 << 28) || V > (1 << 28) || ld > ((int64_t)1 << 32)) return FWB_E_SHAPE;
  if (!(inv_t > 0.0f) || !std::isfinite(inv_t)) return FWB_E_SHAPE;
  return FWB_OK;
}

bool misaligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }

template <class T, int NW>
int launch_score(const ScoreArgs& a, cudaStream_t st) {
  return launch_status(a.k > 0 ? launch_dependent(fw_logprob_kernel<T, NW, true>, a.B, NW * 32, 0, 1, st, a)
                               : launch_dependent(fw_logprob_kernel<T, NW, false>, a.B, NW * 32, 0, 1, st, a));
}

template <class T>
int run_score(const ScoreArgs& a, cudaStream_t st) {
  const int slots = a.V / (16 / (int)sizeof(T));
  if (slots <= 256) return launch_score<T, 1>(a, st);
  if (slots <= 2048) return launch_score<T, 4>(a, st);
  return launch_score<T, 8>(a, st);
}

template <class T>
int run_score_grad(ScoreGradArgs a, cudaStream_t st) {
  const int64_t slots = a.V / (16 / (int)sizeof(T)) + 2;  // whatever the row's start
  a.units = (int)((slots + kGradSlots - 1) / kGradSlots);
  const int64_t need = (a.B * a.units + 7) / 8, cap = (int64_t)sm_count() * 48;
  return launch_status(launch_dependent(fw_logprob_grad_kernel<T>, need < cap ? need : cap, 256, 0, 1, st, a));
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
