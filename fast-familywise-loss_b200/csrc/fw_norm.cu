// Root-mean-square norm of a residual stream: the addition, the norm, its
// gradient, and the form whose output is 8-bit integers with a scale per row
// (the input of the 8-bit output layer).
//
//   s = x + residual, rounded to the stream's type      (s = x without one)
//   y = s * rstd * w,   rstd = 1 / sqrt(mean(s^2) + eps)
//   q = y / scale to the nearest, scale = max|y| / 127  (8-bit form)
//
// s is defined as the stored, rounded sum, so the gradient (which reads the
// stored stream) is the gradient of exactly this function:
//   a = dy * w,  c = sum(a * s) * rstd^2 / D
//   ds = rstd * (a - s * c) + ds_out,  dx = dresidual = ds
//   dw = sum over rows of dy * s * rstd
// Sums, statistics and gains are fp32; each output is rounded once.
//
// Bound by HBM: forward reads x and residual and writes s and y, backward
// reads dy, s and ds_out and writes ds, each once.  A row belongs to a group
// of G threads (a warp, or a CTA of up to 1024), CH slots of 16 bytes per
// thread (fw_rowslots.cuh).  The next kAhead rows of a group are on their way
// into shared memory (cp.async; each thread copies the slots it will read, so
// no barrier is needed) while a row is reduced: a CTA-wide reduction would
// otherwise drain the memory pipe at every row.  The grid is persistent with
// a group count that is a multiple of 8, so that the rows one group visits
// all start at the same distance from a 16-byte boundary: a thread keeps the
// same columns from row to row, hence its gains and its part of dw stay in
// registers for any D.  dw parts are written once per CTA and added in a
// fixed order by a second kernel.
//
// Forward and backward with a residual, 16384 x 4096 bfloat16 (1.07 GB): 193
// to 201 us, 5.3 to 5.6 TB/s; without the copies ahead 202 where it takes 193.  8001 x 7001 (rows at every
// alignment): 174 us, 5.2 TB/s, without them 570.
#include <cuda_runtime.h>

#include <climits>

#include "fw_host.cuh"
#include "fw_rowslots.cuh"

namespace fwb200 {
namespace {

enum { kNormOut = 0, kNormInt8 = 1, kInt8Only = 2 };

struct NormArgs {
  const void* x;
  const void* res;
  const void* w;
  void* s;
  void* y;
  float* rstd;
  int8_t* q;
  float* qscale;
  int64_t ldx, ldr, lds, ldy, ldq;
  int64_t rows, D;
  float eps;
  int w_f32;  // gains are fp32 whatever T is
  int vec;    // x, residual, s and y rows share their distance from a 16-byte boundary
};

struct NormGradArgs {
  const void* dy;
  const void* s;
  const void* dso;
  const void* w;
  const float* rstd;
  void* dx;
  float* part;  // [gridDim.x, D]
  int64_t lddy, lds, ldo, lddx;
  int64_t rows, D;
  int w_f32;
  int vec;
};

template <class T>
__device__ __forceinline__ int row_off(const void* base, int64_t row, int64_t ld, int vec) {
  if (!vec) return 0;
  return (int)((reinterpret_cast<uintptr_t>(base) + (uintptr_t)(row * ld) * sizeof(T)) & 15u) / (int)sizeof(T);
}

// Gains of slot e0.., zero outside the row.
template <class T>
__device__ __forceinline__ void load_gain(const void* w, int w_f32, int64_t e0, int64_t D, float* out) {
  constexpr int V = 16 / sizeof(T);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int64_t e = e0 + j;
    float g = 0.0f;
    if (e >= 0 && e < D) g = w_f32 ? static_cast<const float*>(w)[e] : ld_elem(static_cast<const T*>(w) + e);
    out[j] = g;
  }
}

// Sum (or NaN-propagating maximum) over the G threads of a group; `buf` holds
// one float per warp and alternates between two halves so that one barrier
// per call is enough.
template <int G, bool MAX>
__device__ __forceinline__ float group_reduce(float v, float* buf, int& flip) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float u = __shfl_xor_sync(kFull, v, o);
    v = MAX ? max_nan(v, u) : v + u;
  }
  if constexpr (G > 32) {
    float* b = buf + flip * (G / 32);
    flip ^= 1;
    if ((threadIdx.x & 31) == 0) b[threadIdx.x >> 5] = v;
    __syncthreads();
    // four partial results side by side, then their join: 16-byte loads, short chains
    float t[4];
#pragma unroll
    for (int i = 0; i < G / 128; ++i) {
      const float4 x = reinterpret_cast<const float4*>(b)[i];
      t[0] = i == 0 ? x.x : MAX ? max_nan(t[0], x.x) : t[0] + x.x;
      t[1] = i == 0 ? x.y : MAX ? max_nan(t[1], x.y) : t[1] + x.y;
      t[2] = i == 0 ? x.z : MAX ? max_nan(t[2], x.z) : t[2] + x.z;
      t[3] = i == 0 ? x.w : MAX ? max_nan(t[3], x.w) : t[3] + x.w;
    }
    v = MAX ? max_nan(max_nan(t[0], t[1]), max_nan(t[2], t[3])) : (t[0] + t[1]) + (t[2] + t[3]);
  }
  return v;
}

// Scale of a row whose largest value is m; rounded up where it is subnormal,
// so that no value is more than 127 steps.
__device__ __forceinline__ float int8_scale(float m) {
  const float scale = m / 127.0f;
  return scale < 0x1p-126f ? __fdiv_ru(m, 127.0f) : scale;
}

// Values in steps of their row's scale, to the nearest, as bytes; 0 for a row
// that has no such step (its values may be NaN).  1 / scale does not fit fp32
// for the smallest scales, hence the power of two taken out of it.  Its
// rounding moves a value by less than 2^-17 of a step, so one that close to
// the middle between two steps may take either.  The steps are added to 1.5 *
// 2^23, whose unit is 1: the addition rounds, and the sum's low byte is the
// integer (a third of the instructions of rounding, clamping and converting:
// norm of 16384 x 4096 bfloat16 with residual 95 us, alone 65, the rows
// themselves 47, for 113, 88 and 69; of 32000 x 2048 float32 162, 94 and 73, for
// 158, 114 and 94; of 8000 x 8192 float32 with residual 297 for 348).
struct Int8Steps {
  float up, per_step;
  uint32_t keep;
  __device__ __forceinline__ explicit Int8Steps(float scale) {
    const bool some = scale > 0.0f && scale < CUDART_INF_F;
    up = scale < 0x1p-100f ? 0x1p100f : 1.0f;
    per_step = some ? 1.0f / (scale * up) : 0.0f;
    keep = some ? 0xffffffffu : 0u;
  }
  __device__ __forceinline__ uint32_t word(float y) const {  // low byte
    return __float_as_uint(fmaf(y * up, per_step, 12582912.0f));
  }
  __device__ __forceinline__ int8_t one(float y) const { return (int8_t)(word(y) & keep & 0xffu); }
  __device__ __forceinline__ uint32_t four(const float* y) const {
    return __byte_perm(__byte_perm(word(y[0]), word(y[1]), 0x0040), __byte_perm(word(y[2]), word(y[3]), 0x0040), 0x5410) &
           keep;
  }
};

template <int G>
__host__ __device__ constexpr int cta_threads() {
  return G < 128 ? 128 : G;
}

constexpr int kAhead = 2;  // rows of a group in flight

// A thread's slots of the rows in flight, of NT matrices, in shared memory
// (slot k of stage d of matrix m at [(d * NT + m) * CH + k][t]).
template <class T, int G, int CH, int NT>
struct RowRing {
  static constexpr int V = 16 / sizeof(T);
  uint4* mine;
  int e0, D;   // first element of slot 0 (negative where the row starts inside it), elements of a row
  int vec;

  __device__ __forceinline__ void init(uint4* smem, int grp, int t, int off, int D_, int vec_) {
    mine = smem + (size_t)grp * kAhead * NT * CH * G + t;
    e0 = t * V - off;
    D = D_;
    vec = vec_;
#pragma unroll
    for (int i = 0; i < kAhead * NT * CH; ++i) mine[i * G] = make_uint4(0u, 0u, 0u, 0u);  // slots past the row stay 0
  }
  // Starts matrix m's row (number r of its matrix) on its way into stage d.
  __device__ __forceinline__ void fetch(int d, int m, const T* row, int64_t r) {
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const int e = e0 + k * (G * V);
      if (e >= D) continue;
      uint4* to = mine + ((d * NT + m) * CH + k) * G;
      if (vec && (e >= 0 || r > 0)) {
        // whole slots of memory: what lies before the row is masked when read, behind it is not read
        const uint32_t bytes = min(16, (D - e) * (int)sizeof(T));
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to)), "l"(row + e), "r"(bytes)
                     : "memory");
      } else {
        *to = load_elems(row + e, row, row + D);
      }
    }
  }
  __device__ __forceinline__ static void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
  // The oldest row in flight has landed.
  __device__ __forceinline__ static void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory"); }
  __device__ __forceinline__ void get(int d, int m, int k, float* v) const {
    unpack16<T>(mine[((d * NT + m) * CH + k) * G], v);
    if (k == 0 && e0 < 0) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < -e0) v[j] = 0.0f;
    }
  }
};

template <class T, int G, int CH>
__host__ __device__ constexpr size_t ring_bytes(int nt) {
  return (size_t)(G < 128 ? 128 / G : 1) * kAhead * nt * CH * G * 16;
}

template <class T, int G, int CH, int MODE>
__global__ void __launch_bounds__(cta_threads<G>(), 1024 / cta_threads<G>()) fw_norm_kernel(NormArgs a) {
  constexpr int V = 16 / sizeof(T);
  constexpr int R = cta_threads<G>() / G;
  __shared__ __align__(16) float red[2 * (G / 32)];
  extern __shared__ __align__(16) uint4 norm_smem[];
  const int t = threadIdx.x % G;
  const int grp = threadIdx.x / G;
  const int64_t step = (int64_t)gridDim.x * R;
  const int64_t first = (int64_t)blockIdx.x * R + grp;
  wait_prior_kernel();
  allow_dependent_launch();
  if (first >= a.rows) return;  // a whole group; groups of one CTA share no barrier unless R == 1
  int flip = 0;
  const int off = row_off<T>(a.x, first, a.ldx, a.vec);
  const int D = (int)a.D;  // fits: longer rows take the other kernel
  RowRing<T, G, CH, 2> ring;
  ring.init(norm_smem, grp, t, off, D, a.vec);
  const int e0 = ring.e0;
  auto fetch = [&](int d, int64_t r) {
    if (r < a.rows) {
      ring.fetch(d, 0, static_cast<const T*>(a.x) + r * a.ldx, r);
      if (a.res) ring.fetch(d, 1, static_cast<const T*>(a.res) + r * a.ldr, r);
    }
    ring.commit();
  };
#pragma unroll
  for (int d = 0; d < kAhead; ++d) fetch(d, first + d * step);
  float gain[CH * V];
  if constexpr (MODE != kInt8Only) {
#pragma unroll
    for (int k = 0; k < CH; ++k) load_gain<T>(a.w, a.w_f32, e0 + k * (G * V), D, gain + k * V);
  }
  const float inv_d = 1.0f / (float)a.D;
  int d = 0;
  for (int64_t r = first; r < a.rows; r += step) {
    ring.wait();
    float v[CH * V];
#pragma unroll
    for (int k = 0; k < CH; ++k) ring.get(d, 0, k, v + k * V);
    if (a.res) {
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        float u[V];
        ring.get(d, 1, k, u);
#pragma unroll
        for (int j = 0; j < V; ++j) u[j] += v[k * V + j];
        const uint4 p = pack_slot<T>(u);
        unpack16<T>(p, v + k * V);
        store_slot(static_cast<T*>(a.s) + r * a.lds, e0 + k * (G * V), D, a.vec, p);
      }
    }
    fetch(d, r + kAhead * step);
    d = d + 1 == kAhead ? 0 : d + 1;
    if constexpr (MODE != kInt8Only) {
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < CH * V; ++i) ss = fmaf(v[i], v[i], ss);
      ss = group_reduce<G, false>(ss, red, flip);
      const float rstd = 1.0f / sqrtf(fmaf(ss, inv_d, a.eps));
      if (a.rstd && t == 0) a.rstd[r] = rstd;
#pragma unroll
      for (int i = 0; i < CH * V; ++i) v[i] = v[i] * rstd * gain[i];
    }
    if constexpr (MODE == kNormOut) {
#pragma unroll
      for (int k = 0; k < CH; ++k)
        store_slot(static_cast<T*>(a.y) + r * a.ldy, e0 + k * (G * V), D, a.vec, pack_slot<T>(v + k * V));
    } else {
      float m = 0.0f;
#pragma unroll
      for (int i = 0; i < CH * V; ++i) m = max_nan(m, fabsf(v[i]));  // slots past the row hold 0 * 0
      m = group_reduce<G, true>(m, red, flip);
      const float scale = int8_scale(m);
      if (t == 0) a.qscale[r] = scale;
      // a row of zeros, or not finite, is 0 (or NaN) through its scale
      const Int8Steps steps(scale);
      const int w16 = (D + 15) / 16 * 16;
      static_assert(CH * G * V % 16 == 0, "the slots cover the row's padding");
      if (off == 0) {  // the slots' bytes lie together in q
#pragma unroll
        for (int k = 0; k < CH; ++k) {
          const int e = e0 + k * (G * V);
          if (e >= w16) continue;
          uint32_t b[V / 4];
#pragma unroll
          for (int j = 0; j < V; j += 4) b[j / 4] = steps.four(v + k * V + j);
          if constexpr (V == 8)
            *reinterpret_cast<uint2*>(a.q + r * a.ldq + e) = make_uint2(b[0], b[1]);
          else
            *reinterpret_cast<uint32_t*>(a.q + r * a.ldq + e) = b[0];
        }
      } else {  // through shared memory
        int8_t* qs = reinterpret_cast<int8_t*>(norm_smem) + ring_bytes<T, G, CH>(2) + grp * w16;
        if (t < 16 && D + t < w16) qs[D + t] = 0;
#pragma unroll
        for (int i = 0; i < CH * V; ++i) {
          const int e = e0 + (i / V) * (G * V) + i % V;
          if (e >= 0 && e < D) qs[e] = steps.one(v[i]);
        }
        if constexpr (G > 32)
          __syncthreads();
        else
          __syncwarp();
        for (int i = t; i < w16 / 16; i += G)
          reinterpret_cast<uint4*>(a.q + r * a.ldq)[i] = reinterpret_cast<const uint4*>(qs)[i];
        if constexpr (G > 32)
          __syncthreads();
        else
          __syncwarp();
      }
    }
  }
}

// Rows too long for a CTA's registers: passes over the row in memory.
template <class T, int MODE>
__global__ void __launch_bounds__(1024) fw_norm_long_kernel(NormArgs a) {
  __shared__ __align__(16) float red[2 * 32];
  int flip = 0;
  wait_prior_kernel();
  allow_dependent_launch();
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* xr = static_cast<const T*>(a.x) + r * a.ldx;
    const T* rr = a.res ? static_cast<const T*>(a.res) + r * a.ldr : nullptr;
    auto elem = [&](int64_t e) {
      float v = ld_elem(xr + e);
      return rr ? Elem<T>::to_f(Elem<T>::from_f(v + ld_elem(rr + e))) : v;
    };
    auto gain = [&](int64_t e) {
      return a.w_f32 ? static_cast<const float*>(a.w)[e] : ld_elem(static_cast<const T*>(a.w) + e);
    };
    float rstd = 1.0f;
    if constexpr (MODE != kInt8Only) {
      float ss = 0.0f;
      for (int64_t e = threadIdx.x; e < a.D; e += 1024) {
        const float v = elem(e);
        ss = fmaf(v, v, ss);
      }
      ss = group_reduce<1024, false>(ss, red, flip);
      rstd = 1.0f / sqrtf(ss / (float)a.D + a.eps);
      if (a.rstd && threadIdx.x == 0) a.rstd[r] = rstd;
    }
    float m = 0.0f;
    for (int64_t e = threadIdx.x; e < a.D; e += 1024) {
      float v = elem(e);
      if (rr && a.s) st_elem(static_cast<T*>(a.s) + r * a.lds + e, v);
      if constexpr (MODE != kInt8Only) v = v * rstd * gain(e);
      if constexpr (MODE == kNormOut)
        st_elem(static_cast<T*>(a.y) + r * a.ldy + e, v);
      else
        m = max_nan(m, fabsf(v));
    }
    if constexpr (MODE != kNormOut) {
      m = group_reduce<1024, true>(m, red, flip);
      const float scale = int8_scale(m);
      if (threadIdx.x == 0) a.qscale[r] = scale;
      const Int8Steps steps(scale);
      for (int64_t e = threadIdx.x; e < (a.D + 15) / 16 * 16; e += 1024) {
        float v = 0.0f;
        if (e < a.D) {
          v = elem(e);
          if constexpr (MODE != kInt8Only) v = v * rstd * gain(e);
        }
        a.q[r * a.ldq + e] = steps.one(v);
      }
    }
  }
}

template <class T, int G, int CH>
__global__ void __launch_bounds__(cta_threads<G>(), 1024 / cta_threads<G>()) fw_norm_grad_kernel(NormGradArgs a) {
  constexpr int V = 16 / sizeof(T);
  constexpr int R = cta_threads<G>() / G;
  __shared__ __align__(16) float red[2 * (G / 32)];
  extern __shared__ __align__(16) uint4 norm_smem[];
  wait_prior_kernel();
  allow_dependent_launch();
  const int t = threadIdx.x % G;
  const int grp = threadIdx.x / G;
  const int64_t step = (int64_t)gridDim.x * R;
  const int64_t first = (int64_t)blockIdx.x * R + grp;
  int flip = 0;
  const int off = row_off<T>(a.s, first, a.lds, a.vec);
  const int D = (int)a.D;
  RowRing<T, G, CH, 3> ring;
  ring.init(norm_smem, grp, t, off, D, a.vec);
  const int e0 = ring.e0;
  auto fetch = [&](int d, int64_t r) {
    if (r < a.rows) {
      ring.fetch(d, 0, static_cast<const T*>(a.s) + r * a.lds, r);
      ring.fetch(d, 1, static_cast<const T*>(a.dy) + r * a.lddy, r);
      if (a.dso) ring.fetch(d, 2, static_cast<const T*>(a.dso) + r * a.ldo, r);
    }
    ring.commit();
  };
#pragma unroll
  for (int d = 0; d < kAhead; ++d) fetch(d, first + d * step);
  float gain[CH * V], dw[CH * V];
#pragma unroll
  for (int k = 0; k < CH; ++k) load_gain<T>(a.w, a.w_f32, e0 + k * (G * V), D, gain + k * V);
#pragma unroll
  for (int i = 0; i < CH * V; ++i) dw[i] = 0.0f;
  const float inv_d = 1.0f / (float)a.D;
  float rs_next = first < a.rows ? a.rstd[first] : 0.0f;
  int d = 0;
  for (int64_t r = first; r < a.rows; r += step) {
    const float rs = rs_next;
    if (r + step < a.rows) rs_next = a.rstd[r + step];
    ring.wait();
    float c = 0.0f;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      float s[V], g[V];
      ring.get(d, 0, k, s);
      ring.get(d, 1, k, g);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float n = s[j] * rs;
        c = fmaf(g[j] * gain[k * V + j], n, c);
        dw[k * V + j] = fmaf(g[j], n, dw[k * V + j]);
      }
    }
    c = group_reduce<G, false>(c, red, flip) * inv_d;
    // read again rather than kept: registers are what bounds the rows in flight
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      float s[V], g[V], o[V];
      ring.get(d, 0, k, s);
      ring.get(d, 1, k, g);
      ring.get(d, 2, k, o);  // zero without dsum
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = fmaf(rs, fmaf(-(s[j] * rs), c, g[j] * gain[k * V + j]), o[j]);
      store_slot(static_cast<T*>(a.dx) + r * a.lddx, e0 + k * (G * V), D, a.vec, pack_slot<T>(o));
    }
    fetch(d, r + kAhead * step);
    d = d + 1 == kAhead ? 0 : d + 1;
  }
  if (!a.part) return;
  float* part = a.part + (int64_t)blockIdx.x * a.D;
  if constexpr (R == 1) {
#pragma unroll
    for (int i = 0; i < CH * V; ++i) {
      const int64_t e = (int64_t)((i / V) * G + t) * V - off + i % V;
      if (e >= 0 && e < a.D) part[e] = dw[i];
    }
  } else {
    float* dw_row = reinterpret_cast<float*>(norm_smem);  // the rings are done with
    __syncthreads();
    for (int64_t e = threadIdx.x; e < a.D; e += blockDim.x) dw_row[e] = 0.0f;
    for (int g = 0; g < R; ++g) {  // the CTA's groups in order: their rows start at different distances
      __syncthreads();
      if (grp == g) {
#pragma unroll
        for (int i = 0; i < CH * V; ++i) {
          const int64_t e = (int64_t)((i / V) * G + t) * V - off + i % V;
          if (e >= 0 && e < a.D) dw_row[e] += dw[i];
        }
      }
    }
    __syncthreads();
    for (int64_t e = threadIdx.x; e < a.D; e += blockDim.x) part[e] = dw_row[e];
  }
}

template <class T>
__global__ void __launch_bounds__(1024) fw_norm_grad_long_kernel(NormGradArgs a) {
  __shared__ __align__(16) float red[2 * 32];
  int flip = 0;
  wait_prior_kernel();
  allow_dependent_launch();
  float* part = a.part ? a.part + (int64_t)blockIdx.x * a.D : nullptr;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* sr = static_cast<const T*>(a.s) + r * a.lds;
    const T* gr = static_cast<const T*>(a.dy) + r * a.lddy;
    const float rstd = a.rstd[r];
    auto gain = [&](int64_t e) {
      return a.w_f32 ? static_cast<const float*>(a.w)[e] : ld_elem(static_cast<const T*>(a.w) + e);
    };
    float c = 0.0f;
    for (int64_t e = threadIdx.x; e < a.D; e += 1024) {
      const float n = ld_elem(sr + e) * rstd, g = ld_elem(gr + e);
      c = fmaf(g * gain(e), n, c);
      if (part) part[e] = r == blockIdx.x ? g * n : fmaf(g, n, part[e]);  // this thread's own columns
    }
    c = group_reduce<1024, false>(c, red, flip) / (float)a.D;
    for (int64_t e = threadIdx.x; e < a.D; e += 1024) {
      const float o = a.dso ? ld_elem(static_cast<const T*>(a.dso) + r * a.ldo + e) : 0.0f;
      const float v = fmaf(rstd, fmaf(ld_elem(gr + e), gain(e), -(ld_elem(sr + e) * rstd) * c), o);
      st_elem(static_cast<T*>(a.dx) + r * a.lddx + e, v);
    }
  }
}

// dw[e] = sum over the parts, in a fixed order: 32 columns per CTA, each of
// its 32 warps adds every 32nd part.
template <class T>
__global__ void __launch_bounds__(1024) fw_norm_dw_kernel(const float* part, int64_t n, int64_t D, T* dw) {
  __shared__ float sm[32][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t e = (int64_t)blockIdx.x * 32 + lane;
  wait_prior_kernel();
  allow_dependent_launch();
  float s = 0.0f;
  if (e < D) {
#pragma unroll 8
    for (int64_t p = w; p < n; p += 32) s += part[p * D + e];
  }
  sm[w][lane] = s;
  __syncthreads();
  // warp w takes column w of the block
  s = sm[lane][w];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kFull, s, o);
  const int64_t c = (int64_t)blockIdx.x * 32 + w;
  if (lane == 0 && c < D) st_elem(dw + c, s);
}

// Threads per row by its slots: a warp, or a CTA with one or two
// slots per thread, so that a thread's 64 registers hold its gains and its
// part of dw; the memory-pass kernels beyond 2048 slots.  With 1024 threads
// one CTA fills an SM and nothing covers its barriers, and the gradient's 64
// registers spill a few: 2000 x 16000 bfloat16 takes 76 us forward and 122
// backward, where the bytes take 39 each way; the memory passes, for 2000 x
// 17000, 102 and 286.
struct NormShape {
  int G, CH;
};

// Slots that a row of the matrix covers at most: one more than its elements
// fill where a row may start inside a slot.
int64_t row_slots(const void* base, int64_t ld, int64_t D, int64_t esize, bool vec) {
  const bool inside = vec && (!aligned16(base) || ld * esize % 16 != 0);
  return (D * esize + 15) / 16 + (inside ? 1 : 0);
}

NormShape norm_shape(int64_t n) {
  if (n <= 32) return {32, 1};
  if (n <= 128) return {128, 1};
  if (n <= 256) return {128, 2};
  if (n <= 512) return {256, 2};
  if (n <= 1024) return {512, 2};
  if (n <= 2048) return {1024, 2};
  return {0, 0};
}

// Persistent grid: enough CTAs for about 1024 resident threads per SM, a
// multiple of 8 unless every group has at most one row.
int64_t norm_grid(int64_t rows, int G) {
  const int threads = G == 0 ? 1024 : (G < 128 ? 128 : G);
  const int64_t R = G == 0 ? 1 : threads / G;
  const int64_t need = (rows + R - 1) / R;
  int64_t cap = (int64_t)sm_count() * (G == 0 ? 2 : 1024 / threads);
  cap = (cap + 7) / 8 * 8;
  return need < cap ? need : cap;
}

bool same_slots(const void* p, int64_t ld, const void* q, int64_t ldq, int64_t esize) {
  return ((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(q)) & 15u) == 0 &&
         ((ld - ldq) * esize) % 16 == 0;
}

bool elem_aligned(const void* p, int64_t esize) { return reinterpret_cast<uintptr_t>(p) % esize == 0; }

int esize_of(int dtype) { return dtype == FWB_DTYPE_F32 ? 4 : 2; }

int norm_check(int dtype, int wdtype, int64_t rows, int64_t D) {
  if (dtype != FWB_DTYPE_F32 && dtype != FWB_DTYPE_BF16 && dtype != FWB_DTYPE_F16) return FWB_E_DTYPE;
  if (wdtype != dtype && wdtype != FWB_DTYPE_F32) return FWB_E_DTYPE;
  if (rows < 0 || D < 1 || D > (int64_t)INT_MAX - 64) return FWB_E_SHAPE;
  return FWB_OK;
}

bool ld_ok(int64_t ld, int64_t rows, int64_t D) {
  return ld >= D && (rows <= 0 || ld <= ((int64_t)1 << 60) / rows);
}

// More than 48 KB of shared memory has to be asked for, once per device.
template <class... KArgs, class A>
cudaError_t launch_rows(void (*kernel)(KArgs...), std::atomic<bool>* asked, int64_t grid, int threads, size_t smem,
                        cudaStream_t st, const A& a) {
  if (smem > 40 * 1024) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= kMaxDevices || !asked[dev].load(std::memory_order_acquire)) {
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - 1024);
      if (e != cudaSuccess) return e;
      if (dev < kMaxDevices) asked[dev].store(true, std::memory_order_release);
    }
  }
  return launch_dependent(kernel, grid, threads, smem, 1, st, a);
}

template <class T, int MODE, int G, int CH>
cudaError_t launch_norm(const NormArgs& a, cudaStream_t st) {
  static std::atomic<bool> asked[kMaxDevices] = {};
  const size_t q = MODE == kNormOut ? 0 : (size_t)(G < 128 ? 128 / G : 1) * (size_t)((a.D + 15) / 16 * 16);
  return launch_rows(fw_norm_kernel<T, G, CH, MODE>, asked, norm_grid(a.rows, G), cta_threads<G>(),
                     ring_bytes<T, G, CH>(2) + q, st, a);
}

template <class T, int MODE>
cudaError_t launch_norm(const NormArgs& a, cudaStream_t st) {
  const NormShape sh = norm_shape(row_slots(a.x, a.ldx, a.D, sizeof(T), a.vec));
  if (sh.G == 32) return launch_norm<T, MODE, 32, 1>(a, st);
  if (sh.G == 128 && sh.CH == 1) return launch_norm<T, MODE, 128, 1>(a, st);
  if (sh.G == 128) return launch_norm<T, MODE, 128, 2>(a, st);
  if (sh.G == 256) return launch_norm<T, MODE, 256, 2>(a, st);
  if (sh.G == 512) return launch_norm<T, MODE, 512, 2>(a, st);
  if (sh.G == 1024) return launch_norm<T, MODE, 1024, 2>(a, st);
  return launch_dependent(fw_norm_long_kernel<T, MODE>, norm_grid(a.rows, 0), 1024, 0, 1, st, a);
}

template <class T, int G, int CH>
cudaError_t launch_norm_grad(const NormGradArgs& a, cudaStream_t st) {
  static std::atomic<bool> asked[kMaxDevices] = {};
  size_t smem = ring_bytes<T, G, CH>(3);
  if (G < 128 && smem < (size_t)a.D * 4) smem = (size_t)a.D * 4;
  return launch_rows(fw_norm_grad_kernel<T, G, CH>, asked, norm_grid(a.rows, G), cta_threads<G>(), smem, st, a);
}

template <class T>
cudaError_t launch_norm_grad(const NormGradArgs& a, cudaStream_t st) {
  const NormShape sh = norm_shape(row_slots(a.s, a.lds, a.D, sizeof(T), a.vec));
  if (sh.G == 32) return launch_norm_grad<T, 32, 1>(a, st);
  if (sh.G == 128 && sh.CH == 1) return launch_norm_grad<T, 128, 1>(a, st);
  if (sh.G == 128) return launch_norm_grad<T, 128, 2>(a, st);
  if (sh.G == 256) return launch_norm_grad<T, 256, 2>(a, st);
  if (sh.G == 512) return launch_norm_grad<T, 512, 2>(a, st);
  if (sh.G == 1024) return launch_norm_grad<T, 1024, 2>(a, st);
  return launch_dependent(fw_norm_grad_long_kernel<T>, norm_grid(a.rows, 0), 1024, 0, 1, st, a);
}

template <int MODE>
int run_norm(int dtype, const NormArgs& a, cudaStream_t st) {
  if (dtype == FWB_DTYPE_BF16) return launch_status(launch_norm<__nv_bfloat16, MODE>(a, st));
  if (dtype == FWB_DTYPE_F16) return launch_status(launch_norm<__half, MODE>(a, st));
  return launch_status(launch_norm<float, MODE>(a, st));
}

// Shared by the entry points: argument checks and the slot test.
int norm_args(int dtype, int wdtype, const void* x, int64_t ldx, const void* res, int64_t ldr, const void* w,
              int64_t rows, int64_t D, float eps, void* s, int64_t lds, NormArgs* a) {
  if (int rc = norm_check(dtype, wdtype, rows, D)) return rc;
  if (!ld_ok(ldx, rows, D) || (res && !ld_ok(ldr, rows, D)) || (s && !ld_ok(lds, rows, D))) return FWB_E_SHAPE;
  if (!(eps >= 0.0f)) return FWB_E_SHAPE;
  const int es = esize_of(dtype);
  if (!elem_aligned(x, es) || !elem_aligned(res, es) || !elem_aligned(s, es) || !elem_aligned(w, esize_of(wdtype)))
    return FWB_E_POINTER;
  a->x = x;
  a->res = res;
  a->w = w;
  a->s = s;
  a->ldx = ldx;
  a->ldr = ldr;
  a->lds = lds;
  a->rows = rows;
  a->D = D;
  a->eps = eps;
  a->w_f32 = wdtype == FWB_DTYPE_F32 && dtype != FWB_DTYPE_F32;
  a->vec = (!res || same_slots(x, ldx, res, ldr, es)) && (!s || same_slots(x, ldx, s, lds, es));
  return FWB_OK;
}

int int8_rows_check(const int8_t* q, int64_t ldq, int64_t rows, int64_t D) {
  if (ldq % 16 != 0 || ldq < (D + 15) / 16 * 16 || (rows > 0 && ldq > ((int64_t)1 << 60) / rows)) return FWB_E_SHAPE;
  return aligned16(q) ? FWB_OK : FWB_E_POINTER;
}

}  // namespace
}  // namespace fwb200

using namespace fwb200;

extern "C" {

int fw_rms_norm(int dtype, int wdtype, const void* x, int64_t ldx, const void* residual, int64_t ldr,
                const void* weight, int64_t rows, int64_t D, float eps, void* sum, int64_t lds, void* y, int64_t ldy,
                float* rstd, void* stream) {
  NormArgs a = {};
  if (int rc = norm_args(dtype, wdtype, x, ldx, residual, ldr, weight, rows, D, eps, sum, lds, &a)) return rc;
  if (!ld_ok(ldy, rows, D)) return FWB_E_SHAPE;
  if (rows == 0) return FWB_OK;
  if (!x || !weight || !y || (residual && !sum)) return FWB_E_POINTER;
  const int es = esize_of(dtype);
  if (!elem_aligned(y, es)) return FWB_E_POINTER;
  a.y = y;
  a.ldy = ldy;
  a.rstd = rstd;
  a.vec = a.vec && same_slots(x, ldx, y, ldy, es);
  return run_norm<kNormOut>(dtype, a, static_cast<cudaStream_t>(stream));
}

int fw_rms_norm_int8(int dtype, int wdtype, const void* x, int64_t ldx, const void* residual, int64_t ldr,
                     const void* weight, int64_t rows, int64_t D, float eps, void* sum, int64_t lds, int8_t* q,
                     int64_t ldq, float* scale, void* stream) {
  NormArgs a = {};
  if (int rc = norm_args(dtype, wdtype, x, ldx, residual, ldr, weight, rows, D, eps, sum, lds, &a)) return rc;
  if (rows == 0) return FWB_OK;
  if (!x || !weight || !q || !scale || (residual && !sum)) return FWB_E_POINTER;
  if (int rc = int8_rows_check(q, ldq, rows, D)) return rc;
  a.q = q;
  a.ldq = ldq;
  a.qscale = scale;
  return run_norm<kNormInt8>(dtype, a, static_cast<cudaStream_t>(stream));
}

int fw_quantize_rows_int8(int dtype, const void* x, int64_t ldx, int64_t rows, int64_t D, int8_t* q, int64_t ldq,
                          float* scale, void* stream) {
  NormArgs a = {};
  if (int rc = norm_args(dtype, dtype, x, ldx, nullptr, 0, nullptr, rows, D, 0.0f, nullptr, 0, &a)) return rc;
  if (rows == 0) return FWB_OK;
  if (!x || !q || !scale) return FWB_E_POINTER;
  if (int rc = int8_rows_check(q, ldq, rows, D)) return rc;
  a.q = q;
  a.ldq = ldq;
  a.qscale = scale;
  return run_norm<kInt8Only>(dtype, a, static_cast<cudaStream_t>(stream));
}

// An upper bound on the parts of dweight that fw_rms_norm_grad writes, by the
// largest grid of any shape it may choose.
int64_t fw_rms_norm_grad_parts(int64_t rows) {
  if (rows < 0) return 0;
  const int64_t cap = ((int64_t)sm_count() * 8 + 7) / 8 * 8;
  return rows < cap ? rows : cap;
}

int fw_rms_norm_grad(int dtype, int wdtype, const void* dy, int64_t lddy, const void* sum, int64_t lds,
                     const void* dsum, int64_t ldo, const void* weight, const float* rstd, int64_t rows, int64_t D,
                     void* dx, int64_t lddx, float* parts, int64_t nparts, void* dweight, void* stream) {
  if (int rc = norm_check(dtype, wdtype, rows, D)) return rc;
  if (!ld_ok(lddy, rows, D) || !ld_ok(lds, rows, D) || !ld_ok(lddx, rows, D) || (dsum && !ld_ok(ldo, rows, D)))
    return FWB_E_SHAPE;
  const int es = esize_of(dtype);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dweight && !elem_aligned(dweight, esize_of(wdtype))) return FWB_E_POINTER;
  if (rows == 0) {
    if (dweight && cudaMemsetAsync(dweight, 0, (size_t)D * esize_of(wdtype), st) != cudaSuccess) return FWB_E_LAUNCH;
    return FWB_OK;
  }
  if (!dy || !sum || !weight || !rstd || !dx || (dweight && !parts)) return FWB_E_POINTER;
  if (!elem_aligned(dy, es) || !elem_aligned(sum, es) || !elem_aligned(dsum, es) || !elem_aligned(dx, es) ||
      !elem_aligned(weight, esize_of(wdtype)))
    return FWB_E_POINTER;
  NormGradArgs a = {};
  a.dy = dy;
  a.s = sum;
  a.dso = dsum;
  a.w = weight;
  a.rstd = rstd;
  a.dx = dx;
  a.part = dweight ? parts : nullptr;
  a.lddy = lddy;
  a.lds = lds;
  a.ldo = ldo;
  a.lddx = lddx;
  a.rows = rows;
  a.D = D;
  a.w_f32 = wdtype == FWB_DTYPE_F32 && dtype != FWB_DTYPE_F32;
  a.vec = same_slots(sum, lds, dy, lddy, es) && same_slots(sum, lds, dx, lddx, es) &&
          (!dsum || same_slots(sum, lds, dsum, ldo, es));
  const int64_t grid = norm_grid(rows, norm_shape(row_slots(sum, lds, D, es, a.vec)).G);
  if (dweight && nparts < grid) return FWB_E_CAPACITY;
  cudaError_t e = dtype == FWB_DTYPE_BF16  ? launch_norm_grad<__nv_bfloat16>(a, st)
                  : dtype == FWB_DTYPE_F16 ? launch_norm_grad<__half>(a, st)
                                           : launch_norm_grad<float>(a, st);
  if (e != cudaSuccess || !dweight) return launch_status(e);
  const int64_t g2 = (D + 31) / 32;
  if (wdtype == FWB_DTYPE_BF16)
    e = launch_dependent(fw_norm_dw_kernel<__nv_bfloat16>, g2, 1024, 0, 1, st, parts, grid, D,
                         static_cast<__nv_bfloat16*>(dweight));
  else if (wdtype == FWB_DTYPE_F16)
    e = launch_dependent(fw_norm_dw_kernel<__half>, g2, 1024, 0, 1, st, parts, grid, D, static_cast<__half*>(dweight));
  else
    e = launch_dependent(fw_norm_dw_kernel<float>, g2, 1024, 0, 1, st, parts, grid, D, static_cast<float*>(dweight));
  return launch_status(e);
}

}  // extern "C"
