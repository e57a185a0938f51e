// Global norm of many gradient tensors, and the gradients scaled to it:
//   n = sqrt(sum over tensors and elements of x^2),  x * min(1, max_norm / n).
//
// Bound by HBM: the norm reads every element once; scaling reads them again
// (from L2, where they fit: the second kernel walks each CTA's part backwards,
// so that what was read last is read first) and writes them.  2.9 GB of bfloat16
// scaled into copies: 1.42 ms, 6.2 TB/s of the 8.8 GB moved; 267 MB of bfloat16
// into float32 187 us; the norm alone of 308 MB 50 us, 6.2 TB/s.  The tensors'
// addresses travel in the kernels' arguments, so nothing is copied to the
// device and a captured graph holds them.
//
// All tensors together are cut into tiles of kTile elements, dealt out to the
// CTAs in contiguous, equal parts, whatever tensors those come from.  A thread
// adds 32 squares in fp32, and those sums in fp64; a sum that overflows, or is
// so small that squares may have been lost, is taken again in fp64.  CTAs
// leave one fp64 partial sum each, added in a fixed order: the same tensors
// give the same norm, bit for bit.
#include <cmath>

#include "fw_host.cuh"
#include "fw_rowslots.cuh"

namespace fwb200 {
namespace {

constexpr int kTile = 8192;  // elements: 4 groups of 8 per thread
constexpr int kThreads = 256;
// CTAs per SM of the norm and of the scaling.  3 GB of bfloat16: norm 423 us with
// 4, 411 with 5; norm and scaled copy 1453 and 1487 (1416 with 4 and stores that
// leave L2 first).
constexpr int kNormCtas = 5, kScaleCtas = 4;
constexpr int kGroups = kTile / 8 / kThreads;
constexpr float kLost = 8.0779357e-28f;  // 2^-90: squares under 2^-149 are gone, 2^-59 of this

// Tensors of one launch.  Tile t of the launch is in the tensor i with
// first[i] <= t < first[i + 1]; groups of 8 elements start where the written
// tensor (the read one, for the norm) is aligned to their size, 16 or 32 bytes.
template <int N>
struct Table {
  int n, tiles;
  const void* in[N];
  void* out[N];
  int64_t numel[N];
  int first[N + 1];
  uint8_t type_in[N], type_out[N];
};

__device__ __forceinline__ int groups_off(const void* p, int type) {  // elements before p's first group boundary
  const uintptr_t a = reinterpret_cast<uintptr_t>(p);
  return type == FWB_DTYPE_F32 ? (int)(a & 31u) >> 2 : (int)(a & 15u) >> 1;
}

template <class T>
constexpr int kParts = sizeof(T) / 2;  // 16-byte slots per group

// A group at an aligned address, by one access: whole sectors of 32 bytes.
__device__ __forceinline__ void load_whole(uint4 (&u)[1], const void* p) { u[0] = ld_global16_once(p); }
__device__ __forceinline__ void load_whole(uint4 (&u)[2], const void* p) {
  asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(u[0].x), "=r"(u[0].y), "=r"(u[0].z), "=r"(u[0].w), "=r"(u[1].x), "=r"(u[1].y), "=r"(u[1].z), "=r"(u[1].w)
               : "l"(p)
               : "memory");
}
// What is stored is not read again here, what was loaded may be.
__device__ __forceinline__ void store_whole(void* p, const uint4 (&u)[1]) { __stcs(static_cast<uint4*>(p), u[0]); }
__device__ __forceinline__ void store_whole(void* p, const uint4 (&u)[2]) {
  asm volatile("st.global.L2::evict_first.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(u[0].x), "r"(u[0].y), "r"(u[0].z),
               "r"(u[0].w), "r"(u[1].x), "r"(u[1].y), "r"(u[1].z), "r"(u[1].w)
               : "memory");
}

// Elements e .. e + 8 of x, which may start anywhere; outside [0, n) as zero.
template <class T>
__device__ __forceinline__ void load_group(uint4 (&u)[kParts<T>], const T* x, int64_t e, int64_t n) {
  constexpr int V = 16 / sizeof(T);
  if (e >= 0 && e + 8 <= n && (reinterpret_cast<uintptr_t>(x + e) & (8 * sizeof(T) - 1)) == 0) {
    load_whole(u, x + e);
  } else {
    const Span<T> span(x, 1, n, n);
#pragma unroll
    for (int i = 0; i < kParts<T>; ++i) u[i] = load_slot_shifted(x + e + i * V, 0, span);
  }
}

template <class T>
__device__ __forceinline__ double tile_squares(const T* x, int64_t e0, int64_t n) {
  uint4 u[kGroups][kParts<T>];
#pragma unroll
  for (int g = 0; g < kGroups; ++g) load_group<T>(u[g], x, e0 + (int64_t)(g * kThreads + threadIdx.x) * 8, n);
  float s[2] = {0.0f, 0.0f};
#pragma unroll
  for (int g = 0; g < kGroups; ++g)
#pragma unroll
    for (int i = 0; i < kParts<T>; ++i) {
      float v[16 / sizeof(T)];
      unpack16<T>(u[g][i], v);
#pragma unroll
      for (int j = 0; j < 16 / (int)sizeof(T); ++j) s[j & 1] = fmaf(v[j], v[j], s[j & 1]);
    }
  const float sum = s[0] + s[1];
  if (sum >= kLost && sum < CUDART_INF_F) return (double)sum;
  double d = 0.0;
  uint32_t any = 0u;
#pragma unroll
  for (int g = 0; g < kGroups; ++g)
#pragma unroll
    for (int i = 0; i < kParts<T>; ++i) any |= u[g][i].x | u[g][i].y | u[g][i].z | u[g][i].w;
  if (any == 0u) return d;
#pragma unroll 1
  for (int g = 0; g < kGroups; ++g)
#pragma unroll 1
    for (int j = 0; j < 8; ++j) {
      const int64_t e = e0 + (int64_t)(g * kThreads + threadIdx.x) * 8 + j;
      const double v = e >= 0 && e < n ? (double)Elem<T>::to_f(x[e]) : 0.0;
      d = fma(v, v, d);
    }
  return d;
}

// Tensor of a tile, looked for from `i` on.
template <int N>
__device__ __forceinline__ int tensor_of(const Table<N>& t, int tile) {
  int lo = 0, hi = t.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= tile)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ double block_sum(double d) {
  __shared__ double red[kThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(kFull, d, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = d;
  __syncthreads();
  d = 0.0;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) d += red[i];
  return d;
}

template <int N>
__global__ void __launch_bounds__(kThreads, kNormCtas) fw_grad_squares_kernel(const __grid_constant__ Table<N> t, double* part) {
  wait_prior_kernel();
  allow_dependent_launch();
  const int lo = (int)((int64_t)t.tiles * blockIdx.x / gridDim.x), hi = (int)((int64_t)t.tiles * (blockIdx.x + 1) / gridDim.x);
  double d = 0.0;
  int i = lo < hi ? tensor_of(t, lo) : 0;
  for (int tile = lo; tile < hi; ++tile) {
    while (tile >= t.first[i + 1]) ++i;
    const int type = t.type_in[i];
    const int64_t n = t.numel[i], e0 = (int64_t)(tile - t.first[i]) * kTile - groups_off(t.in[i], type);
    d += type == FWB_DTYPE_F32    ? tile_squares(static_cast<const float*>(t.in[i]), e0, n)
         : type == FWB_DTYPE_BF16 ? tile_squares(static_cast<const __nv_bfloat16*>(t.in[i]), e0, n)
                                  : tile_squares(static_cast<const __half*>(t.in[i]), e0, n);
  }
  d = block_sum(d);
  if (threadIdx.x == 0) part[blockIdx.x] = d;
}

// The norm from the partial sums, in a fixed order; every thread of a CTA.
__device__ __forceinline__ double norm_of(const double* part, int parts) {
  double d = 0.0;
  for (int i = threadIdx.x; i < parts; i += kThreads) d += __ldcg(part + i);
  return sqrt(block_sum(d));
}

__device__ __forceinline__ void give_norm(double n, float* norm, int32_t* status) {
  const float f = (float)n;
  *norm = f;
  if (!(f < CUDART_INF_F)) raise_status(status, FWB_STATUS_NONFINITE);
}

__global__ void __launch_bounds__(kThreads) fw_grad_norm_kernel(const double* part, int parts, float* norm, int32_t* status) {
  wait_prior_kernel();
  allow_dependent_launch();
  const double n = norm_of(part, parts);
  if (threadIdx.x == 0) give_norm(n, norm, status);
}

template <class TI, class TO>
__device__ __forceinline__ void tile_scale(const TI* x, TO* y, int64_t e0, int64_t n, float f) {
  uint4 u[kGroups][kParts<TI>];
#pragma unroll
  for (int g = 0; g < kGroups; ++g) load_group<TI>(u[g], x, e0 + (int64_t)(g * kThreads + threadIdx.x) * 8, n);
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    const int64_t e = e0 + (int64_t)(g * kThreads + threadIdx.x) * 8;
    if (e >= n) continue;
    float v[8];
#pragma unroll
    for (int i = 0; i < kParts<TI>; ++i) unpack16<TI>(u[g][i], v + i * (16 / (int)sizeof(TI)));
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= f;
    constexpr int V = 16 / sizeof(TO);
    uint4 o[kParts<TO>];
#pragma unroll
    for (int i = 0; i < kParts<TO>; ++i) o[i] = pack_slot<TO>(v + i * V);
    if (e >= 0 && e + 8 <= n) {
      store_whole(y + e, o);
    } else {
#pragma unroll
      for (int i = 0; i < kParts<TO>; ++i) store_slot(y, e + i * V, n, false, o[i]);
    }
  }
}

template <class TI>
__device__ __forceinline__ void tile_scale_to(const TI* x, void* y, int type, int64_t e0, int64_t n, float f) {
  if (type == FWB_DTYPE_F32)
    tile_scale(x, static_cast<float*>(y), e0, n, f);
  else if (type == FWB_DTYPE_BF16)
    tile_scale(x, static_cast<__nv_bfloat16*>(y), e0, n, f);
  else
    tile_scale(x, static_cast<__half*>(y), e0, n, f);
}

// `part` NULL: the norm is *norm_in.  `inplace`: nothing is written where the
// factor is 1.
template <int N>
__global__ void __launch_bounds__(kThreads, kScaleCtas)
    fw_grad_scale_kernel(const __grid_constant__ Table<N> t, const double* part, int parts, const float* norm_in,
                         float max_norm, int inplace, float* norm, int32_t* status) {
  wait_prior_kernel();
  allow_dependent_launch();
  const double n = part ? norm_of(part, parts) : (double)*norm_in;
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) give_norm(n, norm, status);
  const float f = n <= (double)max_norm ? 1.0f : (float)((double)max_norm / n);  // NaN where the norm is
  if (inplace && f == 1.0f) return;
  const int lo = (int)((int64_t)t.tiles * blockIdx.x / gridDim.x), hi = (int)((int64_t)t.tiles * (blockIdx.x + 1) / gridDim.x);
  int i = lo < hi ? tensor_of(t, hi - 1) : 0;
  for (int tile = hi - 1; tile >= lo; --tile) {
    while (tile < t.first[i]) --i;
    const int type = t.type_in[i], to = t.type_out[i];
    const int64_t e = t.numel[i], e0 = (int64_t)(tile - t.first[i]) * kTile - groups_off(t.out[i], to);
    if (type == FWB_DTYPE_F32)
      tile_scale_to(static_cast<const float*>(t.in[i]), t.out[i], to, e0, e, f);
    else if (type == FWB_DTYPE_BF16)
      tile_scale_to(static_cast<const __nv_bfloat16*>(t.in[i]), t.out[i], to, e0, e, f);
    else
      tile_scale_to(static_cast<const __half*>(t.in[i]), t.out[i], to, e0, e, f);
  }
}

// ------------------------------------------------------------ host
constexpr int kFew = 64, kMany = 512;  // tensors per launch: 2 or 16 KB of arguments

struct Tensors {
  int64_t n;
  const void* const* in;
  void* const* out;  // NULL: only read
  const int64_t* numel;
  const int32_t *type_in, *type_out;
};

int type_size(int32_t type) { return type == FWB_DTYPE_F32 ? 4 : 2; }

bool type_known(int32_t type) { return type == FWB_DTYPE_F32 || type == FWB_DTYPE_BF16 || type == FWB_DTYPE_F16; }

constexpr int64_t kMostElements = (int64_t)1 << 43;  // of all tensors: 2^30 tiles

int check_tensors(const Tensors& t) {
  if (t.n < 0 || t.n > (1 << 24)) return FWB_E_SHAPE;
  if (t.n > 0 && (!t.in || !t.numel || !t.type_in || (t.out && !t.type_out))) return FWB_E_POINTER;
  int64_t total = 0;
  for (int64_t i = 0; i < t.n; ++i) {
    if (!type_known(t.type_in[i]) || (t.out && !type_known(t.type_out[i]))) return FWB_E_DTYPE;
    if (t.numel[i] < 0 || t.numel[i] > kMostElements || (total += t.numel[i]) > kMostElements) return FWB_E_SHAPE;
    if (t.numel[i] == 0) continue;
    if (!t.in[i] || reinterpret_cast<uintptr_t>(t.in[i]) % type_size(t.type_in[i]) != 0) return FWB_E_POINTER;
    if (t.out && (!t.out[i] || reinterpret_cast<uintptr_t>(t.out[i]) % type_size(t.type_out[i]) != 0)) return FWB_E_POINTER;
  }
  return FWB_OK;
}

int64_t norm_ctas() { return (int64_t)sm_count() * kNormCtas; }

// Fills a launch's table from tensor `at` on and returns the tensor behind it.
template <int N>
int64_t fill(const Tensors& t, int64_t at, Table<N>* out) {
  out->n = 0;
  int64_t tiles = 0;
  for (; at < t.n && out->n < N; ++at) {
    if (t.numel[at] == 0) continue;
    const bool w = t.out != nullptr;
    const int type = w ? t.type_out[at] : t.type_in[at];
    const int size = type_size(type);
    const int64_t off = (int64_t)(reinterpret_cast<uintptr_t>(w ? t.out[at] : t.in[at]) & (uintptr_t)(8 * size - 1)) / size;
    const int64_t more = (t.numel[at] + off + kTile - 1) / kTile;
    const int i = out->n++;
    out->in[i] = t.in[at];
    out->out[i] = w ? t.out[at] : nullptr;
    out->numel[i] = t.numel[at];
    out->type_in[i] = (uint8_t)t.type_in[at];
    out->type_out[i] = (uint8_t)type;
    out->first[i] = (int)tiles;
    tiles += more;
    out->first[i + 1] = (int)tiles;
  }
  out->tiles = (int)tiles;
  return at;
}

template <int N, class Launch>
int for_tables(const Tensors& t, int64_t cap, Launch&& launch) {
  Table<N> table;
  for (int64_t at = 0; at < t.n;) {
    at = fill(t, at, &table);
    if (table.n == 0) break;
    if (launch(table, table.tiles < cap ? table.tiles : cap) != cudaSuccess) return FWB_E_LAUNCH;
  }
  return FWB_OK;
}

template <int N>
int run_squares(const Tensors& t, double* part, int* parts, cudaStream_t st) {
  *parts = 0;
  return for_tables<N>(t, norm_ctas(), [&](const Table<N>& table, int64_t grid) {
    const cudaError_t e = launch_dependent(fw_grad_squares_kernel<N>, grid, kThreads, 0, 1, st, table, part + *parts);
    *parts += (int)grid;
    return e;
  });
}

template <int N>
int run_scale(const Tensors& t, const double* part, int parts, const float* norm_in, float max_norm, float* norm,
              int32_t* status, cudaStream_t st) {
  bool inplace = true;
  for (int64_t i = 0; i < t.n; ++i)
    if (t.numel[i] > 0 && (t.in[i] != t.out[i] || t.type_in[i] != t.type_out[i])) inplace = false;
  return for_tables<N>(t, (int64_t)sm_count() * kScaleCtas, [&](const Table<N>& table, int64_t grid) {
    const cudaError_t e = launch_dependent(fw_grad_scale_kernel<N>, grid, kThreads, 0, 1, st, table, part, parts, norm_in,
                                           max_norm, (int)inplace, norm, status);
    norm = nullptr;  // given by the first launch
    return e;
  });
}

int64_t squares_bytes(int64_t n) { return 8 * norm_ctas() * ((n + kFew - 1) / kFew); }

bool nothing(const Tensors& t) {
  for (int64_t i = 0; i < t.n; ++i)
    if (t.numel[i] > 0) return false;
  return true;
}

}  // namespace
}  // namespace fwb200

using namespace fwb200;

extern "C" {

int64_t fw_grad_norm_workspace(int64_t n) { return n < 0 || n > (1 << 24) ? 0 : squares_bytes(n); }

int fw_grad_norm(int64_t n, const void* const* grads, const int64_t* numel, const int32_t* dtypes, void* workspace,
                 int64_t workspace_bytes, float* norm, int32_t* status, void* stream) {
  const Tensors t = {n, grads, nullptr, numel, dtypes, nullptr};
  if (int rc = check_tensors(t)) return rc;
  if (!norm) return FWB_E_POINTER;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (nothing(t)) return cudaMemsetAsync(norm, 0, 4, st) == cudaSuccess ? FWB_OK : FWB_E_LAUNCH;
  if (!workspace || !aligned16(workspace)) return FWB_E_POINTER;
  if (workspace_bytes < squares_bytes(n)) return FWB_E_CAPACITY;
  double* part = static_cast<double*>(workspace);
  int parts = 0;
  if (int rc = n <= kFew ? run_squares<kFew>(t, part, &parts, st) : run_squares<kMany>(t, part, &parts, st)) return rc;
  return launch_status(launch_dependent(fw_grad_norm_kernel, 1, kThreads, 0, 1, st, (const double*)part, parts, norm, status));
}

int fw_grad_clip(int64_t n, const void* const* grads, void* const* out, const int64_t* numel, const int32_t* dtypes,
                 const int32_t* out_dtypes, float max_norm, const float* norm_in, void* workspace, int64_t workspace_bytes,
                 float* norm, int32_t* status, void* stream) {
  const Tensors t = {n, grads, out, numel, dtypes, out_dtypes};
  if (int rc = check_tensors(t)) return rc;
  if (!(max_norm >= 0.0f)) return FWB_E_SHAPE;
  if (n > 0 && !out) return FWB_E_POINTER;
  if (!norm_in && !norm) return FWB_E_POINTER;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (nothing(t)) {
    if (norm_in) return FWB_OK;
    return cudaMemsetAsync(norm, 0, 4, st) == cudaSuccess ? FWB_OK : FWB_E_LAUNCH;
  }
  double* part = nullptr;
  int parts = 0;
  if (!norm_in) {
    if (!workspace || !aligned16(workspace)) return FWB_E_POINTER;
    if (workspace_bytes < squares_bytes(n)) return FWB_E_CAPACITY;
    part = static_cast<double*>(workspace);
    const Tensors in = {n, grads, nullptr, numel, dtypes, nullptr};
    if (int rc = n <= kFew ? run_squares<kFew>(in, part, &parts, st) : run_squares<kMany>(in, part, &parts, st)) return rc;
  } else {
    norm = nullptr;
  }
  return n <= kFew ? run_scale<kFew>(t, part, parts, norm_in, max_norm, norm, status, st)
                   : run_scale<kMany>(t, part, parts, norm_in, max_norm, norm, status, st);
}

}  // extern "C"
