// Softmax cross entropy of an output layer, logits z = H W^T never stored:
//   lse_r = log sum_j exp z_rj,  loss_r = lse_r - z_r,y(r)
//   G_rj = g_r (exp(z_rj - lse_r) - 1[j = y(r)]),  dH = G W,  dW = G^T H
// for H [B, D] and W [V, D] in bfloat16 or float16; logits, statistics and
// sums in fp32.
//
// Forward: live rows are packed (rows whose label is ignore_index take no
// part in anything, whatever they hold), one tensor-core product gives each
// 256 x 256 logit tile, whose epilogue keeps only each row's maximum and sum
// of exponentials; a second kernel joins the tiles' pairs, takes the losses
// and reduces them in a fixed order.
// Backward, in pieces of the vocabulary: the logits of a piece again, their
// epilogue writing G (16-bit, the products' operand type: the rounding is
// relative to each entry, so it weighs as the rounding of the result does);
// then dH += G W and dW = G^T H of the piece in one launch, G read in both
// orientations from the one buffer (MN-major operands), each row of dW written
// once.
// Bound by the tensor cores, on large sizes by the power they may draw: 2 B V
// D operations for each of the four products.  bfloat16, 4014 live rows, 128256
// x 4096: 13.3 to 13.9 ms, 1.26 PFLOP/s in all (1.41 within the products);
// float16, 1609 live rows, 32000 x 2048: 0.71 to 0.87 ms with the clock.
//
// The upstream factors g_r stay out of the rounding of G, whose label entry
// -g_r would carry the rounding of g_r into a whole row (and, if all g_r are
// 1 / B, into everything).  One factor for all rows is applied in fp32 after
// the sums.  Factors per row are split, g_r = s_r f_r with s_r a power of two:
// s_r goes into G, f_r in [0.5, 1) multiplies the rows of dH in fp32 and the
// rows of H that dW is made of, which are rounded to their type once more: a
// term of dW then carries two roundings, of G and of f_r H.  Its error is 1.3
// to 1.5 times that of a form in 32 bits rounded at the end (2.3e-3 for 1.65e-3
// in bfloat16, 3.2e-4 for 2.4e-4 in float16, 1609 live rows, 32000 x 2048; level
// for one factor).  A second G with g_r whole and H as it is would have it too:
// the label's entry -g_r (1 - p) makes up most of a row of dW and would be
// rounded in the place of f_r H.
//
// float16 G: exp(z - lse) may be under float16's smallest value, so G is
// scaled by 2^15 (over the largest finite s_r), taken out after the sums.
#include "fw_reduce.cuh"
#include "fw_rowslots.cuh"
#include "fw_tc_gemm.cuh"

namespace fwb200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kF16Unit = 32768.0f;
constexpr int kPackThreads = 256;

// Device words at the start of the state.
struct XentHead {
  int32_t rows;    // live rows
  uint32_t done;   // blocks of the joining kernel that have finished
  int32_t status;  // status bits raised inside
};

struct PackArgs {
  const void* hidden;
  const int64_t* y;
  int64_t B, Bp, D, Dp, ldh, V, ignore;
  void* hp;
  int32_t* row_of;   // [Bp] packed -> given row (behind the live ones the ignored ones, then -1)
  int32_t* label;    // [Bp] -1: outside [0, V)
  float* loss_rows;  // zero for ignored rows, per given row; may be NULL
  XentHead* head;
  int32_t* status;
  int per_cta;
};

// Every CTA counts the live rows before its own by reading all labels, so
// packing is one launch.  8 rows per CTA (a warp each) as long as that makes
// no more than four CTAs per SM, so that many rows do not read the labels too
// often (4096 rows, 8000 x 1024: 242 us in all, with 64 rows per CTA 257; 2^20
// rows read their labels 592 times, not 131072).
template <class T>
__global__ void __launch_bounds__(kPackThreads) fw_xent_pack_kernel(PackArgs a) {
  __shared__ int red[2][kPackThreads / 32];
  constexpr int V = 16 / sizeof(T);
  wait_prior_kernel();
  allow_dependent_launch();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t r0 = (int64_t)blockIdx.x * a.per_cta;
  int before = 0, total = 0;
  for (int64_t i = threadIdx.x; i < a.B; i += kPackThreads) {
    const int live = a.y[i] != a.ignore;
    total += live;
    before += i < r0 ? live : 0;
  }
  before = __reduce_add_sync(kFull, before);
  total = __reduce_add_sync(kFull, total);
  if (lane == 0) {
    red[0][w] = before;
    red[1][w] = total;
  }
  __syncthreads();
  before = total = 0;
#pragma unroll
  for (int i = 0; i < kPackThreads / 32; ++i) {
    before += red[0][i];
    total += red[1][i];
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.head->rows = total;
    a.head->done = 0u;
    a.head->status = 0;
  }
  const int64_t rows_up = ((int64_t)total + 255) / 256 * 256;
  const Span<T> span(a.hidden, a.B, a.ldh, a.D);
  for (int i0 = 0; i0 < a.per_cta; i0 += 32) {
    const int64_t rl = r0 + i0 + lane;
    const int64_t yl = rl < a.B ? a.y[rl] : a.ignore;
    const uint32_t live = __ballot_sync(kFull, rl < a.B && yl != a.ignore);
    for (int i = w; i < 32 && i0 + i < a.per_cta; i += kPackThreads / 32) {
      const int64_t r = r0 + i0 + i;
      if (r >= a.Bp) break;
      const bool alive = (live >> i) & 1u;
      const int64_t ahead = before + __popc(live & ((1u << i) - 1u));
      const int64_t dst = alive ? ahead : total + (r - ahead);
      const int64_t y = __shfl_sync(kFull, yl, i);
      if (lane == 0) {
        const bool ok = y >= 0 && y < a.V;
        a.row_of[dst] = r < a.B ? (int32_t)r : -1;
        a.label[dst] = alive && ok ? (int32_t)y : -1;
        if (alive && !ok) raise_status(a.status, FWB_STATUS_LABEL_RANGE);
        if (!alive && r < a.B && a.loss_rows) a.loss_rows[r] = 0.0f;
      }
      if (dst >= rows_up) continue;
      T* out = static_cast<T*>(a.hp) + dst * a.Dp;
      const T* in = static_cast<const T*>(a.hidden) + (alive ? r : 0) * a.ldh;
      for (int64_t e = (int64_t)lane * V; e < a.Dp; e += 32 * V)
        *reinterpret_cast<uint4*>(out + e) = alive ? load_slot_shifted(in, (int)e, span) : make_uint4(0u, 0u, 0u, 0u);
    }
    before += __popc(live);
  }
}

// Rows of an unaligned matrix copied to 16-byte boundaries.  (What lands in
// the columns from D on is never read: the tensor maps end at D.)
template <class T>
__global__ void __launch_bounds__(256) fw_xent_align_kernel(const T* src, int64_t ld, T* dst, int64_t ldd, int64_t rows,
                                                            int64_t D) {
  constexpr int V = 16 / sizeof(T);
  const int lane = threadIdx.x & 31;
  const int64_t slabs = (ldd + 32 * V * 4 - 1) / (32 * V * 4);
  const Span<T> span(src, rows, ld, D);
  const int64_t nw = (int64_t)gridDim.x * 8;
  for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < rows * slabs; i += nw) {
    const int64_t r = i / slabs, e0 = ((i - r * slabs) * 128 + lane) * V;
    uint4 u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t e = e0 + k * 32 * V;
      if (e < ldd) u[k] = load_slot_shifted(src + r * ld, (int)e, span);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t e = e0 + k * 32 * V;
      if (e < ldd) *reinterpret_cast<uint4*>(dst + r * ldd + e) = u[k];
    }
  }
}

// 2^x by the hardware's instruction (relative error 2^-22, results under
// 2^-126 flushed to 0); volatile, so that the compiler does not hold many
// arguments in registers to interleave them.
__device__ __forceinline__ float exp2_hw(float x) {
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr int kTileM = 256, kTileN = 256;  // of a pair of CTAs

__device__ __forceinline__ int row_tiles(const XentHead* h) { return (h->rows + kTileM - 1) / kTileM; }

// Tiles dealt out in turn.
struct TurnPlan {
  TileOrder order;
  int first, step;
  __device__ __forceinline__ void set(int mt, int nt, int group, int groups) {
    order.set(mt, nt, 16);
    first = group;
    step = groups;
  }
  __device__ __forceinline__ bool get(int i, int* m, int* n) const {
    const int w = first + i * step;
    if (w >= order.count()) return false;
    order.get(w, m, n);
    return true;
  }
};

// ------------------------------------------------------------ forward
struct LseArgs {
  const XentHead* head;
  const int32_t* label;
  float2* part;  // [kLseCols columns of V, Bp]: maximum, sum of exp(z - maximum)
  float* zy;     // [Bp]
  int64_t Bp;
  int V, D;
  int32_t* status;
};

// The accumulator is taken over every kLseStages stages of K and added up in
// registers: the tensor cores' fp32 additions round towards zero, so a logit
// shrinks by a part that grows with the length of the sum.  Every 8, 16, 32 or
// all 64 stages (K = 4096): error of the loss 1.2e-7, 2.6e-7, 5.6e-7, 1.2e-6,
// forward and backward 13.5, 13.4, 13.4, 13.4 ms.
constexpr int kLseStages = 8;
constexpr int kLseCols = 128;  // columns of a tile per epilogue thread: they stay in its registers

template <TcKind K>
struct LseTile {
  using Args = LseArgs;
  struct State {
    float z[kLseCols] = {};
    int y;
  };
  static constexpr TcKind KIND = K;
  static constexpr bool A_MN = false, B_MN = false;
  static constexpr bool TWO = false, A_MN2 = false;
  static constexpr int CG = 2, BN = kTileN, STAGES = 7, KC = kLseStages, EW = 4 * BN / kLseCols, A_BOX = 128, AHEAD = 0;
  static constexpr uint32_t EPI_BYTES = 0;
  using Plan = TurnPlan;
  __device__ static void plan(const Args& a, int group, int groups, Plan* p) {
    p->set(row_tiles(a.head), (a.V + BN - 1) / BN, group, groups);
  }
  __device__ static bool get(const Args& a, const Plan& p, int i, TcTile* t) {
    int m, n;
    if (!p.get(i, &m, &n)) return false;
    *t = {m * kTileM, n * BN, 0, 0, (a.D + 63) / 64, 128, 0};
    return true;
  }
  __device__ static void begin(const Args& a, const Plan&, const TcTile& t, const TcPart& p, State& st) {
    st.y = a.label[t.m0 + p.row + p.lane];
  }
  template <bool LOST, class Done>
  __device__ static void epilogue(const Args& a, const Plan&, const TcTile& t, const TcPart& p, State& st, int k,
                                  int parts, Done done) {
    if constexpr (LOST) return;  // the status word in the state makes every loss NaN
#pragma unroll
    for (int c = 0; c < kLseCols; c += 16) {
      float v[16];
      tmem_ld16(p.taddr + p.share * kLseCols + c, v);
#pragma unroll
      for (int i = 0; i < 16; ++i) st.z[c + i] += v[i];
    }
    done();
    if (k < parts - 1) return;
    const int row = t.m0 + p.row + p.lane;  // < Bp
    const int n0 = t.n0 + p.share * kLseCols;
    const int y = st.y - n0;
    const int valid = a.V - n0;
    float m = -CUDART_INF_F, s = 0.0f;
#pragma unroll
    for (int i = 0; i < kLseCols; ++i) {
      if (i >= valid) st.z[i] = -CUDART_INF_F;
      if (i == y) a.zy[row] = st.z[i];
      m = max_nan(m, st.z[i]);
    }
    if (m != -CUDART_INF_F) {  // a NaN maximum, or +inf, makes the sum NaN
      float s4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < kLseCols; ++i) s4[i & 3] += exp2_hw((st.z[i] - m) * kLog2e);
      s = (s4[0] + s4[1]) + (s4[2] + s4[3]);
    }
    a.part[(int64_t)(n0 / kLseCols) * a.Bp + row] = make_float2(m, s);
  }
};

struct JoinArgs {
  XentHead* head;
  const float2* part;
  const float* zy;
  const int32_t* label;
  const int32_t* row_of;
  float* lse;        // [Bp], packed
  float* loss_pack;  // [Bp], packed
  float* loss;       // [B] (reduction none) or one value
  int64_t Bp;
  int ntiles;
  int reduction;
  int32_t* status;
};

constexpr int kJoinWarps = 32;

// 32 rows per CTA, the tiles' pairs split over its warps; the last CTA to
// finish adds the losses in a fixed order.
__global__ void __launch_bounds__(kJoinWarps * 32) fw_xent_join_kernel(JoinArgs a) {
  __shared__ float sm[kJoinWarps][32], ss[kJoinWarps][32];
  __shared__ double sd[kJoinWarps];
  __shared__ bool last;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  wait_prior_kernel();
  const int rows = a.head->rows;
  const int row = blockIdx.x * 32 + lane;
  float m = -CUDART_INF_F, s = 0.0f;
  if (row < rows) {
#pragma unroll 4
    for (int t = w; t < a.ntiles; t += kJoinWarps) {
      const float2 p = a.part[(int64_t)t * a.Bp + row];
      const float to = max_nan(m, p.x);
      if (to == -CUDART_INF_F) continue;
      s = (m == -CUDART_INF_F ? 0.0f : s * exp2f((m - to) * kLog2e)) +
          (p.x == -CUDART_INF_F ? 0.0f : p.y * exp2f((p.x - to) * kLog2e));
      m = to;
    }
  }
  sm[w][lane] = m;
  ss[w][lane] = s;
  __syncthreads();
  if (w == 0 && row < rows) {
    float M = sm[0][lane];
#pragma unroll
    for (int i = 1; i < kJoinWarps; ++i) M = max_nan(M, sm[i][lane]);
    float S = 0.0f;
#pragma unroll
    for (int i = 0; i < kJoinWarps; ++i)
      if (sm[i][lane] != -CUDART_INF_F) S += ss[i][lane] * exp2f((sm[i][lane] - M) * kLog2e);
    const bool ok = a.label[row] >= 0 && a.head->status == 0;
    if (lane == 0 && a.head->status != 0) raise_status(a.status, a.head->status);
    const float lse = ok ? M + logf(S) : CUDART_NAN_F;  // a NaN row stays NaN in the gradient too
    const float loss = ok ? lse - a.zy[row] : CUDART_NAN_F;
    a.lse[row] = lse;
    a.loss_pack[row] = loss;
    if (!(fabsf(lse) < CUDART_INF_F) && a.label[row] >= 0) raise_status(a.status, FWB_STATUS_NONFINITE);
    if (a.reduction == FWB_REDUCE_NONE) a.loss[a.row_of[row]] = loss;
  }
  if (a.reduction == FWB_REDUCE_NONE) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(&a.head->done, 1u) == gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  double d = 0.0;
  for (int i = threadIdx.x; i < rows; i += kJoinWarps * 32) d += (double)__ldcg(a.loss_pack + i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(kFull, d, o);
  if (lane == 0) sd[w] = d;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kJoinWarps; ++i) d += sd[i];
    a.loss[0] = (float)(a.reduction == FWB_REDUCE_MEAN ? d / (double)rows : d);
  }
}

// ------------------------------------------------------------ backward
// The power of two above |g| (|g| itself where there is none: 0, not finite).
__device__ __forceinline__ float pow2_above(float g) {
  const float m = fabsf(g);
  if (!(m > 0.0f && m < CUDART_INF_F)) return m;
  int e;
  frexpf(m, &e);  // m = f 2^e, f in [0.5, 1)
  return ldexpf(1.0f, min(e, 127));
}

// The upstream gradient: the factors of G's rows (powers of two) and what is
// left of it.
struct Upstream {
  const float* go;   // one per given row, or one
  const float* top;  // largest finite s_r of a live row (float16, factors per row)
  int per_row, mean, f16;

  // s_r, scaled to the range of the type; a factor that is not finite stands for itself
  __device__ float in_g(int r) const {
    if (!per_row) return f16 ? kF16Unit : 1.0f;
    const float g = go[r], s = pow2_above(g);
    if (!(s < CUDART_INF_F)) return g;
    return f16 && *top > 0.0f ? s / *top * kF16Unit : s;
  }
  // f_r; 1 where the factor is in G (0, not finite) or common
  __device__ float rest(int r) const {
    if (!per_row) return 1.0f;
    const float g = go[r], s = pow2_above(g);
    return s > 0.0f && s < CUDART_INF_F ? g / s : 1.0f;
  }
  // common factor taken out after the sums
  __device__ float back(const XentHead* h) const {
    if (per_row) return f16 && *top > 0.0f ? *top / kF16Unit : 1.0f;
    const float g = mean ? go[0] / (float)h->rows : go[0];
    return f16 ? g / kF16Unit : g;
  }
};

__global__ void __launch_bounds__(1024) fw_xent_top_kernel(const XentHead* head, const int32_t* row_of, const float* go,
                                                             float* out) {
  __shared__ float red[32];
  const int rows = head->rows;
  float top = 0.0f;
  for (int i = threadIdx.x; i < rows; i += 1024) {
    const float s = pow2_above(go[row_of[i]]);
    if (s < CUDART_INF_F) top = fmaxf(top, s);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 32; ++i) top = fmaxf(top, red[i]);
    *out = top;
  }
}

// The packed rows of H times f_r: dW's operand where the factors differ.
template <class T>
__global__ void __launch_bounds__(256) fw_xent_scale_kernel(const XentHead* head, const int32_t* row_of, Upstream up,
                                                            const T* hp, T* out, int64_t Dp) {
  constexpr int V = 16 / sizeof(T);
  const int rows = head->rows, rows_up = (rows + kTileM - 1) / kTileM * kTileM;
  const int64_t slots = Dp / V;
  for (int r = blockIdx.x; r < rows_up; r += gridDim.x) {
    const float f = r < rows ? up.rest(row_of[r]) : 0.0f;
    for (int64_t i = threadIdx.x; i < slots; i += 256) {
      float v[V];
      unpack16<T>(*reinterpret_cast<const uint4*>(hp + r * Dp + i * V), v);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = r < rows ? v[j] * f : 0.0f;
      *reinterpret_cast<uint4*>(out + r * Dp + i * V) = pack_slot<T>(v);
    }
  }
}

struct GradArgs {
  const XentHead* head;
  const int32_t* label;
  const int32_t* row_of;
  const float* lse;
  Upstream up;
  void* g;  // [Bp, ldg]
  int64_t ldg;
  int V, D;
  int v0, vn;  // first column of the piece, its columns rounded up to 256
  int32_t* status;
};

template <class T, TcKind K>
struct GradTile {
  using Args = GradArgs;
  struct State {
    float lse, coef;
    int y;
  };
  static constexpr TcKind KIND = K;
  static constexpr bool A_MN = false, B_MN = false;
  static constexpr bool TWO = false, A_MN2 = false;
  static constexpr int CG = 2, BN = kTileN, STAGES = 7, KC = 0, EW = 8, A_BOX = 128, AHEAD = 0;
  static constexpr uint32_t EPI_BYTES = 0;
  using Plan = TurnPlan;
  __device__ static void plan(const Args& a, int group, int groups, Plan* p) {
    p->set(row_tiles(a.head), a.vn / BN, group, groups);
  }
  __device__ static bool get(const Args& a, const Plan& p, int i, TcTile* t) {
    int m, n;
    if (!p.get(i, &m, &n)) return false;
    *t = {m * kTileM, a.v0 + n * BN, 0, 0, (a.D + 63) / 64, 128, 0};
    return true;
  }
  __device__ static void begin(const Args& a, const Plan&, const TcTile& t, const TcPart& p, State& st) {
    const int row = t.m0 + p.row + p.lane;
    const bool live = row < a.head->rows;
    st.y = live ? a.label[row] : -2;  // -2: not a live row
    st.lse = live ? a.lse[row] : 0.0f;
    st.coef = live ? a.up.in_g(a.row_of[row]) : 0.0f;
  }
  template <bool LOST, class Done>
  __device__ static void epilogue(const Args& a, const Plan&, const TcTile& t, const TcPart& p, State& st, int, int,
                                  Done done) {
    const int row = t.m0 + p.row + p.lane, y = st.y;
    const bool live = y != -2;
    const float lse = st.lse, coef = st.coef;
    T* g = static_cast<T*>(a.g) + (int64_t)row * a.ldg + (t.n0 - a.v0);
    for (int c = p.share * (BN / 2); c < (p.share + 1) * (BN / 2); c += 32) {
      float v[32];
      if constexpr (!LOST) tmem_ld32(p.taddr + c, v);
      if (c + 32 == (p.share + 1) * (BN / 2)) done();
      const int valid = live ? min(32, a.V - (t.n0 + c)) : 0;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        float q = LOST ? CUDART_NAN_F : exp2_hw((v[i] - lse) * kLog2e);
        if (t.n0 + c + i == y) q -= 1.0f;
        v[i] = i < valid ? q * coef : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(g + c + 8 * i) = pack_slot<T>(v + 8 * i);
    }
  }
};

// dH += G W and dW = G^T H of a piece, in one launch: the few long tiles of dH
// (all of the piece's columns are their K) would leave most of the last round
// of SMs idle, so the tiles of dW fill it up.  Where one of them is longer than
// 1.25 of a CTA pair's share of all stages, K is cut into splits with an fp32
// sum each, which a last small kernel adds in order.  Forward and backward of
// 32000 x 2048 with 1024, 768, 512 rows (1.16, 1.32, 1.54 shares): 432, 379, 324
// us in one piece, 449, 369, 280 split; 50257 x 1024 with 64 rows: 360 and 182.

// A short tile in stages of K: its stages, or its epilogue where that takes longer.
__device__ __forceinline__ int short_cost(int stages) { return max(stages, 16); }

struct ProductArgs {
  const XentHead* head;
  const int32_t* row_of;
  Upstream up;
  float* sum;     // dH so far, [max_splits, Bp, lds]; not there for one piece and one split
  void* dhidden;  // [B, D] or NULL
  void* dweight;  // [V, D] or NULL
  int Bp, V, D, lds;
  int v0, vn;  // first column of the piece, its columns rounded up to 256
  int first, last;
  int piece;       // columns of a whole piece, a multiple of 256
  int max_splits;  // sums there is room for
  int pairs;       // CTA pairs of the launch
  int32_t* status;

  __device__ int v_tiles() const { return dweight ? (min(vn, V - v0) + kTileM - 1) / kTileM : 0; }
  // The same for every piece (whole ones are taken to reckon with).
  __device__ int splits() const {
    if (max_splits == 1 || !dhidden) return 1;
    // in fp32: the share of a pair need not be exact, only the same everywhere
    const float nt = (float)((D + kTileN - 1) / kTileN), k = (float)(piece / 64), mt = (float)row_tiles(head);
    const float rest = dweight ? (float)(piece / kTileM) * (float)short_cost((head->rows + 63) / 64) : 0.0f;
    const float share = fmaxf(nt * (mt * k + rest) / (float)pairs, 16.0f);
    return max(1, min(max_splits, (int)ceilf(k / share - 0.25f)));
  }
};

template <class T, TcKind K>
struct ProductTile {
  using Args = ProductArgs;
  struct State {
    int mine;  // dH: the given row of this lane's row
    float f;   // its factor
    bool zero;
  };
  static constexpr TcKind KIND = K;
  static constexpr bool A_MN = false, A_MN2 = true, B_MN = true, TWO = true;
  static constexpr int CG = 2, BN = kTileN, STAGES = 5, KC = 0, EW = 8, A_BOX = 128, AHEAD = 0;
  static constexpr uint32_t EPI_BYTES = EW * kStageBytes<BN / 2>;

  // Tiles: the long ones of dH with vn / 64 / splits stages each, then the
  // short ones of dW with rows / 64, then (last piece, one split) those of dH
  // that hold only ignored rows.  A CTA group takes its long tiles in turn;
  // with `more` groups having one more than the others, the short ones go to
  // the others first, for `lead` rounds, until all are level, then to all in
  // turn.
  struct Plan {
    TileOrder longs, shorts;
    FastDiv by_tile, by_nt, by_split;
    int group, groups, splits, k_all, k_short, n_one, n_rest, mine, more, lead;
    float back;
  };
  __device__ static void plan(const Args& a, int group, int groups, Plan* p) {
    const int nt = (a.D + BN - 1) / BN, mt = a.dhidden ? row_tiles(a.head) : 0;
    p->splits = a.splits();
    p->k_all = a.vn / 64;
    p->k_short = (a.head->rows + 63) / 64;
    p->longs.set(mt, nt, 8);
    p->shorts.set(a.v_tiles(), nt, 5);
    p->n_one = mt * nt;
    p->by_tile.set(p->n_one);
    p->by_nt.set(nt);
    p->by_split.set(p->splits);
    p->n_rest = p->shorts.count() + (a.dhidden && a.last && p->splits == 1 ? (a.Bp / kTileM - mt) * nt : 0);
    p->group = group;
    p->groups = groups;
    const int n_long = p->n_one * p->splits;
    p->more = n_long % groups;
    p->mine = n_long / groups + (group < p->more ? 1 : 0);
    p->lead = 0;
    if (p->more > 0) {
      const int k_long = (p->k_all + p->splits - 1) / p->splits, cost = short_cost(p->k_short);
      p->lead = min((k_long + cost / 2) / cost, (p->n_rest + groups - p->more - 1) / (groups - p->more));
    }
    p->back = a.up.back(a.head);
  }
  __device__ static bool get(const Args& a, const Plan& p, int i, TcTile* t) {
    int m, n;
    if (i < p.mine) {
      const int w = i * p.groups + p.group, part = p.by_tile.div(w);
      const int k0 = p.by_split.div(p.k_all * part), k1 = p.by_split.div(p.k_all * (part + 1));
      p.longs.get(w - part * p.n_one, &m, &n);
      *t = {m * kTileM, n * BN, k0 * 64, a.v0 + k0 * 64, k1 - k0, part, 0};
      return true;
    }
    i -= p.mine;
    const int others = p.groups - p.more;
    int w;
    if (p.group >= p.more && i < p.lead) {
      w = i * others + (p.group - p.more);
    } else {
      if (p.group >= p.more) i -= p.lead;
      w = p.lead * others + i * p.groups + p.group;
    }
    if (w >= p.n_rest) return false;
    if (w < p.shorts.count()) {
      p.shorts.get(w, &m, &n);
      *t = {m * kTileM, n * BN, 0, 0, p.k_short, 0, 1};
    } else {
      const int d = w - p.shorts.count(), q = p.by_nt.div(d);
      *t = {(p.longs.mt + q) * kTileM, (d - q * p.longs.nt) * BN, 0, 0, 0, 0, 0};
    }
    return true;
  }

  __device__ static void begin(const Args& a, const Plan& plan, const TcTile& t, const TcPart& p, State& st) {
    // without stages of K the accumulator is never written; dH's rows behind the live ones are ignored ones
    const int row = t.m0 + p.row + p.lane;
    const bool dh = t.kind == 0;
    st.mine = dh ? a.row_of[row] : -1;
    st.zero = t.nk == 0 || (dh && row >= a.head->rows);
    st.f = st.zero ? 0.0f : dh ? plan.back * a.up.rest(st.mine) : plan.back;
  }
  template <bool LOST, class Done>
  __device__ static void epilogue(const Args& a, const Plan& plan, const TcTile& t, const TcPart& p, State& st, int,
                                  int, Done done) {
    uint32_t* sm = reinterpret_cast<uint32_t*>(p.smem);
    const int r0 = t.m0 + p.row, s0 = p.share * (BN / 2);
    const int cols = a.D - (t.n0 + s0);
    const bool dh = t.kind == 0, any = t.nk > 0;
    const bool one = plan.splits == 1;
    const bool summed = dh && any && !(one && a.first && a.last);  // t.rows: the split
    const bool store = dh ? one && a.last : true;
    float* sum = summed ? a.sum + ((int64_t)t.rows * a.Bp + r0 + p.lane) * a.lds + t.n0 + s0 : nullptr;
    for (int c = 0; c < BN / 2; c += 32) {
      float v[32];
      if constexpr (LOST) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = CUDART_NAN_F;
      } else {
        tmem_ld32(p.taddr + s0 + c, v);
      }
      if (c + 32 == BN / 2) done();
      if (c >= cols) continue;
      if (summed) {  // this thread's own row of the sum so far; lds is D rounded up to 32
        if (!a.first) {
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 x = *reinterpret_cast<const float4*>(sum + c + i);
            v[i] += x.x, v[i + 1] += x.y, v[i + 2] += x.z, v[i + 3] += x.w;
          }
        }
        if (!store) {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<float4*>(sum + c + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        }
      }
      if (!store) continue;
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = st.zero ? 0.0f : v[i] * st.f;
      stage_block<T, BN / 2>(sm, v, p.lane, c);
    }
    if (!store || cols <= 0) return;
    const int rows = a.V - (a.v0 + r0);  // dW
    T* out = (dh ? static_cast<T*>(a.dhidden) : static_cast<T*>(a.dweight) + (int64_t)(a.v0 + r0) * a.D) + t.n0 + s0;
    store_staged<T, BN / 2>(sm, p.lane, min(cols, BN / 2), [&](int i) -> T* {
      const int r = dh ? __shfl_sync(kFull, st.mine, i) : i < rows ? i : -1;
      return r >= 0 ? out + (int64_t)r * a.D : nullptr;
    });
  }
};

// dH from the sums of its splits; one warp per row and 128 columns.
template <class T>
__global__ void __launch_bounds__(256) fw_xent_dhidden_kernel(ProductArgs a) {
  wait_prior_kernel();
  allow_dependent_launch();
  const int lane = threadIdx.x & 31;
  const int slabs = (a.D + 127) / 128;
  const int64_t work = (int64_t)a.Bp * slabs, nw = (int64_t)gridDim.x * 8;
  const int rows = a.head->rows, splits = a.splits();
  if (splits == 1) return;  // written by the product itself
  const float back = a.up.back(a.head);
  for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < work; i += nw) {
    const int r = (int)(i / slabs), c = (int)(i % slabs) * 128 + lane * 4;
    const int to = a.row_of[r];
    if (to < 0 || c >= a.D) continue;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (r < rows) {
#pragma unroll 4
      for (int q = 0; q < splits; ++q) {
        const float4 x = *reinterpret_cast<const float4*>(a.sum + ((int64_t)q * a.Bp + r) * a.lds + c);
        v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
      }
      const float f = back * a.up.rest(to);
      v.x *= f, v.y *= f, v.z *= f, v.w *= f;
    }
    T* out = static_cast<T*>(a.dhidden) + (int64_t)to * a.D + c;
    const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j < a.D) st_elem(out + j, x[j]);
  }
}

// ------------------------------------------------------------ host
// Bytes of G that one piece of the vocabulary may take: it should still be in
// L2 when the products read it, and short pieces end in part-filled rounds.
// 48, 128, 256, 512 MB: 14.6, 14.0, 13.7, 13.8 ms (4014 rows, 128256 x 4096).
constexpr int64_t kPieceBytes = (int64_t)256 << 20;
// Bytes of dH's sums where they are split.
constexpr int64_t kSumBytes = (int64_t)128 << 20;

int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

struct XentPlan {
  int64_t Bp, Dp;
  bool copy_w;
  // state: what backward needs
  int64_t row_of, label, lse, hp, wp, state_bytes;
  // forward workspace
  int64_t part, zy, loss_pack, fwd_bytes;
  // backward workspace
  int64_t piece, pieces, splits, top, g, sum, hs, bwd_bytes;
};

XentPlan xent_plan(int64_t B, int64_t D, int64_t V, bool copy_w) {
  XentPlan p = {};
  p.Bp = up(B, 256);
  p.Dp = up(D, 8);
  p.copy_w = copy_w;
  int64_t at = 256;
  p.row_of = at, at += up(4 * p.Bp, 256);
  p.label = at, at += up(4 * p.Bp, 256);
  p.lse = at, at += up(4 * p.Bp, 256);
  p.hp = at, at += up(2 * p.Bp * p.Dp, 256);
  p.wp = at, at += copy_w ? up(2 * V * p.Dp, 256) : 0;
  p.state_bytes = at;
  at = 0;
  p.part = at, at += up(8 * p.Bp * up(V, kTileN) / kLseCols, 256);
  p.zy = at, at += up(4 * p.Bp, 256);
  p.loss_pack = at, at += up(4 * p.Bp, 256);
  p.fwd_bytes = at;
  const int64_t Vp = up(V, 256);
  p.pieces = (2 * p.Bp * Vp + kPieceBytes - 1) / kPieceBytes;
  if (p.pieces < 1) p.pieces = 1;
  p.piece = up((Vp + p.pieces - 1) / p.pieces, 256);
  p.pieces = (Vp + p.piece - 1) / p.piece;
  at = 0;
  p.top = at, at += 256;
  p.g = at, at += up(2 * p.Bp * p.piece, 256);
  // as many as one row tile could use, 16 stages of K each, within kSumBytes
  p.splits = sm_count() / 2 / ((D + kTileN - 1) / kTileN);
  const int64_t room = B > 0 ? kSumBytes / (4 * p.Bp * up(D, 32)) : 1;
  if (p.splits > room) p.splits = room;
  if (p.splits > p.piece / 64 / 16) p.splits = p.piece / 64 / 16;
  if (p.splits < 1) p.splits = 1;
  p.sum = at, at += p.pieces > 1 || p.splits > 1 ? up(4 * p.splits * p.Bp * up(D, 32), 256) : 0;
  p.hs = at, at += up(2 * p.Bp * p.Dp, 256);  // factors per row
  p.bwd_bytes = at;
  return p;
}

int xent_check(int dtype, int64_t B, int64_t D, int64_t V) {
  if (dtype != FWB_DTYPE_BF16 && dtype != FWB_DTYPE_F16) return FWB_E_DTYPE;
  if (B < 0 || D < 1 || V < 1 || B > (1 << 26) || D > (1 << 20) || V > (1 << 28)) return FWB_E_SHAPE;
  if ((up(B, 256) / 256) * (up(V, 256) / 256) > (1 << 30)) return FWB_E_SHAPE;
  return FWB_OK;
}

// Rows that a TMA tile load can read in place.
bool tma_rows(const void* p, int64_t ld) { return aligned16(p) && ld % 8 == 0; }

template <class T, TcKind K>
int run_forward(const void* hidden, int64_t ldh, const void* weight, int64_t ldw, const int64_t* y, int64_t B,
                int64_t D, int64_t V, int64_t ignore, int reduction, float* loss, char* state, char* ws,
                int32_t* status, cudaStream_t st) {
  const XentPlan p = xent_plan(B, D, V, !tma_rows(weight, ldw));
  XentHead* head = reinterpret_cast<XentHead*>(state);
  int32_t* row_of = reinterpret_cast<int32_t*>(state + p.row_of);
  int32_t* label = reinterpret_cast<int32_t*>(state + p.label);
  const int64_t per_cta = (p.Bp + 4 * sm_count() - 1) / (4 * sm_count());
  PackArgs pk = {hidden, y, B, p.Bp, D, p.Dp, ldh, V, ignore, state + p.hp, row_of, label,
                 reduction == FWB_REDUCE_NONE ? loss : nullptr, head, status, (int)(per_cta < 8 ? 8 : per_cta)};
  if (launch_dependent(fw_xent_pack_kernel<T>, (p.Bp + pk.per_cta - 1) / pk.per_cta, kPackThreads, 0, 1, st, pk) !=
      cudaSuccess)
    return FWB_E_LAUNCH;
  const void* w = weight;
  if (p.copy_w) {
    const int64_t need = (V * ((p.Dp + 1023) / 1024) + 7) / 8, cap = (int64_t)sm_count() * 16;
    fw_xent_align_kernel<T><<<(unsigned)(need < cap ? need : cap), 256, 0, st>>>(
        static_cast<const T*>(weight), ldw, reinterpret_cast<T*>(state + p.wp), p.Dp, V, D);
    w = state + p.wp;
    ldw = p.Dp;
  }
  if (cudaGetLastError() != cudaSuccess) return FWB_E_LAUNCH;
  CUtensorMap mh, mw;
  if (!tc_map(&mh, K, state + p.hp, p.Bp, D, p.Dp, 128) || !tc_map(&mw, K, w, V, D, ldw, 128)) return FWB_E_LAUNCH;
  LseArgs la = {head, label, reinterpret_cast<float2*>(ws + p.part), reinterpret_cast<float*>(ws + p.zy), p.Bp, (int)V,
                (int)D, &head->status};
  const int64_t nt = (V + 255) / 256;
  if (launch_gemm<LseTile<K>>(mh, mw, la, (p.Bp / 256) * nt, st) != cudaSuccess) return FWB_E_LAUNCH;
  JoinArgs ja = {head, la.part, la.zy, label, row_of, reinterpret_cast<float*>(state + p.lse),
                 reinterpret_cast<float*>(ws + p.loss_pack), loss, p.Bp, (int)((V + kLseCols - 1) / kLseCols), reduction, status};
  return launch_status(launch_dependent(fw_xent_join_kernel, p.Bp / 32, kJoinWarps * 32, 0, 1, st, ja));
}

template <class T, TcKind K>
int run_backward(const void* weight, int64_t ldw, int64_t B, int64_t D, int64_t V, int mean, const float* go,
                 int per_row, const char* state, char* ws, void* dhidden, void* dweight, int32_t* status, cudaStream_t st) {
  const XentPlan p = xent_plan(B, D, V, !tma_rows(weight, ldw));
  const XentHead* head = reinterpret_cast<const XentHead*>(state);
  const int32_t* row_of = reinterpret_cast<const int32_t*>(state + p.row_of);
  const int32_t* label = reinterpret_cast<const int32_t*>(state + p.label);
  const void* w = p.copy_w ? state + p.wp : weight;
  if (p.copy_w) ldw = p.Dp;
  float* top = reinterpret_cast<float*>(ws + p.top);
  const Upstream u = {go, top, per_row, mean, K == kTcF16};
  const char* hw = state + p.hp;  // dW's operand
  if (per_row) {
    if (u.f16) fw_xent_top_kernel<<<1, 1024, 0, st>>>(head, row_of, go, top);
    if (dweight) {
      T* hs = reinterpret_cast<T*>(ws + p.hs);
      const int64_t cap = (int64_t)sm_count() * 8;
      fw_xent_scale_kernel<T><<<(unsigned)(p.Bp < cap ? p.Bp : cap), 256, 0, st>>>(
          head, row_of, u, reinterpret_cast<const T*>(state + p.hp), hs, p.Dp);
      hw = ws + p.hs;
    }
    if (cudaGetLastError() != cudaSuccess) return FWB_E_LAUNCH;
  }
  CUtensorMap mh, mw, mg, wmn, gmn, hmn;
  const char* hp = state + p.hp;
  char* g = ws + p.g;
  if (!tc_map(&mh, K, hp, p.Bp, D, p.Dp, 128) || !tc_map(&mw, K, w, V, D, ldw, 128) ||
      !tc_map(&mg, K, g, p.Bp, p.piece, p.piece, 128) || !tc_map(&wmn, K, w, V, D, ldw, 64) ||
      !tc_map(&gmn, K, g, p.Bp, p.piece, p.piece, 64) || !tc_map(&hmn, K, hw, p.Bp, D, p.Dp, 64))
    return FWB_E_LAUNCH;
  const int64_t Vp = up(V, 256), mb = p.Bp / 256, nd = (D + 255) / 256;
  float* sum = p.pieces > 1 || p.splits > 1 ? reinterpret_cast<float*>(ws + p.sum) : nullptr;
  for (int64_t i = 0; i < p.pieces; ++i) {
    const int v0 = (int)(i * p.piece), vn = (int)(Vp - v0 < p.piece ? Vp - v0 : p.piece);
    const GradArgs ga = {head, label, row_of, reinterpret_cast<const float*>(state + p.lse), u, g, p.piece, (int)V, (int)D,
                         v0, vn, status};
    if (launch_gemm<GradTile<T, K>>(mh, mw, ga, mb * (vn / 256), st) != cudaSuccess) return FWB_E_LAUNCH;
    const int64_t tiles = (dhidden ? mb * nd * p.splits : 0) + (dweight ? vn / 256 * nd : 0);
    const int64_t pairs = sm_count() / 2;
    const ProductArgs pa = {head, row_of, u, sum, dhidden, dweight, (int)p.Bp, (int)V, (int)D, (int)up(D, 32), v0, vn,
                            i == 0, i == p.pieces - 1, (int)p.piece, (int)p.splits,
                            (int)(tiles < pairs ? tiles : pairs), status};
    if (launch_gemm<ProductTile<T, K>>(mg, wmn, pa, tiles, st, &gmn, &hmn) != cudaSuccess) return FWB_E_LAUNCH;
    if (dhidden && pa.last && p.splits > 1) {
      const int64_t need = (p.Bp * ((D + 127) / 128) + 7) / 8, cap = (int64_t)sm_count() * 16;
      if (launch_dependent(fw_xent_dhidden_kernel<T>, need < cap ? need : cap, 256, 0, 1, st, pa) != cudaSuccess)
        return FWB_E_LAUNCH;
    }
  }
  return FWB_OK;
}

}  // namespace
}  // namespace fwb200

using namespace fwb200;

extern "C" {

int64_t fw_xent_state_bytes(int64_t B, int64_t D, int64_t V, const void* weight, int64_t ldw) {
  if (xent_check(FWB_DTYPE_BF16, B, D, V) != FWB_OK) return 0;
  return xent_plan(B, D, V, !tma_rows(weight, ldw)).state_bytes;
}

int64_t fw_xent_workspace(int64_t B, int64_t D, int64_t V, int backward) {
  if (xent_check(FWB_DTYPE_BF16, B, D, V) != FWB_OK) return 0;
  const XentPlan p = xent_plan(B, D, V, false);
  return backward ? p.bwd_bytes : p.fwd_bytes;
}

int fw_xent_forward(int dtype, const void* hidden, int64_t ldh, const void* weight, int64_t ldw, const int64_t* y,
                    int64_t B, int64_t D, int64_t V, int64_t ignore_index, int reduction, float* loss, void* state,
                    int64_t state_bytes, void* workspace, int64_t workspace_bytes, int32_t* status, void* stream) {
  if (int rc = xent_check(dtype, B, D, V)) return rc;
  if (reduction < FWB_REDUCE_NONE || reduction > FWB_REDUCE_SUM || ldh < D || ldw < D || ldh > ((int64_t)1 << 38) ||
      ldw > ((int64_t)1 << 38))
    return FWB_E_SHAPE;
  if (B > 0 && (!hidden || !y)) return FWB_E_POINTER;
  if (!weight || !state || !workspace || (!loss && (B > 0 || reduction != FWB_REDUCE_NONE))) return FWB_E_POINTER;
  if (reinterpret_cast<uintptr_t>(hidden) % 2 || reinterpret_cast<uintptr_t>(weight) % 2 || !aligned16(state) ||
      !aligned16(workspace))
    return FWB_E_POINTER;
  const XentPlan p = xent_plan(B, D, V, !tma_rows(weight, ldw));
  if (state_bytes < p.state_bytes || workspace_bytes < p.fwd_bytes) return FWB_E_CAPACITY;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (B == 0) {  // no rows: the mean is 0 / 0
    if (cudaMemsetAsync(state, 0, sizeof(XentHead), st) != cudaSuccess) return FWB_E_LAUNCH;
    if (reduction == FWB_REDUCE_NONE) return FWB_OK;
    return cudaMemsetAsync(loss, reduction == FWB_REDUCE_MEAN ? 0xff : 0, 4, st) == cudaSuccess ? FWB_OK : FWB_E_LAUNCH;
  }
  char* s = static_cast<char*>(state);
  char* w = static_cast<char*>(workspace);
  return dtype == FWB_DTYPE_BF16 ? run_forward<__nv_bfloat16, kTcBf16>(hidden, ldh, weight, ldw, y, B, D, V, ignore_index,
                                                                       reduction, loss, s, w, status, st)
                                 : run_forward<__half, kTcF16>(hidden, ldh, weight, ldw, y, B, D, V, ignore_index,
                                                               reduction, loss, s, w, status, st);
}

int fw_xent_backward(int dtype, const void* weight, int64_t ldw, int64_t B, int64_t D, int64_t V, int reduction,
                     const float* grad_output, const void* state, int64_t state_bytes, void* workspace,
                     int64_t workspace_bytes, void* dhidden, void* dweight, int32_t* status, void* stream) {
  if (int rc = xent_check(dtype, B, D, V)) return rc;
  if (reduction < FWB_REDUCE_NONE || reduction > FWB_REDUCE_SUM || ldw < D || ldw > ((int64_t)1 << 38))
    return FWB_E_SHAPE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (B == 0) {
    if (dweight && cudaMemsetAsync(dweight, 0, (size_t)(2 * V * D), st) != cudaSuccess) return FWB_E_LAUNCH;
    return FWB_OK;
  }
  if (!weight || !grad_output || !state || !workspace) return FWB_E_POINTER;
  if (reinterpret_cast<uintptr_t>(weight) % 2 || reinterpret_cast<uintptr_t>(dhidden) % 2 ||
      reinterpret_cast<uintptr_t>(dweight) % 2 || !aligned16(state) || !aligned16(workspace))
    return FWB_E_POINTER;
  const XentPlan p = xent_plan(B, D, V, !tma_rows(weight, ldw));
  if (state_bytes < p.state_bytes || workspace_bytes < p.bwd_bytes) return FWB_E_CAPACITY;
  if (!dhidden && !dweight) return FWB_OK;
  const char* s = static_cast<const char*>(state);
  char* w = static_cast<char*>(workspace);
  const int per_row = reduction == FWB_REDUCE_NONE, mean = reduction == FWB_REDUCE_MEAN;
  return dtype == FWB_DTYPE_BF16
             ? run_backward<__nv_bfloat16, kTcBf16>(weight, ldw, B, D, V, mean, grad_output, per_row, s, w, dhidden,
                                                    dweight, status, st)
             : run_backward<__half, kTcF16>(weight, ldw, B, D, V, mean, grad_output, per_row, s, w, dhidden, dweight,
                                            status, st);
}

}  // extern "C"
