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
//
// Log probabilities with entropies take the same kernels (BOTH below).  With a
// temperature T and t = (z - max z) / T the tiles keep sum exp(t) t as well,
// from which the entropy is h_r = log S - (sum exp(t) t) / S, two positive
// terms, and with upstream factors a of logp and b of the entropy the logit
// gradient is, with l = log p,
//   T G_rj = a_r (1[j = y(r)] - p_rj) - b_r p_rj (l_rj + h_r).
// Its factors are in G whole: they have no common power of two to be split off
// where a and b differ, and a row of H is then rounded no further.  What the
// rounding takes from the label's entry, which would show in a whole row of dH
// and in the largest terms of dW, is kept in fp32 and added to both: that much
// of the label's row of W, and of the row of H.  In flat rows their error is that
// of a form in 32 bits rounded at the end.  It grows where another column than
// the label's holds much of the probability, whose entry is as large and rounded
// with nothing kept (512 x 256 into 4000, labels drawn from the rows; mean
// entropies of 8, 5.5, 4, 3, 1.8, 0.7 and 0.4 nats: 1.00, 1.01, 1.04, 1.06, 1.1,
// 1.16 and 1.2 times, with factors of the entropies as large as those of the log
// probabilities 1.00, 1.07, 1.13, 1.13, 1.15, 1.16 and 1.2).
// |p (l + h)| is at most (log V) / 4 + 0.3, under 5.2, hence 2^13 in the place
// of 2^15 for float16.  bfloat16, 4014 live rows, 128256 x 4096: 13.4 to 14.1 ms;
// float16, 1609 live rows, 32000 x 2048: 0.86 to 0.87 ms; at T < 0.5 (see
// GradBothTile) 14.4 and 0.90.
#include <cmath>

#include "fw_reduce.cuh"
#include "fw_rowslots.cuh"
#include "fw_sort.cuh"
#include "fw_tc_gemm.cuh"

namespace fwb200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kF16Unit = 32768.0f, kF16UnitBoth = 8192.0f;
constexpr float kExpFloor = -200.0f;  // 2^kExpFloor is 0 in fp32; keeps 0 * t finite
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
  float* more_rows;  // sorted: the same, entropies
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

// As fw_xent_pack_kernel, the live rows in the order of their labels, equal ones
// by position, those outside [0, V) last: the product finds the rows of a label
// next to each other.  Up to kCountRows rows every CTA counts what comes before
// its own; more are sorted first, and `sorted` has them (key V: out of range, V
// + 1: ignored).  Rows of 512 bfloat16, by counting and by sorting, each kernel
// by itself: 4096 rows 12 us (in the order given: 7), 8192 29 and 38, 65536
// sorted 64 (in the order given: 55).
constexpr int64_t kCountRows = 8192;

template <class T>
__global__ void __launch_bounds__(kPackThreads) fw_xent_pack_sorted_kernel(PackArgs a, const uint2* sorted) {
  __shared__ int red[10][kPackThreads / 32];
  constexpr int V = 16 / sizeof(T);
  wait_prior_kernel();
  allow_dependent_launch();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t r0 = (int64_t)blockIdx.x * a.per_cta;
  const Span<T> span(a.hidden, a.B, a.ldh, a.D);
  const auto key_of = [&](int64_t y, int64_t i) {  // of a live row
    return ((uint64_t)(y >= 0 && y < a.V ? (uint32_t)y : 0xffffffffu) << 32) | (uint64_t)i;
  };
  const auto put = [&](int64_t dst, int64_t r, bool live, int64_t y, int64_t rows_up) {  // one warp
    if (lane == 0) {
      const bool ok = y >= 0 && y < a.V;
      a.row_of[dst] = r < a.B ? (int32_t)r : -1;
      a.label[dst] = live && ok ? (int32_t)y : -1;
      if (live && !ok) raise_status(a.status, FWB_STATUS_LABEL_RANGE);
      if (!live && r < a.B) a.loss_rows[r] = a.more_rows[r] = 0.0f;
    }
    if (dst >= rows_up) return;
    T* out = static_cast<T*>(a.hp) + dst * a.Dp;
    const T* in = static_cast<const T*>(a.hidden) + (live ? r : 0) * a.ldh;
    for (int64_t e0 = (int64_t)lane * V; e0 < a.Dp; e0 += 4 * 32 * V) {
      uint4 x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int64_t e = e0 + k * 32 * V;
        x[k] = live && e < a.Dp ? load_slot_shifted(in, (int)e, span) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (e0 + k * 32 * V < a.Dp) *reinterpret_cast<uint4*>(out + e0 + k * 32 * V) = x[k];
    }
  };
  if (sorted) {
    int64_t lo = 0, hi = a.B;  // live rows: up to the first ignored one
    while (lo < hi) {
      const int64_t mid = (lo + hi) / 2;
      if (sorted[mid].x <= (uint32_t)a.V)
        lo = mid + 1;
      else
        hi = mid;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.head = {(int32_t)lo, 0u, 0};
    for (int64_t i = r0 + w; i < r0 + a.per_cta && i < a.Bp; i += kPackThreads / 32) {
      const uint2 e = i < a.B ? sorted[i] : make_uint2((uint32_t)a.V + 1u, (uint32_t)i);
      put(i, e.y, i < lo, e.x < (uint32_t)a.V ? (int64_t)e.x : -1, (lo + 255) / 256 * 256);
    }
    return;
  }
  for (int g0 = 0; g0 < a.per_cta; g0 += 8) {  // 8 rows, a warp each
    uint64_t key[8];
    int n[10] = {};  // live rows before each in the order of labels; all; before the first by position
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int64_t r = r0 + g0 + k, y = r < a.B ? a.y[r] : a.ignore;
      key[k] = y != a.ignore ? key_of(y, r) : 0u;
    }
    for (int64_t i0 = threadIdx.x; i0 < a.B; i0 += 4 * kPackThreads) {
      int64_t y[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) y[q] = i0 + q * kPackThreads < a.B ? a.y[i0 + q * kPackThreads] : a.ignore;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t i = i0 + q * kPackThreads;
        const bool live = y[q] != a.ignore;
        const uint64_t own = live ? key_of(y[q], i) : ~0ull;
#pragma unroll
        for (int k = 0; k < 8; ++k) n[k] += own < key[k];
        n[8] += live;
        n[9] += live && i < r0 + g0;
      }
    }
#pragma unroll
    for (int k = 0; k < 10; ++k) {
      n[k] = __reduce_add_sync(kFull, n[k]);
      if (lane == 0) red[k][w] = n[k];
    }
    __syncthreads();
    int rank = 0, total = 0, before = 0;  // of this warp's row
#pragma unroll
    for (int i = 0; i < kPackThreads / 32; ++i) {
      rank += red[w][i];
      total += red[8][i];
      before += red[9][i];
    }
    if (g0 == 0 && blockIdx.x == 0 && threadIdx.x == 0) *a.head = {total, 0u, 0};
    const int64_t r = r0 + g0 + w, y = r < a.B ? a.y[r] : a.ignore;
    const bool live = y != a.ignore;
    for (int k = 0; k < w; ++k) {
      const int64_t q = r0 + g0 + k;
      before += q < a.B && a.y[q] != a.ignore;
    }
    if (g0 + w < a.per_cta && r < a.Bp) put(live ? rank : total + (r - before), r, live, y, ((int64_t)total + 255) / 256 * 256);
    __syncthreads();
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
  float* part_t;  // BOTH: sum of 2^t t, t = (z - maximum) c
  float c;        // BOTH: log2(e) / T
};

// The accumulator is taken over every kLseStages stages of K and added up in
// registers: the tensor cores' fp32 additions round towards zero, so a logit
// shrinks by a part that grows with the length of the sum.  Every 8, 16, 32 or
// all 64 stages (K = 4096): error of the loss 1.2e-7, 2.6e-7, 5.6e-7, 1.2e-6,
// forward and backward 13.5, 13.4, 13.4, 13.4 ms.
constexpr int kLseStages = 8;
constexpr int kLseCols = 128;  // columns of a tile per epilogue thread: they stay in its registers

template <TcKind K, bool BOTH>
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
    float m = -CUDART_INF_F, s = 0.0f, u = 0.0f;
#pragma unroll
    for (int i = 0; i < kLseCols; ++i) {
      if (i >= valid) st.z[i] = -CUDART_INF_F;
      if (i == y) a.zy[row] = st.z[i];
      m = max_nan(m, st.z[i]);
    }
    if (m != -CUDART_INF_F) {  // a NaN maximum, or +inf, makes the sum NaN
      float s4[4] = {0.0f, 0.0f, 0.0f, 0.0f}, u2[2] = {0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < kLseCols; ++i) {
        if constexpr (BOTH) {
          const float t2 = fmaxf((st.z[i] - m) * a.c, kExpFloor), e = exp2_hw(t2);
          s4[i & 3] += e;
          u2[i & 1] = fmaf(e, t2, u2[i & 1]);
        } else {
          s4[i & 3] += exp2_hw((st.z[i] - m) * kLog2e);
        }
      }
      s = (s4[0] + s4[1]) + (s4[2] + s4[3]);
      u = u2[0] + u2[1];
    }
    if constexpr (BOTH) a.part_t[(int64_t)(n0 / kLseCols) * a.Bp + row] = u;
    a.part[(int64_t)(n0 / kLseCols) * a.Bp + row] = make_float2(m, s);
  }
};

struct JoinArgs {
  XentHead* head;
  const float2* part;
  const float* zy;
  const int32_t* label;
  const int32_t* row_of;
  float* lse;        // [Bp], packed; BOTH: maximum
  float* loss_pack;  // [Bp], packed
  float* loss;       // [B] (reduction none) or one value
  int64_t Bp;
  int ntiles;
  int reduction;
  int32_t* status;
  const float* part_t;           // BOTH, which writes logp in the place of the loss
  float *entropy, *entropy_pack;  // per given row, packed
  float* log_s;                   // BOTH: log S, packed
  float inv_t;
};

constexpr int kJoinWarps = 32;

// Maximum and sums of BOTH, relative to another maximum (not under it).
__device__ __forceinline__ void raise_sums(float m, float to, float c, float* s, float* u) {
  const float d = fmaxf((m - to) * c, kExpFloor), f = exp2_hw(d);
  *u = f * fmaf(d, *s, *u);
  *s *= f;
}

// As fw_xent_join_kernel, for log probabilities and entropies.
__global__ void __launch_bounds__(kJoinWarps * 32) fw_xent_join_both_kernel(JoinArgs a) {
  __shared__ float sm[kJoinWarps][33], ss[kJoinWarps][33], su[kJoinWarps][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  wait_prior_kernel();
  const int rows = a.head->rows;
  const int row = blockIdx.x * 32 + lane;
  const float c = a.inv_t * kLog2e;
  float m = -CUDART_INF_F, s = 0.0f, u = 0.0f;
  if (row < rows) {
    constexpr int N = 8;  // parts in flight, joined by their largest maximum
    for (int t0 = w; t0 < a.ntiles; t0 += N * kJoinWarps) {
      float2 p[N];
      float pu[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int t = t0 + i * kJoinWarps;
        p[i] = t < a.ntiles ? a.part[(int64_t)t * a.Bp + row] : make_float2(-CUDART_INF_F, 0.0f);
        pu[i] = t < a.ntiles ? a.part_t[(int64_t)t * a.Bp + row] : 0.0f;
      }
      float to = m;
#pragma unroll
      for (int i = 0; i < N; ++i) to = max_nan(to, p[i].x);
      if (to == -CUDART_INF_F) continue;
      if (m != -CUDART_INF_F) raise_sums(m, to, c, &s, &u);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (p[i].x == -CUDART_INF_F) continue;
        raise_sums(p[i].x, to, c, &p[i].y, &pu[i]);
        s += p[i].y;
        u += pu[i];
      }
      m = to;
    }
  }
  sm[w][lane] = m;
  ss[w][lane] = s;
  su[w][lane] = u;
  __syncthreads();
  // a warp per row, a lane per part
  const int mine = blockIdx.x * 32 + w;
  if (mine >= rows) return;
  m = sm[lane][w], s = ss[lane][w], u = su[lane][w];
  const float M = warp_max_nan(m);
  if (m != -CUDART_INF_F) raise_sums(m, M, c, &s, &u);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(kFull, s, o);
    u += __shfl_xor_sync(kFull, u, o);
  }
  if (lane != 0) return;
  const float S = s, U = u;
  const bool label = a.label[mine] >= 0, ok = label && a.head->status == 0 && fabsf(M) < CUDART_INF_F;
  if (w == 0 && a.head->status != 0) raise_status(a.status, a.head->status);
  if (label && !(fabsf(M) < CUDART_INF_F)) raise_status(a.status, FWB_STATUS_NONFINITE);
  const float log_s = logf(S), nan = CUDART_NAN_F;
  const int to = a.row_of[mine];
  const float h = ok ? log_s - U * kLn2 / S : nan;
  a.lse[mine] = ok ? M : nan;
  a.log_s[mine] = ok ? log_s : nan;
  a.entropy_pack[mine] = h;
  a.entropy[to] = h;
  a.loss[to] = ok ? (a.zy[mine] - M) * a.inv_t - log_s : nan;
}

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
  int both;             // go is logp's, either may be NULL
  const float* go_ent;  // the entropy's
  float inv_t;

  // g_r; of BOTH the larger of the two
  __device__ float factor(int r) const {
    return both ? max_nan(go ? fabsf(go[r]) : 0.0f, go_ent ? fabsf(go_ent[r]) : 0.0f) : go[r];
  }
  // s_r, scaled to the range of the type; a factor that is not finite stands for itself
  __device__ float in_g(int r) const {
    if (!per_row) return f16 ? kF16Unit : 1.0f;
    const float g = go[r], s = pow2_above(g);
    if (!(s < CUDART_INF_F)) return g;
    return f16 && *top > 0.0f ? s / *top * kF16Unit : s;
  }
  // BOTH: -a_r and -b_r, scaled to the range of the type (float16: by kF16UnitBoth / top); NaN where either is not finite
  __device__ float top_both() const { return f16 && *top > 0.0f ? *top : 0.0f; }
  __device__ float2 in_g_both(float a, float b, float top) const {
    if (!(fabsf(a) < CUDART_INF_F && fabsf(b) < CUDART_INF_F)) return make_float2(CUDART_NAN_F, CUDART_NAN_F);
    return top > 0.0f ? make_float2(-a / top * kF16UnitBoth, -b / top * kF16UnitBoth) : make_float2(-a, -b);
  }
  // f_r; 1 where the factor is in G (0, not finite, BOTH) or common
  __device__ float rest(int r) const {
    if (!per_row || both) return 1.0f;
    const float g = go[r], s = pow2_above(g);
    return s > 0.0f && s < CUDART_INF_F ? g / s : 1.0f;
  }
  // common factor taken out after the sums
  __device__ float back(const XentHead* h) const {
    if (both) return f16 && *top > 0.0f ? *top / kF16UnitBoth * inv_t : inv_t;
    if (per_row) return f16 && *top > 0.0f ? *top / kF16Unit : 1.0f;
    const float g = mean ? go[0] / (float)h->rows : go[0];
    return f16 ? g / kF16Unit : g;
  }
};

__global__ void __launch_bounds__(1024) fw_xent_top_kernel(const XentHead* head, const int32_t* row_of, Upstream up,
                                                             float* out) {
  __shared__ float red[32];
  wait_prior_kernel();
  allow_dependent_launch();
  const int rows = head->rows;
  float top = 0.0f;
  for (int i = threadIdx.x; i < rows; i += 1024) {
    const float s = pow2_above(up.factor(row_of[i]));
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
  const float* entropy;  // BOTH: packed
  const float* log_s;    // BOTH: log S, packed; `lse` has the maxima
  float* label_rest;     // BOTH: what rounding took from the label's entry, packed
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
        float q;
        if constexpr (LOST) {
          q = CUDART_NAN_F;
        } else {
          q = exp2_hw((v[i] - lse) * kLog2e);
          if (t.n0 + c + i == y) q -= 1.0f;
        }
        v[i] = i < valid ? q * coef : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(g + c + 8 * i) = pack_slot<T>(v + 8 * i);
    }
  }
};

// BOTH: with l = (z - max z) / T - log S, and the maximum and log S apart: M / T
// + log S in one number would be off by half an ulp of M / T, by 2e-5 at T = 0.1
// and 2e-3 at T = 1e-3 where the winning logit is 50.
// A sum over all of K in the accumulator (KC 0) shrinks a logit more than the
// forward's does (kLseStages), by up to D / 8 ulps of its terms, which T
// divides too: of a winning logit of 50, D = 2048, a probability of 1 came out
// 2e-4 too small at T = 1, 2 % at T = 0.01.  Down to kLowT that is under
// the rounding of G (2^-8 of an entry in bfloat16, 2^-11 in float16).  At lower
// temperatures z is made as in the forward: the same bits, of which the maximum
// is one, and the probabilities add up to 1 within fp32's rounding whatever T is.
// Parts are short, and the epilogue of a tile's last one is then waited for: 1609
// live rows, 32000 x 2048 float16 172 and 217 us, 4014 rows, 128256 x 4096
// bfloat16 3.32 and 3.96 ms.
// Nothing in `begin` waits: a row's factors, which are behind row_of, are asked
// for after the first part, and worked out after the last (with parts: 226 us
// where the labels' entries are looked at one by one, 217 all at once).
constexpr float kLowT = 0.5f;

template <class T, TcKind K, bool LOW>
struct GradBothTile {
  using Args = GradArgs;
  static constexpr int COLS = 128;  // of a tile per epilogue thread
  struct State {
    int y, row;      // -2: not a live row; the given row
    float m, log_s, h;
    float lo, en;    // the upstream factors
    float z[COLS] = {};  // the logits so far
  };
  static constexpr TcKind KIND = K;
  static constexpr bool A_MN = false, B_MN = false;
  static constexpr bool TWO = false, A_MN2 = false;
  static constexpr int CG = 2, BN = kTileN, STAGES = 7, KC = LOW ? kLseStages : 0, EW = 4 * BN / COLS, A_BOX = 128, AHEAD = 0;
  static constexpr uint32_t EPI_BYTES = 0;
  struct Plan {
    TurnPlan turn;
    int rows;
    float top;  // of the factors, float16
  };
  __device__ static void plan(const Args& a, int group, int groups, Plan* p) {
    p->turn.set(row_tiles(a.head), a.vn / BN, group, groups);
    p->rows = a.head->rows;
    p->top = a.up.top_both();
  }
  __device__ static bool get(const Args& a, const Plan& p, int i, TcTile* t) {
    int m, n;
    if (!p.turn.get(i, &m, &n)) return false;
    *t = {m * kTileM, a.v0 + n * BN, 0, 0, (a.D + 63) / 64, 128, 0};
    return true;
  }
  __device__ static void begin(const Args& a, const Plan& plan, const TcTile& t, const TcPart& p, State& st) {
    const int row = t.m0 + p.row + p.lane;
    st.y = -2;
    st.row = -1;
    st.m = st.log_s = st.h = st.lo = st.en = 0.0f;
    if (row < plan.rows) {
      st.y = a.label[row];
      st.row = a.row_of[row];
      st.m = a.lse[row];
      st.log_s = a.log_s[row];
      st.h = a.entropy[row];
    }
  }
  template <bool LOST, class Done>
  __device__ static void epilogue(const Args& a, const Plan& plan, const TcTile& t, const TcPart& p, State& st, int k,
                                  int parts, Done done) {
    const int row = t.m0 + p.row + p.lane, n0 = t.n0 + p.share * COLS;
    if constexpr (!LOST) {
#pragma unroll
      for (int c = 0; c < COLS; c += 16) {
        float v[16];
        tmem_ld16(p.taddr + p.share * COLS + c, v);
#pragma unroll
        for (int i = 0; i < 16; ++i) st.z[c + i] += v[i];
      }
      done();
      if (k == 0 && st.row >= 0) {
        if (a.up.go) st.lo = a.up.go[st.row];
        if (a.up.go_ent) st.en = a.up.go_ent[st.row];
      }
      if (k < parts - 1) return;
    }
    T* g = static_cast<T*>(a.g) + (int64_t)row * a.ldg + (n0 - a.v0);
    const float2 f = a.up.in_g_both(st.lo, st.en, plan.top);
    const int y = st.y - n0, valid = st.y != -2 ? a.V - n0 : 0;
    const auto entry = [&](float z) {  // of a bad row m, log_s and h are NaN, and so is what comes of them
      const float l = fmaxf(fmaf(z - st.m, a.up.inv_t, -st.log_s), kExpFloor * kLn2);
      return exp2_hw(l * kLog2e) * fmaf(f.y, l + st.h, f.x);
    };
    float zy = 0.0f;
#pragma unroll
    for (int c = 0; c < COLS; c += 8) {
      if (!LOST && (unsigned)(y - c) < 8u) {
#pragma unroll
        for (int i = 0; i < 8; ++i) zy = c + i == y ? st.z[c + i] : zy;
      }
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = LOST ? CUDART_NAN_F : entry(st.z[c + i]);
        v[i] = c + i < valid ? v[i] : 0.0f;
      }
      *reinterpret_cast<uint4*>(g + c) = pack_slot<T>(v);
    }
    if (!LOST && (unsigned)y < (unsigned)COLS) {
      const float q = entry(zy) - f.x;
      const T r = Elem<T>::from_f(q);
      g[y] = r;
      a.label_rest[row] = q - Elem<T>::to_f(r);
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
  // BOTH: dH takes label_rest of the label's row of the weight,
  const float* label_rest;
  const int32_t* label;
  const void* w;
  int64_t ldw;
  // and dW that of the rows of H with this label: their sum is in the row of
  // `sums` with the number of the first of them, first_row[v - v0] (-1: none)
  const void* hp;
  int64_t ldh;
  __nv_bfloat16* sums;
  int64_t lds2;
  int32_t* first_row;

  // 8 columns of it from c on, times `by`, added to v
  template <class T>
  __device__ void add_label(int y, int c, float by, float* v) const {
    const T* p = static_cast<const T*>(w) + (int64_t)y * ldw + c;
    float x[8];
    unpack16<T>(c + 8 <= D ? ld_global16(p) : load_elems(p, p, p + (D - c)), x);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = fmaf(by, x[i], v[i]);
  }

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

template <class T, TcKind K, bool BOTH>
struct ProductTile {
  using Args = ProductArgs;
  struct State {
    int mine;  // dH: the given row of this lane's row
    float f;   // its factor
    bool zero;
    float rest;  // BOTH: its label_rest, 0 without a label
    int label;
    bool any;  // BOTH, dW: there are sums for one of the warp's 32 rows
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
    if constexpr (BOTH) {
      st.label = dh && !st.zero ? a.label[row] : -1;
      st.rest = st.label >= 0 ? a.label_rest[row] : 0.0f;
      st.any = !dh && fetch(a, p, t.m0 + p.row, t.n0 + p.share * (BN / 2));
    }
  }

  // BOTH: dW's rows take what is in `sums`.  While the tile's products run, the
  // warp leaves its rows' in the staging rows that the epilogue takes them from
  // before it writes there.  (Loads wait here behind the operands' copies, some
  // 5000 clocks, so that many are in flight and none depends on another.)
  __device__ static bool fetch(const Args& a, const TcPart& p, int v, int c0) {
    if (c0 >= a.D) return false;
    const int first = a.first_row[v + p.lane];
    uint32_t who = __ballot_sync(kFull, first >= 0);
    if (who == 0u) return false;
    uint32_t* sm = reinterpret_cast<uint32_t*>(p.smem);
    constexpr int kWords = kStageWords<BN / 2>;
    for (int i = p.lane; i < 32 * kWords; i += 32) sm[i] = 0u;
    __syncwarp();
    while (who) {
      uint2 u[16];
      int to[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        to[i] = __ffs(who) - 1;  // -1: no more
        who &= who - 1;
        const int64_t row = __shfl_sync(kFull, first, to[i] & 31);
        if (to[i] >= 0) u[i] = *reinterpret_cast<const uint2*>(a.sums + row * a.lds2 + c0 + 4 * p.lane);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (to[i] >= 0) {
          sm[to[i] * kWords + 2 * p.lane] = u[i].x;
          sm[to[i] * kWords + 2 * p.lane + 1] = u[i].y;
        }
    }
    __syncwarp();
    return true;
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
      if constexpr (BOTH && !LOST) {
        if (st.rest != 0.0f) {
#pragma unroll
          for (int i = 0; i < 32; i += 8)
            if (c + i < cols) a.template add_label<T>(st.label, t.n0 + s0 + c + i, st.rest, v + i);
        }
        if (st.any) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint32_t u = sm[p.lane * kStageWords<BN / 2> + c / 2 + i];
            v[2 * i] += __uint_as_float(u << 16);
            v[2 * i + 1] += __uint_as_float(u & 0xffff0000u);
          }
        }
      }
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

// First of the packed rows, in the order of their labels, whose label is at least v: 33 parts a step, by a warp.
__device__ __forceinline__ int first_at(const int32_t* label, int rows, uint32_t v, int lane) {
  int lo = 0, hi = rows;  // labels before lo are under v, those from hi on are not
  while (lo < hi) {
    const int step = (hi - lo + 32) / 33, at = lo + (lane + 1) * step - 1;
    const bool under = at < hi && (uint32_t)label[at] < v;
    const int n = __popc(__ballot_sync(kFull, under));  // the first n of them
    if (n < 32) hi = min(hi, lo + (n + 1) * step - 1);
    lo += n * step;
  }
  return lo;
}

// BOTH: label_rest times the rows of H, summed over the rows of every label:
// what rounding took from dW's largest terms (bfloat16 has the range of the
// sums, and rounds what is itself the rest of a rounding).  Packed rows are in
// the order of their labels, so a label's are next to each other.  A CTA takes
// the labels that begin in 32 rows, and 128 columns: a warp those that begin in
// four of the rows, all warps the one that may go on beyond the 32, if it is long
// (the commonest tokens are those of a tenth of the rows).  The grid's last CTAs look for the
// first row of every v of the piece.  (Summed by the warps of the product's
// tiles instead: labels that fall off as 1 / rank, 1609 live rows, 32000 x 2048
// bfloat16, gradient 828 us, so 623; 65536 x 256 into 1000 3719 and 658.)
template <class T>
__global__ void __launch_bounds__(256) fw_xent_labels_kernel(ProductArgs a) {
  __shared__ float4 part[8][32];
  wait_prior_kernel();
  allow_dependent_launch();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int rows = a.head->rows, slabs = (a.D + 127) / 128, summing = a.Bp / 32 * slabs;
  if ((int)blockIdx.x >= summing) {
    const int i = ((int)blockIdx.x - summing) * 256 + threadIdx.x;
    if (i >= a.vn) return;
    const uint32_t v = (uint32_t)(a.v0 + i);
    int lo = 0, hi = rows;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if ((uint32_t)a.label[mid] < v)
        lo = mid + 1;
      else
        hi = mid;
    }
    a.first_row[i] = lo < rows && (uint32_t)a.label[lo] == v ? lo : -1;
    return;
  }
  const int r0 = (int)blockIdx.x / slabs * 32, c = (int)blockIdx.x % slabs * 128 + 4 * lane;
  if (r0 >= rows) return;
  const int n = min(32, rows - r0);
  const int y = lane < n ? a.label[r0 + lane] : -1, before = r0 + lane > 0 && lane < n ? a.label[r0 + lane - 1] : -2;
  const uint32_t starts = __ballot_sync(kFull, lane < n && y != before);
  if (starts == 0u) return;
  const T* h = static_cast<const T*>(a.hp) + c;
  const auto load = [&](int64_t row, float& by, uint2& u) {
    by = a.label_rest[row];
    u = c < a.ldh ? *reinterpret_cast<const uint2*>(h + row * a.ldh) : make_uint2(0u, 0u);
  };
  const auto add_row = [&](float by, uint2 u, float (&x)[4]) {
    x[0] = fmaf(by, Elem<T>::bits_to_f(u.x & 0xffffu), x[0]);
    x[1] = fmaf(by, Elem<T>::bits_to_f(u.x >> 16), x[1]);
    x[2] = fmaf(by, Elem<T>::bits_to_f(u.y & 0xffffu), x[2]);
    x[3] = fmaf(by, Elem<T>::bits_to_f(u.y >> 16), x[3]);
  };
  const auto add = [&](int from, int to, float (&x)[4]) {  // rows from .. to
    for (int r = from; r < to; r += 8) {
      uint2 u[8];
      float by[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) load(min(r + i, to - 1), by[i], u[i]);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (r + i < to) add_row(by[i], u[i], x);
    }
  };
  const auto give = [&](int row, const float (&x)[4]) {
    *reinterpret_cast<uint2*>(a.sums + (int64_t)row * a.lds2 + c) =
        make_uint2(pack2<__nv_bfloat16>(x[0], x[1]), pack2<__nv_bfloat16>(x[2], x[3]));
  };
  const auto wanted = [&](int at) {  // its label is of this piece
    const int v = __shfl_sync(kFull, y, at);
    return v >= a.v0 && v < a.v0 + a.vn;
  };
  const int last = 31 - __clz((int)starts);
  if (const uint32_t mine = starts & (0xfu << 4 * w) & ~(1u << last)) {  // labels that begin in the warp's 4 rows
    int at = __ffs(mine) - 1;
    const int end = __ffs(starts & ~((2u << (31 - __clz((int)mine))) - 1u)) - 1;
    float x[4] = {};
    for (int r = at; r < end; r += 8) {
      uint2 u[8];
      float by[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) load(r0 + min(r + i, end - 1), by[i], u[i]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (r + i >= end) break;
        if (r + i != at && (starts >> (r + i) & 1u)) {
          if (wanted(at)) give(r0 + at, x);
          at = r + i;
          x[0] = x[1] = x[2] = x[3] = 0.0f;
        }
        add_row(by[i], u[i], x);
      }
    }
    if (wanted(at)) give(r0 + at, x);
  }
  if (!wanted(last)) return;
  const int from = r0 + last, yl = __shfl_sync(kFull, y, last);
  int to = r0 + n;
  if (to < rows && a.label[to] == yl) to = first_at(a.label, rows, (uint32_t)yl + 1u, lane);
  float x[4] = {};
  if (to - from <= 32) {
    if (last / 4 != w) return;
    add(from, to, x);
    give(from, x);
    return;
  }
  add(from + (int)((int64_t)(to - from) * w / 8), from + (int)((int64_t)(to - from) * (w + 1) / 8), x);
  part[w][lane] = make_float4(x[0], x[1], x[2], x[3]);
  __syncthreads();
  if (w != 0) return;
#pragma unroll
  for (int q = 1; q < 8; ++q) {
    const float4 o = part[q][lane];
    x[0] += o.x, x[1] += o.y, x[2] += o.z, x[3] += o.w;
  }
  give(from, x);
}

// dH from the sums of its splits; one warp per row and 128 columns.
template <class T, bool BOTH>
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
      if constexpr (BOTH) {
        const int y = a.label[r];
        if (y >= 0) {
          const float by = a.label_rest[r];
          const T* w = static_cast<const T*>(a.w) + (int64_t)y * a.ldw + c;
          v.x = fmaf(by, ld_elem(w), v.x);
          if (c + 1 < a.D) v.y = fmaf(by, ld_elem(w + 1), v.y);
          if (c + 2 < a.D) v.z = fmaf(by, ld_elem(w + 2), v.z);
          if (c + 3 < a.D) v.w = fmaf(by, ld_elem(w + 3), v.w);
        }
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
  int64_t row_of, label, lse, entropy, log_s, hp, wp, state_bytes;
  // forward workspace
  int64_t part, part_t, zy, loss_pack, sorted, hist, fwd_bytes;
  // backward workspace
  int64_t piece, pieces, splits, top, label_rest, sums, first, g, sum, hs, bwd_bytes;
};

XentPlan xent_plan(int64_t B, int64_t D, int64_t V, bool copy_w, bool both = false) {
  XentPlan p = {};
  p.Bp = up(B, 256);
  p.Dp = up(D, 8);
  p.copy_w = copy_w;
  int64_t at = 256;
  p.row_of = at, at += up(4 * p.Bp, 256);
  p.label = at, at += up(4 * p.Bp, 256);
  p.lse = at, at += up(4 * p.Bp, 256);
  p.entropy = at, at += both ? up(4 * p.Bp, 256) : 0;
  p.log_s = at, at += both ? up(4 * p.Bp, 256) : 0;
  p.hp = at, at += up(2 * p.Bp * p.Dp, 256);
  p.wp = at, at += copy_w ? up(2 * V * p.Dp, 256) : 0;
  p.state_bytes = at;
  at = 0;
  p.part = at, at += up(8 * p.Bp * up(V, kTileN) / kLseCols, 256);
  p.part_t = at, at += both ? up(4 * p.Bp * up(V, kTileN) / kLseCols, 256) : 0;
  p.zy = at, at += up(4 * p.Bp, 256);
  p.loss_pack = at, at += up(4 * p.Bp, 256);
  if (both && B > kCountRows) {
    int passes, bits;
    sort_digits(V + 1, &passes, &bits);
    p.sorted = at, at += up(16 * B, 256);
    p.hist = at, at += up((B + kSortTile - 1) / kSortTile * ((int64_t)4 << bits), 256);
  }
  p.fwd_bytes = at;
  const int64_t Vp = up(V, 256);
  p.pieces = (2 * p.Bp * Vp + kPieceBytes - 1) / kPieceBytes;
  if (p.pieces < 1) p.pieces = 1;
  p.piece = up((Vp + p.pieces - 1) / p.pieces, 256);
  p.pieces = (Vp + p.piece - 1) / p.piece;
  at = 0;
  p.top = at, at += 256;
  p.label_rest = at, at += both ? up(4 * p.Bp, 256) : 0;
  p.sums = at, at += both ? up(2 * p.Bp * up(D, 128), 256) : 0;
  p.first = at, at += both ? up(4 * p.piece, 256) : 0;
  p.g = at, at += up(2 * p.Bp * p.piece, 256);
  // as many as one row tile could use, 16 stages of K each, within kSumBytes
  p.splits = sm_count() / 2 / ((D + kTileN - 1) / kTileN);
  const int64_t room = B > 0 ? kSumBytes / (4 * p.Bp * up(D, 32)) : 1;
  if (p.splits > room) p.splits = room;
  if (p.splits > p.piece / 64 / 16) p.splits = p.piece / 64 / 16;
  if (p.splits < 1) p.splits = 1;
  p.sum = at, at += p.pieces > 1 || p.splits > 1 ? up(4 * p.splits * p.Bp * up(D, 32), 256) : 0;
  p.hs = at, at += both ? 0 : up(2 * p.Bp * p.Dp, 256);  // factors per row
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

// BOTH: log probabilities in the place of losses, FWB_REDUCE_NONE.
template <class T, TcKind K, bool BOTH>
int run_forward(const void* hidden, int64_t ldh, const void* weight, int64_t ldw, const int64_t* y, int64_t B,
                int64_t D, int64_t V, int64_t ignore, int reduction, float* loss, float* entropy, float inv_t,
                char* state, char* ws, int32_t* status, cudaStream_t st) {
  const XentPlan p = xent_plan(B, D, V, !tma_rows(weight, ldw), BOTH);
  XentHead* head = reinterpret_cast<XentHead*>(state);
  int32_t* row_of = reinterpret_cast<int32_t*>(state + p.row_of);
  int32_t* label = reinterpret_cast<int32_t*>(state + p.label);
  const int64_t per_cta = (p.Bp + 4 * sm_count() - 1) / (4 * sm_count());
  PackArgs pk = {hidden, y, B, p.Bp, D, p.Dp, ldh, V, ignore, state + p.hp, row_of, label,
                 reduction == FWB_REDUCE_NONE ? loss : nullptr, head, status, (int)(per_cta < 8 ? 8 : per_cta), entropy};
  const int64_t ctas = (p.Bp + pk.per_cta - 1) / pk.per_cta;
  if constexpr (BOTH) {
    const uint2* sorted = nullptr;
    if (B > kCountRows) {
      SortArgs s = {};
      s.ids = y, s.T = B, s.V = V, s.padding = ignore, s.tail = 1;
      s.hist = reinterpret_cast<uint32_t*>(ws + p.hist);
      s.tiles = (int)((B + kSortTile - 1) / kSortTile);
      int passes;
      sort_digits(V + 1, &passes, &s.bits);
      uint2* ent = reinterpret_cast<uint2*>(ws + p.sorted);
      sorted = sort_launch(s, ent, ent + B, passes, st);
      if (cudaGetLastError() != cudaSuccess) return FWB_E_LAUNCH;
    }
    if (launch_dependent(fw_xent_pack_sorted_kernel<T>, ctas, kPackThreads, 0, 1, st, pk, sorted) != cudaSuccess)
      return FWB_E_LAUNCH;
  } else {
    if (launch_dependent(fw_xent_pack_kernel<T>, ctas, kPackThreads, 0, 1, st, pk) != cudaSuccess) return FWB_E_LAUNCH;
  }
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
                (int)D, &head->status, reinterpret_cast<float*>(ws + p.part_t), inv_t * kLog2e};
  const int64_t nt = (V + 255) / 256;
  if (launch_gemm<LseTile<K, BOTH>>(mh, mw, la, (p.Bp / 256) * nt, st) != cudaSuccess) return FWB_E_LAUNCH;
  JoinArgs ja = {head, la.part, la.zy, label, row_of, reinterpret_cast<float*>(state + p.lse),
                 reinterpret_cast<float*>(ws + p.loss_pack), loss, p.Bp, (int)((V + kLseCols - 1) / kLseCols), reduction, status,
                 la.part_t, entropy, reinterpret_cast<float*>(state + p.entropy), reinterpret_cast<float*>(state + p.log_s), inv_t};
  return launch_status(launch_dependent(BOTH ? fw_xent_join_both_kernel : fw_xent_join_kernel, p.Bp / 32, kJoinWarps * 32, 0, 1, st, ja));
}

template <class T, TcKind K, bool BOTH>
int run_backward(const void* weight, int64_t ldw, int64_t B, int64_t D, int64_t V, int mean, const float* go,
                 const float* go_ent, float inv_t, int per_row, const char* state, char* ws, void* dhidden, void* dweight,
                 int32_t* status, cudaStream_t st) {
  const XentPlan p = xent_plan(B, D, V, !tma_rows(weight, ldw), BOTH);
  const XentHead* head = reinterpret_cast<const XentHead*>(state);
  const int32_t* row_of = reinterpret_cast<const int32_t*>(state + p.row_of);
  const int32_t* label = reinterpret_cast<const int32_t*>(state + p.label);
  const void* w = p.copy_w ? state + p.wp : weight;
  if (p.copy_w) ldw = p.Dp;
  float* top = reinterpret_cast<float*>(ws + p.top);
  const Upstream u = {go, top, per_row, mean, K == kTcF16, BOTH, go_ent, inv_t};
  const char* hw = state + p.hp;  // dW's operand
  if (per_row) {
    if (u.f16 && launch_dependent(fw_xent_top_kernel, 1, 1024, 0, 1, st, head, row_of, u, top) != cudaSuccess)
      return FWB_E_LAUNCH;
    if (dweight && !BOTH) {
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
                         v0, vn, status, reinterpret_cast<const float*>(state + p.entropy),
                         reinterpret_cast<const float*>(state + p.log_s),
                         reinterpret_cast<float*>(ws + p.label_rest)};
    const int64_t logit_tiles = mb * (vn / 256);
    cudaError_t e;
    if constexpr (!BOTH)
      e = launch_gemm<GradTile<T, K>>(mh, mw, ga, logit_tiles, st);
    else if (inv_t > 1.0f / kLowT)
      e = launch_gemm<GradBothTile<T, K, true>>(mh, mw, ga, logit_tiles, st);
    else
      e = launch_gemm<GradBothTile<T, K, false>>(mh, mw, ga, logit_tiles, st);
    if (e != cudaSuccess) return FWB_E_LAUNCH;
    const int64_t tiles = (dhidden ? mb * nd * p.splits : 0) + (dweight ? vn / 256 * nd : 0);
    const int64_t pairs = sm_count() / 2;
    const ProductArgs pa = {head, row_of, u, sum, dhidden, dweight, (int)p.Bp, (int)V, (int)D, (int)up(D, 32), v0, vn,
                            i == 0, i == p.pieces - 1, (int)p.piece, (int)p.splits,
                            (int)(tiles < pairs ? tiles : pairs), status, ga.label_rest, label, w, ldw,
                            hp, p.Dp, reinterpret_cast<__nv_bfloat16*>(ws + p.sums), up(D, 128),
                            reinterpret_cast<int32_t*>(ws + p.first)};
    if (BOTH && dweight) {
      const int64_t ctas = p.Bp / 32 * ((D + 127) / 128) + vn / 256;
      if (launch_dependent(fw_xent_labels_kernel<T>, ctas, 256, 0, 1, st, pa) != cudaSuccess) return FWB_E_LAUNCH;
    }
    if (launch_gemm<ProductTile<T, K, BOTH>>(mg, wmn, pa, tiles, st, &gmn, &hmn) != cudaSuccess) return FWB_E_LAUNCH;
    if (dhidden && pa.last && p.splits > 1) {
      const int64_t need = (p.Bp * ((D + 127) / 128) + 7) / 8, cap = (int64_t)sm_count() * 16;
      if (launch_dependent(fw_xent_dhidden_kernel<T, BOTH>, need < cap ? need : cap, 256, 0, 1, st, pa) != cudaSuccess)
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
  return dtype == FWB_DTYPE_BF16
             ? run_forward<__nv_bfloat16, kTcBf16, false>(hidden, ldh, weight, ldw, y, B, D, V, ignore_index, reduction,
                                                          loss, nullptr, 1.0f, s, w, status, st)
             : run_forward<__half, kTcF16, false>(hidden, ldh, weight, ldw, y, B, D, V, ignore_index, reduction, loss,
                                                  nullptr, 1.0f, s, w, status, st);
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
             ? run_backward<__nv_bfloat16, kTcBf16, false>(weight, ldw, B, D, V, mean, grad_output, nullptr, 1.0f, per_row,
                                                           s, w, dhidden, dweight, status, st)
             : run_backward<__half, kTcF16, false>(weight, ldw, B, D, V, mean, grad_output, nullptr, 1.0f, per_row, s, w,
                                                   dhidden, dweight, status, st);
}

static int head_check(int dtype, int64_t B, int64_t D, int64_t V, float inv_t) {
  if (int rc = xent_check(dtype, B, D, V)) return rc;
  if (!(inv_t > 0.0f) || !std::isfinite(inv_t * kLog2e)) return FWB_E_SHAPE;
  return FWB_OK;
}

int64_t fw_lm_head_log_probs_state(int64_t B, int64_t D, int64_t V, const void* weight, int64_t ldw) {
  if (xent_check(FWB_DTYPE_BF16, B, D, V) != FWB_OK) return 0;
  return xent_plan(B, D, V, !tma_rows(weight, ldw), true).state_bytes;
}

int64_t fw_lm_head_log_probs_workspace(int64_t B, int64_t D, int64_t V, int backward) {
  if (xent_check(FWB_DTYPE_BF16, B, D, V) != FWB_OK) return 0;
  const XentPlan p = xent_plan(B, D, V, false, true);
  return backward ? p.bwd_bytes : p.fwd_bytes;
}

int fw_lm_head_log_probs(int dtype, const void* hidden, int64_t ldh, const void* weight, int64_t ldw, const int64_t* y,
                         int64_t B, int64_t D, int64_t V, float inv_t, int64_t ignore_index, float* logp, float* entropy,
                         void* state, int64_t state_bytes, void* workspace, int64_t workspace_bytes, int32_t* status,
                         void* stream) {
  if (int rc = head_check(dtype, B, D, V, inv_t)) return rc;
  if (ldh < D || ldw < D || ldh > ((int64_t)1 << 38) || ldw > ((int64_t)1 << 38)) return FWB_E_SHAPE;
  if (!weight || !state || !workspace) return FWB_E_POINTER;
  if (B > 0 && (!hidden || !y || !logp || !entropy)) return FWB_E_POINTER;
  if (reinterpret_cast<uintptr_t>(hidden) % 2 || reinterpret_cast<uintptr_t>(weight) % 2 || !aligned16(state) ||
      !aligned16(workspace))
    return FWB_E_POINTER;
  const XentPlan p = xent_plan(B, D, V, !tma_rows(weight, ldw), true);
  if (state_bytes < p.state_bytes || workspace_bytes < p.fwd_bytes) return FWB_E_CAPACITY;
  if (B == 0) return FWB_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  char* s = static_cast<char*>(state);
  char* w = static_cast<char*>(workspace);
  return dtype == FWB_DTYPE_BF16
             ? run_forward<__nv_bfloat16, kTcBf16, true>(hidden, ldh, weight, ldw, y, B, D, V, ignore_index,
                                                         FWB_REDUCE_NONE, logp, entropy, inv_t, s, w, status, st)
             : run_forward<__half, kTcF16, true>(hidden, ldh, weight, ldw, y, B, D, V, ignore_index, FWB_REDUCE_NONE,
                                                 logp, entropy, inv_t, s, w, status, st);
}

int fw_lm_head_log_probs_grad(int dtype, const void* weight, int64_t ldw, int64_t B, int64_t D, int64_t V, float inv_t,
                              const float* dlogp, const float* dentropy, const void* state, int64_t state_bytes,
                              void* workspace, int64_t workspace_bytes, void* dhidden, void* dweight, int32_t* status,
                              void* stream) {
  if (int rc = head_check(dtype, B, D, V, inv_t)) return rc;
  if (ldw < D || ldw > ((int64_t)1 << 38)) return FWB_E_SHAPE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (B == 0) {
    if (dweight && cudaMemsetAsync(dweight, 0, (size_t)(2 * V * D), st) != cudaSuccess) return FWB_E_LAUNCH;
    return FWB_OK;
  }
  if (!weight || !state || !workspace) return FWB_E_POINTER;
  if (reinterpret_cast<uintptr_t>(weight) % 2 || reinterpret_cast<uintptr_t>(dhidden) % 2 ||
      reinterpret_cast<uintptr_t>(dweight) % 2 || !aligned16(state) || !aligned16(workspace))
    return FWB_E_POINTER;
  const XentPlan p = xent_plan(B, D, V, !tma_rows(weight, ldw), true);
  if (state_bytes < p.state_bytes || workspace_bytes < p.bwd_bytes) return FWB_E_CAPACITY;
  if (!dhidden && !dweight) return FWB_OK;
  const char* s = static_cast<const char*>(state);
  char* w = static_cast<char*>(workspace);
  return dtype == FWB_DTYPE_BF16
             ? run_backward<__nv_bfloat16, kTcBf16, true>(weight, ldw, B, D, V, 0, dlogp, dentropy, inv_t, 1, s, w,
                                                          dhidden, dweight, status, st)
             : run_backward<__half, kTcF16, true>(weight, ldw, B, D, V, 0, dlogp, dentropy, inv_t, 1, s, w, dhidden,
                                                  dweight, status, st);
}

}  // extern "C"
