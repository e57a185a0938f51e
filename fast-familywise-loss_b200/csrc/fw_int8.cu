// Output layer in 8-bit integers:
//   out[t, n] = (sum_k q[t, k] * wq[n, k]) * q_scale[t] * w_scale[n]
// with an exact 32-bit integer sum on the tensor cores (tcgen05 kind::i8),
// two fp32 multiplications and one rounding to the output's type.
//
// Two layouts of the same product:
//   many tokens  tokens are the rows of a tile, weight rows its columns: 256 x
//                256 tiles by two CTAs, bound by the tensor cores (4096 x 4096
//                into 32000 columns: 395 us, 2.7 Pop/s), or, where 128 x 128
//                tiles by one CTA are no more than the SMs, those (333 x 4096
//                into 5001: 17.4 us against 20.3; 300 x 4096 into 8000, more
//                tiles than SMs: 27.1 against 20.0);
//   few tokens   weight rows are the 128 rows of a tile and the tokens its
//                16 .. 128 columns: every weight is read once, bound by HBM
//                (48 x 4096 into 128256: 95 us, 5.7 TB/s).
//                The rows that do not make a whole round of tiles are dealt
//                out evenly over the SMs in steps of 8 (a last round of whole
//                tiles would leave up to all but one of them idle), loading
//                only the 32-row boxes they need, and the first weights are brought
//                into L2 while the kernel before (the norm that makes q) still
//                runs.  Past 16 tokens it takes a whole round of tiles, past 64
//                three (64 x 4096 into 10000: 20.9 us against 16.5 with tiles of
//                tokens, into 20000: 30.4 against 32.9; 128 tokens into 32000:
//                37.2 against 35.8, into 128256: 102 against 107).  Columns for
//                the tokens there are: one token into 128256 86 us, with 128
//                columns 122.
#include "fw_tc_gemm.cuh"

namespace fwb200 {
namespace {

struct Int8Args {
  const float* qs;
  const float* ws;
  void* out;
  int64_t ldo;
  int T, N, K;
  int vec;  // fp32 rows of out start on 16-byte boundaries
  int per;  // few tokens: weight rows per CTA behind the whole tiles
  int32_t* status;
};

template <class TO, int SIDE>
struct Int8Many {
  using Args = Int8Args;
  static constexpr int COLS = SIDE / 2;  // per epilogue warp
  struct State {
    float qs, ws[COLS / 32];
  };
  static constexpr TcKind KIND = kTcS8;
  static constexpr bool A_MN = false, B_MN = false;
  static constexpr bool TWO = false, A_MN2 = false;
  static constexpr int CG = SIDE / 128, BN = SIDE, STAGES = 5, KC = 0, EW = 8, A_BOX = 128, AHEAD = 0;
  static constexpr uint32_t EPI_BYTES = EW * (sizeof(TO) == 2 ? kStageBytes<COLS> : 32 * 33 * 4);
  struct Plan {
    TileOrder order;
    int first, step;
  };
  __device__ static void plan(const Args& a, int group, int groups, Plan* p) {
    p->order.set((a.T + SIDE - 1) / SIDE, (a.N + SIDE - 1) / SIDE, 16);  // token blocks that share the weight tiles in flight
    p->first = group;
    p->step = groups;
  }
  __device__ static bool get(const Args& a, const Plan& p, int i, TcTile* t) {
    const int w = p.first + i * p.step;
    if (w >= p.order.count()) return false;
    int m, n;
    p.order.get(w, &m, &n);
    *t = {m * SIDE, n * SIDE, 0, 0, (a.K + 127) / 128, 128, 0};
    return true;
  }
  __device__ static void begin(const Args& a, const Plan&, const TcTile& t, const TcPart& p, State& st) {
    const int row = t.m0 + p.row + p.lane, col = t.n0 + p.share * COLS + p.lane;
    st.qs = row < a.T ? a.qs[row] : 0.0f;
#pragma unroll
    for (int k = 0; k < COLS / 32; ++k) st.ws[k] = col + 32 * k < a.N ? a.ws[col + 32 * k] : 0.0f;
  }
  template <bool LOST, class Done>
  __device__ static void epilogue(const Args& a, const Plan&, const TcTile& t, const TcPart& p, State& st, int, int,
                                  Done done) {
    const int r0 = t.m0 + p.row, rows = a.T - r0, s0 = p.share * COLS;
    TO* out = static_cast<TO*>(a.out) + t.n0 + s0;
#pragma unroll
    for (int c = 0; c < COLS; c += 32) {
      float v[32];
      if constexpr (!LOST) tmem_ld32(p.taddr + s0 + c, v);
      if (c + 32 == COLS) done();
#pragma unroll
      for (int i = 0; i < 32; ++i)
        v[i] = LOST ? CUDART_NAN_F : (float)__float_as_int(v[i]) * st.qs * __shfl_sync(kFull, st.ws[c / 32], i);
      if constexpr (sizeof(TO) == 2)
        stage_block<TO, COLS>(reinterpret_cast<uint32_t*>(p.smem), v, p.lane, c);
      else
        store_block(reinterpret_cast<float*>(p.smem), v, p.lane, a.N - (t.n0 + s0 + c), a.vec,
                    [&](int i) -> float* { return i < rows ? out + (int64_t)(r0 + i) * a.ldo + c : nullptr; });
    }
    if constexpr (sizeof(TO) == 2)
      store_staged<TO, COLS>(reinterpret_cast<uint32_t*>(p.smem), p.lane, min(COLS, a.N - (t.n0 + s0)),
                       [&](int i) -> TO* { return i < rows ? out + (int64_t)(r0 + i) * a.ldo : nullptr; });
  }
};

template <class TO, int NT>
struct Int8Few {
  using Args = Int8Args;
  struct State {
    float ws, qs[(NT + 31) / 32];  // lane i: tokens i, i + 32, ...
  };
  static constexpr TcKind KIND = kTcS8;
  static constexpr bool A_MN = false, B_MN = false;
  static constexpr bool TWO = false, A_MN2 = false;
  static constexpr int CG = 1, BN = NT, KC = 0, EW = 4, A_BOX = 32, AHEAD = 16;
  static constexpr int STAGES = NT <= 32 ? 10 : NT <= 64 ? 8 : 6;
  static constexpr uint32_t EPI_BYTES = 0;
  struct Plan {
    int group, groups, rounds;
  };
  __device__ static void plan(const Args& a, int group, int groups, Plan* p) {
    p->group = group;
    p->groups = groups;
    p->rounds = a.N / 128 / groups;
  }
  // whole tiles in turn, then what is left in equal parts
  __device__ static bool get(const Args& a, const Plan& p, int i, TcTile* t) {
    int m0 = (i * p.groups + p.group) * 128, rows = 128;
    if (i >= p.rounds) {
      if (i > p.rounds) return false;
      m0 = p.rounds * p.groups * 128 + p.group * a.per;
      rows = min(a.per, a.N - m0);
      if (rows <= 0) return false;
    }
    *t = {m0, 0, 0, 0, (a.K + 127) / 128, rows, 0};
    return true;
  }
  __device__ static void begin(const Args& a, const Plan&, const TcTile& t, const TcPart& p, State& st) {
    const int row = p.row + p.lane;
    st.ws = row < t.rows ? a.ws[t.m0 + row] : 0.0f;
#pragma unroll
    for (int k = 0; k < (NT + 31) / 32; ++k) st.qs[k] = k * 32 + p.lane < a.T ? a.qs[k * 32 + p.lane] : 0.0f;
  }
  template <bool LOST, class Done>
  __device__ static void epilogue(const Args& a, const Plan&, const TcTile& t, const TcPart& p, State& st, int, int,
                                  Done done) {
    const int n = t.m0 + p.row + p.lane;
    const bool mine = p.row + p.lane < t.rows;
    TO* out = static_cast<TO*>(a.out) + n;
    constexpr int STEP = NT < 32 ? 16 : 32;
#pragma unroll
    for (int c = 0; c < NT; c += STEP) {
      float v[STEP];
      if constexpr (LOST) {
      } else if constexpr (STEP == 32) {
        tmem_ld32(p.taddr + c, v);
      } else {
        tmem_ld16(p.taddr + c, v);
      }
      if (c + STEP == NT) done();
#pragma unroll
      for (int i = 0; i < STEP; ++i) {
        const int tok = c + i;
        const float x =
            LOST ? CUDART_NAN_F : (float)__float_as_int(v[i]) * __shfl_sync(kFull, st.qs[tok / 32], tok % 32) * st.ws;
        if (mine && tok < a.T) st_elem(out + (int64_t)tok * a.ldo, x);
      }
    }
  }
};

template <class P>
cudaError_t run_int8(const void* a, int64_t rows_a, int64_t lda, const void* b, int64_t rows_b, int64_t ldb,
                     const Int8Args& args, int64_t tiles, cudaStream_t st) {
  CUtensorMap ma, ma2, mb;
  if (!tc_map(&ma, kTcS8, a, rows_a, args.K, lda, kGemmBM) || !tc_map(&ma2, kTcS8, a, rows_a, args.K, lda, P::A_BOX) ||
      !tc_map(&mb, kTcS8, b, rows_b, args.K, ldb, P::BN / P::CG))
    return cudaErrorInvalidValue;
  return launch_gemm<P>(ma, mb, args, tiles, st, &ma2);
}

template <class TO>
cudaError_t run_int8_linear(const int8_t* q, int64_t ldq, const int8_t* w, int64_t ldw, Int8Args a,
                            cudaStream_t st) {
  const int sms = sm_count(), left = a.N % (128 * sms);
  a.per = ((left + sms - 1) / sms + 7) / 8 * 8;
  const int64_t nt = a.N / 128 >= sms ? sms : (left + a.per - 1) / a.per;  // CTAs
  const int64_t rounds = a.N / 128 / sms;  // of whole tiles of weight rows
  if (a.T <= 16) return run_int8<Int8Few<TO, 16>>(w, a.N, ldw, q, a.T, ldq, a, nt, st);
  if (a.T <= 32 && rounds >= 1) return run_int8<Int8Few<TO, 32>>(w, a.N, ldw, q, a.T, ldq, a, nt, st);
  if (a.T <= 64 && rounds >= 1) return run_int8<Int8Few<TO, 64>>(w, a.N, ldw, q, a.T, ldq, a, nt, st);
  if (a.T <= 128 && rounds >= 3) return run_int8<Int8Few<TO, 128>>(w, a.N, ldw, q, a.T, ldq, a, nt, st);
  const int64_t small = (((int64_t)a.T + 127) / 128) * (((int64_t)a.N + 127) / 128);
  if (small <= sms) return run_int8<Int8Many<TO, 128>>(q, a.T, ldq, w, a.N, ldw, a, small, st);
  const int64_t big = (((int64_t)a.T + 255) / 256) * (((int64_t)a.N + 255) / 256);
  return run_int8<Int8Many<TO, 256>>(q, a.T, ldq, w, a.N, ldw, a, big, st);
}

}  // namespace
}  // namespace fwb200

using namespace fwb200;

extern "C" {

int fw_int8_linear(int out_dtype, const int8_t* q, int64_t ldq, const float* q_scale, const int8_t* wq, int64_t ldw,
                   const float* w_scale, int64_t T, int64_t N, int64_t K, void* out, int64_t ldo, int32_t* status,
                   void* stream) {
  if (out_dtype != FWB_DTYPE_F32 && out_dtype != FWB_DTYPE_BF16 && out_dtype != FWB_DTYPE_F16) return FWB_E_DTYPE;
  if (T < 0 || N < 1 || K < 1 || T > (1 << 30) || N > (1 << 30)) return FWB_E_SHAPE;
  if (K > FWB_INT8_MAX_K || ((T + 127) / 128) * ((N + 255) / 256) > (1 << 30)) return FWB_E_CAPACITY;
  if (ldq % 16 != 0 || ldw % 16 != 0 || ldq < K || ldw < K || ldo < N || ldq > ((int64_t)1 << 39) ||
      ldw > ((int64_t)1 << 39) || ldo > ((int64_t)1 << 60) / (T > 0 ? T : 1))
    return FWB_E_SHAPE;
  if (T == 0) return FWB_OK;
  if (!q || !q_scale || !wq || !w_scale || !out) return FWB_E_POINTER;
  if (!aligned16(q) || !aligned16(wq)) return FWB_E_POINTER;
  if (reinterpret_cast<uintptr_t>(out) % (out_dtype == FWB_DTYPE_F32 ? 4 : 2)) return FWB_E_POINTER;
  const int64_t es = out_dtype == FWB_DTYPE_F32 ? 4 : 2;
  const int vec = aligned16(out) && ldo * es % 16 == 0 && N * es % 16 == 0;
  const Int8Args a = {q_scale, w_scale, out, ldo, (int)T, (int)N, (int)K, vec, 0, status};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (out_dtype == FWB_DTYPE_BF16) return launch_status(run_int8_linear<__nv_bfloat16>(q, ldq, wq, ldw, a, st));
  if (out_dtype == FWB_DTYPE_F16) return launch_status(run_int8_linear<__half>(q, ldq, wq, ldw, a, st));
  return launch_status(run_int8_linear<float>(q, ldq, wq, ldw, a, st));
}

}  // extern "C"
