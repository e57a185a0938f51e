// Rows cut into 16-byte slots of memory, for kernels that keep a row in
// registers whatever its length and start address.
//
// A row of D elements that starts `off` elements past a 16-byte boundary is
// covered by slots k = 0, 1, ...; slot k holds elements k * V - off + j,
// j < V = 16 / sizeof(T).  Slots inside the row are one 16-byte access; the
// first and the last touch only the row's own elements, one by one.  Tensors
// whose rows start at the same distance from a boundary share the slots; if
// they do not (`vec` false), off is 0 and every slot is read element by
// element.
#pragma once

#include "fw_device.cuh"

namespace fwb200 {

// 16 bytes of global memory.  Not the non-coherent form, which wants memory
// that nobody writes while the kernel runs: a programmatic dependent has
// started while the kernel before it still writes what it will read.
__device__ __forceinline__ uint4 ld_global16(const void* p) {
  uint4 r;
  asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p)
               : "memory");
  return r;
}

// The same for what is read once.
__device__ __forceinline__ uint4 ld_global16_once(const void* p) {
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p)
               : "memory");
  return r;
}

template <class T>
__device__ __forceinline__ void store_slot(T* row, int64_t e0, int64_t D, bool vec, const uint4& u) {
  constexpr int V = 16 / sizeof(T);
  if (vec && e0 >= 0 && e0 + V <= D) {
    *reinterpret_cast<uint4*>(row + e0) = u;
    return;
  }
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int64_t e = e0 + j;
    if (e >= 0 && e < D) {
      if constexpr (sizeof(T) == 4)
        row[e] = __uint_as_float(w[j]);
      else
        *reinterpret_cast<unsigned short*>(row + e) = (unsigned short)(w[j >> 1] >> (16 * (j & 1)));
    }
  }
}

// Two values in one word, rounded to nearest by one instruction.
template <class T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  static_assert(sizeof(T) == 2, "16-bit types");
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

template <class T>
__device__ __forceinline__ uint4 pack_slot(const float* v) {
  if constexpr (sizeof(T) == 4)
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  else
    return make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
}

// First element of a matrix and the one behind its last.
template <class T>
struct Span {
  const T* lo;
  const T* hi;
  __device__ __forceinline__ Span(const void* base, int64_t rows, int64_t ld, int64_t D)
      : lo(static_cast<const T*>(base)), hi(lo + (rows - 1) * ld + D) {}
};

// Elements p .. p + V one by one, those outside [lo, hi) as zero.
template <class T>
__device__ __forceinline__ uint4 load_elems(const T* p, const T* lo, const T* hi) {
  constexpr int V = 16 / sizeof(T);
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (p + j >= lo && p + j < hi) {
      if constexpr (sizeof(T) == 4)
        w[j] = __float_as_uint(p[j]);
      else
        w[j >> 1] |= (uint32_t)*reinterpret_cast<const unsigned short*>(p + j) << (16 * (j & 1));
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The slot at row + e0 of a row that may start anywhere: its 16 bytes through
// the two aligned neighbours they lie in and a funnel shift.  Elements outside
// the row are whatever lies there (zero outside the span).
template <class T>
__device__ __forceinline__ uint4 load_slot_shifted(const T* row, int e0, const Span<T>& span) {
  const T* p = row + e0;
  const uintptr_t addr = reinterpret_cast<uintptr_t>(p);
  const uint32_t m = (uint32_t)(addr & 15u);
  const uintptr_t lo = addr - m;
  if (lo < reinterpret_cast<uintptr_t>(span.lo) || lo + (m ? 32 : 16) > reinterpret_cast<uintptr_t>(span.hi))
    return load_elems(p, span.lo, span.hi);
  const uint4 a = ld_global16(reinterpret_cast<const void*>(lo));
  if (m == 0) return a;
  const uint4 b = ld_global16(reinterpret_cast<const void*>(lo + 16));
  const uint32_t s = (m & 3u) * 8u;
  uint32_t w[5];
  switch (m >> 2) {  // the same for the whole row
    case 0: w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x; break;
    case 1: w[0] = a.y, w[1] = a.z, w[2] = a.w, w[3] = b.x, w[4] = b.y; break;
    case 2: w[0] = a.z, w[1] = a.w, w[2] = b.x, w[3] = b.y, w[4] = b.z; break;
    default: w[0] = a.w, w[1] = b.x, w[2] = b.y, w[3] = b.z, w[4] = b.w; break;
  }
  return make_uint4(__funnelshift_r(w[0], w[1], s), __funnelshift_r(w[1], w[2], s), __funnelshift_r(w[2], w[3], s),
                    __funnelshift_r(w[3], w[4], s));
}

}  // namespace fwb200
