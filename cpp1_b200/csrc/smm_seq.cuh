// Helpers of the sequence operators (short convolution, selective scan, 4-bit
// matrix-vector product): vectors of fp32 or bf16 elements widened to fp32,
// sequence boundaries and state slots, host-side overlap checks.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "smm_device.cuh"
#include "smm_host.h"

namespace smm {

// Two fp32 lanes in one 64-bit register: one instruction does two multiply-adds, each
// rounded as a scalar one is.
__device__ __forceinline__ unsigned long long pack2(float a, float b) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(unsigned long long x, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x));
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// The two elements of a bf16 pair.
__device__ __forceinline__ unsigned long long widen2(uint32_t w) {
  return pack2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
__device__ __forceinline__ uint32_t narrow2(unsigned long long v) {
  float a, b;
  unpack2(v, a, b);
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  return static_cast<float>(v);
}
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// N consecutive elements as fp32.  With VEC they are moved in pieces of 16 bytes, or of
// 8 where N elements are no multiple of 16 bytes; the pointer is aligned to a piece.
template <int BYTES>
struct Piece {
  using type = uint4;
};
template <>
struct Piece<8> {
  using type = uint2;
};
// The raw pieces, and their elements.
template <typename T, int N, int PB>
struct RawVec {
  static_assert(N * sizeof(T) % PB == 0, "whole pieces");
  typename Piece<PB>::type q[N * sizeof(T) / PB];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < int(N * sizeof(T) / PB); ++i) q[i] = reinterpret_cast<const typename Piece<PB>::type*>(p)[i];
  }
  __device__ __forceinline__ void get(float (&v)[N]) const {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(q);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (sizeof(T) == 4)
        v[i] = __uint_as_float(w[i]);
      else
        v[i] = __uint_as_float((i & 1) ? (w[i / 2] & 0xFFFF0000u) : (w[i / 2] << 16));
    }
  }
};
template <typename T, int N, bool VEC, int PB = (N * sizeof(T) % 16 == 0 ? 16 : 8)>
__device__ __forceinline__ void load_f32(const T* p, float (&v)[N]) {
  if constexpr (VEC) {
    RawVec<T, N, PB> r;
    r.load(p);
    r.get(v);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = to_f32(p[i]);
  }
}
template <typename T, int N, bool VEC, int PB = (N * sizeof(T) % 16 == 0 ? 16 : 8)>
__device__ __forceinline__ void store_f32(T* p, const float (&v)[N]) {
  if constexpr (VEC) {
    constexpr int Q = N * sizeof(T) / PB;
    typename Piece<PB>::type q[Q];
    uint32_t* w = reinterpret_cast<uint32_t*>(q);
#pragma unroll
    for (int i = 0; i < int(N * sizeof(T) / 4); ++i) {
      if constexpr (sizeof(T) == 4) {
        w[i] = __float_as_uint(v[i]);
      } else {
        const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&b);
      }
    }
#pragma unroll
    for (int i = 0; i < Q; ++i) reinterpret_cast<typename Piece<PB>::type*>(p)[i] = q[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = from_f32<T>(v[i]);
  }
}

// v * sigmoid(v) in five instructions: exp(-v) as a power of two and the reciprocal by
// the fast units, 2 units in the last place each.  (The IEEE quotient made an
// epilogue of 64 of them ten times as long.)  It is 0, the right limit, once
// 1 + exp(-v) passes 2^126 (v below -87).
__device__ __forceinline__ float silu(float v) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-1.4426950408889634f * v));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return v * r;
}
__device__ __forceinline__ unsigned long long silu2(unsigned long long v) {
  float a, b, ra, rb;
  unpack2(mul2(v, pack2(-1.4426950408889634f, -1.4426950408889634f)), a, b);
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(a));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(b));
  unpack2(add2(pack2(a, b), pack2(1.0f, 1.0f)), a, b);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(ra) : "f"(a));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(rb) : "f"(b));
  return mul2(v, pack2(ra, rb));
}
// log(1 + exp(v)); above 20 the correction is below half a step of v.
__device__ __forceinline__ float softplus(float v) { return v > 20.0f ? v : log1pf(expf(v)); }

// Rows [begin, end) of sequence s, kept inside [0, tokens) whatever the
// offsets hold.
__device__ __forceinline__ void seq_range(const int* __restrict__ offsets, int s, long long tokens, long long* begin,
                                          long long* end) {
  if (!offsets) {
    *begin = 0;
    *end = tokens;
    return;
  }
  long long b = __ldg(offsets + s), e = __ldg(offsets + s + 1);
  b = b < 0 ? 0 : (b > tokens ? tokens : b);
  e = e < b ? b : (e > tokens ? tokens : e);
  *begin = b;
  *end = e;
}

// State entry of sequence s, or -1 when it has none.
__device__ __forceinline__ int seq_slot(const int* __restrict__ slots, int s, int nslots, uint32_t* status) {
  const int i = slots ? __ldg(slots + s) : s;
  if (i >= nslots) {
    if (status) atomicOr(status, kDevErrBounds | kBoundsSlot);
    return -1;
  }
  return i < 0 ? -1 : i;
}

// ---------------------------------------------------------------- host checks
// Memory that a call touches: rows of `width` bytes, ld apart (one row: contiguous bytes).
struct Span {
  const void* p;
  size_t width;
  long long rows = 1;
  size_t ld = 0;
};
inline Span row_span(const void* p, long long rows, long long width, long long ld, size_t esz) {
  return {p, static_cast<size_t>(width) * esz, rows, static_cast<size_t>(ld) * esz};
}
// Whether two spans share a byte.  Columns of the same rows of one matrix may lie side
// by side; rows of different strides count as whole.
inline bool overlaps(const Span& a, const Span& b) {
  if (!a.p || !b.p || !a.width || !b.width || a.rows <= 0 || b.rows <= 0) return false;
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
  const size_t an = (a.rows - 1) * a.ld + a.width, bn = (b.rows - 1) * b.ld + b.width;
  if (x >= y + bn || y >= x + an) return false;
  if ((a.rows == 1 && b.rows == 1) || (a.rows > 1 && b.rows > 1 && a.ld != b.ld)) return true;
  const long long ld = a.rows > 1 ? a.ld : b.ld, aw = a.width, bw = b.width;
  if (aw > ld || bw > ld) return true;
  // b's row j begins d + (j - i) ld behind a's row i: some k = j - i with -bw < d + k ld < aw?
  const long long d = static_cast<long long>(y - x);
  for (long long k = -d / ld - 2; k <= -d / ld + 2; ++k)
    if (k > -a.rows && k < b.rows && d + k * ld > -bw && d + k * ld < aw) return true;
  return false;
}
inline bool aligned_to(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
// All of these pointers lie on a multiple of n bytes, an element's size (null does).
template <typename... P>
inline bool all_aligned_to(size_t n, P... p) {
  return (aligned_to(p, n) && ...);
}
inline bool valid_dtype(int d) { return d == SMM_DTYPE_F32 || d == SMM_DTYPE_BF16; }
inline size_t dtype_size(int d) { return d == SMM_DTYPE_F32 ? 4 : 2; }

}  // namespace smm
