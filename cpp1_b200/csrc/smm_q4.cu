// y = x W^T for a few rows x and a matrix W held in 4 bits with group scales
// (and zero points): W[r][k] = (code[r][k] - zero[r][k/group]) scale[r][k/group].
//
// Bound by reading the codes once (half a byte per two operations and row of
// x).  To leave the issue slots to that, the products run on the tensor
// cores through mma.sync m16n8k16 with W as the 16-row operand and up to eight
// rows of x as the 8-column one: at 8 columns the tensor cores' 5th-generation
// tiles (128 rows, operands staged in shared memory) would add a trip through
// shared memory and save nothing, as the matrix pipe is far from busy.
//
// The order of k inside a product is free as long as both operands agree.  Lane
// (g, t) of a warp loads 4 V bytes of rows g and g+8 at k = 8 V t: V words of
// eight codes with consecutive k.  Masking a word and its shifts by 4, 8 and 12
// bits yields the code pairs (0,4), (1,5), (2,6), (3,7); OR 0x4300 makes each the
// bf16 number 128 + code, and subtracting 128 + zero leaves code - zero, exactly.
// x's pairs are picked in the same order from one 16-byte load.  So products are
// exact, and a group's sum is scaled in fp32 when the group's last product is
// done, which also keeps the tensor cores' truncating additions to one group.
// fp32 x is the exact sum of three bf16 numbers and takes three products.
//
// The warps of a CTA share 16 rows and take chunks of 32 V columns in turn; their
// sums are added through shared memory in a fixed order.
#include "smm_seq.cuh"

#include <algorithm>

namespace smm {
namespace {

struct Q4Params {
  const uint8_t* q;
  const void* scales;
  const uint8_t* zeros;
  const void* x;
  void* y;
  int batch, rows, cols, group, scale_f32;
  long long ldx, ldy;
};

__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The code pair (i, i+4) of a word, as bf16 code - zero (off = 128 + zero twice).
__device__ __forceinline__ uint32_t code_pair(uint32_t w, int i, __nv_bfloat162 off) {
  const uint32_t u = ((w >> (4 * i)) & 0x000F000Fu) | 0x43004300u;
  const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), off);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Pairs (x[i], x[i+4]), i = 0..3, of eight consecutive elements: PARTS bf16
// terms whose sum is x exactly.
template <typename T>
struct XWord;
template <>
struct XWord<__nv_bfloat16> {
  static constexpr int kParts = 1;
  uint32_t b[1][4];
  __device__ __forceinline__ void load(const __nv_bfloat16* p, bool ok) {
    const uint4 v = ok ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
    b[0][0] = __byte_perm(v.x, v.z, 0x5410);
    b[0][1] = __byte_perm(v.x, v.z, 0x7632);
    b[0][2] = __byte_perm(v.y, v.w, 0x5410);
    b[0][3] = __byte_perm(v.y, v.w, 0x7632);
  }
};
template <>
struct XWord<float> {
  static constexpr int kParts = 3;
  uint32_t b[3][4];
  __device__ __forceinline__ void load(const float* p, bool ok) {
    float v[8];
    if (ok) {
      load_f32<float, 8, true>(p, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    }
#pragma unroll
    for (int part = 0; part < 3; ++part) {
      uint32_t hi[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        hi[i] = __float_as_uint(v[i]) & 0xFFFF0000u;  // 8 of the 24 significant bits, truncated
        // an infinity or NaN is all in its first term
        v[i] = (hi[i] & 0x7F800000u) == 0x7F800000u ? 0.0f : v[i] - __uint_as_float(hi[i]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) b[part][i] = __byte_perm(hi[i], hi[i + 4], 0x7632);
    }
  }
};

template <int V>
struct Words {
  uint32_t w[V];
  __device__ __forceinline__ void load(const uint8_t* p) {
    if constexpr (V == 4) {
      const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p));
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (V == 2) {
      const uint2 v = __ldcs(reinterpret_cast<const uint2*>(p));
      w[0] = v.x, w[1] = v.y;
    } else {
      w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
    }
  }
};

template <typename T, int V, int NT>
__global__ void __launch_bounds__(512) q4_kernel(const Q4Params p) {
  constexpr int kChunk = 32 * V;
  constexpr int U = V == 4 ? 2 : 4;  // chunks in flight per warp
  extern __shared__ float red[];     // [warp][NT][16][8]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int r0 = blockIdx.x * 16;
  const int ra = r0 + g < p.rows ? r0 + g : p.rows - 1;
  const int rb = r0 + g + 8 < p.rows ? r0 + g + 8 : p.rows - 1;
  const int b0 = blockIdx.y * 8 * NT;
  const int groups = p.cols / p.group;
  const uint8_t* qa = p.q + static_cast<long long>(ra) * (p.cols / 2) + 4 * V * t;
  const uint8_t* qb = p.q + static_cast<long long>(rb) * (p.cols / 2) + 4 * V * t;
  const T* xp[NT];
  bool xok[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int n = b0 + 8 * j + g;
    xok[j] = n < p.batch;
    xp[j] = static_cast<const T*>(p.x) + (xok[j] ? n : 0) * p.ldx + 8 * V * t;
  }
  auto scale_at = [&](long long i) {
    return p.scale_f32 ? __ldg(static_cast<const float*>(p.scales) + i)
                       : to_f32(static_cast<const __nv_bfloat16*>(p.scales)[i]);
  };
  float tot[NT][4] = {};
  const int chunks = p.cols / kChunk;
  for (int c0 = warp; c0 < chunks; c0 += U * warps) {
    Words<V> wa[U], wb[U];
    float sa[U], sb[U];
    __nv_bfloat162 oa[U], ob[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + u * warps;
      if (c < chunks) {
        wa[u].load(qa + static_cast<long long>(c) * (kChunk / 2));
        wb[u].load(qb + static_cast<long long>(c) * (kChunk / 2));
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + u * warps;
      if (c < chunks) {
        const int gr = c * kChunk / p.group;
        const long long ia = static_cast<long long>(ra) * groups + gr, ib = static_cast<long long>(rb) * groups + gr;
        sa[u] = scale_at(ia);
        sb[u] = scale_at(ib);
        oa[u] = __float2bfloat162_rn(128.0f + (p.zeros ? p.zeros[ia] & 15 : 8));
        ob[u] = __float2bfloat162_rn(128.0f + (p.zeros ? p.zeros[ib] & 15 : 8));
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + u * warps;
      if (c >= chunks) break;
      float acc[NT][4] = {};
#pragma unroll
      for (int v = 0; v < V; ++v) {
        uint32_t lo[4], hi[4];
        lo[0] = code_pair(wa[u].w[v], 0, oa[u]);
        lo[1] = code_pair(wb[u].w[v], 0, ob[u]);
        lo[2] = code_pair(wa[u].w[v], 1, oa[u]);
        lo[3] = code_pair(wb[u].w[v], 1, ob[u]);
        hi[0] = code_pair(wa[u].w[v], 2, oa[u]);
        hi[1] = code_pair(wb[u].w[v], 2, ob[u]);
        hi[2] = code_pair(wa[u].w[v], 3, oa[u]);
        hi[3] = code_pair(wb[u].w[v], 3, ob[u]);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          XWord<T> x;
          x.load(xp[j] + static_cast<long long>(c) * kChunk + 8 * v, xok[j]);
#pragma unroll
          for (int part = XWord<T>::kParts - 1; part >= 0; --part) {
            mma_16816(acc[j], lo, x.b[part][0], x.b[part][1]);
            mma_16816(acc[j], hi, x.b[part][2], x.b[part][3]);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        tot[j][0] = fmaf(sa[u], acc[j][0], tot[j][0]);
        tot[j][1] = fmaf(sa[u], acc[j][1], tot[j][1]);
        tot[j][2] = fmaf(sb[u], acc[j][2], tot[j][2]);
        tot[j][3] = fmaf(sb[u], acc[j][3], tot[j][3]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    float* o = red + (warp * NT + j) * 128;  // [column][row]
    o[(2 * t) * 16 + g] = tot[j][0];
    o[(2 * t + 1) * 16 + g] = tot[j][1];
    o[(2 * t) * 16 + g + 8] = tot[j][2];
    o[(2 * t + 1) * 16 + g + 8] = tot[j][3];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < NT * 128; e += blockDim.x) {
    float s = 0.0f;
    for (int w = 0; w < warps; ++w) s += red[w * NT * 128 + e];
    const int n = b0 + e / 16, r = r0 + e % 16;
    if (n < p.batch && r < p.rows) static_cast<T*>(p.y)[n * p.ldy + r] = from_f32<T>(s);
  }
}

template <typename T, int V>
void launch_q4(const Q4Params& p, int warps, cudaStream_t st) {
  const unsigned gx = (p.rows + 15) / 16;
  auto go = [&](auto nt) {
    constexpr int NT = decltype(nt)::value;
    q4_kernel<T, V, NT><<<dim3(gx, (p.batch + 8 * NT - 1) / (8 * NT)), warps * 32, warps * NT * 512, st>>>(p);
  };
  if (p.batch <= 8) return go(std::integral_constant<int, 1>{});
  if (p.batch <= 16) return go(std::integral_constant<int, 2>{});
  go(std::integral_constant<int, 4>{});
}

}  // namespace
}  // namespace smm

using namespace smm;

extern "C" int smm_q4_matvec(const void* q, const void* scales, const void* zeros, const void* x, void* y, int batch,
                             int rows, int cols, int group, long long ldx, long long ldy, int dtype, int scale_dtype,
                             void* stream) {
  SMM_RANGE("smm_q4_matvec");
  if (batch < 0 || rows < 0 || cols < 0) return set_error(SMM_ERR_INVALID, "smm_q4_matvec: negative shape");
  if (group < 32 || group % 32 != 0 || cols % group != 0)
    return set_error(SMM_ERR_INVALID, "smm_q4_matvec: group %d is not a multiple of 32 that divides %d columns", group,
                     cols);
  if (!valid_dtype(dtype) || !valid_dtype(scale_dtype))
    return set_error(SMM_ERR_INVALID, "smm_q4_matvec: unknown element type %d or %d", dtype, scale_dtype);
  if (ldx < cols || ldy < rows) return set_error(SMM_ERR_INVALID, "smm_q4_matvec: row stride shorter than a row");
  if (batch == 0 || rows == 0) return SMM_OK;
  if (!y || (cols > 0 && (!q || !scales || !x))) return set_error(SMM_ERR_INVALID, "smm_q4_matvec: null pointer");
  const size_t e = dtype_size(dtype);
  const size_t groups = static_cast<size_t>(rows) * (cols / group);
  const Span ys{y, span_bytes(batch, rows, ldy, e)};
  if (overlaps(ys, {x, span_bytes(batch, cols, ldx, e)}) || overlaps(ys, {q, static_cast<size_t>(rows) * (cols / 2)}) ||
      overlaps(ys, {scales, groups * dtype_size(scale_dtype)}) || overlaps(ys, {zeros, groups}))
    return set_error(SMM_ERR_INVALID, "smm_q4_matvec: y overlaps an input");
  if (!aligned_to(q, 16) || !aligned_to(x, 16) || (batch > 1 && ldx * e % 16 != 0))
    return set_error(SMM_ERR_INVALID, "smm_q4_matvec: q, x and x's rows must be 16-byte aligned");
  if (batch > 65535 * 32) return set_error(SMM_ERR_INVALID, "smm_q4_matvec: batch %d too large", batch);
  Q4Params p{static_cast<const uint8_t*>(q), scales, static_cast<const uint8_t*>(zeros), x, y, batch, rows, cols,
             group, scale_dtype == SMM_DTYPE_F32, ldx, ldy};
  const int warps = 8;
  cudaStream_t st = as_stream(stream);
  const int v = group % 128 == 0 ? 4 : group % 64 == 0 ? 2 : 1;
  if (dtype == SMM_DTYPE_F32) {
    if (v == 4) launch_q4<float, 4>(p, warps, st);
    else if (v == 2) launch_q4<float, 2>(p, warps, st);
    else launch_q4<float, 1>(p, warps, st);
  } else {
    if (v == 4) launch_q4<__nv_bfloat16, 4>(p, warps, st);
    else if (v == 2) launch_q4<__nv_bfloat16, 2>(p, warps, st);
    else launch_q4<__nv_bfloat16, 1>(p, warps, st);
  }
  count_launch();
  SMM_CUDA_TRY(cudaGetLastError(), "q4_matvec launch");
  return SMM_OK;
}
