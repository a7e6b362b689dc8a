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
// bf16 number 128 + code, and subtracting 128 + zero leaves code - zero, exactly (for zero
// points up to 127: 16 is common where a format keeps zero - 1 in four bits).
// x's pairs are picked in the same order from one 16-byte load.  So products are
// exact, and a group's sum is scaled in fp32 when the group's last product is
// done, which also keeps the tensor cores' truncating additions to one group.
// fp32 x is the exact sum of three bf16 numbers and takes three products.
//
// A CTA of 1024 threads (512 for more than eight rows of x) is four (two) teams of eight
// warps.  A team takes a tile of 16 rows of W, its warps the tile's columns in
// runs of U chunks of 32 V, and adds their sums through shared memory in a fixed
// order; then it takes its next tile.  x is laid out once per CTA in shared memory in the order
// that the products take it.  64 registers a thread leave little to prefetch with:
// the 32 warps' loads cover for one another.  8192 x 4096 with one row takes 9.3 us (1.2
// for the launch, 0.7 for x, 4.3 until the codes are there, then the unpacking),
// 8200 x 8192 with eight rows and zero points 19 us (with two sets of codes in turn 8.9 and 21.1
// where a set is one chunk, 10.6 and 23.3 where it is two).  Of the instances for fp32 x those of 1024
// threads spill (4 to 124 bytes a thread).
#include "smm_seq.cuh"

#include <algorithm>
#include <mutex>

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

__device__ __forceinline__ void mma_16816_zero(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

// The code pair (i, i+4) of a word as bf16 code - zero: off is the bf16 pair 128 + zero,
// whose bits are 0x4300 | zero.
__device__ __forceinline__ uint32_t code_pair(uint32_t w, int i, uint32_t off) {
  const uint32_t u = ((w >> (4 * i)) & 0x000F000Fu) | 0x43004300u;
  const __nv_bfloat162 v =
      __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), *reinterpret_cast<const __nv_bfloat162*>(&off));
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Pairs (x[i], x[i+4]), i = 0..3, of eight consecutive elements: kParts bf16
// terms whose sum is x exactly.
template <typename T>
struct XWord;
template <>
struct XWord<__nv_bfloat16> {
  static constexpr int kParts = 1;
  uint4 b[1];
  __device__ __forceinline__ void load(const __nv_bfloat16* p) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
    b[0] = make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                      __byte_perm(v.y, v.w, 0x7632));
  }
};
template <>
struct XWord<float> {
  static constexpr int kParts = 3;
  uint4 b[3];
  __device__ __forceinline__ void load(const float* p) {
    float v[8];
    load_f32<float, 8, true>(p, v);
#pragma unroll
    for (int part = 0; part < 3; ++part) {
      uint32_t hi[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        hi[i] = __float_as_uint(v[i]) & 0xFFFF0000u;  // 8 of the 24 significant bits, truncated
        // an infinity or NaN is all in its first term (a NaN may lie in the bits that were cut)
        if (part == 0 && v[i] != v[i]) hi[i] = 0x7FC00000u;
        v[i] = (hi[i] & 0x7F800000u) == 0x7F800000u ? 0.0f : v[i] - __uint_as_float(hi[i]);
      }
      b[part] = make_uint4(__byte_perm(hi[0], hi[4], 0x7632), __byte_perm(hi[1], hi[5], 0x7632),
                           __byte_perm(hi[2], hi[6], 0x7632), __byte_perm(hi[3], hi[7], 0x7632));
    }
  }
};

// V words of codes of rows g and g + 8 of up to four chunks.  Lane (g, t) holds the scales and
// zero points of chunk t alone, for the four lanes of its rows: a load by each for
// each chunk had touched three times the lines that the codes lie in.
template <int V>
constexpr int kRun = V == 4 ? 2 : 4;  // chunks fetched together: four of 16 bytes a lane spilled (10.3 and 9.3 us)

template <int V>
struct Codes {
  uint32_t wa[kRun<V>][V], wb[kRun<V>][V];
  uint32_t sa, sb;  // scales as loaded: an fp32 or, in the low half, a bf16
  uint32_t za, zb;
};
template <int V>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[V]) {
  if constexpr (V == 4) {
    const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p));
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (V == 2) {
    const uint2 v = __ldcs(reinterpret_cast<const uint2*>(p));
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = __ldcs(reinterpret_cast<const uint32_t*>(p));
  }
}

constexpr int kTeam = 8;                  // warps that share a tile
constexpr size_t kQ4XBytes = 192 * 1024;  // most of shared memory for x; the sums take up to 16 KB

// XS: x in shared memory (else, for rows of x too long for it, read beside the products)
template <typename T, int V, int NT, bool XS>
__global__ void __launch_bounds__(NT == 1 ? 1024 : 512, 1) q4_kernel(const Q4Params p, int nb) {
  constexpr int kTeams = (NT == 1 ? 1024 : 512) / (32 * kTeam);
  constexpr int kChunk = 32 * V, U = kRun<V>, kParts = XWord<T>::kParts;
  extern __shared__ uint4 q4_smem[];
  // x by words of 8 columns, in the order in which lanes (g, t) take them: [chunk][v][part][row of x][t]
  uint4* sx = q4_smem;
  const int words = p.cols / 8;
  // (from a shuffle, so that the compiler knows them, and all loops, to be the warp's)
  const int wid = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31, warp = wid % kTeam, team = wid / kTeam;
  float* red = reinterpret_cast<float*>(sx + (XS ? static_cast<size_t>(words) * kParts * nb : 0)) +
               team * (kTeam * NT * 128);  // [warp][NT][8][16]
  const int g = lane >> 2, t = lane & 3;
  const int b0 = blockIdx.y * nb;
  const int nx = p.batch - b0 < nb ? p.batch - b0 : nb;  // rows of x here
  const int tiles = (p.rows - 1) / 16 + 1;  // (rows + 15 may pass 31 bits)
  const int groups = p.cols / p.group;
  const int chunks = p.cols / kChunk;
  const int ratio = p.group / kChunk;  // chunks per group
  // this warp's chunks of every tile
  const int per_warp = (chunks + kTeam - 1) / kTeam;
  const int c_first = warp * per_warp, c_end = c_first + per_warp < chunks ? c_first + per_warp : chunks;

  // Columns of the product behind the last row of x are not stored: lanes there repeat the last row.
  const uint4* xs[NT];
  const T* xg[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int n = 8 * j + g < nx ? 8 * j + g : nx - 1;
    xs[j] = sx + n * 4 + t;
    xg[j] = static_cast<const T*>(p.x) + (b0 + n) * p.ldx + 8 * V * t;
  }

  Codes<V> k;
  const uint8_t *qa, *qb, *za, *zb;
  const char *sa, *sb;
  // a lane's rows of a tile, at this warp's first column
  auto seek = [&](int tile) {
    const int ra = tile * 16 + g < p.rows ? tile * 16 + g : p.rows - 1;
    const int rb = tile * 16 + g + 8 < p.rows ? tile * 16 + g + 8 : p.rows - 1;
    qa = p.q + static_cast<long long>(ra) * (p.cols / 2) + 4 * V * t;
    qb = p.q + static_cast<long long>(rb) * (p.cols / 2) + 4 * V * t;
    const long long ia = static_cast<long long>(ra) * groups, ib = static_cast<long long>(rb) * groups;
    sa = static_cast<const char*>(p.scales) + ia * (p.scale_f32 ? 4 : 2);
    sb = static_cast<const char*>(p.scales) + ib * (p.scale_f32 ? 4 : 2);
    za = p.zeros + ia;
    zb = p.zeros + ib;
  };
  auto fetch = [&](int c) {
    // scales first: the first chunk's sum wants them, the last chunk's codes are in no hurry
    const int ct = c + t < c_end ? c + t : c;
    const int gr = ratio == 1 ? ct : ct / ratio;
    if (p.scale_f32) {
      k.sa = __ldg(reinterpret_cast<const uint32_t*>(sa) + gr);
      k.sb = __ldg(reinterpret_cast<const uint32_t*>(sb) + gr);
    } else {
      k.sa = __ldg(reinterpret_cast<const unsigned short*>(sa) + gr);
      k.sb = __ldg(reinterpret_cast<const unsigned short*>(sb) + gr);
    }
    if (p.zeros) {
      k.za = __ldg(za + gr);
      k.zb = __ldg(zb + gr);
    }
    const uint8_t* a = qa + c * (kChunk / 2);
    const uint8_t* b = qb + c * (kChunk / 2);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c + u < c_end) {
        load_words<V>(a + u * (kChunk / 2), k.wa[u]);
        load_words<V>(b + u * (kChunk / 2), k.wb[u]);
      }
  };
  const int tstep = gridDim.x * kTeams;
  int tile = team * gridDim.x + blockIdx.x;
  if (tile < tiles) {
    seek(tile);
    if (c_first < c_end) fetch(c_first);
  }
  if constexpr (XS) {
    // over rows and words alike, so that four loads of a thread are in flight
    const int all = nx * words;
#pragma unroll 4
    for (int i = threadIdx.x; i < all; i += blockDim.x) {
      const int n = i / words, w = i - n * words;
      XWord<T> x;
      x.load(static_cast<const T*>(p.x) + (b0 + n) * p.ldx + 8 * w);
#pragma unroll
      for (int part = 0; part < kParts; ++part)
        sx[(((w / (4 * V) * V + w % V) * kParts + part) * nb + n) * 4 + w / V % 4] = x.b[part];
    }
    __syncthreads();
  }
  const int xstep = kParts * nb * 4;  // from one word to the next
  for (; tile < tiles; tile += tstep) {
    float tot[NT][4] = {};
    for (int c0 = c_first; c0 < c_end; c0 += U) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = c0 + u;
        if (c >= c_end) break;
        uint32_t oa = 0x43084308u, ob = 0x43084308u;
        if (p.zeros) {
          oa = 0x43004300u | ((__shfl_sync(0xFFFFFFFFu, k.za, u, 4) & 127u) * 0x10001u);
          ob = 0x43004300u | ((__shfl_sync(0xFFFFFFFFu, k.zb, u, 4) & 127u) * 0x10001u);
        }
        float acc[NT][4];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const uint32_t wa = k.wa[u][v], wb = k.wb[u][v];
          const uint32_t lo[4] = {code_pair(wa, 0, oa), code_pair(wb, 0, ob), code_pair(wa, 1, oa), code_pair(wb, 1, ob)};
          const uint32_t hi[4] = {code_pair(wa, 2, oa), code_pair(wb, 2, ob), code_pair(wa, 3, oa), code_pair(wb, 3, ob)};
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            XWord<T> x;
            if constexpr (XS) {
#pragma unroll
              for (int part = 0; part < kParts; ++part) x.b[part] = xs[j][(c * V + v) * xstep + part * nb * 4];
            } else {
              x.load(xg[j] + static_cast<long long>(c) * kChunk + 8 * v);
            }
#pragma unroll
            for (int part = kParts - 1; part >= 0; --part) {
              if (v == 0 && part == kParts - 1)
                mma_16816_zero(acc[j], lo, x.b[part].x, x.b[part].y);
              else
                mma_16816(acc[j], lo, x.b[part].x, x.b[part].y);
              mma_16816(acc[j], hi, x.b[part].z, x.b[part].w);
            }
          }
        }
        const uint32_t ua = __shfl_sync(0xFFFFFFFFu, k.sa, u, 4), ub = __shfl_sync(0xFFFFFFFFu, k.sb, u, 4);
        const float fa = __uint_as_float(p.scale_f32 ? ua : ua << 16);
        const float fb = __uint_as_float(p.scale_f32 ? ub : ub << 16);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          tot[j][0] = fmaf(fa, acc[j][0], tot[j][0]);
          tot[j][1] = fmaf(fa, acc[j][1], tot[j][1]);
          tot[j][2] = fmaf(fb, acc[j][2], tot[j][2]);
          tot[j][3] = fmaf(fb, acc[j][3], tot[j][3]);
        }
      }
      if (c0 + U < c_end) fetch(c0 + U);
    }
    if (tile + tstep < tiles) {
      seek(tile + tstep);
      if (c_first < c_end) fetch(c_first);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      float* o = red + (warp * NT + j) * 128;  // [column][row]
      o[(2 * t) * 16 + g] = tot[j][0];
      o[(2 * t + 1) * 16 + g] = tot[j][1];
      o[(2 * t) * 16 + g + 8] = tot[j][2];
      o[(2 * t + 1) * 16 + g + 8] = tot[j][3];
    }
    // a team's barrier: its number is the team's, its count the team's threads
    asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(32 * kTeam) : "memory");
    const int e = threadIdx.x % (32 * kTeam);
    if (e < NT * 128) {
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < kTeam; ++w) s += red[w * NT * 128 + e];
      const int n = e / 16, row = tile * 16 + e % 16;
      if (n < nx && row < p.rows) static_cast<T*>(p.y)[(b0 + n) * p.ldy + row] = from_f32<T>(s);
    }
    asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(32 * kTeam) : "memory");
  }
}

template <typename T, int V, int NT, bool XS>
int launch_q4(const Q4Params& p, int nb, cudaStream_t st) {
  auto kern = q4_kernel<T, V, NT, XS>;
  constexpr int kThreads = NT == 1 ? 1024 : 512, kTeams = kThreads / (32 * kTeam);
  constexpr size_t sums = kTeams * kTeam * NT * 128 * sizeof(float);
  const size_t smem = (XS ? static_cast<size_t>(p.cols) / 8 * XWord<T>::kParts * nb * sizeof(uint4) : 0) + sums;
  if constexpr (XS) {
    // The largest size, once: were it each call's own, another thread's smaller one could
    // take its place before this launch.
    static std::once_flag once[64];
    int dev = 0;
    SMM_CUDA_TRY(cudaGetDevice(&dev), "cudaGetDevice");
    cudaError_t err = cudaSuccess;
    auto set = [&] {
      err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kQ4XBytes + sums));
    };
    if (dev < 64) std::call_once(once[dev], set);
    else set();
    SMM_CUDA_TRY(err, "q4_matvec shared memory size");
  }
  const int tiles = (p.rows - 1) / 16 + 1;  // (rows + 15 may pass 31 bits)
  // One CTA an SM.  Few tiles are spread over the SMs, one to a CTA.
  const dim3 grid(std::min(tiles, 148), (p.batch + nb - 1) / nb);
  kern<<<grid, kThreads, smem, st>>>(p, nb);
  return SMM_OK;
}

template <typename T, int V>
int launch_q4_rows(const Q4Params& p, cudaStream_t st) {
  // up to 16 rows of x to a CTA, 8 where 16 do not fit, fewer of long rows
  const size_t row = static_cast<size_t>(p.cols) / 8 * XWord<T>::kParts * sizeof(uint4);
  if (p.batch > 8 && 16 * row <= kQ4XBytes) return launch_q4<T, V, 2, true>(p, std::min(p.batch, 16), st);
  const int fit = row ? static_cast<int>(std::min<size_t>(kQ4XBytes / row, 8)) : 8;
  if (fit >= 1) {
    // equal shares: 9 rows by at most 8 are 5 and 4
    const int parts = (p.batch + fit - 1) / fit;
    return launch_q4<T, V, 1, true>(p, (p.batch + parts - 1) / parts, st);
  }
  return launch_q4<T, V, 1, false>(p, 8, st);
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
  if (!aligned_to(y, e) || !aligned_to(scales, dtype_size(scale_dtype)))
    return set_error(SMM_ERR_INVALID, "smm_q4_matvec: a pointer is not aligned to its elements");
  const size_t groups = static_cast<size_t>(rows) * (cols / group);
  const Span ys = row_span(y, batch, rows, ldy, e);
  if (overlaps(ys, row_span(x, batch, cols, ldx, e)) || overlaps(ys, {q, static_cast<size_t>(rows) * (cols / 2)}) ||
      overlaps(ys, {scales, groups * dtype_size(scale_dtype)}) || overlaps(ys, {zeros, groups}))
    return set_error(SMM_ERR_INVALID, "smm_q4_matvec: y overlaps an input");
  if (!aligned_to(q, 16) || !aligned_to(x, 16) || (batch > 1 && ldx * e % 16 != 0))
    return set_error(SMM_ERR_INVALID, "smm_q4_matvec: q, x and x's rows must be 16-byte aligned");
  if (batch > 65535) return set_error(SMM_ERR_INVALID, "smm_q4_matvec: batch %d too large", batch);
  Q4Params p{static_cast<const uint8_t*>(q), scales, static_cast<const uint8_t*>(zeros), x, y, batch, rows, cols,
             group, scale_dtype == SMM_DTYPE_F32, ldx, ldy};
  cudaStream_t st = as_stream(stream);
  // the widest load whose columns lie in one group
  const int v = group % 128 == 0 ? 4 : group % 64 == 0 ? 2 : 1;
  int rc;
  if (dtype == SMM_DTYPE_F32)
    rc = v == 4   ? launch_q4_rows<float, 4>(p, st)
         : v == 2 ? launch_q4_rows<float, 2>(p, st)
                  : launch_q4_rows<float, 1>(p, st);
  else
    rc = v == 4   ? launch_q4_rows<__nv_bfloat16, 4>(p, st)
         : v == 2 ? launch_q4_rows<__nv_bfloat16, 2>(p, st)
                  : launch_q4_rows<__nv_bfloat16, 1>(p, st);
  if (rc) return rc;
  count_launch();
  SMM_CUDA_TRY(cudaGetLastError(), "q4_matvec launch");
  return SMM_OK;
}
