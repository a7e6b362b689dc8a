// Selective state space scan (per head a lower-triangular semiseparable
// matrix times x): the recurrence on the fp32 pipes for prompts, the
// single-token step, and the C entries.
#include "smm_scan.cuh"

#include <algorithm>
#include <type_traits>

namespace smm {
namespace {

using F2 = unsigned long long;  // two fp32 lanes

// ------------------------------------------------------------ prompts
// The recurrence itself, for fp32 elements (whose accuracy bf16 products do
// not reach) and for shapes the tensor-core kernel does not take.  Three
// packed multiply-adds per two state elements and token; bound by their issue.
//
// A CTA holds the states of one head and 8 dims per warp in registers: lane
// (pg, ng) has 2 dims x NPL state elements, in 16-byte pieces strided by the 8
// lanes ng so that reading B and C from shared memory has no bank conflict and
// each value serves four lanes.  Tokens pass in tiles of 16: the next tile's B, C,
// x, z and dt are loaded into registers while the present one is computed, four
// tokens at a time, whose eight sums over the lanes ng are made together.  (Token by
// token, the chain of one token's sum and its shuffles showed: 4096 tokens of 64
// heads of 64 x 128 took 1.21 ms.)
constexpr int kTile = 16;

template <typename T, int NPL, int THREADS, bool STATES>
__global__ void __launch_bounds__(THREADS) scan_kernel(const ScanParams p, int ptiles) {
  constexpr int NP = 8 * NPL;                  // padded state_dim
  constexpr int PT = THREADS / 4;              // dims per CTA
  constexpr int NE = kTile * NP / THREADS > 0 ? kTile * NP / THREADS : 1;
  constexpr int XE = kTile * PT / THREADS;     // 4
  constexpr int CH = NPL >= 4 ? 4 : 2;         // consecutive state elements of a lane
  constexpr int NC = NPL / CH;
  extern __shared__ float sm[];
  float* sB = sm;                              // [kTile][NP]
  float* sC = sB + kTile * NP;
  float* sx = sC + (STATES ? 0 : kTile * NP);  // [kTile][PT]
  float* sy = sx + kTile * PT;
  float2* sad = reinterpret_cast<float2*>(sy + (STATES ? 0 : kTile * PT));  // decay, d
  __shared__ Segment sseg;

  const int pt = static_cast<int>(blockIdx.x % ptiles);
  const int hs = static_cast<int>(blockIdx.x / ptiles);
  const int h = hs % p.heads, seg = hs / p.heads;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int ng = lane & 7, pg = lane >> 3;
  if (warp == 0) {
    const Segment s = find_segment(p, seg);
    if (lane == 0) sseg = s;
  }
  __syncthreads();
  const Segment sg = sseg;
  if (!sg.valid) return;
  const int g = h / (p.heads / p.groups);
  const int p0 = pt * PT;
  const int pl = p0 + warp * 8 + pg * 2;       // this lane's first dim
  const int N = p.state_dim;
  const float A = __ldg(p.A + h);
  const bool last = sg.j == sg.count - 1;
  const int slot = (p.state_in || p.state_out) ? seq_slot(p.slots, sg.seq, p.nslots, p.status) : -1;

  auto n_of = [&](int c, int i) { return c * 8 * CH + ng * CH + i; };
  auto state_at = [&](int pp, int n) {
    return (static_cast<long long>(h) * p.dim + pl + pp) * N + n;
  };
  const long long per_slot = static_cast<long long>(p.heads) * p.dim * N;

  // state before the segment
  float hv[2][NPL];
#pragma unroll
  for (int pp = 0; pp < 2; ++pp)
#pragma unroll
    for (int i = 0; i < NPL; ++i) hv[pp][i] = 0.0f;
  auto add_state = [&](const float* src, float decay) {
#pragma unroll
    for (int pp = 0; pp < 2; ++pp)
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        const int n = n_of(i / CH, i % CH);
        if (pl + pp < p.dim && n < N) hv[pp][i] = fmaf(hv[pp][i], decay, src[state_at(pp, n)]);
      }
  };
  auto put_state = [&](float* dst) {
#pragma unroll
    for (int pp = 0; pp < 2; ++pp)
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        const int n = n_of(i / CH, i % CH);
        if (pl + pp < p.dim && n < N) dst[state_at(pp, n)] = hv[pp][i];
      }
  };
  const float* in = p.state_in && slot >= 0 ? p.state_in + slot * per_slot : nullptr;
  if constexpr (STATES) {
    // The last segment's place keeps the state the sequence started from: the
    // second launch may overwrite it while other segments still need it.
    if (last) {
      if (sg.count > 1) {
        if (in) add_state(in, 0.0f);
        put_state(p.seg_state + seg * per_slot);
      }
      return;
    }
  } else if (sg.count == 1) {
    if (in) add_state(in, 0.0f);
  } else {
    add_state(p.seg_state + (sg.first + sg.count - 1) * per_slot, 0.0f);
    for (int k = 0; k < sg.j; ++k)
      add_state(p.seg_state + (sg.first + k) * per_slot,
                expf(p.seg_log[static_cast<long long>(sg.first + k) * p.heads + h]));
  }
  F2 hst[2][NPL / 2];
#pragma unroll
  for (int pp = 0; pp < 2; ++pp)
#pragma unroll
    for (int i = 0; i < NPL / 2; ++i) hst[pp][i] = pack2(hv[pp][2 * i], hv[pp][2 * i + 1]);

  const T* gB = static_cast<const T*>(p.B) + static_cast<long long>(g) * N;
  const T* gC = static_cast<const T*>(p.C) + static_cast<long long>(g) * N;
  const T* gx = static_cast<const T*>(p.x) + static_cast<long long>(h) * p.dim + p0;
  const T* gz = p.z ? static_cast<const T*>(p.z) + static_cast<long long>(h) * p.dim + p0 : nullptr;
  // elements as loaded: nothing waits for them before stage() widens them
  T rB[NE], rC[NE], rx[XE], rz[XE], cx[XE], cz[XE];
  uint32_t rd = 0;
  float la = 0.0f;
  const float bias = p.dt_bias ? __ldg(p.dt_bias + h) : 0.0f;
  const T zero = from_f32<T>(0.0f);
  const int pdims = p.dim - p0 < PT ? p.dim - p0 : PT;
  auto fetch = [&](long long t0) {
    const int nt = sg.end - t0 < kTile ? static_cast<int>(sg.end - t0) : kTile;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const int e = tid + i * THREADS, t = e / NP, n = e % NP;
      const bool ok = t < nt && n < N;
      rB[i] = ok ? gB[(t0 + t) * p.ldb + n] : zero;
      if constexpr (!STATES) rC[i] = ok ? gC[(t0 + t) * p.ldc + n] : zero;
    }
#pragma unroll
    for (int i = 0; i < XE; ++i) {
      const int e = tid + i * THREADS, t = e / PT, q = e % PT;
      const bool ok = t < nt && q < pdims;
      rx[i] = ok ? gx[(t0 + t) * p.ldx + q] : zero;
      if constexpr (!STATES) rz[i] = ok && gz ? gz[(t0 + t) * p.ldz + q] : zero;
    }
    if (tid < nt) rd = scan_dt_raw(p, t0 + tid, h);
  };
  auto stage = [&](int nt) {
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const int e = tid + i * THREADS;
      if (e < kTile * NP) {
        sB[e] = to_f32(rB[i]);
        if constexpr (!STATES) sC[e] = to_f32(rC[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < XE; ++i) {
      sx[tid + i * THREADS] = to_f32(rx[i]);
      cx[i] = rx[i];
      if constexpr (!STATES) cz[i] = rz[i];
    }
    if (tid < kTile) {
      const float d = tid < nt ? scan_dt(p, rd, bias) : 0.0f;
      sad[tid] = tid < nt ? make_float2(expf(d * A), d) : make_float2(1.0f, 0.0f);
      la += d * A;
    }
  };

  const float Dh = p.D ? __ldg(p.D + h) : 0.0f;
  T* gy = static_cast<T*>(p.y) + static_cast<long long>(h) * p.dim + p0;
  if (sg.begin < sg.end) {
    fetch(sg.begin);
    stage(sg.end - sg.begin < kTile ? static_cast<int>(sg.end - sg.begin) : kTile);
  }
  __syncthreads();
  for (long long t0 = sg.begin; t0 < sg.end; t0 += kTile) {
    const int nt = sg.end - t0 < kTile ? static_cast<int>(sg.end - t0) : kTile;
    const bool more = t0 + kTile < sg.end;
    if (more) fetch(t0 + kTile);
#pragma unroll 1
    for (int t = 0; t < nt; t += 4) {  // tokens behind the last one do nothing: decay 1, d 0
      float ys[8];                     // [token][dim]
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float2 ad = sad[t + u];
        const float2 xv = *reinterpret_cast<const float2*>(sx + (t + u) * PT + warp * 8 + pg * 2);
        const F2 a2 = pack2(ad.x, ad.x);
        const F2 d0 = pack2(xv.x * ad.y, xv.x * ad.y), d1 = pack2(xv.y * ad.y, xv.y * ad.y);
        F2 y0 = pack2(0.0f, 0.0f), y1 = y0;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          F2 b[CH / 2], cc[CH / 2];
          if constexpr (CH == 4) {
            *reinterpret_cast<float4*>(b) = *reinterpret_cast<const float4*>(sB + (t + u) * NP + n_of(c, 0));
            if constexpr (!STATES)
              *reinterpret_cast<float4*>(cc) = *reinterpret_cast<const float4*>(sC + (t + u) * NP + n_of(c, 0));
          } else {
            b[0] = *reinterpret_cast<const F2*>(sB + (t + u) * NP + n_of(c, 0));
            if constexpr (!STATES) cc[0] = *reinterpret_cast<const F2*>(sC + (t + u) * NP + n_of(c, 0));
          }
#pragma unroll
          for (int q = 0; q < CH / 2; ++q) {
            const int k = c * (CH / 2) + q;
            hst[0][k] = fma2(hst[0][k], a2, mul2(d0, b[q]));
            hst[1][k] = fma2(hst[1][k], a2, mul2(d1, b[q]));
            if constexpr (!STATES) {
              y0 = fma2(hst[0][k], cc[q], y0);
              y1 = fma2(hst[1][k], cc[q], y1);
            }
          }
        }
        float lo, hi;
        unpack2(y0, lo, hi);
        ys[2 * u] = lo + hi;
        unpack2(y1, lo, hi);
        ys[2 * u + 1] = lo + hi;
      }
      if constexpr (!STATES) {
        // sums over the 8 lanes ng, of which lane ng keeps the one of token ng / 2, dim ng % 2
        float s4[4], s2[2];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          s4[i] = ((ng & 4) ? ys[4 + i] : ys[i]) + __shfl_xor_sync(0xFFFFFFFFu, (ng & 4) ? ys[i] : ys[4 + i], 4);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          s2[i] = ((ng & 2) ? s4[2 + i] : s4[i]) + __shfl_xor_sync(0xFFFFFFFFu, (ng & 2) ? s4[i] : s4[2 + i], 2);
        const float sum = ((ng & 1) ? s2[1] : s2[0]) + __shfl_xor_sync(0xFFFFFFFFu, (ng & 1) ? s2[0] : s2[1], 1);
        sy[(t + (ng >> 1)) * PT + warp * 8 + pg * 2 + (ng & 1)] = sum;
      }
    }
    __syncthreads();
    if constexpr (!STATES) {
#pragma unroll
      for (int i = 0; i < XE; ++i) {
        const int e = tid + i * THREADS, t = e / PT, q = e % PT;
        if (t < nt && q < pdims) {
          float v = fmaf(Dh, to_f32(cx[i]), sy[e]);
          if (gz) v *= silu(to_f32(cz[i]));
          gy[(t0 + t) * p.ldy + q] = from_f32<T>(v);
        }
      }
    }
    if (more) {
      const long long left = sg.end - t0 - kTile;
      stage(left < kTile ? static_cast<int>(left) : kTile);
    }
    __syncthreads();
  }
#pragma unroll
  for (int pp = 0; pp < 2; ++pp)
#pragma unroll
    for (int i = 0; i < NPL / 2; ++i) unpack2(hst[pp][i], hv[pp][2 * i], hv[pp][2 * i + 1]);
  if constexpr (STATES) {
    put_state(p.seg_state + seg * per_slot);
    if (warp == 0 && pt == 0) {
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) la += __shfl_down_sync(0xFFFFFFFFu, la, o);
      if (lane == 0) p.seg_log[static_cast<long long>(seg) * p.heads + h] = la;
    }
  } else if (last && p.state_out && slot >= 0) {
    put_state(p.state_out + slot * per_slot);
  }
}

template <typename T, int NPL, int THREADS>
int launch_scan(const ScanParams& p, long long segs, cudaStream_t st) {
  constexpr int NP = 8 * NPL, PT = THREADS / 4;
  const int ptiles = (p.dim + PT - 1) / PT;
  const long long blocks = segs * p.heads * ptiles;
  if (blocks > 0x7FFFFFFFLL) return set_error(SMM_ERR_INVALID, "selective scan too large for one launch");
  const unsigned grid = static_cast<unsigned>(blocks);
  const size_t full = sizeof(float) * kTile * (2 * NP + 2 * PT + 2);
  if (p.split) {
    scan_kernel<T, NPL, THREADS, true><<<grid, THREADS, full, st>>>(p, ptiles);
    count_launch();
  }
  scan_kernel<T, NPL, THREADS, false><<<grid, THREADS, full, st>>>(p, ptiles);
  count_launch();
  SMM_CUDA_TRY(cudaGetLastError(), "selective scan launch");
  return SMM_OK;
}

template <typename T>
int launch_scan_type(const ScanParams& p, long long segs, cudaStream_t st) {
  auto go = [&](auto npl) {
    constexpr int NPL = decltype(npl)::value;
    // 32 dims to a CTA where 64 would leave SMs without one (or a head has no more)
    const bool small = p.dim <= 32 || segs * p.heads * ((p.dim + 63) / 64) < 2 * 148;
    return small ? launch_scan<T, NPL, 128>(p, segs, st) : launch_scan<T, NPL, 256>(p, segs, st);
  };
  if (p.state_dim <= 16) return go(std::integral_constant<int, 2>{});
  if (p.state_dim <= 32) return go(std::integral_constant<int, 4>{});
  if (p.state_dim <= 64) return go(std::integral_constant<int, 8>{});
  if (p.state_dim <= 128) return go(std::integral_constant<int, 16>{});
  return go(std::integral_constant<int, 32>{});
}

// ------------------------------------------------------------ one token
// S = exp(d A) S + d x (outer) B, y = S C: the state is read once and written
// once (8 bytes per element against 5 operations), which bounds it.  A warp takes
// whole rows of the state (16 bytes per lane; several rows side by side where
// state_dim is short), four at a time so that their loads are in flight
// together, before anything that depends on dt is computed.
constexpr int kStepThreads = 128;
constexpr int kStepRows = 4;  // rows in flight per lane

template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(kStepThreads) step_kernel(const ScanParams p, int lanes, int rows_per_cta,
                                                            int ptiles) {
  const int pt = static_cast<int>(blockIdx.x % ptiles);
  const int hb = static_cast<int>(blockIdx.x / ptiles);
  const int h = hb % p.heads, b = hb / p.heads;
  const int g = h / (p.heads / p.groups);
  const int N = p.state_dim;
  const int sub = threadIdx.x % lanes, row0 = threadIdx.x / lanes, rstep = kStepThreads / lanes;
  const int slot = seq_slot(p.slots, b, p.nslots, p.status);
  const long long base = (static_cast<long long>(slot) * p.heads + h) * p.dim * N;
  const float* in = p.state_in && slot >= 0 ? p.state_in + base : nullptr;
  float* out = p.state_out && slot >= 0 ? p.state_out + base : nullptr;
  const int pend = (pt + 1) * rows_per_cta < p.dim ? (pt + 1) * rows_per_cta : p.dim;

  float hv[kStepRows][NV][VEC], xv[kStepRows], bv[NV][VEC], cv[NV][VEC];
  auto load_rows = [&](int r0) {
#pragma unroll
    for (int r = 0; r < kStepRows; ++r) {
      const int q = r0 + r * rstep;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int n = (k * lanes + sub) * VEC;
        if (in && q < pend && n < N) {
          if constexpr (VEC == 4) {
            const float4 f = __ldcs(reinterpret_cast<const float4*>(in + static_cast<long long>(q) * N + n));
            hv[r][k][0] = f.x, hv[r][k][1] = f.y, hv[r][k][2] = f.z, hv[r][k][3] = f.w;
          } else {
            hv[r][k][0] = in[static_cast<long long>(q) * N + n];
          }
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i) hv[r][k][i] = 0.0f;
        }
      }
    }
#pragma unroll
    for (int r = 0; r < kStepRows; ++r) {
      const int q = r0 + r * rstep;
      xv[r] = q < pend ? to_f32(static_cast<const T*>(p.x)[b * p.ldx + static_cast<long long>(h) * p.dim + q]) : 0.0f;
    }
  };
  load_rows(pt * rows_per_cta + row0);
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int n = (k * lanes + sub) * VEC + i;
      bv[k][i] = n < N ? to_f32(static_cast<const T*>(p.B)[b * p.ldb + static_cast<long long>(g) * N + n]) : 0.0f;
      cv[k][i] = n < N ? to_f32(static_cast<const T*>(p.C)[b * p.ldc + static_cast<long long>(g) * N + n]) : 0.0f;
    }
  const float d = scan_dt(p, scan_dt_raw(p, b, h), p.dt_bias ? __ldg(p.dt_bias + h) : 0.0f);
  const float a = expf(d * __ldg(p.A + h));
  const float Dh = p.D ? __ldg(p.D + h) : 0.0f;
  // every thread of the CTA makes the same number of turns (the shuffles)
  for (int base_row = pt * rows_per_cta; base_row < pend; base_row += kStepRows * rstep) {
    if (base_row != pt * rows_per_cta) load_rows(base_row + row0);
#pragma unroll
    for (int r = 0; r < kStepRows; ++r) {
      const int q = base_row + row0 + r * rstep;
      const float dx = d * xv[r];
      float y = 0.0f;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          hv[r][k][i] = fmaf(hv[r][k][i], a, dx * bv[k][i]);
          y = fmaf(hv[r][k][i], cv[k][i], y);
        }
        const int n = (k * lanes + sub) * VEC;
        if (out && q < pend && n < N) {
          if constexpr (VEC == 4)
            __stcs(reinterpret_cast<float4*>(out + static_cast<long long>(q) * N + n),
                   make_float4(hv[r][k][0], hv[r][k][1], hv[r][k][2], hv[r][k][3]));
          else
            out[static_cast<long long>(q) * N + n] = hv[r][k][0];
        }
      }
      for (int o = lanes >> 1; o > 0; o >>= 1) y += __shfl_xor_sync(0xFFFFFFFFu, y, o);
      if (sub == 0 && q < pend) {
        y = fmaf(Dh, xv[r], y);
        const long long col = static_cast<long long>(h) * p.dim + q;
        if (p.z) y *= silu(to_f32(static_cast<const T*>(p.z)[b * p.ldz + col]));
        static_cast<T*>(p.y)[b * p.ldy + col] = from_f32<T>(y);
      }
    }
  }
}

template <typename T>
int launch_step(const ScanParams& p, int batch, cudaStream_t st) {
  const bool vec = p.state_dim % 4 == 0 && aligned_to(p.state_in, 16) && aligned_to(p.state_out, 16);
  const int pieces = vec ? p.state_dim / 4 : p.state_dim;
  int lanes = 1;
  while (lanes < 32 && lanes < pieces) lanes *= 2;
  const int nv = (pieces + lanes - 1) / lanes;
  // one round of rows per CTA: the most CTAs, and the shortest wait for one token
  const int rows = kStepRows * kStepThreads / lanes;
  const int ptiles = (p.dim + rows - 1) / rows;
  const long long blocks = static_cast<long long>(batch) * p.heads * ptiles;
  if (blocks > 0x7FFFFFFFLL) return set_error(SMM_ERR_INVALID, "selective step too large for one launch");
  const unsigned grid = static_cast<unsigned>(blocks);
  if (vec && nv == 1)
    step_kernel<T, 4, 1><<<grid, kStepThreads, 0, st>>>(p, lanes, rows, ptiles);
  else if (vec)
    step_kernel<T, 4, 2><<<grid, kStepThreads, 0, st>>>(p, lanes, rows, ptiles);
  else if (nv == 1)
    step_kernel<T, 1, 1><<<grid, kStepThreads, 0, st>>>(p, lanes, rows, ptiles);
  else
    step_kernel<T, 1, 8><<<grid, kStepThreads, 0, st>>>(p, lanes, rows, ptiles);
  count_launch();
  SMM_CUDA_TRY(cudaGetLastError(), "selective step launch");
  return SMM_OK;
}

// ------------------------------------------------------------ checks
int check_scan(const char* who, const ScanParams& p, int dtype, int dt_dtype, bool step) {
  if (p.tokens < 0 || p.nseq < 0 || p.nslots < 0 || p.heads < 0)
    return set_error(SMM_ERR_INVALID, "%s: negative size", who);
  if (p.tokens > 0x7FFFFFFFLL) return set_error(SMM_ERR_INVALID, "%s: %lld tokens exceed 31 bits", who, p.tokens);
  if (p.dim < 1 || p.dim > 256 || p.state_dim < 1 || p.state_dim > 256)
    return set_error(SMM_ERR_INVALID, "%s: dim %d or state_dim %d is not in 1..256", who, p.dim, p.state_dim);
  if (p.groups < 1 || p.heads % p.groups != 0)
    return set_error(SMM_ERR_INVALID, "%s: %d heads do not divide into %d groups", who, p.heads, p.groups);
  if (!valid_dtype(dtype) || !valid_dtype(dt_dtype))
    return set_error(SMM_ERR_INVALID, "%s: unknown element type %d or %d", who, dtype, dt_dtype);
  const long long hp = static_cast<long long>(p.heads) * p.dim, gn = static_cast<long long>(p.groups) * p.state_dim;
  if (hp * p.state_dim > 0x7FFFFFFFLL)
    return set_error(SMM_ERR_INVALID, "%s: one state of %lld elements exceeds 31 bits", who, hp * p.state_dim);
  if (p.ldx < hp || p.ldy < hp || (p.z && p.ldz < hp) || p.ldb < gn || p.ldc < gn || p.lddt < p.heads)
    return set_error(SMM_ERR_INVALID, "%s: row stride shorter than a row", who);
  if (!step && !p.offsets && p.nseq > 1)
    return set_error(SMM_ERR_INVALID, "%s: %d sequences without offsets", who, p.nseq);
  if ((p.state_in || p.state_out) && !p.slots && p.nslots < p.nseq)
    return set_error(SMM_ERR_INVALID, "%s: %d states for %d sequences", who, p.nslots, p.nseq);
  if (p.heads == 0 || p.nseq == 0) return SMM_OK;
  if (!p.A || (p.tokens > 0 && (!p.x || !p.dt || !p.B || !p.C || !p.y)))
    return set_error(SMM_ERR_INVALID, "%s: null pointer", who);
  const size_t e = dtype_size(dtype);
  const size_t sb = static_cast<size_t>(p.nslots) * hp * p.state_dim * sizeof(float);
  const Span y{p.y, span_bytes(p.tokens, hp, p.ldy, e)}, so{p.state_out, sb}, si{p.state_in, sb};
  const Span in[] = {{p.x, span_bytes(p.tokens, hp, p.ldx, e)},
                     {p.z, span_bytes(p.tokens, hp, p.ldz, e)},
                     {p.B, span_bytes(p.tokens, gn, p.ldb, e)},
                     {p.C, span_bytes(p.tokens, gn, p.ldc, e)},
                     {p.dt, span_bytes(p.tokens, p.heads, p.lddt, dtype_size(dt_dtype))},
                     {p.A, p.heads * sizeof(float)},
                     {p.D, p.heads * sizeof(float)},
                     {p.dt_bias, p.heads * sizeof(float)},
                     {p.offsets, (static_cast<size_t>(p.nseq) + 1) * sizeof(int)},
                     {p.slots, p.nseq * sizeof(int)}};
  bool bad = overlaps(y, si) || overlaps(y, so) || (p.state_in != p.state_out && overlaps(si, so));
  for (const Span& s : in) bad = bad || overlaps(y, s) || overlaps(so, s);
  if (bad) return set_error(SMM_ERR_INVALID, "%s: an output overlaps an input", who);
  return SMM_OK;
}

size_t round256(size_t b) { return (b + 255) & ~size_t(255); }

// Segment length on the fp32 pipes.  The first launch costs over half of the
// second, so a split pays once it makes three times the warps, and only while
// they are fewer than the GPU's 592 schedulers.
int simt_seg_len(long long tokens, int nseq, int heads, int dim) {
  const long long whole = std::max<long long>(tokens, 1);
  if (nseq < 1 || heads < 1) return static_cast<int>(whole);
  const long long warps = static_cast<long long>(heads) * ((dim + 7) / 8) * nseq;
  const long long parts = std::min(592 / warps, tokens / nseq / 64);
  if (parts < 3) return static_cast<int>(whole);
  const long long len = (tokens / nseq + parts - 1) / parts;
  return static_cast<int>((len + kTile - 1) / kTile * kTile);
}

}  // namespace

// smm_scan_umma.cu
int umma_seg_len(long long tokens, int nseq, int heads, int dim);

}  // namespace smm

using namespace smm;

namespace {
size_t split_bytes(long long tokens, int nseq, int heads, int dim, int state_dim, int seg_len) {
  if (seg_len >= tokens) return 0;
  const size_t segs = static_cast<size_t>(max_segments(tokens, nseq, seg_len));
  return round256(segs * heads * dim * state_dim * sizeof(float)) + round256(segs * heads * sizeof(float));
}
}  // namespace

extern "C" size_t smm_selective_scan_workspace_size(long long tokens, int nseq, int heads, int dim, int groups,
                                                    int state_dim, int dtype) {
  (void)groups;
  if (tokens <= 0 || nseq <= 0 || heads <= 0 || dim <= 0 || state_dim <= 0) return 0;
  size_t need = split_bytes(tokens, nseq, heads, dim, state_dim, simt_seg_len(tokens, nseq, heads, dim));
  if (dtype == SMM_DTYPE_BF16)
    need = std::max(need, split_bytes(tokens, nseq, heads, dim, state_dim, umma_seg_len(tokens, nseq, heads, dim)));
  return need;
}

extern "C" int smm_selective_scan(const void* x, const void* dt, const float* A, const void* B, const void* C,
                                  const float* D, const void* z, const float* dt_bias, const int* offsets,
                                  const float* state_in, float* state_out, const int* slots, void* y,
                                  long long tokens, int nseq, int nslots, int heads, int dim, int groups,
                                  int state_dim, long long ldx, long long lddt, long long ldb, long long ldc,
                                  long long ldz, long long ldy, int dtype, int dt_dtype, int dt_softplus, void* ws,
                                  size_t ws_bytes, void* stream) {
  SMM_RANGE("smm_selective_scan");
  ScanParams p{x,  dt,     A,   B,    C,   D,   z,   dt_bias, offsets, state_in, state_out, slots, y,
               tokens, ldx, lddt, ldb, ldc, ldz, ldy, nseq,    nslots,  heads,    dim,       groups, state_dim};
  p.dt_f32 = dt_dtype == SMM_DTYPE_F32;
  p.softplus = dt_softplus != 0;
  if (int rc = check_scan("smm_selective_scan", p, dtype, dt_dtype, false)) return rc;
  if (heads == 0 || nseq == 0) return SMM_OK;
  p.wait_limit_ns = wait_limit_ns();
  const bool umma = scan_umma_fits(p, dtype);
  p.seg_len = umma ? umma_seg_len(tokens, nseq, heads, dim) : simt_seg_len(tokens, nseq, heads, dim);
  p.split = p.seg_len < tokens;
  const long long segs = max_segments(tokens, nseq, p.seg_len);
  const size_t need = split_bytes(tokens, nseq, heads, dim, state_dim, p.seg_len);
  if (need) {
    if (!ws || ws_bytes < need)
      return set_error(SMM_ERR_WORKSPACE, "smm_selective_scan: workspace %zu bytes < %zu required", ws_bytes, need);
    if (!aligned_to(ws, 16)) return set_error(SMM_ERR_INVALID, "smm_selective_scan: workspace not 16-byte aligned");
    p.seg_state = static_cast<float*>(ws);
    p.seg_log = reinterpret_cast<float*>(
        static_cast<uint8_t*>(ws) + round256(static_cast<size_t>(segs) * heads * dim * state_dim * sizeof(float)));
  }
  p.status = device_status_word();
  if (!p.status) return set_error(SMM_ERR_CUDA, "device status word unavailable");
  if (umma) return scan_umma_launch(p, as_stream(stream));
  return dtype == SMM_DTYPE_F32 ? launch_scan_type<float>(p, segs, as_stream(stream))
                                : launch_scan_type<__nv_bfloat16>(p, segs, as_stream(stream));
}

extern "C" int smm_selective_step(const void* x, const void* dt, const float* A, const void* B, const void* C,
                                  const float* D, const void* z, const float* dt_bias, const float* state_in,
                                  float* state_out, const int* slots, void* y, int batch, int nslots, int heads,
                                  int dim, int groups, int state_dim, long long ldx, long long lddt, long long ldb,
                                  long long ldc, long long ldz, long long ldy, int dtype, int dt_dtype,
                                  int dt_softplus, void* stream) {
  SMM_RANGE("smm_selective_step");
  ScanParams p{x,     dt,  A,    B,   C,   D,   z,   dt_bias, nullptr, state_in, state_out, slots, y,
               batch, ldx, lddt, ldb, ldc, ldz, ldy, batch,   nslots,  heads,    dim,       groups, state_dim};
  p.dt_f32 = dt_dtype == SMM_DTYPE_F32;
  p.softplus = dt_softplus != 0;
  if (int rc = check_scan("smm_selective_step", p, dtype, dt_dtype, true)) return rc;
  if (heads == 0 || batch == 0) return SMM_OK;
  p.status = device_status_word();
  if (!p.status) return set_error(SMM_ERR_CUDA, "device status word unavailable");
  return dtype == SMM_DTYPE_F32 ? launch_step<float>(p, batch, as_stream(stream))
                                : launch_step<__nv_bfloat16>(p, batch, as_stream(stream));
}
