// Selective state space scan (per head a lower-triangular semiseparable
// matrix times x): the recurrence on the fp32 pipes for prompts, the
// single-token step, and the C entries.
#include "smm_scan.cuh"

#include <algorithm>
#include <mutex>
#include <type_traits>

namespace smm {
namespace {

using F2 = unsigned long long;  // two fp32 lanes

// ------------------------------------------------------------ prompts
// The recurrence itself, for fp32 elements (whose accuracy bf16 products do
// not reach) and for shapes the tensor-core kernel does not take.  Three
// packed multiply-adds per two state elements and token; bound by their issue.
//
// A CTA holds the states of one head and 4 PPL dims per warp in registers: lane
// (pg, ng) has PPL dims x NPL state elements, in 16-byte pieces strided by the 8
// lanes ng so that reading B and C from shared memory has no bank conflict and
// each value serves four lanes.  Tokens pass in tiles of 16: the next tile's B, C,
// x, z and dt are loaded into registers while the present one is computed, four
// tokens at a time, whose sums over the lanes ng are made together: 4096 tokens of 64
// heads of 64 x 128 take 0.77 ms.  (Token by token, the chain of one token's sum and its
// shuffles showed: 1.21 ms.)
constexpr int kTile = 16;

// bf16 comes here with short sequences, whose start and end want a second CTA on the SM (TWO;
// 16 tokens of 64 heads, 32 sequences: 188 -> 121 us); fp32 wants the registers.
template <typename T, int NPL, int THREADS, int PPL, bool STATES, bool TWO>
__global__ void __launch_bounds__(THREADS, TWO ? 512 / THREADS : 1) scan_kernel(const ScanParams p, int ptiles) {
  constexpr int NP = 8 * NPL;                  // padded state_dim
  constexpr int PT = THREADS / 8 * PPL;        // dims per CTA
  constexpr int NE = kTile * NP / THREADS > 0 ? kTile * NP / THREADS : 1;
  constexpr int XE = kTile * PT / THREADS;
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
  const int pw = warp * 4 * PPL + pg * PPL;    // this lane's first dim in the CTA's
  const int pl = p0 + pw;
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
  float hv[PPL][NPL];
#pragma unroll
  for (int pp = 0; pp < PPL; ++pp)
#pragma unroll
    for (int i = 0; i < NPL; ++i) hv[pp][i] = 0.0f;
  // (a multiply-add to zero where a load would do: with the plain load the compiler
  // schedules the whole loop differently, and 4096 tokens of 64 heads take 0.87 ms, not 0.77)
  auto get_state = [&](const float* src) {
#pragma unroll
    for (int pp = 0; pp < PPL; ++pp)
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        const int n = n_of(i / CH, i % CH);
        if (pl + pp < p.dim && n < N) hv[pp][i] = fmaf(hv[pp][i], 0.0f, src[state_at(pp, n)]);
      }
  };
  auto put_state = [&](float* dst) {
#pragma unroll
    for (int pp = 0; pp < PPL; ++pp)
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
        if (in) get_state(in);
        put_state(p.seg_state + seg * per_slot);
      }
      return;
    }
  } else if (sg.count > 1) {
    get_state(p.seg_state + seg * per_slot);
  } else if (in) {
    get_state(in);
  }
  F2 hst[PPL][NPL / 2];
#pragma unroll
  for (int pp = 0; pp < PPL; ++pp)
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
      float ys[4 * PPL];               // [token][dim]
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float2 ad = sad[t + u];
        const F2 a2 = pack2(ad.x, ad.x);
        F2 d[PPL], y[PPL][2];
#pragma unroll
        for (int pp = 0; pp < PPL; ++pp) {
          const float dx = sx[(t + u) * PT + pw + pp] * ad.y;
          d[pp] = pack2(dx, dx);
          y[pp][0] = y[pp][1] = pack2(0.0f, 0.0f);
        }
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
#pragma unroll
            for (int pp = 0; pp < PPL; ++pp) {
              hst[pp][k] = fma2(hst[pp][k], a2, mul2(d[pp], b[q]));
              if constexpr (!STATES) y[pp][q] = fma2(hst[pp][k], cc[q], y[pp][q]);
            }
          }
        }
        if constexpr (!STATES) {
#pragma unroll
          for (int pp = 0; pp < PPL; ++pp) {
            float lo, hi;
            unpack2(add2(y[pp][0], y[pp][1]), lo, hi);
            ys[PPL * u + pp] = lo + hi;
          }
        }
      }
      if constexpr (!STATES) {
        // sums over the 8 lanes ng, of which lane ng keeps the one of token ng / 2 (and dim ng % 2)
        constexpr int H = 2 * PPL, Q = PPL;
        float s4[H], s2[Q];
#pragma unroll
        for (int i = 0; i < H; ++i)
          s4[i] = ((ng & 4) ? ys[H + i] : ys[i]) + __shfl_xor_sync(0xFFFFFFFFu, (ng & 4) ? ys[i] : ys[H + i], 4);
#pragma unroll
        for (int i = 0; i < Q; ++i)
          s2[i] = ((ng & 2) ? s4[Q + i] : s4[i]) + __shfl_xor_sync(0xFFFFFFFFu, (ng & 2) ? s4[i] : s4[Q + i], 2);
        const float mine = (PPL == 2 && (ng & 1)) ? s2[Q - 1] : s2[0];
        const float sum = mine + __shfl_xor_sync(0xFFFFFFFFu, (PPL == 2 && !(ng & 1)) ? s2[Q - 1] : s2[0], 1);
        if (PPL == 2 || !(ng & 1)) sy[(t + (ng >> 1)) * PT + pw + (PPL == 2 ? (ng & 1) : 0)] = sum;
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
  for (int pp = 0; pp < PPL; ++pp)
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

template <typename T, int NPL, int THREADS, int PPL, bool TWO>
int launch_scan_ctas(const ScanParams& p, unsigned grid, int ptiles, cudaStream_t st) {
  constexpr int NP = 8 * NPL, PT = THREADS / 8 * PPL;
  const size_t full = sizeof(float) * kTile * (2 * NP + 2 * PT + 2);
  if (p.split) {
    scan_kernel<T, NPL, THREADS, PPL, true, TWO><<<grid, THREADS, full, st>>>(p, ptiles);
    count_launch();
    SMM_CUDA_TRY(cudaGetLastError(), "selective scan launch");
    if (int rc = scan_combine(p, st)) return rc;
  }
  scan_kernel<T, NPL, THREADS, PPL, false, TWO><<<grid, THREADS, full, st>>>(p, ptiles);
  count_launch();
  SMM_CUDA_TRY(cudaGetLastError(), "selective scan launch");
  return SMM_OK;
}

template <typename T, int NPL, int THREADS, int PPL>
int launch_scan(const ScanParams& p, long long segs, cudaStream_t st) {
  constexpr int PT = THREADS / 8 * PPL;
  const int ptiles = (p.dim + PT - 1) / PT;
  const long long blocks = segs * p.heads * ptiles;
  if (blocks > 0x7FFFFFFFLL) return set_error(SMM_ERR_INVALID, "selective scan too large for one launch");
  const unsigned grid = static_cast<unsigned>(blocks);
  // Half of the registers spill for state_dim above 128, which a second CTA on the SM makes up for, if
  // there is one (64 heads of state_dim 256: one sequence of 4000 tokens 3.6 ms with half, 1.8 with all
  // of them, two of 600 577 and 382 us, but eight of 500 898 and 956, 32 of 64 497 and 593).
  if constexpr (sizeof(T) == 2 && NPL == 32) {
    if (blocks * THREADS <= 148 * 256) return launch_scan_ctas<T, NPL, THREADS, PPL, false>(p, grid, ptiles, st);
  }
  return launch_scan_ctas<T, NPL, THREADS, PPL, sizeof(T) == 2>(p, grid, ptiles, st);
}

template <typename T>
int launch_scan_type(const ScanParams& p, long long segs, cudaStream_t st) {
  auto go = [&](auto npl) {
    constexpr int NPL = decltype(npl)::value;
    // Two dims to a lane read B and C half as often; one makes twice the warps, which is faster
    // for small states while a scheduler has one warp of two dims at most (592 of them; state_dim
    // 16, sequences of 200 tokens, 256 to 512 warps: 19.2 us against 20.2, of 800: 68 against 72; 624
    // warps: 24.9 against 22.9; state_dim 32, 512 warps: 23.8 against 22.7, with 128 49 against 46).
    // Then 32 dims to a CTA where 64 would leave SMs without one.
    if constexpr (NPL == 2) {
      if (segs * p.heads * ((p.dim + 7) / 8) <= 592) return launch_scan<T, NPL, 256, 1>(p, segs, st);
    }
    if (p.dim <= 32 || segs * p.heads * ((p.dim + 63) / 64) < 2 * 148) return launch_scan<T, NPL, 128, 2>(p, segs, st);
    return launch_scan<T, NPL, 256, 2>(p, segs, st);
  };
  if (p.state_dim <= 16) return go(std::integral_constant<int, 2>{});
  if (p.state_dim <= 32) return go(std::integral_constant<int, 4>{});
  if (p.state_dim <= 64) return go(std::integral_constant<int, 8>{});
  if (p.state_dim <= 128) return go(std::integral_constant<int, 16>{});
  return go(std::integral_constant<int, 32>{});
}

// ------------------------------------------------------------ one token
// S = exp(d A) S + d x (outer) B, y = S C: the state is read once and written
// once (8 bytes per element against 5 operations), which bounds it.  A row of the
// state takes LANES lanes with 16 bytes each (twice where NV is 2).  A warp walks a
// run of tiles of 4 KB, a few rows of one head each, its lanes copying their own
// pieces up to two tiles ahead into shared memory (cp.async: no register holds them,
// and as a lane reads back only what it copied, no barrier is needed).  671 MB of
// states take 122 us, 85 % of a copy's rate; a short CTA for every few rows, which
// waits for slot, states, then dt, B and C, took 164 us, and 4.5 instead of 4.1 for
// 4 MB.  Sums over a row's lanes are made for all rows together: 9 exchanges, not 40
// (122 us against 149, with two tiles of loads in flight and x and z one tile ahead).
constexpr int kStepThreads = 256, kStepCtas = 2, kStepStages = 3, kStepTile = 4096;
constexpr int kStepSmem = kStepThreads / 32 * kStepStages * kStepTile;

template <typename T, int LANES, int NV>
__global__ void __launch_bounds__(kStepThreads, kStepCtas) step_kernel(const ScanParams p, int tph,
                                                                       long long tiles) {
  constexpr int R = kStepTile / 512 / NV;         // rows of a lane in a tile, LANES lanes to a row
  constexpr int H = R < LANES ? R : LANES;        // lanes that end with sums of their own
  constexpr int KEEP = R / H, SHARE = LANES / H;  // rows of each, lanes with the same ones
  constexpr int rstep = 32 / LANES;
  extern __shared__ __align__(16) unsigned char smem[];
  const int lane = threadIdx.x & 31, sub = lane % LANES, row0 = lane / LANES, mine = sub / SHARE * KEEP;
  const int N = p.state_dim, per_group = p.heads / p.groups;
  const long long warp = static_cast<long long>(blockIdx.x) * (kStepThreads / 32) + (threadIdx.x >> 5);
  const long long warps = static_cast<long long>(gridDim.x) * (kStepThreads / 32);
  const long long t0 = tiles * warp / warps, t1 = tiles * (warp + 1) / warps;
  if (t0 >= t1) return;
  float4* const ring = reinterpret_cast<float4*>(smem + (threadIdx.x >> 5) * kStepStages * kStepTile) + lane;
  constexpr int kPieces = kStepTile / 16;

  struct Place {
    int b, h, pt, slot;
  };
  auto place = [&](long long t) {
    Place c;
    c.pt = static_cast<int>(t % tph);
    const long long hb = t / tph;
    c.h = static_cast<int>(hb % p.heads);
    c.b = static_cast<int>(hb / p.heads);
    c.slot = p.state_in || p.state_out ? seq_slot(p.slots, c.b, p.nslots, p.status) : -1;
    return c;
  };
  auto advance = [&](Place& c, bool live) {
    if (++c.pt < tph) return;
    c.pt = 0;
    if (++c.h < p.heads) return;
    c.h = 0;
    ++c.b;
    if (live && (p.state_in || p.state_out)) c.slot = seq_slot(p.slots, c.b, p.nslots, p.status);
  };
  auto state_at = [&](const Place& c) {
    return (static_cast<long long>(c.slot) * p.heads + c.h) * p.dim * N;
  };
  Place ahead = place(t0), cur = ahead;
  int fill = 0;
  auto issue = [&](long long t) {
    if (t < t1) {
      const float* in = p.state_in && ahead.slot >= 0 ? p.state_in + state_at(ahead) : nullptr;
      float4* dst = ring + fill * kPieces;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int q = ahead.pt * R * rstep + r * rstep + row0;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          const int n = (k * LANES + sub) * 4;
          if (in && q < p.dim && n < N)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst + (r * NV + k) * 32)),
                         "l"(in + static_cast<long long>(q) * N + n)
                         : "memory");
          else
            dst[(r * NV + k) * 32] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
      }
      fill = fill + 1 == kStepStages ? 0 : fill + 1;
      advance(ahead, t + 1 < t1);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kStepStages - 1; ++i) issue(t0 + i);

  // x and z of the rows that this lane finishes, one tile ahead
  T xn[KEEP], zn[KEEP];
  auto load_xz = [&](const Place& c) {
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
      const int q = (c.pt * R + mine + i) * rstep + row0;
      const long long col = static_cast<long long>(c.h) * p.dim + q;
      xn[i] = zn[i] = from_f32<T>(0.0f);
      if (q < p.dim) xn[i] = static_cast<const T*>(p.x)[c.b * p.ldx + col];
      if (q < p.dim && p.z) zn[i] = static_cast<const T*>(p.z)[c.b * p.ldz + col];
    }
  };
  load_xz(cur);
  float bv[NV][4], cv[NV][4], d = 0.0f, a = 0.0f, Dh = 0.0f;
  int stage = 0;
  for (long long t = t0; t < t1; ++t) {
    issue(t + kStepStages - 1);
    float xs[KEEP], zs[KEEP];
#pragma unroll
    for (int i = 0; i < KEEP; ++i) xs[i] = to_f32(xn[i]), zs[i] = to_f32(zn[i]);
    if (t == t0 || cur.pt == 0) {
      const int g = cur.h / per_group;
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int n = (k * LANES + sub) * 4 + i;
          const long long col = static_cast<long long>(g) * N + n;
          bv[k][i] = n < N ? to_f32(static_cast<const T*>(p.B)[cur.b * p.ldb + col]) : 0.0f;
          cv[k][i] = n < N ? to_f32(static_cast<const T*>(p.C)[cur.b * p.ldc + col]) : 0.0f;
        }
      d = scan_dt(p, scan_dt_raw(p, cur.b, cur.h), p.dt_bias ? __ldg(p.dt_bias + cur.h) : 0.0f);
      a = expf(d * __ldg(p.A + cur.h));
      Dh = p.D ? __ldg(p.D + cur.h) : 0.0f;
    }
    const Place at = cur;
    advance(cur, t + 1 < t1);
    if (t + 1 < t1) load_xz(cur);
    float* out = p.state_out && at.slot >= 0 ? p.state_out + state_at(at) : nullptr;
    asm volatile("cp.async.wait_group %0;" ::"n"(kStepStages - 1) : "memory");
    const float4* src = ring + stage * kPieces;
    float ys[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int q = (at.pt * R + r) * rstep + row0;
      const float dx = d * __shfl_sync(0xFFFFFFFFu, xs[r % KEEP], row0 * LANES + r / KEEP * SHARE);
      float y = 0.0f;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int n = (k * LANES + sub) * 4;
        float4 f = src[(r * NV + k) * 32];
        f.x = fmaf(f.x, a, dx * bv[k][0]), f.y = fmaf(f.y, a, dx * bv[k][1]);
        f.z = fmaf(f.z, a, dx * bv[k][2]), f.w = fmaf(f.w, a, dx * bv[k][3]);
        y = fmaf(f.x, cv[k][0], y), y = fmaf(f.y, cv[k][1], y);
        y = fmaf(f.z, cv[k][2], y), y = fmaf(f.w, cv[k][3], y);
        if (out && q < p.dim && n < N) __stcs(reinterpret_cast<float4*>(out + static_cast<long long>(q) * N + n), f);
      }
      ys[r] = y;
    }
    // Sums over the LANES lanes of all rows together: each exchange halves the rows
    // of a lane, then the lanes that share a row add up.
    int o = LANES / 2;
#pragma unroll
    for (int half = R / 2; half >= KEEP; half /= 2, o /= 2) {
      const bool up = sub & o;
#pragma unroll
      for (int i = 0; i < half; ++i) {
        const float got = __shfl_xor_sync(0xFFFFFFFFu, up ? ys[i] : ys[i + half], o);
        ys[i] = (up ? ys[i + half] : ys[i]) + got;
      }
    }
#pragma unroll
    for (; o > 0; o /= 2) ys[0] += __shfl_xor_sync(0xFFFFFFFFu, ys[0], o);
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
      const int q = (at.pt * R + mine + i) * rstep + row0;
      if (sub % SHARE != 0 || q >= p.dim) continue;
      float y = fmaf(Dh, xs[i], ys[i]);
      if (p.z) y *= silu(zs[i]);
      static_cast<T*>(p.y)[at.b * p.ldy + static_cast<long long>(at.h) * p.dim + q] = from_f32<T>(y);
    }
    stage = stage + 1 == kStepStages ? 0 : stage + 1;
  }
}

template <typename T, int LANES, int NV>
int launch_step_tiles(const ScanParams& p, long long heads, cudaStream_t st) {
  auto kern = step_kernel<T, LANES, NV>;
  constexpr int rows = kStepTile / 512 / NV * (32 / LANES);
  const int tph = (p.dim + rows - 1) / rows;
  static std::once_flag once[64];
  int dev = 0;
  SMM_CUDA_TRY(cudaGetDevice(&dev), "cudaGetDevice");
  cudaError_t err = cudaSuccess;
  auto set = [&] { err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kStepSmem); };
  if (dev < 64) std::call_once(once[dev], set);
  else set();
  SMM_CUDA_TRY(err, "selective step shared memory size");
  const int grid = static_cast<int>(std::min<long long>(heads * tph, kStepCtas * 148));
  kern<<<grid, kStepThreads, kStepSmem, st>>>(p, tph, heads * tph);
  count_launch();
  SMM_CUDA_TRY(cudaGetLastError(), "selective step launch");
  return SMM_OK;
}


// Any other state_dim, one element at a time.
constexpr int kOddThreads = 128, kOddRows = 4;
template <typename T, int NV>
__global__ void __launch_bounds__(kOddThreads) step_odd_kernel(const ScanParams p, int lanes, int rows_per_cta,
                                                                int ptiles) {
  const int pt = static_cast<int>(blockIdx.x % ptiles);
  const int hb = static_cast<int>(blockIdx.x / ptiles);
  const int h = hb % p.heads, b = hb / p.heads;
  const int g = h / (p.heads / p.groups);
  const int N = p.state_dim;
  const int sub = threadIdx.x % lanes, row0 = threadIdx.x / lanes, rstep = kOddThreads / lanes;
  const int slot = p.state_in || p.state_out ? seq_slot(p.slots, b, p.nslots, p.status) : -1;
  const long long base = (static_cast<long long>(slot) * p.heads + h) * p.dim * N;
  const float* in = p.state_in && slot >= 0 ? p.state_in + base : nullptr;
  float* out = p.state_out && slot >= 0 ? p.state_out + base : nullptr;
  const int pend = (pt + 1) * rows_per_cta < p.dim ? (pt + 1) * rows_per_cta : p.dim;

  float hv[kOddRows][NV], xv[kOddRows], bv[NV], cv[NV];
  auto load_rows = [&](int r0) {
#pragma unroll
    for (int r = 0; r < kOddRows; ++r) {
      const int q = r0 + r * rstep;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int n = k * lanes + sub;
        hv[r][k] = in && q < pend && n < N ? in[static_cast<long long>(q) * N + n] : 0.0f;
      }
    }
#pragma unroll
    for (int r = 0; r < kOddRows; ++r) {
      const int q = r0 + r * rstep;
      xv[r] = q < pend ? to_f32(static_cast<const T*>(p.x)[b * p.ldx + static_cast<long long>(h) * p.dim + q]) : 0.0f;
    }
  };
  load_rows(pt * rows_per_cta + row0);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int n = k * lanes + sub;
    bv[k] = n < N ? to_f32(static_cast<const T*>(p.B)[b * p.ldb + static_cast<long long>(g) * N + n]) : 0.0f;
    cv[k] = n < N ? to_f32(static_cast<const T*>(p.C)[b * p.ldc + static_cast<long long>(g) * N + n]) : 0.0f;
  }
  const float d = scan_dt(p, scan_dt_raw(p, b, h), p.dt_bias ? __ldg(p.dt_bias + h) : 0.0f);
  const float a = expf(d * __ldg(p.A + h));
  const float Dh = p.D ? __ldg(p.D + h) : 0.0f;
  // every thread of the CTA makes the same number of turns (the shuffles)
  for (int base_row = pt * rows_per_cta; base_row < pend; base_row += kOddRows * rstep) {
    if (base_row != pt * rows_per_cta) load_rows(base_row + row0);
#pragma unroll
    for (int r = 0; r < kOddRows; ++r) {
      const int q = base_row + row0 + r * rstep;
      const float dx = d * xv[r];
      float y = 0.0f;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        hv[r][k] = fmaf(hv[r][k], a, dx * bv[k]);
        y = fmaf(hv[r][k], cv[k], y);
        const int n = k * lanes + sub;
        if (out && q < pend && n < N) out[static_cast<long long>(q) * N + n] = hv[r][k];
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
  const long long heads = static_cast<long long>(batch) * p.heads;
  if (p.state_dim % 4 == 0 && p.state_dim > 8 && aligned_to(p.state_in, 16) && aligned_to(p.state_out, 16)) {
    if (p.state_dim <= 16) return launch_step_tiles<T, 4, 1>(p, heads, st);
    if (p.state_dim <= 32) return launch_step_tiles<T, 8, 1>(p, heads, st);
    if (p.state_dim <= 64) return launch_step_tiles<T, 16, 1>(p, heads, st);
    return p.state_dim <= 128 ? launch_step_tiles<T, 32, 1>(p, heads, st) : launch_step_tiles<T, 32, 2>(p, heads, st);
  }
  int lanes = 1;
  while (lanes < 32 && lanes < p.state_dim) lanes *= 2;
  const int rows = kOddRows * kOddThreads / lanes;
  const int ptiles = (p.dim + rows - 1) / rows;
  if (heads * ptiles > 0x7FFFFFFFLL) return set_error(SMM_ERR_INVALID, "selective step too large for one launch");
  const unsigned grid = static_cast<unsigned>(heads * ptiles);
  if (p.state_dim <= 32)
    step_odd_kernel<T, 1><<<grid, kOddThreads, 0, st>>>(p, lanes, rows, ptiles);
  else
    step_odd_kernel<T, 8><<<grid, kOddThreads, 0, st>>>(p, lanes, rows, ptiles);
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
  if (!all_aligned_to(e, p.x, p.z, p.B, p.C, p.y) || !aligned_to(p.dt, dtype_size(dt_dtype)) ||
      !all_aligned_to(4, p.A, p.D, p.dt_bias, p.state_in, p.state_out, p.offsets, p.slots))
    return set_error(SMM_ERR_INVALID, "%s: a pointer is not aligned to its elements", who);
  const size_t sb = static_cast<size_t>(p.nslots) * hp * p.state_dim * sizeof(float);
  const Span y = row_span(p.y, p.tokens, hp, p.ldy, e), so{p.state_out, sb}, si{p.state_in, sb};
  const Span in[] = {row_span(p.x, p.tokens, hp, p.ldx, e),
                     row_span(p.z, p.tokens, hp, p.ldz, e),
                     row_span(p.B, p.tokens, gn, p.ldb, e),
                     row_span(p.C, p.tokens, gn, p.ldc, e),
                     row_span(p.dt, p.tokens, p.heads, p.lddt, dtype_size(dt_dtype)),
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

// The state before segment j from the final states F_k of those before it (each from
// zero) and S_in, which lies in the last one's place: a thread walks one element's
// segments, eight elements' loads at a time.  Memory-bound: 8 bytes an element and segment.
constexpr int kCombineThreads = 256;

template <int V>  // elements of a thread
__global__ void __launch_bounds__(kCombineThreads) combine_kernel(const ScanParams p, int tiles, long long nsegs) {
  __shared__ int sfirst;
  const int s = static_cast<int>(blockIdx.x / tiles);
  const int per_head = p.dim * p.state_dim;
  const long long per_slot = static_cast<long long>(p.heads) * per_head;
  const long long e = (static_cast<long long>(blockIdx.x % tiles) * kCombineThreads + threadIdx.x) * V;
  long long first = 0;
  if (s > 0) {
    if (threadIdx.x == 0) sfirst = 0;
    __syncthreads();
    int before = 0;
    for (int q = threadIdx.x; q < s; q += kCombineThreads) {
      long long b, end;
      seq_range(p.offsets, q, p.tokens, &b, &end);
      before += segments_of(p, b, end);
    }
    if (before) atomicAdd(&sfirst, before);
    __syncthreads();
    first = sfirst;
  }
  long long b, end;
  seq_range(p.offsets, s, p.tokens, &b, &end);
  const int count = segments_of(p, b, end);
  // sequences that overlap (offsets that decrease) may count past the workspace's segments
  if (count == 1 || first + count > nsegs || e >= per_slot) return;
  using E = typename std::conditional<V == 4, float4, float>::type;
  const float* log = p.seg_log + first * p.heads + e / per_head;
  float* at = p.seg_state + first * per_slot + e;
  auto get = [&](int j, float(&v)[V]) { *reinterpret_cast<E*>(v) = *reinterpret_cast<const E*>(at + j * per_slot); };
  auto put = [&](int j, const float(&v)[V]) { *reinterpret_cast<E*>(at + j * per_slot) = *reinterpret_cast<const E*>(v); };
  alignas(16) float run[V];
  get(count - 1, run);
  constexpr int U = 8 / V;
  for (int j0 = 0; j0 < count - 1; j0 += U) {
    alignas(16) float f[U][V];
    float a[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (j0 + u < count - 1) {
        get(j0 + u, f[u]);
        a[u] = log[static_cast<long long>(j0 + u) * p.heads];
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (j0 + u < count - 1) {
        put(j0 + u, run);
        const float decay = expf(a[u]);
#pragma unroll
        for (int i = 0; i < V; ++i) run[i] = fmaf(run[i], decay, f[u][i]);
      }
  }
  put(count - 1, run);
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

int scan_combine(const ScanParams& p, cudaStream_t st) {
  const bool vec = p.dim * p.state_dim % 4 == 0;  // the workspace's alignment is checked
  const long long per_cta = kCombineThreads * (vec ? 4 : 1);
  const long long tiles = (static_cast<long long>(p.heads) * p.dim * p.state_dim + per_cta - 1) / per_cta;
  if (tiles * p.nseq > 0x7FFFFFFFLL) return set_error(SMM_ERR_INVALID, "selective scan too large for one launch");
  const unsigned grid = static_cast<unsigned>(tiles * p.nseq);
  const long long nsegs = max_segments(p.tokens, p.nseq, p.seg_len);
  if (vec)
    combine_kernel<4><<<grid, kCombineThreads, 0, st>>>(p, static_cast<int>(tiles), nsegs);
  else
    combine_kernel<1><<<grid, kCombineThreads, 0, st>>>(p, static_cast<int>(tiles), nsegs);
  count_launch();
  SMM_CUDA_TRY(cudaGetLastError(), "selective scan combine launch");
  return SMM_OK;
}

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
  if (umma) {
    p.wait_limit_ns = take_wait_limit_ns();
    return scan_umma_launch(p, as_stream(stream));
  }
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
