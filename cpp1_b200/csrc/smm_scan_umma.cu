// Selective scan of bf16 prompts on the tensor cores (tcgen05, TMEM, TMA).
//
// With cum_t the sum of d A over a chunk of 128 tokens up to t, and H the state
// before the chunk, a chunk of one head is four products:
//   S  = C B^T                               128 x 128 x state_dim
//   Y  = G x,  G[t][s] = S[t][s] exp(cum_t - cum_s) d_s for s <= t, else 0
//   Yo = C H^T,  y_t = Y_t + exp(cum_t) Yo_t + D x_t
//   dS = B^T Xw,  Xw[s] = exp(cum_127 - cum_s) d_s x_s,  H' = exp(cum_127) H + dS
// Only H' = ... is serial along the tokens.  One CTA walks the chunks of one
// (segment, head, 64 dims), with S double-buffered in tensor memory so that the
// next chunk's S and G are under way while this one's products run.
//
// Decays are products of factors exp(<= 0 when A <= 0) whose exponents are sums over
// at most 128 tokens that lie between s and t, never differences of long sums:
// within blocks of 32 tokens u_t = exp(sum from the block's start to t),
// f[b][s] = d_s exp(sum from behind s to the start of block b).  G is S u_t f[b][s]
// off the diagonal blocks, and exp(l_t - l_s) d_s on them, l being sums within
// the block; w_s = f[4][s].  So a quarter of the exponentials remains.
//
// Roundings: G and H to bf16 as operands of products (relative 2^-8 of
// each term of y, which is itself rounded to bf16); Xw as the sum of two bf16 terms
// (2^-16), because the state is an fp32 result that is carried on.  The state
// itself stays in fp32 registers, S, Y, Yo and dS are fp32 in tensor memory.
//
// Warps: 0 loads (TMA), 1 issues the products, 2 computes the decays, 4-7 and 8-11
// form G and write y of the even and the odd chunks, 12-15 form Xw, 16-19 carry
// the state.  Every wait is bounded; on expiry the CTA records it and leaves.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>

#include "smm_scan.cuh"

namespace smm {

void* tensor_map_encoder();  // smm_lib.cu

namespace {

constexpr int kQ = 128;         // tokens per chunk
constexpr int kP = 64;          // dims per CTA
constexpr int kThreads = 640;
constexpr uint32_t kAtom = kQ * 128;  // one 64-element wide tile of 128 rows: 16 KiB
// tensor memory columns; G[k] overlays the first half of S[k]
constexpr uint32_t kColS = 0, kColY = 256, kColYo = 384, kColDs = 448, kCols = 512;

struct Scal {
  float f[4][kQ];  // f[b-1][s], b = 1..4
  float l[kQ];     // log2 of the decay from the block's start through t
  float u[kQ];     // its value
  float e[kQ];     // decay from the chunk's start through t
  float d[kQ];
  float total;     // decay of the whole chunk
  float pad[3];
};

struct Bars {
  uint64_t full_bc[2], full_x[2], done[2], xfree[2], s_full[2], g_full[2];
  uint64_t xw_full, ds_full, ds_free, h_full, yo_free;
  uint64_t sc_full[3], sc_free[3];
  uint64_t drain;
  uint32_t tmem;
  int abort_flag;
};

// NA: 64-wide tiles that state_dim takes (1 or 2)
template <int NA>
struct Smem {
  static constexpr uint32_t kStage = (2 * NA + 1) * kAtom;  // C, B, x
  static constexpr uint32_t kXw = 2 * kStage;               // high and low terms
  static constexpr uint32_t kH = kXw + 2 * kAtom;
  static constexpr uint32_t kScal = kH + NA * 64 * 128;
  static constexpr uint32_t kBars = kScal + 3 * sizeof(Scal);
  static constexpr uint32_t kBytes = kBars + sizeof(Bars) + 1024;  // + alignment
};

struct Tmaps {
  CUtensorMap x, b, c;
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1,
                                            int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  umma_lohi<false, true>(d, static_cast<uint32_t>(a), static_cast<uint32_t>(a >> 32), static_cast<uint32_t>(b),
                         static_cast<uint32_t>(b >> 32), idesc, acc ? 1u : 0u);
}
// A from tensor memory (bf16, two per column), B from shared memory
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc ? 1u : 0u)
      : "memory");
}
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long x, y, r;
  float2 o;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(b.x), "f"(b.y));
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(o.x), "=f"(o.y) : "l"(r));
  return o;
}
__device__ __forceinline__ void st_shared_v4(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}

// STATES: the first launch of a split scan (B, x and the state only).
template <int NA, bool STATES>
__global__ void __launch_bounds__(kThreads, 1)
    scan_umma_kernel(const __grid_constant__ Tmaps maps, const ScanParams p, int ptiles) {
  using L = Smem<NA>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Segment sseg;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  Scal* scal = reinterpret_cast<Scal*>(smem + L::kScal);
  Bars* bars = reinterpret_cast<Bars*>(smem + L::kBars);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pt = static_cast<int>(blockIdx.x % ptiles);
  const int hs = static_cast<int>(blockIdx.x / ptiles);
  const int h = hs % p.heads, seg = hs / p.heads;
  if (warp == 0) {
    const Segment s = find_segment(p, seg);
    if (lane == 0) sseg = s;
  }
  __syncthreads();
  const Segment sg = sseg;
  if (!sg.valid) return;
  const int g = h / (p.heads / p.groups);
  const int p0 = pt * kP;
  const int pdims = p.dim - p0 < kP ? p.dim - p0 : kP;
  const int N = p.state_dim;
  const bool last = sg.j == sg.count - 1;
  const long long per_slot = static_cast<long long>(p.heads) * p.dim * N;
  const long long head_at = (static_cast<long long>(h) * p.dim + p0) * N;
  const int slot = (p.state_in || p.state_out) ? seq_slot(p.slots, sg.seq, p.nslots, p.status) : -1;
  const float* in = p.state_in && slot >= 0 ? p.state_in + slot * per_slot + head_at : nullptr;
  if constexpr (STATES) {
    // The last segment's place keeps the state the sequence started from: the
    // second launch may overwrite it while other segments still need it.
    if (last) {
      if (sg.count > 1)
        for (int i = threadIdx.x; i < pdims * N; i += kThreads)
          p.seg_state[seg * per_slot + head_at + i] = in ? in[i] : 0.0f;
      return;
    }
  }
  const int nc = static_cast<int>((sg.end - sg.begin + kQ - 1) / kQ);

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->full_bc[i], 1);
      mbar_init(&bars->full_x[i], 1);
      mbar_init(&bars->done[i], 1);
      mbar_init(&bars->xfree[i], 4);
      mbar_init(&bars->s_full[i], 1);
      mbar_init(&bars->g_full[i], 4);
    }
    mbar_init(&bars->xw_full, 4);
    mbar_init(&bars->ds_full, 1);
    mbar_init(&bars->ds_free, 4);
    mbar_init(&bars->h_full, 4);
    mbar_init(&bars->yo_free, 4);
    for (int i = 0; i < 3; ++i) {
      mbar_init(&bars->sc_full[i], 1);
      mbar_init(&bars->sc_free[i], STATES ? 8 : 12);
    }
    mbar_init(&bars->drain, 1);
    bars->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(&bars->tmem, kCols);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = bars->tmem;

  WaitCtx w{&bars->abort_flag, p.status, p.wait_limit_ns, 0};
  const uint32_t stage_c = 0, stage_b = NA * kAtom, stage_x = 2 * NA * kAtom;

  if (warp == 0) {
    // ------------------------------------------------------------ loads
    if (lane == 0) {
      w.where = kWaitProducer;
      tma_prefetch_desc(&maps.x);
      tma_prefetch_desc(&maps.b);
      if (!STATES) tma_prefetch_desc(&maps.c);
      int issued = 0;
      for (int c = 0; c < nc; ++c) {
        const int s = c & 1;
        if (c >= 2 && !mbar_wait(&bars->done[s], ((c >> 1) - 1) & 1, w)) break;
        const uint32_t st = sbase + s * L::kStage;
        const int t0 = static_cast<int>(sg.begin) + c * kQ;
        mbar_arrive_expect_tx(&bars->full_bc[s], (STATES ? 1 : 2) * NA * kAtom);
#pragma unroll
        for (int a = 0; a < NA; ++a) {
          if (!STATES) tma_load_3d(st + stage_c + a * kAtom, &maps.c, &bars->full_bc[s], a * 64, g, t0);
          tma_load_3d(st + stage_b + a * kAtom, &maps.b, &bars->full_bc[s], a * 64, g, t0);
        }
        issued = c + 1;
        if (!STATES && c >= 2 && !mbar_wait(&bars->xfree[s], ((c >> 1) - 1) & 1, w)) break;
        mbar_arrive_expect_tx(&bars->full_x[s], kAtom);
        tma_load_3d(st + stage_x, &maps.x, &bars->full_x[s], p0, h, t0);
      }
      // after an abort, copies in flight land before the CTA leaves
      if (bars->abort_flag) {
        int none = 0;
        WaitCtx dw{&none, p.status, p.wait_limit_ns > 1000000000ull ? p.wait_limit_ns : 1000000000ull, kWaitDrain};
        for (int c = issued >= 2 ? issued - 2 : 0; c < issued; ++c) {
          mbar_wait(&bars->full_bc[c & 1], (c >> 1) & 1, dw);
          // x's copy of the newest chunk may not have been issued
          if (c < issued - 1) mbar_wait(&bars->full_x[c & 1], (c >> 1) & 1, dw);
        }
        const int c = issued - 1;
        if (c >= 0) {
          none = 0;
          dw.limit_ns = 1000000;
          dw.status = nullptr;
          mbar_wait(&bars->full_x[c & 1], (c >> 1) & 1, dw);
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ products
    if (lane == 0) {
      constexpr uint32_t idS = make_idesc(kFmtBF16, 128, 128, 0, 0);
      constexpr uint32_t idY = make_idesc(kFmtBF16, 128, kP, 0, 1);
      constexpr uint32_t idD = make_idesc(kFmtBF16, 128, kP, 1, 1);
      const int ksteps = (N + 15) / 16;
      int s_next = STATES ? nc : 0, g_next = 0, sub = 0;
      uint64_t t_idle = 0;
      while (g_next < nc) {
        bool did = false;
        if (!STATES && s_next < nc && s_next < g_next + 2 &&
            mbar_test(&bars->full_bc[s_next & 1], (s_next >> 1) & 1)) {
          // the loads of chunk c waited for every product of chunk c - 2, so S and G are free
          tc_fence_after_sync();
          const int s = s_next & 1;
          const uint32_t st = sbase + s * L::kStage;
          for (int k = 0; k < ksteps; ++k) {
            const uint32_t off = (k >> 2) * kAtom + (k & 3) * 32;
            umma_ss(tmem + kColS + s * 128, make_smem_desc(st + stage_c + off, 16, 1024, kLayoutSw128),
                    make_smem_desc(st + stage_b + off, 16, 1024, kLayoutSw128), idS, k > 0);
          }
          umma_commit(&bars->s_full[s]);
          ++s_next;
          did = true;
        } else if (STATES || g_next < s_next) {
          const int c = g_next, s = c & 1;
          const uint32_t st = sbase + s * L::kStage;
          if (sub == 0) {
            if (mbar_test(&bars->xw_full, c & 1) && (c == 0 || mbar_test(&bars->ds_free, (c - 1) & 1)) &&
                mbar_test(&bars->full_bc[s], (c >> 1) & 1) && mbar_test(&bars->full_x[s], (c >> 1) & 1)) {
              tc_fence_after_sync();
              for (int k = 0; k < 16; ++k) {
                const uint32_t kk = (k & 7) * 2048;
                umma_ss(tmem + kColDs, make_smem_desc(st + stage_b + kk, kAtom, 1024, kLayoutSw128),
                        make_smem_desc(sbase + L::kXw + (k >> 3) * kAtom + kk, kAtom, 1024, kLayoutSw128), idD, k > 0);
              }
              umma_commit(&bars->ds_full);
              if (STATES) {
                umma_commit(&bars->done[s]);
                ++g_next;
              } else {
                sub = 1;
              }
              did = true;
            }
          } else if (sub == 1) {
            if (mbar_test(&bars->g_full[s], (c >> 1) & 1)) {
              tc_fence_after_sync();
              for (int k = 0; k < 8; ++k)
                umma_ts(tmem + kColY + s * kP, tmem + kColS + s * 128 + k * 8,
                        make_smem_desc(st + stage_x + k * 2048, kAtom, 1024, kLayoutSw128), idY, k > 0);
              sub = 2;
              did = true;
            }
          } else {
            if (mbar_test(&bars->h_full, c & 1) && (c == 0 || mbar_test(&bars->yo_free, (c - 1) & 1))) {
              tc_fence_after_sync();
              for (int k = 0; k < ksteps; ++k) {
                const uint32_t off = (k >> 2) * kAtom + (k & 3) * 32;
                umma_ss(tmem + kColYo, make_smem_desc(st + stage_c + off, 16, 1024, kLayoutSw128),
                        make_smem_desc(sbase + L::kH + k * 2048, kAtom, 1024, kLayoutSw128), idY, k > 0);
              }
              umma_commit(&bars->done[s]);
              sub = 0;
              ++g_next;
              did = true;
            }
          }
        }
        if (did) {
          t_idle = 0;
        } else {
          if (t_idle == 0) t_idle = globaltimer_ns();
          if (*w.abort_flag) break;
          if (globaltimer_ns() - t_idle > w.limit_ns) {
            *w.abort_flag = 1;
            if (w.status) atomicOr(w.status, kDevErrTimeout | kWaitMma);
            break;
          }
        }
      }
      // every product has completed, and its arrivals have landed, before the CTA leaves
      int none = 0;
      WaitCtx dw{&none, p.status, p.wait_limit_ns > 1000000000ull ? p.wait_limit_ns : 1000000000ull, kWaitDrain};
      umma_commit(&bars->drain);
      mbar_wait(&bars->drain, 0, dw);
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------ decays
    w.where = kWaitTransform;
    const float A2 = __ldg(p.A + h) * kLog2e;
    float log_sum = 0.0f;  // log2 of the segment's decay
    bool ok = true;
    const float bias = p.dt_bias ? __ldg(p.dt_bias + h) : 0.0f;
    uint32_t raw[4] = {};
    auto fetch = [&](int c) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long long t = sg.begin + static_cast<long long>(c) * kQ + lane * 4 + i;
        if (t < sg.end) raw[i] = scan_dt_raw(p, t, h);
      }
    };
    if (nc > 0) fetch(0);
    for (int c = 0; c < nc; ++c) {
      const int b3 = c % 3;
      if (c >= 3) {
        ok = mbar_wait(&bars->sc_free[b3], (c / 3 - 1) & 1, w);
        if (!ok) break;
      }
      Scal& sc = scal[b3];
      float d[4], inc[4], suf[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long long t = sg.begin + static_cast<long long>(c) * kQ + lane * 4 + i;
        d[i] = t < sg.end ? scan_dt(p, raw[i], bias) : 0.0f;
      }
      if (c + 1 < nc) fetch(c + 1);
      // sums within blocks of 32 tokens (8 lanes): inclusive before, exclusive behind
      float run = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) inc[i] = (run += d[i] * A2);
      float back = 0.0f;
#pragma unroll
      for (int i = 3; i >= 0; --i) {
        suf[i] = back;
        back += d[i] * A2;
      }
      float pre = run, post = back;  // scans of the lanes' sums
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        const float a = __shfl_up_sync(0xFFFFFFFFu, pre, o, 8), z = __shfl_down_sync(0xFFFFFFFFu, post, o, 8);
        if ((lane & 7) >= o) pre += a;
        if ((lane & 7) + o < 8) post += z;
      }
      const float before = __shfl_up_sync(0xFFFFFFFFu, pre, 1, 8), behind = __shfl_down_sync(0xFFFFFFFFu, post, 1, 8);
      if (lane & 7) {
#pragma unroll
        for (int i = 0; i < 4; ++i) inc[i] += before;
      }
      if ((lane & 7) != 7) {
#pragma unroll
        for (int i = 0; i < 4; ++i) suf[i] += behind;
      }
      float bt[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) bt[k] = __shfl_sync(0xFFFFFFFFu, pre, 8 * k + 7);
      const int blk = lane >> 3;
      const float head = (blk > 0 ? bt[0] : 0.0f) + (blk > 1 ? bt[1] : 0.0f) + (blk > 2 ? bt[2] : 0.0f);
      float4 v;
      v = make_float4(inc[0], inc[1], inc[2], inc[3]);
      reinterpret_cast<float4*>(sc.l)[lane] = v;
      reinterpret_cast<float4*>(sc.u)[lane] = make_float4(ex2(v.x), ex2(v.y), ex2(v.z), ex2(v.w));
      reinterpret_cast<float4*>(sc.e)[lane] =
          make_float4(ex2(head + v.x), ex2(head + v.y), ex2(head + v.z), ex2(head + v.w));
      reinterpret_cast<float4*>(sc.d)[lane] = make_float4(d[0], d[1], d[2], d[3]);
      float between = 0.0f;
#pragma unroll
      for (int b = 1; b <= 4; ++b) {
        if (b > blk) {
          if (b - 1 > blk) between += bt[b - 1];
          reinterpret_cast<float4*>(sc.f[b - 1])[lane] =
              make_float4(d[0] * ex2(suf[0] + between), d[1] * ex2(suf[1] + between), d[2] * ex2(suf[2] + between),
                          d[3] * ex2(suf[3] + between));
        }
      }
      const float total = bt[0] + bt[1] + bt[2] + bt[3];
      log_sum += total;
      if (lane == 0) sc.total = ex2(total);
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->sc_full[b3]);
    }
    if (STATES && ok && pt == 0 && lane == 0)
      p.seg_log[static_cast<long long>(seg) * p.heads + h] = log_sum * (1.0f / kLog2e);
  } else if (warp >= 4 && warp < 12) {
    // ------------------------------------------------------------ G, then y
    if constexpr (!STATES) {
      w.where = kWaitEpilogue;
      const int wg = (warp - 4) >> 2, q = warp & 3;
      const int t = 32 * q + lane;
      const uint32_t lanes = static_cast<uint32_t>(32 * q) << 16;
      const uint32_t sS = tmem + lanes + kColS + wg * 128, sY = tmem + lanes + kColY + wg * kP;
      const uint32_t sYo = tmem + lanes + kColYo;
      const float Dh = p.D ? __ldg(p.D + h) : 0.0f;
      __nv_bfloat16* gy = static_cast<__nv_bfloat16*>(p.y) + static_cast<long long>(h) * p.dim + p0;
      const __nv_bfloat16* gz =
          p.z ? static_cast<const __nv_bfloat16*>(p.z) + static_cast<long long>(h) * p.dim + p0 : nullptr;
      for (int c = wg; c < nc; c += 2) {
        const int b3 = c % 3;
        const uint32_t par = (c >> 1) & 1;
        if (!mbar_wait(&bars->sc_full[b3], (c / 3) & 1, w)) break;
        if (!mbar_wait(&bars->s_full[wg], par, w)) break;
        tc_fence_after_sync();
        const Scal& sc = scal[b3];
        const float u = sc.u[t], lt = sc.l[t];
        for (int b = 0; b < 4; ++b) {
          uint32_t o[16];
          if (b <= q) {
            uint32_t r[2][16];
            tmem_ld_32x32b_x16(sS + 32 * b, r[0]);
            tmem_ld_32x32b_x16(sS + 32 * b + 16, r[1]);
            tmem_wait_ld();
            if (b < q) {
              const float2* f = reinterpret_cast<const float2*>(sc.f[q - 1] + 32 * b);
              const float2 u2 = make_float2(u, u);
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float2 s2 = make_float2(__uint_as_float(r[i >> 3][2 * (i & 7)]),
                                              __uint_as_float(r[i >> 3][2 * (i & 7) + 1]));
                const float2 v = mul2(mul2(s2, f[i]), u2);
                o[i] = bf16_pair(v.x, v.y);
              }
            } else {
              const float2* ls = reinterpret_cast<const float2*>(sc.l + 32 * b);
              const float2* ds = reinterpret_cast<const float2*>(sc.d + 32 * b);
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float2 l2 = ls[i], d2 = ds[i];
                const float a = __uint_as_float(r[i >> 3][2 * (i & 7)]) * (ex2(lt - l2.x) * d2.x);
                const float z = __uint_as_float(r[i >> 3][2 * (i & 7) + 1]) * (ex2(lt - l2.y) * d2.y);
                o[i] = bf16_pair(2 * i <= lane ? a : 0.0f, 2 * i + 1 <= lane ? z : 0.0f);
              }
            }
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = 0;
          }
          // columns 16 b .. 16 b + 15 of S have been read by this lane already
          tmem_st_32x32b_x16(sS + 16 * b, o);
        }
        tmem_wait_st();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->g_full[wg]);

        const long long row = sg.begin + static_cast<long long>(c) * kQ + t;
        const bool live = row < sg.end;
        uint4 zv[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (gz && live && 8 * i < pdims) zv[i] = __ldcs(reinterpret_cast<const uint4*>(gz + row * p.ldz) + i);
        if (!mbar_wait(&bars->done[wg], par, w)) break;
        tc_fence_after_sync();
        const float e = sc.e[t];
        const uint32_t xrow = sbase + wg * L::kStage + stage_x;
#pragma unroll
        for (int pc = 0; pc < 4; ++pc) {
          uint32_t ry[16], ro[16];
          tmem_ld_32x32b_x16(sY + 16 * pc, ry);
          tmem_ld_32x32b_x16(sYo + 16 * pc, ro);
          uint4 xv[2];
          xv[0] = ld_shared_v4(xrow + swz_offset(t, 2 * pc, 128));
          xv[1] = ld_shared_v4(xrow + swz_offset(t, 2 * pc + 1, 128));
          tmem_wait_ld();
          uint32_t out[8];
          const uint32_t* xw = reinterpret_cast<const uint32_t*>(xv);
          const uint32_t* zw = reinterpret_cast<const uint32_t*>(zv) + 8 * pc;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float a = fmaf(e, __uint_as_float(ro[2 * i]), __uint_as_float(ry[2 * i]));
            float b = fmaf(e, __uint_as_float(ro[2 * i + 1]), __uint_as_float(ry[2 * i + 1]));
            a = fmaf(Dh, bf_lo(xw[i]), a);
            b = fmaf(Dh, bf_hi(xw[i]), b);
            if (gz) {
              a *= silu(bf_lo(zw[i]));
              b *= silu(bf_hi(zw[i]));
            }
            out[i] = bf16_pair(a, b);
          }
          if (live) {
            uint4* dst = reinterpret_cast<uint4*>(gy + row * p.ldy + 16 * pc);
            if (16 * pc < pdims) dst[0] = make_uint4(out[0], out[1], out[2], out[3]);
            if (16 * pc + 8 < pdims) dst[1] = make_uint4(out[4], out[5], out[6], out[7]);
          }
          if (pc == 3) {
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(&bars->yo_free);
              mbar_arrive(&bars->xfree[wg]);
              mbar_arrive(&bars->sc_free[b3]);
            }
          }
        }
      }
    }
  } else if (warp >= 12 && warp < 16) {
    // ------------------------------------------------------------ Xw
    w.where = kWaitTransform;
    const int s = threadIdx.x - 384;  // row
    const uint32_t hi = sbase + L::kXw, lo = hi + kAtom;
    for (int c = 0; c < nc; ++c) {
      const int b3 = c % 3, sb = c & 1;
      const uint32_t st = sbase + sb * L::kStage;
      const long long left = sg.end - sg.begin - static_cast<long long>(c) * kQ;
      if (!mbar_wait(&bars->sc_full[b3], (c / 3) & 1, w)) break;
      if (!mbar_wait(&bars->full_x[sb], (c >> 1) & 1, w)) break;
      const float ws = scal[b3].f[3][s];
      uint32_t vh[32], vl[32];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint4 x = ld_shared_v4(st + stage_x + swz_offset(s, i, 128));
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float a = 0.0f, b = 0.0f;
          if (s < left) a = ws * bf_lo(xs[k]), b = ws * bf_hi(xs[k]);
          const uint32_t hp = bf16_pair(a, b);
          vh[4 * i + k] = hp;
          vl[4 * i + k] = bf16_pair(a - bf_lo(hp), b - bf_hi(hp));
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->sc_free[b3]);
      if (c >= 1 && !mbar_wait(&bars->ds_full, (c - 1) & 1, w)) break;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t off = swz_offset(s, i, 128);
        st_shared_v4(hi + off, vh[4 * i], vh[4 * i + 1], vh[4 * i + 2], vh[4 * i + 3]);
        st_shared_v4(lo + off, vl[4 * i], vl[4 * i + 1], vl[4 * i + 2], vl[4 * i + 3]);
      }
      if (left < kQ) {
        // rows behind the sequence hold what lies there; a zero factor would not stop a NaN
        if (!mbar_wait(&bars->full_bc[sb], (c >> 1) & 1, w)) break;
        if (s >= left) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t off = swz_offset(s, i, 128);
            st_shared_v4(st + stage_x + off, 0, 0, 0, 0);
#pragma unroll
            for (int a = 0; a < NA; ++a) st_shared_v4(st + stage_b + a * kAtom + off, 0, 0, 0, 0);
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->xw_full);
    }
  } else if (warp >= 16) {
    // ------------------------------------------------------------ state
    w.where = kWaitTransform;
    const int n = threadIdx.x - 512;  // state element (lane of tensor memory)
    const int q = warp & 3;
    const bool wlive = 32 * q < N;    // this warp has state elements
    const bool live = n < N;
    const uint32_t sD = tmem + (static_cast<uint32_t>(32 * q) << 16) + kColDs;
    float hv[kP];
#pragma unroll
    for (int i = 0; i < kP; ++i) hv[i] = 0.0f;
    auto add_state = [&](const float* src, float decay) {
#pragma unroll
      for (int i = 0; i < kP; ++i)
        if (live && i < pdims) hv[i] = fmaf(hv[i], decay, src[i * N + n]);
    };
    if (!STATES) {
      if (sg.count == 1) {
        if (in) add_state(in, 0.0f);
      } else {
        add_state(p.seg_state + (sg.first + sg.count - 1) * per_slot + head_at, 0.0f);
        for (int k = 0; k < sg.j; ++k)
          add_state(p.seg_state + (sg.first + k) * per_slot + head_at,
                    expf(p.seg_log[static_cast<long long>(sg.first + k) * p.heads + h]));
      }
    }
    auto put_h = [&]() {
      if (n < 64 * NA) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          st_shared_v4(sbase + L::kH + swz_offset(n, i, 128), bf16_pair(hv[8 * i], hv[8 * i + 1]),
                       bf16_pair(hv[8 * i + 2], hv[8 * i + 3]), bf16_pair(hv[8 * i + 4], hv[8 * i + 5]),
                       bf16_pair(hv[8 * i + 6], hv[8 * i + 7]));
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->h_full);
    };
    if (!STATES && nc > 0) put_h();
    bool ok = true;
    for (int c = 0; c < nc; ++c) {
      const int b3 = c % 3;
      ok = mbar_wait(&bars->sc_full[b3], (c / 3) & 1, w);
      if (!ok) break;
      const float decay = scal[b3].total;
      ok = mbar_wait(&bars->ds_full, c & 1, w);
      if (!ok) break;
      tc_fence_after_sync();
      if (wlive) {
#pragma unroll
        for (int pc = 0; pc < 4; ++pc) {
          uint32_t r[16];
          tmem_ld_32x32b_x16(sD + 16 * pc, r);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i)
            hv[16 * pc + i] = live ? fmaf(hv[16 * pc + i], decay, __uint_as_float(r[i])) : 0.0f;
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&bars->ds_free);
        mbar_arrive(&bars->sc_free[b3]);
      }
      if (!STATES && c + 1 < nc) {
        ok = mbar_wait(&bars->done[c & 1], (c >> 1) & 1, w);  // the product that reads the old H
        if (!ok) break;
        put_h();
      }
    }
    if (ok) {
      float* dst = STATES ? p.seg_state + seg * per_slot + head_at
                          : (last && p.state_out && slot >= 0 ? p.state_out + slot * per_slot + head_at : nullptr);
      if (dst && live) {
#pragma unroll
        for (int i = 0; i < kP; ++i)
          if (i < pdims) dst[i * N + n] = hv[i];
      }
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 1) tmem_dealloc(tmem, kCols);
}

int make_map(CUtensorMap* m, const void* base, int inner, int mid, long long rows, long long ld, const char* what) {
  auto fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(tensor_map_encoder());
  if (!fn) return set_error(SMM_ERR_CUDA, "cuTensorMapEncodeTiled unavailable from the driver");
  // (element, head or group, token); elements past a head's end read as zero
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(mid), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(inner) * 2, static_cast<cuuint64_t>(ld) * 2};
  cuuint32_t box[3] = {64, 1, kQ};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return set_error(SMM_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d) for %s: %d x %d x %lld, row stride %lld",
                     int(r), what, inner, mid, rows, ld);
  return SMM_OK;
}

template <int NA, bool STATES>
int launch_one(const Tmaps& maps, const ScanParams& p, unsigned grid, int ptiles, cudaStream_t st) {
  auto kern = scan_umma_kernel<NA, STATES>;
  static std::once_flag once[64];
  int dev = 0;
  SMM_CUDA_TRY(cudaGetDevice(&dev), "cudaGetDevice");
  cudaError_t err = cudaSuccess;
  auto set = [&] { err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<NA>::kBytes); };
  if (dev < 64) std::call_once(once[dev], set);
  else set();
  SMM_CUDA_TRY(err, "selective scan shared memory size");
  kern<<<grid, kThreads, Smem<NA>::kBytes, st>>>(maps, p, ptiles);
  count_launch();
  SMM_CUDA_TRY(cudaGetLastError(), "selective scan (tensor core) launch");
  return SMM_OK;
}

}  // namespace

// bf16, whole 16-byte pieces everywhere, state_dim of one 128-row tile, and prompts
// long enough that tiles of 128 tokens are not mostly empty.
bool scan_umma_fits(const ScanParams& p, int dtype) {
  return dtype == SMM_DTYPE_BF16 && p.dim % 8 == 0 && p.state_dim % 8 == 0 && p.state_dim <= 128 && p.ldx % 8 == 0 &&
         p.ldb % 8 == 0 && p.ldc % 8 == 0 && p.ldy % 8 == 0 && (!p.z || p.ldz % 8 == 0) && aligned_to(p.x, 16) &&
         aligned_to(p.B, 16) && aligned_to(p.C, 16) && aligned_to(p.y, 16) && aligned_to(p.z, 16) &&
         p.tokens >= 16LL * p.nseq;
}

// Segment length of the tensor-core kernel: whole chunks, so that the waves of
// CTAs (one per SM) times the chunks of each are fewest.  A split adds the
// states' launch, about half the work of the outputs'.
int umma_seg_len(long long tokens, int nseq, int heads, int dim) {
  const int whole = static_cast<int>(std::max<long long>(tokens, 1));
  if (nseq < 1 || heads < 1) return whole;
  const long long ctas = static_cast<long long>(heads) * ((dim + kP - 1) / kP) * nseq;
  const long long chunks = (tokens / nseq + kQ - 1) / kQ;
  long long best = 0;
  int best_parts = 1;
  for (int parts = 1; parts <= 32 && parts <= chunks; ++parts) {
    const long long len = (chunks + parts - 1) / parts;
    const long long waves = (ctas * parts + 147) / 148;
    const long long waves_st = (ctas * (parts - 1) + 147) / 148;
    // in half chunks; 2 for a CTA's start
    const long long cost = waves * (2 * len + 4) + (parts > 1 ? waves_st * (len + 4) + 4 : 0);
    if (parts == 1 || cost < best) best = cost, best_parts = parts;
  }
  if (best_parts == 1) return whole;
  return static_cast<int>((chunks + best_parts - 1) / best_parts) * kQ;
}

int scan_umma_launch(ScanParams& p, cudaStream_t st) {
  const int ptiles = (p.dim + kP - 1) / kP;
  const long long blocks = max_segments(p.tokens, p.nseq, p.seg_len) * p.heads * ptiles;
  if (blocks > 0x7FFFFFFFLL) return set_error(SMM_ERR_INVALID, "selective scan too large for one launch");
  Tmaps maps;
  if (int rc = make_map(&maps.x, p.x, p.dim, p.heads, p.tokens, p.ldx, "x")) return rc;
  if (int rc = make_map(&maps.b, p.B, p.state_dim, p.groups, p.tokens, p.ldb, "B")) return rc;
  if (int rc = make_map(&maps.c, p.C, p.state_dim, p.groups, p.tokens, p.ldc, "C")) return rc;
  const unsigned grid = static_cast<unsigned>(blocks);
  if (p.state_dim <= 64) {
    if (p.split)
      if (int rc = launch_one<1, true>(maps, p, grid, ptiles, st)) return rc;
    return launch_one<1, false>(maps, p, grid, ptiles, st);
  }
  if (p.split)
    if (int rc = launch_one<2, true>(maps, p, grid, ptiles, st)) return rc;
  return launch_one<2, false>(maps, p, grid, ptiles, st);
}

}  // namespace smm
