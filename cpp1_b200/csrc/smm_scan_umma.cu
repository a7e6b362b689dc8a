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
// Warps: 0 loads (TMA), 1 issues the products, 2 and 3 compute the decays in turn, 4-7 and 8-11
// form G and write y of the even and the odd chunks, 12-19 form Xw, 20-23 carry
// the state.  Every wait is bounded; on expiry the CTA records it and leaves.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>
#include <type_traits>
#include <utility>

#include "smm_scan.cuh"

namespace smm {

void* tensor_map_encoder();  // smm_lib.cu

namespace {

constexpr int kQ = 128;         // tokens per chunk
constexpr int kP = 64;          // dims per CTA
constexpr int kThreads = 768;
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
  uint64_t full_bc[2], full_x[2], full_z[2], done[2], xfree[2], bfree[2], zfree[2], s_full[2], g_full[2];
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
  CUtensorMap x, b, c, y, z;
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1,
                                            int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
// Tile in shared memory -> global; returns once the tile has been read.
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];\n\t"
      "cp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group.read 0;" ::"l"(reinterpret_cast<uint64_t>(map)),
      "r"(src), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
// The whole warp reaches these together and only lane `leader` issues: with the
// predicate on the instruction, control flow stays uniform and the compiler
// keeps the descriptors in uniform registers.  (From one lane's branch, each
// product cost 65 to 110 cycles of register moves, 2600 and more a chunk.)
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b32 t;\n\telect.sync t|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(r));
  return r;
}
// The descriptors are given as their low word of the stage's first product and
// their high word; the step's offset is added inside, so that the compiler
// does not keep a register for every step of every product.
template <uint32_t OA, uint32_t OB, bool FIRST>
__device__ __forceinline__ void umma_ss(uint32_t leader, uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo,
                                        uint32_t b_hi, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b32 x, y;\n\t.reg .b64 da, db;\n\t"
      "add.u32 x, %1, %7;\n\tadd.u32 y, %3, %8;\n\tmov.b64 da, {x, %2};\n\tmov.b64 db, {y, %4};\n\t"
      "setp.ne.b32 p, %9, 0;\n\tsetp.ne.b32 e, %6, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n\t}\n" ::"r"(d),
      "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(leader), "n"(OA), "n"(OB), "n"(FIRST ? 0 : 1)
      : "memory");
}
// A from tensor memory (bf16, two per column), B from shared memory
template <uint32_t OA, uint32_t OB, bool FIRST>
__device__ __forceinline__ void umma_ts(uint32_t leader, uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi,
                                        uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b32 x, y;\n\t.reg .b64 db;\n\t"
      "add.u32 x, %1, %6;\n\tadd.u32 y, %2, %7;\n\tmov.b64 db, {y, %3};\n\t"
      "setp.ne.b32 p, %8, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [x], db, %4, p;\n\t}\n" ::"r"(d),
      "r"(a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(leader), "n"(OA), "n"(OB), "n"(FIRST ? 0 : 1)
      : "memory");
}
template <int... K, typename F>
__device__ __forceinline__ void steps_of(std::integer_sequence<int, K...>, F&& f) {
  (f(std::integral_constant<int, K>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void steps(F&& f) {
  steps_of(std::make_integer_sequence<int, N>{}, f);
}
__device__ __forceinline__ void umma_commit_by(uint32_t leader, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar)),
      "r"(leader)
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
// Whether to give up a wait (called every 64 tries, out of line: a dozen roles' waits
// share it).  t0 is 0 before the first call.
__device__ __forceinline__ bool give_up(const WaitCtx& w, uint64_t& t0) {
  if (*w.abort_flag) return true;
  const uint64_t t = globaltimer_ns();
  if (t0 == 0) t0 = t;
  if (t - t0 <= w.limit_ns) return false;
  *w.abort_flag = 1;
  if (w.status) atomicOr(w.status, kDevErrTimeout | w.where);
  return true;
}
// mbar_wait with a short inline path.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, const WaitCtx& w) {
  const uint32_t a = smem_u32(bar);
  if (mbar_try_wait(a, parity)) return true;
  uint64_t t0 = 0;
  uint32_t n = 0;
  while (!mbar_try_wait(a, parity))
    if ((++n & 63u) == 0 && give_up(w, t0)) return false;
  return true;
}
template <int R>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R));
}
template <int R>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R));
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
// Registers into 32 lanes x 8 consecutive columns of tensor memory.
__device__ __forceinline__ void tmem_st_32x32b_x8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void st_shared_v4(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// STATES: the first launch of a split scan (B, x and the state only).
template <int NA, bool STATES>
__global__ void __launch_bounds__(kThreads, 1)
    scan_umma_kernel(const __grid_constant__ Tmaps maps, const ScanParams p, int ptiles) {
  using L = Smem<NA>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Segment sseg;
  __shared__ float seg_sum[2];
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
      mbar_init(&bars->full_z[i], 1);
      mbar_init(&bars->xfree[i], 1);
      mbar_init(&bars->bfree[i], 1);
      mbar_init(&bars->zfree[i], 4);
      mbar_init(&bars->s_full[i], 1);
      mbar_init(&bars->g_full[i], 4);
    }
    mbar_init(&bars->xw_full, 8);
    mbar_init(&bars->ds_full, 1);
    mbar_init(&bars->ds_free, 4);
    mbar_init(&bars->h_full, 4);
    mbar_init(&bars->yo_free, 4);
    for (int i = 0; i < 3; ++i) {
      mbar_init(&bars->sc_full[i], 1);
      mbar_init(&bars->sc_free[i], STATES ? 12 : 16);
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
  constexpr uint32_t stage_c = 0, stage_b = NA * kAtom, stage_x = 2 * NA * kAtom;

  // The launch's 6 x 80 registers per warpgroup's thread, shared out by need:
  // 64 (loads, products, decays), 2 x 96 (G and y), 2 x 64 (Xw), 96 (state) = 480.
  // A spill costs a trip to L2 here: shared memory leaves L1 too small for the stacks.
  if (warp < 4) {
    regs_dec<64>();
  if (warp == 0) {
    // ------------------------------------------------------------ loads
    if (lane == 0) {
      w.where = kWaitProducer;
      const bool gated = !STATES && p.z != nullptr;
      // next chunk of each kind of load; z goes where B was, once dS has read it
      int c_bc = 0, c_x = 0, c_z = 0;
      uint32_t idle = 0;
      uint64_t t0 = 0;
      const int row0 = static_cast<int>(sg.begin);
      while (c_bc < nc || c_x < nc || (gated && c_z < nc)) {
        bool did = false;
        if (gated && c_z < c_bc && mbar_test(&bars->bfree[c_z & 1], (c_z >> 1) & 1)) {
          const int s = c_z & 1;
          mbar_arrive_expect_tx(&bars->full_z[s], kAtom);
          tma_load_3d(sbase + s * L::kStage + stage_b, &maps.z, &bars->full_z[s], p0, h, row0 + c_z * kQ);
          ++c_z;
          did = true;
        }
        if (c_bc < nc &&
            (c_bc < 2 || (mbar_test(&bars->done[c_bc & 1], ((c_bc >> 1) - 1) & 1) &&
                          (!gated || (c_z > c_bc - 2 && mbar_test(&bars->zfree[c_bc & 1], ((c_bc >> 1) - 1) & 1)))))) {
          const int s = c_bc & 1;
          const uint32_t st = sbase + s * L::kStage;
          mbar_arrive_expect_tx(&bars->full_bc[s], (STATES ? 1 : 2) * NA * kAtom);
#pragma unroll
          for (int a = 0; a < NA; ++a) {
            if (!STATES) tma_load_3d(st + stage_c + a * kAtom, &maps.c, &bars->full_bc[s], a * 64, g, row0 + c_bc * kQ);
            tma_load_3d(st + stage_b + a * kAtom, &maps.b, &bars->full_bc[s], a * 64, g, row0 + c_bc * kQ);
          }
          ++c_bc;
          did = true;
        }
        if (c_x < c_bc && (c_x < 2 || STATES || mbar_test(&bars->xfree[c_x & 1], ((c_x >> 1) - 1) & 1))) {
          const int s = c_x & 1;
          mbar_arrive_expect_tx(&bars->full_x[s], kAtom);
          tma_load_3d(sbase + s * L::kStage + stage_x, &maps.x, &bars->full_x[s], p0, h, row0 + c_x * kQ);
          ++c_x;
          did = true;
        }
        if (did)
          idle = 0, t0 = 0;
        else if ((++idle & 255u) == 0 && give_up(w, t0))
          break;
      }
      // after an abort, copies in flight land before the CTA leaves
      if (*w.abort_flag) {
        int none = 0;
        WaitCtx dw{&none, p.status, p.wait_limit_ns > 1000000000ull ? p.wait_limit_ns : 1000000000ull, kWaitDrain};
        for (int c = c_bc > 2 ? c_bc - 2 : 0; c < c_bc; ++c) wait_bar(&bars->full_bc[c & 1], (c >> 1) & 1, dw);
        for (int c = c_x > 2 ? c_x - 2 : 0; c < c_x; ++c) wait_bar(&bars->full_x[c & 1], (c >> 1) & 1, dw);
        for (int c = c_z > 2 ? c_z - 2 : 0; c < c_z; ++c) wait_bar(&bars->full_z[c & 1], (c >> 1) & 1, dw);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ products
    constexpr uint32_t idS = make_idesc(kFmtBF16, 128, 128, 0, 0);
    constexpr uint32_t idY = make_idesc(kFmtBF16, 128, kP, 0, 1);
    constexpr uint32_t idD = make_idesc(kFmtBF16, 128, kP, 1, 1);
    const int ksteps = (N + 15) / 16;
    const uint32_t leader = elect_one();
    // descriptors of stage 0; a stage is kSt further.  Only the low word, the
    // start address in 16-byte units, changes with stage and step.
    constexpr uint32_t kSt = L::kStage >> 4;
    auto lo = [](uint64_t d) { return static_cast<uint32_t>(d); };
    const uint64_t dK = make_smem_desc(sbase, 16, 1024, kLayoutSw128);      // K-major
    const uint64_t dM = make_smem_desc(sbase, kAtom, 1024, kLayoutSw128);   // MN-major
    const uint32_t hK = static_cast<uint32_t>(dK >> 32), hM = static_cast<uint32_t>(dM >> 32);
    auto ready = [&](uint64_t* bar, uint32_t parity) { return __any_sync(0xFFFFFFFFu, mbar_test(bar, parity)) != 0; };
    int s_next = STATES ? nc : 0, g_next = 0, sub = 0;
    uint32_t idle = 0;
    uint64_t t_idle = 0;
    while (g_next < nc) {
      bool did = false;
      if (!STATES && s_next < nc && s_next < g_next + 2 && ready(&bars->full_bc[s_next & 1], (s_next >> 1) & 1)) {
        // the loads of chunk c waited for every product of chunk c - 2, so S and G are free
        tc_fence_after_sync();
        const int s = s_next & 1;
        const uint32_t base = lo(dK) + s * kSt;
        steps<4 * NA>([&](auto kc) {
          constexpr int k = decltype(kc)::value;
          constexpr uint32_t off = ((k >> 2) * kAtom + (k & 3) * 32) >> 4;
          if (k < ksteps)
            umma_ss<off + (stage_c >> 4), off + (stage_b >> 4), k == 0>(leader, tmem + kColS + s * 128, base, hK, base, hK,
                                                                       idS);
        });
        umma_commit_by(leader, &bars->s_full[s]);
        ++s_next;
        did = true;
      } else if (STATES || g_next < s_next) {
        const int c = g_next, s = c & 1;
        if (sub == 0) {
          if (ready(&bars->xw_full, c & 1) && (c == 0 || ready(&bars->ds_free, (c - 1) & 1)) &&
              ready(&bars->full_bc[s], (c >> 1) & 1) && ready(&bars->full_x[s], (c >> 1) & 1)) {
            tc_fence_after_sync();
            const uint32_t base = lo(dM) + s * kSt;
            steps<16>([&](auto kc) {
              constexpr int k = decltype(kc)::value;
              constexpr uint32_t kk = (k & 7) * 128;
              umma_ss<(stage_b >> 4) + kk, (L::kXw >> 4) + (k >> 3) * (kAtom >> 4) + kk, k == 0>(
                  leader, tmem + kColDs, base, hM, lo(dM), hM, idD);
            });
            umma_commit_by(leader, &bars->ds_full);
            if (!STATES) umma_commit_by(leader, &bars->bfree[s]);
            if (STATES) {
              umma_commit_by(leader, &bars->done[s]);
              ++g_next;
            } else {
              sub = 1;
            }
            did = true;
          }
        } else if (sub == 1) {
          if (ready(&bars->g_full[s], (c >> 1) & 1)) {
            tc_fence_after_sync();
            const uint32_t base = lo(dM) + s * kSt;
            steps<8>([&](auto kc) {
              constexpr int k = decltype(kc)::value;
              umma_ts<k * 8, (stage_x >> 4) + k * 128, k == 0>(leader, tmem + kColY + s * kP, tmem + kColS + s * 128, base,
                                                               hM, idY);
            });
            sub = 2;
            did = true;
          }
        } else {
          if (ready(&bars->h_full, c & 1) && (c == 0 || ready(&bars->yo_free, (c - 1) & 1))) {
            tc_fence_after_sync();
            const uint32_t base = lo(dK) + s * kSt;
            steps<4 * NA>([&](auto kc) {
              constexpr int k = decltype(kc)::value;
              constexpr uint32_t off = ((k >> 2) * kAtom + (k & 3) * 32) >> 4;
              if (k < ksteps)
                umma_ss<off + (stage_c >> 4), (L::kH >> 4) + k * 128, k == 0>(leader, tmem + kColYo, base, hK, lo(dM), hM,
                                                                             idY);
            });
            umma_commit_by(leader, &bars->done[s]);
            sub = 0;
            ++g_next;
            did = true;
          }
        }
      }
      if (did) {
        idle = 0;
      } else if ((++idle & 1023u) == 0) {
        // the timer is slow to read: now and then is enough for the limit
        if (__any_sync(0xFFFFFFFFu, *w.abort_flag != 0)) break;
        if (idle == 1024u) t_idle = globaltimer_ns();
        if (__any_sync(0xFFFFFFFFu, globaltimer_ns() - t_idle > w.limit_ns)) {
          *w.abort_flag = 1;
          if (w.status && lane == 0) atomicOr(w.status, kDevErrTimeout | kWaitMma);
          break;
        }
      }
    }
    // every product has completed, and its arrivals have landed, before the CTA leaves
    int none = 0;
    WaitCtx dw{&none, p.status, p.wait_limit_ns > 1000000000ull ? p.wait_limit_ns : 1000000000ull, kWaitDrain};
    umma_commit_by(leader, &bars->drain);
    wait_bar(&bars->drain, 0, dw);
  } else {
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
    if (warp - 2 < nc) fetch(warp - 2);
    for (int c = warp - 2; c < nc; c += 2) {
      const int b3 = c % 3;
      if (c >= 3) {
        ok = wait_bar(&bars->sc_free[b3], (c / 3 - 1) & 1, w);
        if (!ok) break;
      }
      Scal& sc = scal[b3];
      float d[4], inc[4], suf[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long long t = sg.begin + static_cast<long long>(c) * kQ + lane * 4 + i;
        d[i] = t < sg.end ? scan_dt(p, raw[i], bias) : 0.0f;
      }
      if (c + 2 < nc) fetch(c + 2);
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
    if (lane == 0) seg_sum[warp - 2] = log_sum;
  }
  } else if (warp < 12) {
    regs_inc<96>();
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
      const bool gated = p.z != nullptr;
      for (int c = wg; c < nc; c += 2) {
        const int b3 = c % 3;
        const uint32_t par = (c >> 1) & 1;
        if (!wait_bar(&bars->sc_full[b3], (c / 3) & 1, w)) break;
        if (!wait_bar(&bars->s_full[wg], par, w)) break;
        tc_fence_after_sync();
        const Scal& sc = scal[b3];
        const float u = sc.u[t], lt = sc.l[t];
        // 16 columns at a time: the block of columns b is off the diagonal for b < q
#pragma unroll 1
        for (int j = 0; j < 8; ++j) {
          const int b = j >> 1;
          uint32_t o[8];
          if (b <= q) {
            uint32_t r[16];
            tmem_ld_32x32b_x16(sS + 16 * j, r);
            const float2* f = reinterpret_cast<const float2*>((b < q ? sc.f[q - 1] : sc.d) + 16 * j);
            if (b < q) {
              const float2 u2 = make_float2(u, u);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float2 v = mul2(
                    mul2(make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), f[i]), u2);
                o[i] = bf16_pair(v.x, v.y);
              }
            } else {
              const float2* ls = reinterpret_cast<const float2*>(sc.l + 16 * j);
              const int top = lane - 16 * (j & 1);  // columns up to here are at or before this row
              float2 g2[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float2 l2 = ls[i], d2 = f[i];
                g2[i] = make_float2(ex2(lt - l2.x) * d2.x, ex2(lt - l2.y) * d2.y);
              }
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 8; ++i)
                o[i] = bf16_pair(2 * i <= top ? __uint_as_float(r[2 * i]) * g2[i].x : 0.0f,
                                 2 * i + 1 <= top ? __uint_as_float(r[2 * i + 1]) * g2[i].y : 0.0f);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = 0;
          }
          // columns 8 j .. 8 j + 7 of S have been read by this lane already
          tmem_st_32x32b_x8(sS + 8 * j, o);
        }
        tmem_wait_st();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->g_full[wg]);

        // y takes x's place in shared memory, row by row, and leaves as one tile (or by
        // rows where the chunk ends before the tile)
        if (!wait_bar(&bars->full_x[wg], par, w)) break;
        if (gated && !wait_bar(&bars->full_z[wg], par, w)) break;
        if (!wait_bar(&bars->done[wg], par, w)) break;
        tc_fence_after_sync();
        const float e = sc.e[t];
        uint8_t* xt = smem + wg * L::kStage + stage_x;
        const uint8_t* zt = smem + wg * L::kStage + stage_b;
#pragma unroll 1
        for (int k = 0; k < 4; ++k) {
          uint32_t ry[16], ro[16], xw[8], zw[8], out[8];
          tmem_ld_32x32b_x16(sY + 16 * k, ry);
          tmem_ld_32x32b_x16(sYo + 16 * k, ro);
          const uint32_t o0 = swz_offset(t, 2 * k, 128), o1 = swz_offset(t, 2 * k + 1, 128);
          *reinterpret_cast<uint4*>(xw) = *reinterpret_cast<const uint4*>(xt + o0);
          *reinterpret_cast<uint4*>(xw + 4) = *reinterpret_cast<const uint4*>(xt + o1);
          if (gated) {
            *reinterpret_cast<uint4*>(zw) = *reinterpret_cast<const uint4*>(zt + o0);
            *reinterpret_cast<uint4*>(zw + 4) = *reinterpret_cast<const uint4*>(zt + o1);
          }
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float a = fmaf(Dh, bf_lo(xw[i]), fmaf(e, __uint_as_float(ro[2 * i]), __uint_as_float(ry[2 * i])));
            float b = fmaf(Dh, bf_hi(xw[i]), fmaf(e, __uint_as_float(ro[2 * i + 1]), __uint_as_float(ry[2 * i + 1])));
            if (gated) {
              a *= silu(bf_lo(zw[i]));
              b *= silu(bf_hi(zw[i]));
            }
            out[i] = bf16_pair(a, b);
          }
          *reinterpret_cast<uint4*>(xt + o0) = make_uint4(out[0], out[1], out[2], out[3]);
          *reinterpret_cast<uint4*>(xt + o1) = make_uint4(out[4], out[5], out[6], out[7]);
        }
        tc_fence_before_sync();
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bars->yo_free);
          mbar_arrive(&bars->sc_free[b3]);
          if (gated) mbar_arrive(&bars->zfree[wg]);
        }
        const long long t0 = sg.begin + static_cast<long long>(c) * kQ;
        if (t0 + kQ <= sg.end) {
          asm volatile("bar.sync %0, 128;" ::"r"(1 + wg) : "memory");  // the four warps' rows are written
          if (q == 0 && lane == 0) {
            tma_store_3d(&maps.y, sbase + wg * L::kStage + stage_x, p0, h, static_cast<int>(t0));
            mbar_arrive(&bars->xfree[wg]);
          }
        } else {
          if (t0 + t < sg.end) {
            __nv_bfloat16* yr = gy + (t0 + t) * p.ldy;
#pragma unroll 1
            for (int i = 0; 8 * i < pdims; ++i)
              *reinterpret_cast<uint4*>(yr + 8 * i) = *reinterpret_cast<const uint4*>(xt + swz_offset(t, i, 128));
          }
          // a partial chunk is the last: nothing waits for its x tile
        }
      }
    }
  } else if (warp < 20) {
    regs_dec<64>();
    // ------------------------------------------------------------ Xw
    w.where = kWaitTransform;
    const int s = (threadIdx.x - 384) & 127;     // row
    const int i0 = warp < 16 ? 0 : 4;            // first of this thread's 16-byte pieces
    for (int c = 0; c < nc; ++c) {
      const int b3 = c % 3, sb = c & 1;
      const uint32_t st = sbase + sb * L::kStage;
      const long long left = sg.end - sg.begin - static_cast<long long>(c) * kQ;
      if (!wait_bar(&bars->sc_full[b3], (c / 3) & 1, w)) break;
      if (!wait_bar(&bars->full_x[sb], (c >> 1) & 1, w)) break;
      const float ws = scal[b3].f[3][s];
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->sc_free[b3]);
      if (c >= 1 && !wait_bar(&bars->ds_full, (c - 1) & 1, w)) break;
      const bool live = s < left;
#pragma unroll 2
      for (int i = i0; i < i0 + 4; ++i) {
        const uint32_t off = swz_offset(s, i, 128);
        const uint4 x = *reinterpret_cast<const uint4*>(smem + sb * L::kStage + stage_x + off);
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
        uint32_t vh[4], vl[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float a = live ? ws * bf_lo(xs[k]) : 0.0f, b = live ? ws * bf_hi(xs[k]) : 0.0f;
          vh[k] = bf16_pair(a, b);
          vl[k] = bf16_pair(a - bf_lo(vh[k]), b - bf_hi(vh[k]));
        }
        *reinterpret_cast<uint4*>(smem + L::kXw + off) = make_uint4(vh[0], vh[1], vh[2], vh[3]);
        *reinterpret_cast<uint4*>(smem + L::kXw + kAtom + off) = make_uint4(vl[0], vl[1], vl[2], vl[3]);
      }
      if (left < kQ) {
        // rows behind the sequence hold what lies there; a zero factor would not stop a NaN
        if (!wait_bar(&bars->full_bc[sb], (c >> 1) & 1, w)) break;
        if (s >= left) {
#pragma unroll
          for (int i = i0; i < i0 + 4; ++i) {
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
  } else {
    regs_inc<96>();
    // ------------------------------------------------------------ state
    w.where = kWaitTransform;
    const int n = threadIdx.x - 640;  // state element (lane of tensor memory)
    const int q = warp & 3;
    const bool wlive = 32 * q < N;    // this warp has state elements
    const bool live = n < N;
    const uint32_t sD = tmem + (static_cast<uint32_t>(32 * q) << 16) + kColDs;
    float hv[kP];
#pragma unroll
    for (int i = 0; i < kP; ++i) hv[i] = 0.0f;
    // eight rows at a time (pdims is a multiple of 8): more loads in flight would not fit the registers
    auto add_state = [&](const float* src, float decay) {
#pragma unroll
      for (int g8 = 0; g8 < kP / 8; ++g8) {
        if (live && 8 * g8 < pdims) {
          const float* at = src + 8 * g8 * N + n;
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = at[i * N];
#pragma unroll
          for (int i = 0; i < 8; ++i) hv[8 * g8 + i] = fmaf(hv[8 * g8 + i], decay, v[i]);
        }
        asm volatile("" ::: "memory");
      }
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
    bool ok = true;
    for (int c = 0; c < nc; ++c) {
      const int b3 = c % 3;
      if (!STATES) {
        // the product that reads the old H is done
        ok = c == 0 || wait_bar(&bars->done[(c - 1) & 1], ((c - 1) >> 1) & 1, w);
        if (!ok) break;
        put_h();
      }
      ok = wait_bar(&bars->sc_full[b3], (c / 3) & 1, w);
      if (!ok) break;
      const float decay = scal[b3].total;
      ok = wait_bar(&bars->ds_full, c & 1, w);
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
    }
    if (ok) {
      float* dst = STATES ? p.seg_state + seg * per_slot + head_at
                          : (last && p.state_out && slot >= 0 ? p.state_out + slot * per_slot + head_at : nullptr);
#pragma unroll
      for (int g8 = 0; g8 < kP / 8; ++g8) {
        if (dst && live && 8 * g8 < pdims) {
          float* at = dst + 8 * g8 * N + n;
#pragma unroll
          for (int i = 0; i < 8; ++i) at[i * N] = hv[8 * g8 + i];
        }
        asm volatile("" ::: "memory");
      }
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 1) tmem_dealloc(tmem, kCols);
  if (STATES && pt == 0 && threadIdx.x == 0)
    p.seg_log[static_cast<long long>(seg) * p.heads + h] = (seg_sum[0] + seg_sum[1]) * (1.0f / kLog2e);
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
  Tmaps maps{};
  if (int rc = make_map(&maps.x, p.x, p.dim, p.heads, p.tokens, p.ldx, "x")) return rc;
  if (int rc = make_map(&maps.b, p.B, p.state_dim, p.groups, p.tokens, p.ldb, "B")) return rc;
  if (int rc = make_map(&maps.c, p.C, p.state_dim, p.groups, p.tokens, p.ldc, "C")) return rc;
  if (int rc = make_map(&maps.y, p.y, p.dim, p.heads, p.tokens, p.ldy, "y")) return rc;
  if (p.z)
    if (int rc = make_map(&maps.z, p.z, p.dim, p.heads, p.tokens, p.ldz, "z")) return rc;
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
