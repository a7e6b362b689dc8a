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
// at most 128 tokens that lie between s and t: within blocks of 32 tokens
// u_t = exp(sum from the block's start to t),
// f[b][s] = d_s exp(sum from behind s to the start of block b).  G is S u_t f[b][s]
// off the diagonal blocks; w_s = f[4][s].  On the diagonal blocks it is exp(l_t - l_s) d_s, l being sums
// within the block: differences, so a token's exponent is cut at -130 binary orders, below which its
// factor is zero in any case, and l stays small enough for the tokens behind a
// strong one (uncut, |d A| of 1e5 put an error of 1e-2 on them).  So a quarter of the exponentials remains.
//
// Roundings: G and H as operands of products are the sum of two bf16 terms (2^-17 of each
// term of y, which is itself rounded to bf16; one term, 2^-9, added up to 1e-3 to y's error of
// 1.7e-3 from its own rounding); Xw is the sum of three (2^-24; two left an error of 2.3e-6 in the
// states, an fp32 result that is carried on, where the plain fp32 form has 0.2 to 1.7e-6).  The state itself stays in fp32
// registers, S, Y, Yo and dS are fp32 in tensor memory.
//
// A CTA takes one (segment, head, 64 dims), the hardware hands out the next as an SM
// becomes free.  (A CTA an SM that walked a fixed share of them as one stream of chunks
// saved their starts but shared out ragged ones badly: prompts of 16 tokens 195 -> 170 us,
// but 8190 ragged tokens of 24 sequences 107 -> 126, in an earlier form.)  Warps: 0 loads (TMA), 1 issues the products, 2 and 3 compute the
// decays in turn, 4-11 form G and write y of the chunk before, half of the columns each,
// 12-19 form Xw, 20-23 carry the state.  Every wait is bounded; on expiry the CTA records
// it and leaves.
//
// 4096 tokens of 64 heads of 64 x 128 take 112 us, 8190 ragged ones of 32 heads 93 us,
// 32768 of 80 heads 0.86 ms.  No one unit's time (tensor pipe 28 % busy, issue slots 44 %, shared
// memory 46 %) but a chunk's way through the roles.  (With one bf16 term for G and H, and NaN of x
// reaching the tokens before it: 101, 83 and 0.78.)
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
// Tensor memory columns.  S is 128 wide and double; G takes the place of the first
// quarter and the third one of S, each written by the warps that have read its half.
constexpr uint32_t kColS = 0, kColY = 256, kColDs = 384, kColYo = 448, kCols = 512;

constexpr int kNapLoad = 32, kNapMma = 20, kNapDecay = 100, kNapG = 32, kNapXw = 32, kNapState = 32;

struct Scal {
  float f[4][kQ];  // f[b-1][s], b = 1..4
  float l[kQ];     // log2 of the decay from the block's start through t
  float u[kQ];     // its value
  float e[kQ];     // decay from the chunk's start through t
  float d[kQ];
  float total;     // decay of the whole chunk
  float log2;      // its logarithm
  float pad[2];
};

struct Bars {
  uint64_t full_bc[2], full_x[2], xfree[2], done[2], s_full[2], g_full[2];
  uint64_t xw_full[2], ds_full[2], ds_free[2];  // by the chunk's parity
  uint64_t h_full, yo_free;
  uint64_t sc_full[3], sc_free[3];
  uint64_t drain;
  uint32_t tmem;
  int abort_flag;
  // Non-finite elements of x, by the chunk's parity: the last chunk that has one (plus 1), and by
  // dim the chunk (x 256) and 128 less its first such row.  Higher is later, so nothing is reset.
  uint32_t bad[2], bad_from[2][kP];
};

// NA: 64-wide tiles that state_dim takes (1 or 2).  The first launch of a split scan
// needs no C and no H; it has two places for Xw and dS, so that a chunk's Xw is formed
// while the product of the one before runs.
template <int NA, bool STATES>
struct Smem {
  static constexpr uint32_t kC = 0, kB = STATES ? 0 : NA * kAtom, kX = kB + NA * kAtom;  // in a stage
  static constexpr uint32_t kStage = kX + kAtom;
  static constexpr uint32_t kXw = 2 * kStage;                  // three terms
  static constexpr uint32_t kXwNext = STATES ? 3 * kAtom : 0;  // from one place to the other
  static constexpr uint32_t kH = NA * kAtom / 2;               // a term of H: two fill B's place in the stage
  static constexpr uint32_t kScal = kXw + 3 * kAtom + kXwNext;
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
// Descriptors are given as two words; a step's offset is added to the low one (the start
// address) inside, so that the compiler keeps no register for each step of each product.
// Unrolled: in a loop, a product took 65 to 80 cycles to issue, here 28.
template <uint32_t OA, uint32_t OB, bool ACC>
__device__ __forceinline__ void umma_ss(uint32_t leader, uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo,
                                        uint32_t b_hi, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b32 x, y;\n\t.reg .b64 da, db;\n\t"
      "add.u32 x, %1, %7;\n\tadd.u32 y, %3, %8;\n\tmov.b64 da, {x, %2};\n\tmov.b64 db, {y, %4};\n\t"
      "setp.ne.b32 p, %9, 0;\n\tsetp.ne.b32 e, %6, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n\t}\n" ::"r"(d),
      "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(leader), "n"(OA), "n"(OB), "n"(ACC ? 1 : 0)
      : "memory");
}
// A from tensor memory (bf16, two per column), B from shared memory
template <uint32_t OA, uint32_t OB, bool ACC>
__device__ __forceinline__ void umma_ts(uint32_t leader, uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi,
                                        uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b32 x, y;\n\t.reg .b64 db;\n\t"
      "add.u32 x, %1, %6;\n\tadd.u32 y, %2, %7;\n\tmov.b64 db, {y, %3};\n\t"
      "setp.ne.b32 p, %8, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [x], db, %4, p;\n\t}\n" ::"r"(d),
      "r"(a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(leader), "n"(OA), "n"(OB), "n"(ACC ? 1 : 0)
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
// Waits of all roles.  A sleep follows every fruitless try: the tries return at once, and
// a dozen waiting warps' loops would take issue slots from those that compute.  Every
// wait depends on loads or products still to come, so the warp that issues the products
// keeps the time, and raises the flag for all: the code of a dozen timers is
// what instruction fetches have no room for.  The answer is the whole warp's: lanes that saw the
// flag and lanes that saw the phase must not part, as what follows (tcgen05.ld and .st, shuffles)
// needs them all.
template <int NS>
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  const uint32_t a = smem_u32(bar);
  while (!__all_sync(0xFFFFFFFFu, mbar_try_wait(a, parity))) {
    __nanosleep(NS);
    if (__any_sync(0xFFFFFFFFu, *abort_flag != 0)) return false;
  }
  return true;
}
// Until what has been issued has landed; gives up (for all) after the limit, a second at least.
__device__ __forceinline__ void drain_bar(uint64_t* bar, uint32_t parity, const ScanParams& p, volatile int* abort_flag) {
  const uint32_t a = smem_u32(bar);
  const uint64_t t0 = globaltimer_ns(), limit = p.wait_limit_ns > 1000000000ull ? p.wait_limit_ns : 1000000000ull;
  while (!mbar_try_wait(a, parity))
    if (globaltimer_ns() - t0 > limit) {
      *abort_flag = 1;
      if (p.status) atomicOr(p.status, kDevErrTimeout | kWaitDrain);
      break;
    }
}
template <int R>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R));
}
template <int R>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R));
}
template <int R>
__device__ __forceinline__ void regs_to() {
  if constexpr (R < 80)
    regs_dec<R>();
  else
    regs_inc<R>();
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two bf16 terms of a pair: their sum is within 2^-17 of it, relative.
__device__ __forceinline__ void split2(unsigned long long v, uint32_t& hi, uint32_t& lo) {
  hi = narrow2(v);
  lo = narrow2(fma2(pack2(-1.0f, -1.0f), widen2(hi), v));
}
// 32 lanes x 32 consecutive columns of tensor memory into registers.
__device__ __forceinline__ void tmem_ld_32x32b_x32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void st_shared_v4(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// One (segment, head, 64 dims) of the work.
struct Item {
  Segment sg;
  int seg, h, p0, pdims, nc;  // nc: chunks (none for the last segment in the first launch of a split scan)
  long long head_at;          // of this head's and these dims' state in an entry
  bool last;                  // the sequence's last segment
};
// Called by a full warp.
template <bool STATES>
__device__ __forceinline__ Item get_item(const ScanParams& p, int it, int ptiles) {
  Item w;
  const int hs = it / ptiles;
  w.h = hs % p.heads;
  w.seg = hs / p.heads;
  w.p0 = (it - hs * ptiles) * kP;
  w.pdims = p.dim - w.p0 < kP ? p.dim - w.p0 : kP;
  w.sg = find_segment(p, w.seg);
  w.last = w.sg.j == w.sg.count - 1;
  w.head_at = (static_cast<long long>(w.h) * p.dim + w.p0) * p.state_dim;
  w.nc = !(STATES && w.last) ? static_cast<int>((w.sg.end - w.sg.begin + kQ - 1) / kQ) : 0;
  return w;
}

// STATES: the first launch of a split scan (B, x and the state only).
template <int NA, bool STATES>
__global__ void __launch_bounds__(kThreads, 1)
    scan_umma_kernel(const __grid_constant__ Tmaps maps, const ScanParams p, int ptiles) {
  using L = Smem<NA, STATES>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  Scal* scal = reinterpret_cast<Scal*>(smem + L::kScal);
  Bars* bars = reinterpret_cast<Bars*>(smem + L::kBars);

  // a shuffle from a fixed lane tells the compiler that the warp's role, and all that
  // follows from it, is uniform
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int N = p.state_dim;
  const long long per_slot = static_cast<long long>(p.heads) * p.dim * N;
  const Item w = get_item<STATES>(p, blockIdx.x, ptiles);
  if (!w.sg.valid) return;  // the grid provides for more segments than there are
  if (w.nc == 0) {
    // An empty sequence's state passes through (a padded batch has many: 16 sequences of 64 heads with 64
    // empty ones behind took 147 us when these went the whole way, now 121).  The first launch of a
    // split scan copies the sequence's start into the last segment's place, as the last launch may
    // overwrite it while other segments still need it.
    const int slot = p.state_in || p.state_out ? seq_slot(p.slots, w.sg.seq, p.nslots, p.status) : -1;
    const float* src = p.state_in && slot >= 0 ? p.state_in + slot * per_slot + w.head_at : nullptr;
    float* dst = nullptr;
    if (STATES && w.sg.count > 1) dst = p.seg_state + w.seg * per_slot + w.head_at;
    if (!STATES && p.state_out && slot >= 0) dst = p.state_out + slot * per_slot + w.head_at;
    if (dst && dst != src)
      for (int i = threadIdx.x; i < w.pdims * N; i += kThreads) dst[i] = src ? src[i] : 0.0f;
    return;
  }

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->full_bc[i], 1);
      mbar_init(&bars->full_x[i], 1);
      mbar_init(&bars->xfree[i], 8);
      mbar_init(&bars->done[i], 1);
      mbar_init(&bars->s_full[i], 1);
      mbar_init(&bars->g_full[i], 8);
      mbar_init(&bars->xw_full[i], 8);
      mbar_init(&bars->ds_full[i], 1);
      mbar_init(&bars->ds_free[i], 4);
    }
    mbar_init(&bars->h_full, 4);
    mbar_init(&bars->yo_free, 8);
    for (int i = 0; i < 3; ++i) {
      mbar_init(&bars->sc_full[i], 1);
      mbar_init(&bars->sc_free[i], STATES ? 12 : 20);
    }
    mbar_init(&bars->drain, 1);
    bars->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(&bars->tmem, kCols);
  if (warp >= 4 && threadIdx.x < 128 + 2 * kP) bars->bad_from[0][threadIdx.x - 128] = 0;
  if (threadIdx.x >= 64 && threadIdx.x < 66) bars->bad[threadIdx.x - 64] = 0;
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, bars->tmem, 0);

  volatile int* const flag = &bars->abort_flag;
  constexpr uint32_t stage_c = L::kC, stage_b = L::kB, stage_x = L::kX;
  constexpr int kDs = STATES ? 2 : 1;  // places for Xw and dS: a chunk's is free kDs chunks later

  // In every role below, stages, buffers and barriers' phases go by the chunk c.
  //
  // The launch's 6 x 80 registers per warpgroup's thread, shared out by need.
  // A spill costs a trip to L2 here: shared memory leaves L1 too small for the stacks (64 bytes a
  // thread remain in the last launch; splits that left 88 and 132 took 4 and 3 % longer).
  constexpr int kRegsMisc = 48, kRegsG = STATES ? 24 : 112, kRegsXw = 56, kRegsState = STATES ? 152 : 96;
  static_assert(kRegsMisc + 2 * kRegsG + 2 * kRegsXw + kRegsState <= 6 * 80, "more registers than the launch has");
  if (warp < 4) {
    regs_dec<kRegsMisc>();
    if (warp == 0) {
      // ---------------------------------------------------------- loads
      // in the order in which the places become free: B and C after all products of their
      // chunk (in the first launch of a split scan after dS, the only one), x after its part in y
      int n_bc = 0, n_x = 0;  // loads issued
      bool ok = true;
      const int g = w.h / (p.heads / p.groups);
      int row = static_cast<int>(w.sg.begin);
#pragma unroll 1
      for (int c = 0; c < w.nc; ++c, row += kQ) {
        const int s = c & 1;
        const uint32_t st = sbase + s * L::kStage, par = ((c >> 1) - 1) & 1;
        const bool first = c < 2;
        ok = first || wait_bar<kNapLoad>(STATES ? &bars->ds_full[s] : &bars->done[s], par, flag);
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&bars->full_bc[s], (STATES ? 1 : 2) * NA * kAtom);
#pragma unroll
          for (int a = 0; a < NA; ++a) {
            tma_load_3d(st + stage_b + a * kAtom, &maps.b, &bars->full_bc[s], a * 64, g, row);
            if (!STATES) tma_load_3d(st + stage_c + a * kAtom, &maps.c, &bars->full_bc[s], a * 64, g, row);
          }
        }
        ++n_bc;
        if (!STATES) {
          ok = first || wait_bar<kNapLoad>(&bars->xfree[s], par, flag);
          if (!ok) break;
        }
        if (lane == 0) {
          mbar_arrive_expect_tx(&bars->full_x[s], kAtom);
          tma_load_3d(st + stage_x, &maps.x, &bars->full_x[s], w.p0, w.h, row);
        }
        ++n_x;
      }
      // Copies in flight land before the CTA leaves, whichever role gives up and when; without
      // that, all have been waited for by those that read them.
      if (lane == 0) {
        const int n[2] = {n_bc, n_x};
#pragma unroll 1
        for (int k = 0; k < 4; ++k) {  // full_bc, full_x, two of each
          const int last_use = ((n[k >> 1] - (k & 1) + 1) >> 1) - 1;
          if (last_use >= 0) drain_bar(&bars->full_bc[0] + k, last_use & 1, p, flag);
        }
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------- products
      constexpr uint32_t idS = make_idesc(kFmtBF16, 128, 128, 0, 0);
      constexpr uint32_t idY = make_idesc(kFmtBF16, 128, kP, 0, 1);
      constexpr uint32_t idD = make_idesc(kFmtBF16, 128, kP, 1, 1);
      const uint32_t ksteps = (N + 15) / 16;
      const uint32_t leader = elect_one();
      // descriptors of stage 0; a stage is kSt further.  Only the low word, the
      // start address in 16-byte units, changes with stage and step.
      constexpr uint32_t kSt = L::kStage >> 4;
      auto lo = [](uint64_t d) { return static_cast<uint32_t>(d); };
      const uint64_t dK = make_smem_desc(sbase, 16, 1024, kLayoutSw128);     // K-major
      const uint64_t dM = make_smem_desc(sbase, kAtom, 1024, kLayoutSw128);  // MN-major
      const uint32_t hK = static_cast<uint32_t>(dK >> 32), hM = static_cast<uint32_t>(dM >> 32);
      auto ready = [&](uint64_t* bar, uint32_t parity) { return __any_sync(0xFFFFFFFFu, mbar_test(bar, parity)) != 0; };
      // one of the three terms of dS = B^T Xw
      auto ds_term = [&](int s, uint32_t xw, uint32_t ds, auto tc) {
        constexpr uint32_t term = decltype(tc)::value * (kAtom >> 4);
        constexpr bool more = decltype(tc)::value > 0;
        const uint32_t base = lo(dM) + s * kSt;
        steps<8>([&](auto kc) {
          constexpr uint32_t k = decltype(kc)::value;
          umma_ss<(stage_b >> 4) + k * 128, (L::kXw >> 4) + term + k * 128, more || (k > 0)>(leader, ds, base, hM,
                                                                                          xw, hM, idD);
        });
      };
      // Whatever has its operands: S up to a chunk ahead of the rest (the order fixed at its
      // usual one, with blocking waits, was a tenth slower).  A chunk's dS never goes before its
      // S: the commit behind dS gives B's place to H, and has to cover both products that read B.
      int s_next = STATES ? w.nc : 0, c = 0, sub = 0;
      // the timer is slow to read: every so many idle turns, unless the limit is a short one
      const uint32_t look = p.wait_limit_ns < 1000000ull ? 0u : 255u;
      uint32_t idle = 0;
      uint64_t t0 = 0;
      while (c < w.nc) {
        bool did = true;
        const int s = c & 1;
        const uint32_t par = (c >> 1) & 1;
        const uint32_t xw = lo(dM) + s * (L::kXwNext >> 4), ds = tmem + kColDs + (STATES ? s * kP : 0);
        if (!STATES && s_next < w.nc && s_next < c + 2 && ready(&bars->full_bc[s_next & 1], (s_next >> 1) & 1)) {
          // C was loaded once every product of chunk c - 2 was done: S's place, where its G was, is free
          tc_fence_after_sync();
          const int sn = s_next & 1;
          const uint32_t base = lo(dK) + sn * kSt;
          steps<4 * NA>([&](auto kc) {
            constexpr uint32_t k = decltype(kc)::value, off = (k >> 2) * (kAtom >> 4) + (k & 3) * 2;
            if (k < ksteps)
              umma_ss<(stage_c >> 4) + off, (stage_b >> 4) + off, (k > 0)>(leader, tmem + kColS + sn * 128, base, hK, base,
                                                                           hK, idS);
          });
          umma_commit_by(leader, &bars->s_full[sn]);
          ++s_next;
        } else if (sub == 0 && s_next > c && ready(&bars->xw_full[s], par) &&
                   (c < kDs || ready(&bars->ds_free[(c - kDs) & 1], ((c - kDs) >> 1) & 1)) &&
                   ready(&bars->full_bc[s], par) && ready(&bars->full_x[s], par)) {
          tc_fence_after_sync();
          ds_term(s, xw, ds, std::integral_constant<int, 0>{});
          ds_term(s, xw, ds, std::integral_constant<int, 1>{});
          ds_term(s, xw, ds, std::integral_constant<int, 2>{});
          umma_commit_by(leader, &bars->ds_full[s]);
          if (STATES)
            ++c;
          else
            sub = 1;
        } else if (sub == 1 && ready(&bars->g_full[s], par)) {
          tc_fence_after_sync();
          const uint32_t base = lo(dM) + s * kSt;
          steps<16>([&](auto kc) {  // both terms of G
            constexpr uint32_t k = decltype(kc)::value & 7, term = decltype(kc)::value >> 3;
            umma_ts<(k >> 1) * 32 + (k & 1) * 8 + term * 16, (stage_x >> 4) + k * 128, (term + k > 0)>(
                leader, tmem + kColY + s * kP, tmem + kColS + s * 128, base, hM, idY);
          });
          sub = 2;
        } else if (sub == 2 && ready(&bars->h_full, c & 1) && (c == 0 || ready(&bars->yo_free, (c - 1) & 1))) {
          tc_fence_after_sync();
          const uint32_t base = lo(dK) + s * kSt, base_h = lo(dM) + s * kSt;
          steps<8 * NA>([&](auto kc) {  // both terms of H
            constexpr uint32_t k = decltype(kc)::value % (4 * NA), term = decltype(kc)::value / (4 * NA);
            constexpr uint32_t off = (k >> 2) * (kAtom >> 4) + (k & 3) * 2;
            if (k < ksteps)
              umma_ss<(stage_c >> 4) + off, ((stage_b + term * L::kH) >> 4) + k * 128, (term + k > 0)>(
                  leader, tmem + kColYo, base, hK, base_h, hM, idY);
          });
          umma_commit_by(leader, &bars->done[s]);
          sub = 0;
          ++c;
        } else {
          did = false;
        }
        if (did) {
          idle = 0;
          t0 = 0;
        } else {
          __nanosleep(kNapMma);
          if ((++idle & look) == 0) {
            if (__any_sync(0xFFFFFFFFu, *flag != 0)) break;
            const uint64_t now = globaltimer_ns();
            if (t0 == 0) t0 = now;
            if (__any_sync(0xFFFFFFFFu, now - t0 > p.wait_limit_ns)) {
              *flag = 1;
              if (p.status && lane == 0) atomicOr(p.status, kDevErrTimeout | kWaitMma);
              break;
            }
          }
        }
      }
      // every product has completed, and its arrivals have landed, before the CTA leaves
      umma_commit_by(leader, &bars->drain);
      drain_bar(&bars->drain, 0, p, flag);
    } else {
      // ---------------------------------------------------------- decays
      // lane -> token 32 b + lane of each block b; even chunks by warp 2, odd ones by warp 3
      bool ok = true;
      const float A2 = __ldg(p.A + w.h) * kLog2e;
      const float bias = p.dt_bias ? __ldg(p.dt_bias + w.h) : 0.0f;
      uint32_t raw[4] = {};
      auto fetch = [&](int c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const long long t = w.sg.begin + static_cast<long long>(c) * kQ + 32 * i + lane;
          if (t < w.sg.end) raw[i] = scan_dt_raw(p, t, w.h);
        }
      };
      const int first = warp & 1;
      if (first < w.nc) fetch(first);
#pragma unroll 1
      for (int c = first; c < w.nc; c += 2) {
        const int b3 = c % 3;
        ok = c < 3 || wait_bar<kNapDecay>(&bars->sc_free[b3], (c / 3 - 1) & 1, flag);
        if (!ok) break;
        Scal& sc = scal[b3];
        const long long left = w.sg.end - w.sg.begin - static_cast<long long>(c) * kQ - lane;
        float bt[4], head = 0.0f;
#pragma unroll 1
        for (int b = 0; b < 4; ++b) {
          const float d = 32 * b < left ? scan_dt(p, raw[0], bias) : 0.0f;
          raw[0] = raw[1], raw[1] = raw[2], raw[2] = raw[3];
          // sums within the block: inclusive up to the token, exclusive behind it
          // 2^-130 counts as zero already; a stronger decay would only take bits from the sums
          // whose differences are the decays of the tokens behind it
          float inc = d * A2;
          if (inc < -130.0f) inc = -130.0f;
          float suf = inc;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const float x = __shfl_up_sync(0xFFFFFFFFu, inc, o), z = __shfl_down_sync(0xFFFFFFFFu, suf, o);
            if (lane >= o) inc += x;
            if (lane + o < 32) suf += z;
          }
          bt[0] = bt[1], bt[1] = bt[2], bt[2] = bt[3], bt[3] = __shfl_sync(0xFFFFFFFFu, inc, 31);
          suf = __shfl_down_sync(0xFFFFFFFFu, suf, 1);
          const int t = 32 * b + lane;
          sc.l[t] = inc;
          sc.u[t] = ex2(inc);
          sc.e[t] = ex2(head + inc);
          sc.d[t] = d;
          sc.f[3][t] = lane < 31 ? suf : 0.0f;  // the exponent, until the blocks' sums are known
          head += bt[3];
        }
        if (c + 2 < w.nc) fetch(c + 2);
#pragma unroll 1
        for (int b = 0; b < 4; ++b) {
          const int t = 32 * b + lane;
          const float suf = sc.f[3][t], d = sc.d[t];
          float between = 0.0f;
#pragma unroll
          for (int k = 1; k <= 4; ++k) {
            if (k > b) {
              if (k - 1 > b) between += bt[k - 1];
              sc.f[k - 1][t] = d * ex2(suf + between);
            }
          }
        }
        if (lane == 0) {
          sc.total = ex2(head);
          sc.log2 = head;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->sc_full[b3]);
      }
    }
  } else if (warp < 12) {
    regs_to<kRegsG>();
    // ------------------------------------------------------------ G, and y of the chunk before
    if constexpr (!STATES) {
      const int half = (warp - 4) >> 2, q = warp & 3;  // columns 64 half.. of G, 32 half.. of y
      const int t = 32 * q + lane;
      const uint32_t lanes = static_cast<uint32_t>(32 * q) << 16;
      const uint32_t sYo = tmem + lanes + kColYo + 32 * half;
      const bool gated = p.z != nullptr;
      const long long zstep = 8 * p.ldz, ystep = 8 * p.ldy;  // eight rows
      const int col8 = 8 * (lane & 3);
      bool ok = true;
      const float Dh = p.D ? __ldg(p.D + w.h) : 0.0f;
      const unsigned long long D2 = pack2(Dh, Dh);
      const long long col = static_cast<long long>(w.h) * p.dim + w.p0 + 32 * half;
      const long long row = w.sg.begin + 32 * q + (lane >> 2);
      const __nv_bfloat16* gz = static_cast<const __nv_bfloat16*>(p.z) + row * p.ldz + col + col8;
      __nv_bfloat16* gy = static_cast<__nv_bfloat16*>(p.y) + row * p.ldy + col + col8;
      const int rows = static_cast<int>(w.sg.end - w.sg.begin);
      const int wdims = w.pdims - 32 * half;  // columns of this half
#pragma unroll 1
      for (int c = 0; c <= w.nc; ++c) {
        // z of the chunk before, on its way while G is formed: four lanes to the 64 bytes of
        // a row, eight rows at a time
        uint4 zv[4];
        const int r0 = (c - 1) * kQ + 32 * q + (lane >> 2);  // this lane's first row in the segment
        if (gated && c > 0) {
          const __nv_bfloat16* zr = gz;
#pragma unroll
          for (int i = 0; i < 4; ++i, zr += zstep)
            zv[i] = col8 < wdims && r0 + 8 * i < rows ? __ldg(reinterpret_cast<const uint4*>(zr))
                                                      : make_uint4(0, 0, 0, 0);
          gz = zr + 12 * zstep;
        }
        if (c < w.nc) {
          const int b3 = c % 3, s = c & 1;
          ok = wait_bar<kNapG>(&bars->sc_full[b3], (c / 3) & 1, flag) &&
               wait_bar<kNapG>(&bars->s_full[s], (c >> 1) & 1, flag);
          if (!ok) break;
          tc_fence_after_sync();
          const Scal& sc = scal[b3];
          const float u = sc.u[t], lt = sc.l[t];
          const uint32_t sS = tmem + lanes + kColS + s * 128 + 64 * half;
#pragma unroll 1
          for (int i2 = 0; i2 < 2; ++i2) {
            const int b = 2 * half + i2;  // block of 32 columns: off the diagonal for b < q
            uint32_t o[16], ol[16];        // G's first and second term
            if (b <= q) {
              uint32_t r[32];
              tmem_ld_32x32b_x32(sS + 32 * i2, r);
              const unsigned long long* f =
                  reinterpret_cast<const unsigned long long*>((b < q ? sc.f[q - 1] : sc.d) + 32 * b);
              if (b < q) {
                const unsigned long long u2 = pack2(u, u);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  const unsigned long long s2 = pack2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
                  split2(mul2(mul2(s2, f[i]), u2), o[i], ol[i]);
                }
              } else {
                const unsigned long long* ls = reinterpret_cast<const unsigned long long*>(sc.l + 32 * b);
                const unsigned long long lt2 = pack2(lt, lt), neg = pack2(-1.0f, -1.0f);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  // Columns up to this row.  The factors are formed for all of them and the rest is
                  // selected away: an exponential inside a condition becomes a branch of its own.
                  float a, z;
                  unpack2(fma2(ls[i], neg, lt2), a, z);
                  const unsigned long long w2 = mul2(pack2(ex2(a), ex2(z)), f[i]);
                  unpack2(mul2(pack2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), w2), a, z);
                  split2(pack2(2 * i <= lane ? a : 0.0f, 2 * i + 1 <= lane ? z : 0.0f), o[i], ol[i]);
                }
              }
            } else {
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = ol[i] = 0;
            }
            // these columns of S have been read by this lane already
            tmem_st_32x32b_x16(sS + 32 * i2, o);
            tmem_st_32x32b_x16(sS + 32 * i2 + 16, ol);
          }
          tmem_wait_st();
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->g_full[s]);
        }
        if (c > 0) {
          const int d = c - 1, b3 = d % 3, s = d & 1;
          ok = wait_bar<kNapG>(&bars->full_x[s], (d >> 1) & 1, flag) &&
               wait_bar<kNapG>(&bars->xw_full[s], (d >> 1) & 1, flag) &&
               wait_bar<kNapG>(&bars->done[s], (d >> 1) & 1, flag);
          if (!ok) break;
          tc_fence_after_sync();
          const bool bad = bars->bad[s] == d + 1u;
          // x's own row for D x.  Its place then takes z and after that y on their way between
          // the layout of global memory and a row to a lane (a lane's own row of z and y
          // to and from global memory touched four times the lines).
          uint8_t* xt = smem + s * L::kStage + stage_x;
          uint4 xv[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) xv[i] = *reinterpret_cast<const uint4*>(xt + swz_offset(t, 4 * half + i, 128));
          const float e = scal[b3].e[t];
          const unsigned long long e2 = pack2(e, e);
          const uint32_t sY = tmem + lanes + kColY + s * kP + 32 * half;
          __syncwarp();
          if (gated) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *reinterpret_cast<uint4*>(xt + swz_offset(32 * q + 8 * i + (lane >> 2), 4 * half + (lane & 3), 128)) = zv[i];
            __syncwarp();
          }
#pragma unroll 1
          for (int k = 0; k < 2; ++k) {
            uint32_t ry[16], ro[16], out[8], zw[8];
            tmem_ld_32x32b_x16(sY + 16 * k, ry);
            tmem_ld_32x32b_x16(sYo + 16 * k, ro);
            const uint32_t o0 = swz_offset(t, 4 * half + 2 * k, 128), o1 = swz_offset(t, 4 * half + 2 * k + 1, 128);
            const uint32_t xw[8] = {xv[0].x, xv[0].y, xv[0].z, xv[0].w, xv[1].x, xv[1].y, xv[1].z, xv[1].w};
            xv[0] = xv[2], xv[1] = xv[3];
            if (gated) {
              *reinterpret_cast<uint4*>(zw) = *reinterpret_cast<const uint4*>(xt + o0);
              *reinterpret_cast<uint4*>(zw + 4) = *reinterpret_cast<const uint4*>(xt + o1);
            }
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              unsigned long long v = fma2(e2, pack2(__uint_as_float(ro[2 * i]), __uint_as_float(ro[2 * i + 1])),
                                          pack2(__uint_as_float(ry[2 * i]), __uint_as_float(ry[2 * i + 1])));
              v = fma2(D2, widen2(xw[i]), v);
              if (gated) v = mul2(v, silu2(widen2(zw[i])));
              out[i] = narrow2(v);
            }
            *reinterpret_cast<uint4*>(xt + o0) = make_uint4(out[0], out[1], out[2], out[3]);
            *reinterpret_cast<uint4*>(xt + o1) = make_uint4(out[4], out[5], out[6], out[7]);
          }
          if (bad) {
#pragma unroll 1
            for (int i = 32 * half; i < 32 * half + 32; ++i) {
              const uint32_t from = bars->bad_from[s][i];
              if ((from >> 8) == d && t >= 128 - static_cast<int>(from & 255))
                *reinterpret_cast<unsigned short*>(xt + t * 128 + ((2 * i) ^ ((t & 7) << 4))) = 0x7FFF;
            }
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i, gy += ystep)
            if (col8 < wdims && r0 + 8 * i < rows)
              *reinterpret_cast<uint4*>(gy) =
                  *reinterpret_cast<const uint4*>(xt + swz_offset(32 * q + 8 * i + (lane >> 2), 4 * half + (lane & 3), 128));
          gy += 12 * ystep;
          fence_proxy_async_smem();  // the tile's next content comes by TMA
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&bars->yo_free);
            mbar_arrive(&bars->xfree[s]);
            mbar_arrive(&bars->sc_free[b3]);
          }
        }
      }
    }
  } else if (warp < 20) {
    regs_dec<kRegsXw>();
    // ------------------------------------------------------------ Xw
    const int s = (threadIdx.x - 384) & 127;     // row
    const int i0 = warp < 16 ? 0 : 4;            // first of this thread's 16-byte pieces
    bool ok = true;
#pragma unroll 1
    for (int c = 0; c < w.nc; ++c) {
      const int b3 = c % 3, sb = c & 1;
      const uint32_t st = sbase + sb * L::kStage;
      const int left = static_cast<int>(w.sg.end - w.sg.begin) - c * kQ;
      ok = wait_bar<kNapXw>(&bars->sc_full[b3], (c / 3) & 1, flag) &&
           wait_bar<kNapXw>(&bars->full_x[sb], (c >> 1) & 1, flag);
      if (!ok) break;
      const float ws = scal[b3].f[3][s];
      ok = c < kDs || wait_bar<kNapXw>(&bars->ds_full[(c - kDs) & 1], ((c - kDs) >> 1) & 1, flag);
      if (!ok) break;
      const uint32_t xw = L::kXw + sb * L::kXwNext;
      const unsigned long long w2 = pack2(ws, ws), neg = pack2(-1.0f, -1.0f);
      unsigned long long chk = 0;  // stays zero while all products are finite
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t off = swz_offset(s, i0 + i, 128);
        const uint4 x = *reinterpret_cast<const uint4*>(smem + sb * L::kStage + stage_x + off);
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
        uint32_t vh[4], vm[4], vl[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const unsigned long long v = mul2(w2, widen2(xs[k]));
          if (!STATES) chk = fma2(v, 0ull, chk);
          vh[k] = narrow2(v);
          split2(fma2(neg, widen2(vh[k]), v), vm[k], vl[k]);
        }
        *reinterpret_cast<uint4*>(smem + xw + off) = make_uint4(vh[0], vh[1], vh[2], vh[3]);
        *reinterpret_cast<uint4*>(smem + xw + kAtom + off) = make_uint4(vm[0], vm[1], vm[2], vm[3]);
        *reinterpret_cast<uint4*>(smem + xw + 2 * kAtom + off) = make_uint4(vl[0], vl[1], vl[2], vl[3]);
      }
      if (!STATES) {
        // In G x every row of x meets zeros of G, for the tokens before it, and a non-finite
        // element would pass them.  It is taken out here (the state gets it through Xw), and y is
        // made NaN in its dim from its token on.
        float c0, c1;
        unpack2(chk, c0, c1);
        if (c0 + c1 != 0.0f && s < left) {
#pragma unroll 1
          for (int e = 8 * i0; e < 8 * i0 + 32; ++e) {
            unsigned short* x = reinterpret_cast<unsigned short*>(smem + sb * L::kStage + stage_x +
                                                                  swz_offset(s, e / 8, 128) + 2 * (e % 8));
            if ((*x & 0x7F80) != 0x7F80) continue;
            *x = 0;
            atomicMax(&bars->bad_from[sb][e], (static_cast<uint32_t>(c) << 8) | (128u - s));
            bars->bad[sb] = c + 1u;
          }
        }
      }
      if (left < kQ) {
        // rows behind the sequence hold what lies there; a zero factor would not stop a NaN
        ok = wait_bar<kNapXw>(&bars->full_bc[sb], (c >> 1) & 1, flag);
        if (!ok) break;
        if (s >= left) {
#pragma unroll 1
          for (int i = i0; i < i0 + 4; ++i) {
            const uint32_t off = swz_offset(s, i, 128);
            st_shared_v4(st + stage_x + off, 0, 0, 0, 0);
            st_shared_v4(sbase + xw + off, 0, 0, 0, 0);
            st_shared_v4(sbase + xw + kAtom + off, 0, 0, 0, 0);
            st_shared_v4(sbase + xw + 2 * kAtom + off, 0, 0, 0, 0);
#pragma unroll
            for (int a = 0; a < NA; ++a) st_shared_v4(st + stage_b + a * kAtom + off, 0, 0, 0, 0);
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&bars->xw_full[sb]);
        mbar_arrive(&bars->sc_free[b3]);
      }
    }
  } else {
    regs_inc<kRegsState>();
    // ------------------------------------------------------------ state
    const int n = threadIdx.x - 640;  // state element (lane of tensor memory)
    const int q = warp & 3;
    const bool wlive = 32 * q < N;    // this warp has state elements
    const bool live = n < N;
    const uint32_t sD = tmem + (static_cast<uint32_t>(32 * q) << 16) + kColDs;
    bool ok = true;
    const int slot = (p.state_in || p.state_out) ? seq_slot(p.slots, w.sg.seq, p.nslots, p.status) : -1;
    const float* in = p.state_in && slot >= 0 ? p.state_in + slot * per_slot + w.head_at : nullptr;
    float hv[kP];
#pragma unroll
    for (int i = 0; i < kP; ++i) hv[i] = 0.0f;
    // what the state starts from: in the first launch of a split scan, zero
    const float* src = w.sg.count == 1 ? in : p.seg_state + w.seg * per_slot + w.head_at;
    if (!STATES && src && live) {
      src += n;
#pragma unroll
      for (int i = 0; i < kP; ++i)
        if (i < w.pdims) hv[i] = src[i * N];
    }
    float log_sum = 0.0f;
#pragma unroll 1
    for (int c = 0; c < w.nc; ++c) {
      const int b3 = c % 3;
      ok = wait_bar<kNapState>(&bars->ds_full[c & 1], (c >> 1) & 1, flag);
      if (!ok) break;
      if (!STATES) {
        // H, the state before the chunk, in the place of B, which has been read
        // (hidden from the compiler, or it keeps eight offsets in registers through the loop)
        uint32_t row = n, at = sbase + (c & 1) * L::kStage + stage_b;
        asm volatile("" : "+r"(row), "+r"(at));
        if (row < 64 * NA) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            uint32_t vh[4], vl[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) split2(pack2(hv[8 * i + 2 * k], hv[8 * i + 2 * k + 1]), vh[k], vl[k]);
            const uint32_t off = swz_offset(row, i, 128);
            st_shared_v4(at + off, vh[0], vh[1], vh[2], vh[3]);
            st_shared_v4(at + L::kH + off, vl[0], vl[1], vl[2], vl[3]);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->h_full);
      }
      ok = wait_bar<kNapState>(&bars->sc_full[b3], (c / 3) & 1, flag);
      if (!ok) break;
      const float decay = scal[b3].total;
      log_sum += scal[b3].log2;
      const unsigned long long decay2 = pack2(decay, decay);
      tc_fence_after_sync();
      if (wlive) {
#pragma unroll
        for (int pc = 0; pc < 4; ++pc) {
          uint32_t r[16];
          tmem_ld_32x32b_x16(sD + (STATES ? (c & 1) * kP : 0) + 16 * pc, r);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 8; ++i)
            unpack2(fma2(pack2(hv[16 * pc + 2 * i], hv[16 * pc + 2 * i + 1]), decay2,
                         pack2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]))),
                    hv[16 * pc + 2 * i], hv[16 * pc + 2 * i + 1]);
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&bars->ds_free[c & 1]);
        mbar_arrive(&bars->sc_free[b3]);
      }
    }
    float* dst = nullptr;  // stays null if the CTA gave up
    if (STATES && ok) {
      dst = p.seg_state + w.seg * per_slot + w.head_at;
      if (n == 0 && w.p0 == 0)
        p.seg_log[static_cast<long long>(w.seg) * p.heads + w.h] = log_sum * (1.0f / kLog2e);
    } else if (ok && w.last && p.state_out && slot >= 0) {
      dst = p.state_out + slot * per_slot + w.head_at;
    }
    if (dst && live) {
      dst += n;
#pragma unroll
      for (int i = 0; i < kP; ++i)
        if (i < w.pdims) dst[i * N] = hv[i];
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
  auto set = [&] { err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<NA, STATES>::kBytes); };
  if (dev < 64) std::call_once(once[dev], set);
  else set();
  SMM_CUDA_TRY(err, "selective scan shared memory size");
  kern<<<grid, kThreads, Smem<NA, STATES>::kBytes, st>>>(maps, p, ptiles);
  count_launch();
  SMM_CUDA_TRY(cudaGetLastError(), "selective scan (tensor core) launch");
  return SMM_OK;
}

}  // namespace

// bf16, whole 16-byte pieces everywhere, state_dim of one 128-row tile, and sequences
// long enough.  Time here goes with the chunks, a started one counting in full (32 sequences
// of 64 heads of 64 x 128: 151 to 157 us for 16 to 32 tokens each), on the fp32 pipes
// with the tokens, and state_dim adds to it.  The two cross near 25 tokens with state_dim 128
// (fp32 pipes against this kernel: 138 and 151 us at 20 tokens, 149 and 152 at 24, 186 and 157
// at 32) and near 120 with 16 (127 and 156 us at 96, 160 and 165 at 128, 214 and 177 at 160; 220 and 88
// for 4 sequences of 1024); for one sequence no later (9.9 and 12.0 us at 16 tokens, 12.7 and 12.2 at 24).
bool scan_umma_fits(const ScanParams& p, int dtype) {
  if (dtype != SMM_DTYPE_BF16 || p.dim % 8 || p.state_dim % 8 || p.state_dim > 128) return false;
  if (p.ldx % 8 || p.ldb % 8 || p.ldc % 8 || p.ldy % 8 || (p.z && p.ldz % 8)) return false;
  if (!aligned_to(p.x, 16) || !aligned_to(p.B, 16) || !aligned_to(p.C, 16) || !aligned_to(p.y, 16) ||
      !aligned_to(p.z, 16))
    return false;
  const long long ptiles = (p.dim + kP - 1) / kP;
  return p.tokens * (p.state_dim + 15) * p.dim >= 3500 * static_cast<long long>(p.nseq) * kP * ptiles;
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
  const unsigned grid = static_cast<unsigned>(blocks);
  if (p.state_dim <= 64) {
    if (p.split) {
      if (int rc = launch_one<1, true>(maps, p, grid, ptiles, st)) return rc;
      if (int rc = scan_combine(p, st)) return rc;
    }
    return launch_one<1, false>(maps, p, grid, ptiles, st);
  }
  if (p.split) {
    if (int rc = launch_one<2, true>(maps, p, grid, ptiles, st)) return rc;
    if (int rc = scan_combine(p, st)) return rc;
  }
  return launch_one<2, false>(maps, p, grid, ptiles, st);
}

}  // namespace smm
