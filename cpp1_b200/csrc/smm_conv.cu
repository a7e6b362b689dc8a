// Short causal convolution: y[t][c] = act(bias[c] + sum_j w[c][j] x[t-W+1+j][c]),
// per channel a banded lower-triangular Toeplitz matrix of W diagonals.  For
// packed prompts, and for one new token of each sequence.
//
// Bound by memory: each element is read once and written once (W multiplies
// per element), with the activation's exponential and reciprocal next (59 % of their
// pipe's time).  A thread owns four channels and walks down a run of
// consecutive tokens with the last W-1 rows in registers, so a row is read
// from memory once and W-1 rows per run again from L2.  While it computes the rows
// that it has, the next ones are on their way: 8192 tokens of 4352 bf16 channels take
// 33 us, 67 % of a copy's rate (40 us without), 8192 of 2176 fp32 ones 30.5 us.
//
// The first min(W-1, length) tokens of a sequence need the state it starts
// from, and the state it ends with may overwrite that.  Both are done by the
// threads whose run holds the sequence's last token: they read the old state
// first and write the new one last, so an update in place has no race, and
// needs no second launch.  Empty sequences are dealt out over the runs, whatever their
// position: a padded batch has hundreds of them in one place (2048 tokens of 16
// sequences with 240 empty ones behind took 115 us when one run walked them all).
#include "smm_seq.cuh"

#include <type_traits>

namespace smm {
namespace {

struct ConvParams {
  const void* x;
  const void* w;
  const void* bias;
  const int* offsets;
  const void* state_in;
  void* state_out;
  const int* slots;
  void* y;
  long long tokens, ldx, ldy;
  int channels, nseq, nslots, run, nruns, ctiles, silu;
  uint32_t* status;
};

// Small CTAs: 1088 channel quads are 17 times 64, and 9 times 128 with a CTA half empty
// (33 against 34 us for 8192 tokens).
constexpr int kConvThreads = 64;

// VEC channels of a thread, in pairs where there are pairs.  Four: with the eight of a
// 16-byte bf16 vector, registers left nine warps on an SM and the loads' latency showed.
template <typename T, int VEC, int W>
struct ConvLane {
  static constexpr bool kVec = VEC > 1;
  static constexpr int kPiece = VEC * sizeof(T) % 16 == 0 ? 16 : 8;  // bytes of one access
  static constexpr int NP = kVec ? VEC / 2 : 1;
  using E = typename std::conditional<kVec, unsigned long long, float>::type;
  E w[W][NP];  // tap j of each channel
  E bias[NP];

  static __device__ __forceinline__ void put(E (&d)[NP], const float (&v)[VEC]) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      if constexpr (kVec)
        d[i] = pack2(v[2 * i], v[2 * i + 1]);
      else
        d[i] = v[i];
    }
  }
  static __device__ __forceinline__ void get(const E (&d)[NP], float (&v)[VEC]) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      if constexpr (kVec)
        unpack2(d[i], v[2 * i], v[2 * i + 1]);
      else
        v[i] = d[i];
    }
  }
  __device__ void load(const ConvParams& p, int c) {
    float wt[VEC * W], one[VEC];  // [channel][tap]
    load_f32<T, VEC * W, kVec, kPiece>(static_cast<const T*>(p.w) + static_cast<long long>(c) * W, wt);
#pragma unroll
    for (int j = 0; j < W; ++j) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) one[i] = wt[i * W + j];
      put(w[j], one);
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) one[i] = 0.0f;
    if (p.bias) load_f32<T, VEC, kVec>(static_cast<const T*>(p.bias) + c, one);
    put(bias, one);
  }
  // a row's channels as they lie (narrower than fp32 pairs while on their way)
  using Raw = typename std::conditional<kVec, RawVec<T, kVec ? VEC : 16 / sizeof(T), kPiece>, T>::type;
  static __device__ __forceinline__ void load_raw(const T* x, Raw& r) {
    if constexpr (kVec)
      r.load(x);
    else
      r = *x;
  }
  static __device__ __forceinline__ void from_raw(const Raw& r, E (&d)[NP]) {
    if constexpr (kVec) {
      float v[VEC];
      r.get(v);
      put(d, v);
    } else {
      d[0] = to_f32(r);
    }
  }
  static __device__ __forceinline__ void load_row(const T* x, E (&d)[NP]) {
    Raw r;
    load_raw(x, r);
    from_raw(r, d);
  }
  // One output row from the W-1 rows before it and its own; the window moves on.
  __device__ __forceinline__ void row(E (&win)[W - 1][NP], const E (&cur)[NP], T* y, bool act) const {
    E a[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      a[i] = bias[i];
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const E in = j < W - 1 ? win[j < W - 1 ? j : 0][i] : cur[i];
        if constexpr (kVec)
          a[i] = fma2(w[j][i], in, a[i]);
        else
          a[i] = fmaf(w[j][i], in, a[i]);
      }
#pragma unroll
      for (int j = 0; j < W - 2; ++j) win[j][i] = win[j + 1][i];
      win[W - 2][i] = cur[i];
    }
    float out[VEC];
    get(a, out);
    if (act) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) out[i] = silu(out[i]);
    }
    store_f32<T, VEC, kVec>(y, out);
  }
  // The window to and from a state's [channel][W-1] elements.
  static __device__ __forceinline__ void from_state(const float (&old)[VEC * (W - 1)], E (&win)[W - 1][NP]) {
    float v[VEC];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = old[i * (W - 1) + j];
      put(win[j], v);
    }
  }
  static __device__ __forceinline__ void to_state(const E (&win)[W - 1][NP], float (&old)[VEC * (W - 1)]) {
    float v[VEC];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
      get(win[j], v);
#pragma unroll
      for (int i = 0; i < VEC; ++i) old[i * (W - 1) + j] = v[i];
    }
  }
};

template <typename T, int VEC, int W>
__global__ void __launch_bounds__(kConvThreads) conv_kernel(const ConvParams p) {
  constexpr bool kVec = VEC > 1;
  const int ctile = static_cast<int>(blockIdx.x % p.ctiles);
  const long long r = static_cast<long long>(blockIdx.x / p.ctiles) * blockDim.y + threadIdx.y;
  const int c = (ctile * blockDim.x + threadIdx.x) * VEC;
  if (c >= p.channels || r >= p.nruns) return;
  const long long t0 = r * p.run;
  const long long t1 = t0 + p.run < p.tokens ? t0 + p.run : p.tokens;
  const T* x = static_cast<const T*>(p.x) + c;
  T* y = static_cast<T*>(p.y) + c;
  const bool act = p.silu != 0;
  using Lane = ConvLane<T, VEC, W>;
  Lane lane;
  lane.load(p, c);

  // first sequence that ends in this run or behind it
  int s = 0;
  if (p.offsets) {
    int lo = 0, hi = p.nseq;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (__ldg(p.offsets + mid + 1) > t0)
        hi = mid;
      else
        lo = mid + 1;
    }
    s = lo;
  }
  for (; s < p.nseq; ++s) {
    long long b, e;
    seq_range(p.offsets, s, p.tokens, &b, &e);
    if (b >= t1) break;
    if (e == b) continue;
    typename Lane::E win[W - 1][Lane::NP];
    const long long lo = b + W - 1 > t0 ? b + W - 1 : t0;
    const long long hi = e < t1 ? e : t1;
    if (lo < hi) {
#pragma unroll
      for (int j = 0; j < W - 1; ++j) Lane::load_row(x + (lo - (W - 1) + j) * p.ldx, win[j]);
      long long t = lo;
      // U rows on their way while the U before them are computed
      constexpr int U = 16 / sizeof(T);
      typename Lane::Raw raw[U], next[U];
      auto fetch = [&](long long row) {
#pragma unroll
        for (int u = 0; u < U; ++u) Lane::load_raw(x + (row + u) * p.ldx, next[u]);
      };
      if (t + U <= hi) fetch(t);
      for (; t + U <= hi; t += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = next[u];
        if (t + 2 * U <= hi) fetch(t + U);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          typename Lane::E cur[Lane::NP];
          Lane::from_raw(raw[u], cur);
          lane.row(win, cur, y + (t + u) * p.ldy, act);
        }
      }
      for (; t < hi; ++t) {
        typename Lane::E cur[Lane::NP];
        Lane::load_row(x + t * p.ldx, cur);
        lane.row(win, cur, y + t * p.ldy, act);
      }
    }
    if (e > t1) continue;  // another run has the last token
    const int slot = (p.state_in || p.state_out) ? seq_slot(p.slots, s, p.nslots, p.status) : -1;
    const long long at = (static_cast<long long>(slot) * p.channels + c) * (W - 1);
    float old[VEC * (W - 1)];
    if (p.state_in && slot >= 0) {
      load_f32<T, VEC*(W - 1), kVec, Lane::kPiece>(static_cast<const T*>(p.state_in) + at, old);
    } else {
#pragma unroll
      for (int i = 0; i < VEC * (W - 1); ++i) old[i] = 0.0f;
    }
    Lane::from_state(old, win);
    const long long len = e - b;
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
      if (j < len) {
        typename Lane::E cur[Lane::NP];
        Lane::load_row(x + (b + j) * p.ldx, cur);
        lane.row(win, cur, y + (b + j) * p.ldy, act);
      }
    }
    if (p.state_out && slot >= 0) {
      // the window now ends at row b + min(len, W-1); a longer sequence ends later
      if (len > W - 1) {
#pragma unroll
        for (int j = 0; j < W - 1; ++j) Lane::load_row(x + (e - (W - 1) + j) * p.ldx, win[j]);
      }
      Lane::to_state(win, old);
      store_f32<T, VEC*(W - 1), kVec, Lane::kPiece>(static_cast<T*>(p.state_out) + at, old);
    }
  }
  // empty sequences: the state they start from is what they end with
  if (!p.state_out) return;
#pragma unroll 1
  for (unsigned q = static_cast<unsigned>(r); q < static_cast<unsigned>(p.nseq); q += p.nruns) {
    long long b, e;
    seq_range(p.offsets, q, p.tokens, &b, &e);
    if (e > b) continue;
    const int slot = seq_slot(p.slots, q, p.nslots, p.status);
    if (slot < 0 || p.state_in == p.state_out) continue;
    const long long at = (static_cast<long long>(slot) * p.channels + c) * (W - 1);
    float old[VEC * (W - 1)] = {};
    if (p.state_in) load_f32<T, VEC*(W - 1), kVec, Lane::kPiece>(static_cast<const T*>(p.state_in) + at, old);
    store_f32<T, VEC*(W - 1), kVec, Lane::kPiece>(static_cast<T*>(p.state_out) + at, old);
  }
}

// One token of each sequence: a thread per four channels of one row.
template <typename T, int VEC, int W>
__global__ void __launch_bounds__(kConvThreads) conv_step_kernel(const ConvParams p) {
  constexpr bool kVec = VEC > 1;
  const int b = static_cast<int>(blockIdx.x / p.ctiles);
  const int c = (static_cast<int>(blockIdx.x % p.ctiles) * blockDim.x + threadIdx.x) * VEC;
  if (c >= p.channels) return;
  const int slot = p.state_in || p.state_out ? seq_slot(p.slots, b, p.nslots, p.status) : -1;
  const long long at = (static_cast<long long>(slot) * p.channels + c) * (W - 1);
  using Lane = ConvLane<T, VEC, W>;
  float old[VEC * (W - 1)];
  typename Lane::E win[W - 1][Lane::NP], cur[Lane::NP];
  if (p.state_in && slot >= 0) {
    load_f32<T, VEC*(W - 1), kVec, Lane::kPiece>(static_cast<const T*>(p.state_in) + at, old);
  } else {
#pragma unroll
    for (int i = 0; i < VEC * (W - 1); ++i) old[i] = 0.0f;
  }
  Lane::load_row(static_cast<const T*>(p.x) + b * p.ldx + c, cur);
  Lane lane;
  lane.load(p, c);
  Lane::from_state(old, win);
  lane.row(win, cur, static_cast<T*>(p.y) + b * p.ldy + c, p.silu != 0);
  if (p.state_out && slot >= 0) {
    Lane::to_state(win, old);
    store_f32<T, VEC*(W - 1), kVec, Lane::kPiece>(static_cast<T*>(p.state_out) + at, old);
  }
}

template <typename T, int VEC, bool STEP>
void launch_width(int width, dim3 grid, dim3 block, const ConvParams& p, cudaStream_t st) {
  auto go = [&](auto w) {
    constexpr int W = decltype(w)::value;
    if constexpr (STEP)
      conv_step_kernel<T, VEC, W><<<grid, block, 0, st>>>(p);
    else
      conv_kernel<T, VEC, W><<<grid, block, 0, st>>>(p);
  };
  switch (width) {
    case 2: return go(std::integral_constant<int, 2>{});
    case 3: return go(std::integral_constant<int, 3>{});
    case 4: return go(std::integral_constant<int, 4>{});
    case 5: return go(std::integral_constant<int, 5>{});
    case 6: return go(std::integral_constant<int, 6>{});
    case 7: return go(std::integral_constant<int, 7>{});
    default: return go(std::integral_constant<int, 8>{});
  }
}

// Checks shared by both entries; rows is tokens or batch, nseq sequences.
int check_conv(const char* who, const ConvParams& p, int width, int dtype, int act, bool step) {
  if (p.tokens < 0 || p.channels < 0 || p.nseq < 0 || p.nslots < 0)
    return set_error(SMM_ERR_INVALID, "%s: negative size", who);
  if (width < 2 || width > 8) return set_error(SMM_ERR_INVALID, "%s: width %d is not in 2..8", who, width);
  if (!valid_dtype(dtype)) return set_error(SMM_ERR_INVALID, "%s: unknown element type %d", who, dtype);
  if (act != SMM_ACT_NONE && act != SMM_ACT_SILU)
    return set_error(SMM_ERR_INVALID, "%s: unknown activation %d", who, act);
  if (p.ldx < p.channels || p.ldy < p.channels)
    return set_error(SMM_ERR_INVALID, "%s: row stride shorter than %d channels", who, p.channels);
  if (!step && !p.offsets && p.nseq > 1)
    return set_error(SMM_ERR_INVALID, "%s: %d sequences without offsets", who, p.nseq);
  if ((p.state_in || p.state_out) && !p.slots && p.nslots < p.nseq)
    return set_error(SMM_ERR_INVALID, "%s: %d states for %d sequences", who, p.nslots, p.nseq);
  if (p.channels == 0 || (p.tokens == 0 && p.nseq == 0)) return SMM_OK;
  if (!p.w || (p.tokens > 0 && (!p.x || !p.y))) return set_error(SMM_ERR_INVALID, "%s: null pointer", who);
  const size_t e = dtype_size(dtype);
  if (!all_aligned_to(e, p.x, p.w, p.bias, p.state_in, p.state_out, p.y) || !all_aligned_to(4, p.offsets, p.slots))
    return set_error(SMM_ERR_INVALID, "%s: a pointer is not aligned to its elements", who);
  const Span x = row_span(p.x, p.tokens, p.channels, p.ldx, e), y = row_span(p.y, p.tokens, p.channels, p.ldy, e);
  const size_t sb = static_cast<size_t>(p.nslots) * p.channels * (width - 1) * e;
  const Span si{p.state_in, sb}, so{p.state_out, sb};
  const Span wv{p.w, static_cast<size_t>(p.channels) * width * e}, bv{p.bias, p.channels * e};
  const Span off{p.offsets, (static_cast<size_t>(p.nseq) + 1) * 4}, sl{p.slots, static_cast<size_t>(p.nseq) * 4};
  if (overlaps(y, x) || overlaps(y, si) || overlaps(y, so) || overlaps(y, wv) || overlaps(y, bv) ||
      overlaps(y, off) || overlaps(y, sl) || overlaps(so, x) || overlaps(so, wv) || overlaps(so, bv) ||
      overlaps(so, off) || overlaps(so, sl) || (p.state_in != p.state_out && overlaps(si, so)))
    return set_error(SMM_ERR_INVALID, "%s: an output overlaps an input", who);
  return SMM_OK;
}

template <bool STEP>
int run_conv(ConvParams& p, int width, int dtype, cudaStream_t st) {
  if (p.channels == 0 || p.nseq == 0) return SMM_OK;
  p.status = device_status_word();
  if (!p.status) return set_error(SMM_ERR_CUDA, "device status word unavailable");
  // accesses of four channels where every row, the weights and the states keep to them
  const size_t al = 4 * dtype_size(dtype);
  const bool vec = p.channels % 4 == 0 && p.ldx % 4 == 0 && p.ldy % 4 == 0 && aligned_to(p.x, al) &&
                   aligned_to(p.y, al) && aligned_to(p.w, al) && aligned_to(p.bias, al) && aligned_to(p.state_in, al) &&
                   aligned_to(p.state_out, al);
  const int cv = vec ? p.channels / 4 : p.channels;
  int bx = 32;
  while (bx < kConvThreads && bx < cv) bx *= 2;
  const int by = STEP ? 1 : kConvThreads / bx;
  p.ctiles = (cv + bx - 1) / bx;
  long long blocks;
  if (STEP) {
    blocks = static_cast<long long>(p.ctiles) * p.nseq;
  } else {
    // Runs of 64 rows read W-1 of 64 rows twice and start the pipeline once;
    // shorter ones where the GPU would otherwise be short of threads (12.1 us against
    // 13.7 for 3001 ragged rows with a threshold of 512).
    p.run = 64;
    while (p.run > 4 && static_cast<long long>(cv) * (p.tokens / p.run) < 148LL * 768) p.run /= 2;
    p.nruns = static_cast<int>(p.tokens > 0 ? (p.tokens + p.run - 1) / p.run : 1);
    blocks = static_cast<long long>(p.ctiles) * ((p.nruns + by - 1) / by);
  }
  if (blocks > 0x7FFFFFFFLL) return set_error(SMM_ERR_INVALID, "convolution too large for one launch");
  const dim3 grid(static_cast<unsigned>(blocks)), block(bx, by);
  if (dtype == SMM_DTYPE_F32) {
    if (vec)
      launch_width<float, 4, STEP>(width, grid, block, p, st);
    else
      launch_width<float, 1, STEP>(width, grid, block, p, st);
  } else {
    if (vec)
      launch_width<__nv_bfloat16, 4, STEP>(width, grid, block, p, st);
    else
      launch_width<__nv_bfloat16, 1, STEP>(width, grid, block, p, st);
  }
  count_launch();
  SMM_CUDA_TRY(cudaGetLastError(), STEP ? "conv_step launch" : "conv launch");
  return SMM_OK;
}

}  // namespace
}  // namespace smm

using namespace smm;

extern "C" int smm_causal_conv(const void* x, const void* w, const void* bias, const int* offsets,
                               const void* state_in, void* state_out, const int* slots, void* y, long long tokens,
                               int channels, int width, int nseq, int nslots, long long ldx, long long ldy, int dtype,
                               int act, void* stream) {
  SMM_RANGE("smm_causal_conv");
  ConvParams p{x, w, bias, offsets, state_in, state_out, slots, y, tokens, ldx, ldy, channels, nseq, nslots};
  p.silu = act == SMM_ACT_SILU;
  if (int rc = check_conv("smm_causal_conv", p, width, dtype, act, false)) return rc;
  if (tokens > 0x7FFFFFFFLL) return set_error(SMM_ERR_INVALID, "smm_causal_conv: %lld tokens exceed 31 bits", tokens);
  return run_conv<false>(p, width, dtype, as_stream(stream));
}

extern "C" int smm_causal_conv_step(const void* x, const void* w, const void* bias, const void* state_in,
                                    void* state_out, const int* slots, void* y, int batch, int channels, int width,
                                    int nslots, long long ldx, long long ldy, int dtype, int act, void* stream) {
  SMM_RANGE("smm_causal_conv_step");
  ConvParams p{x, w, bias, nullptr, state_in, state_out, slots, y, batch, ldx, ldy, channels, batch, nslots};
  p.silu = act == SMM_ACT_SILU;
  if (int rc = check_conv("smm_causal_conv_step", p, width, dtype, act, true)) return rc;
  if (batch == 0) return SMM_OK;
  return run_conv<true>(p, width, dtype, as_stream(stream));
}
