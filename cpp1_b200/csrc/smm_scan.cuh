// Selective state space scan: what the two prompt kernels (smm_scan.cu on the
// fp32 pipes, smm_scan_umma.cu on the tensor cores) share.
//
// Long sequences are split into segments of seg_len tokens so that few heads
// still fill the GPU.  A segment's work needs the state before it, which is
// linear in the states that the earlier segments would end with when started
// from zero:  S_before(j) = exp(a_0+..+a_{j-1}) S_in + sum_k exp(a_{k+1}+..+a_{j-1}) F_k
// with a_k the sum of d A over segment k and F_k its final state from zero.
// A first launch writes every F_k and a_k (all but the last segment of each
// sequence, in whose place it puts S_in), a second one turns them into the states
// before each segment, a third one computes the outputs.  (Each CTA of the last launch
// summing its own state's terms instead read up to as many of them as there are parts,
// one after another: 24 heads of 8192 tokens in six parts took 88 us that way, 77 this way.)
#pragma once
#include "smm_seq.cuh"

namespace smm {

struct ScanParams {
  const void* x;
  const void* dt;
  const float* A;
  const void* B;
  const void* C;
  const float* D;
  const void* z;
  const float* dt_bias;
  const int* offsets;
  const float* state_in;
  float* state_out;
  const int* slots;
  void* y;
  long long tokens, ldx, lddt, ldb, ldc, ldz, ldy;
  int nseq, nslots, heads, dim, groups, state_dim;
  int dt_f32, softplus;
  int seg_len;       // tokens per segment (tokens or more: no sequence is split)
  int split;         // seg_len < tokens
  float* seg_state;  // [segment][head][dim][state_dim]: F_k
  float* seg_log;    // [segment][head]: a_k
  uint32_t* status;
  unsigned long long wait_limit_ns;
};

constexpr float kLog2e = 1.4426950408889634f;

// dt as it lies (the 16 bits of a bf16 element, or an fp32 one), and d from it
// and the head's bias: loads stay ahead of the arithmetic that waits for them.
__device__ __forceinline__ uint32_t scan_dt_raw(const ScanParams& p, long long t, int h) {
  const long long i = t * p.lddt + h;
  return p.dt_f32 ? __ldg(static_cast<const uint32_t*>(p.dt) + i)
                  : static_cast<uint32_t>(__ldg(static_cast<const unsigned short*>(p.dt) + i));
}
__device__ __forceinline__ float scan_dt(const ScanParams& p, uint32_t raw, float bias) {
  const float d = __uint_as_float(p.dt_f32 ? raw : raw << 16) + bias;
  return p.softplus ? softplus(d) : d;
}

__device__ __forceinline__ int segments_of(const ScanParams& p, long long begin, long long end) {
  return end > begin ? static_cast<int>((end - begin + p.seg_len - 1) / p.seg_len) : 1;
}

// One segment: sequence, its index in the sequence, how many the sequence
// has, and the rows.
struct Segment {
  int seq, j, count;
  long long begin, end;
  bool valid;
};

// Finds segment `seg`: sequences have max(1, ceil(length / seg_len)) each.
// Called by one full warp.
__device__ __forceinline__ Segment find_segment(const ScanParams& p, int seg) {
  Segment r;
  r.valid = false;
  r.seq = r.j = 0;
  r.count = 1;
  r.begin = r.end = 0;
  if (!p.split) {
    if (seg >= p.nseq) return r;
    r.seq = seg;
    seq_range(p.offsets, seg, p.tokens, &r.begin, &r.end);
    r.valid = true;
    return r;
  }
  const int lane = threadIdx.x & 31;
  int base = 0;
  for (int s0 = 0; s0 < p.nseq; s0 += 32) {
    long long b = 0, e = 0;
    int n = 0;
    if (s0 + lane < p.nseq) {
      seq_range(p.offsets, s0 + lane, p.tokens, &b, &e);
      n = segments_of(p, b, e);
    }
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
      if (lane >= o) incl += v;
    }
    const unsigned hit = __ballot_sync(0xFFFFFFFFu, seg < base + incl && n > 0);
    if (hit) {
      const int src = __ffs(hit) - 1;
      const int end_incl = __shfl_sync(0xFFFFFFFFu, incl, src);
      r.count = __shfl_sync(0xFFFFFFFFu, n, src);
      b = __shfl_sync(0xFFFFFFFFu, b, src);
      e = __shfl_sync(0xFFFFFFFFu, e, src);
      r.seq = s0 + src;
      r.j = seg - (base + end_incl - r.count);
      r.begin = b + static_cast<long long>(r.j) * p.seg_len;
      r.end = r.begin + p.seg_len < e ? r.begin + p.seg_len : e;
      r.valid = true;
      return r;
    }
    base += __shfl_sync(0xFFFFFFFFu, incl, 31);
  }
  return r;
}

// Segments that the grid and the workspace provide for.
inline long long max_segments(long long tokens, int nseq, int seg_len) {
  return seg_len >= tokens ? nseq : nseq + tokens / seg_len;
}

// smm_scan.cu: between the two launches of a split scan
int scan_combine(const ScanParams& p, cudaStream_t st);

// smm_scan_umma.cu
bool scan_umma_fits(const ScanParams& p, int dtype);
int scan_umma_launch(ScanParams& p, cudaStream_t st);

}  // namespace smm
