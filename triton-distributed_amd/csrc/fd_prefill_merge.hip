// Merge of the partials of prompt attention and of a shared-prefix decode step (gfx950).
//
// A row's partials (O_s, LSE_s) of disjoint key ranges merge to out = sum_s w_s O_s / sum_s w_s, w_s = e^{LSE_s - M},
// M = max_s LSE_s, LSE = M + log sum_s w_s.  In a shared-prefix step the ranges of the group's prefix come first and those of
// the sequence's own keys behind them.  A wave has a row: its lanes take one LSE each, and 64 / (D / 4) groups of lanes, 128
// bits a lane, share the partials among them.  The first of those are requested together with the LSEs -- an empty range's
// partial may hold anything, its weight of 0 is never multiplied.  A NaN LSE -- a row that met a NaN -- makes the row NaN, in
// out and LSE, as it does where one range is stored without a merge.  Bound: a launch and a dependent round trip or two where
// there are few rows (4.6 us: 1280 rows of 8 partials), the partials' bytes else (6.5 us: 2048 rows of 17, 18 MB; 9.5 us with
// D / 4 lanes a row and the partials requested behind the LSEs).
#include "fd_prefill.h"

namespace {

template <int D>
__global__ void __launch_bounds__(256) fd_prefill_merge_kernel(const PrefillArgs a, int out_dtype) {
  constexpr int L = D / 4, H = 64 / L;         // lanes of a partial row, groups of them in a wave
  constexpr int kAhead = 8;                    // partial rows that a group requests together
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = lane / L, col = lane % L * 4;
  if (row >= (int64_t)a.total_q * a.Hq) return;
  const int tok = (int)(row / a.Hq), head = (int)(row - (int64_t)tok * a.Hq);
  const int NP = a.splits + a.own_splits;
  const float* lses = a.part_lse + row * NP;
  const float* parts = a.part + row * NP * D + col;
  f32x4 x[kAhead];
  auto request = [&](int s0, int n) {          // this group's partials of [s0, n)
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int s = s0 + k * H + group;
      if (s < n) x[k] = *(const f32x4*)(parts + (int64_t)s * D);
    }
  };
  float mine = lane < NP ? lses[lane] : -INFINITY;
  request(0, min(64, NP));
  // the sequence (or group) that holds the token: the last one that starts at or before it
  bool inside = false;
  {
    int lo = 0;                                // sequences that end at or before it, 64 offsets at a time
    if (a.cu_q) {
      for (int b0 = 0; b0 < a.batch; b0 += 64)
        lo += __popcll(__ballot(b0 + lane < a.batch && a.cu_q[b0 + lane + 1] <= tok));
    }
    if (lo < a.batch) {
      int start, count;
      fd_prefill_span(a, lo, start, count);
      inside = tok >= start && tok < start + count;
    }
  }
  if (!inside && a.own_splits == 0) return;    // a row behind the last sequence, or padding: left as it is
  const int first = inside ? 0 : a.splits;     // a row outside every group has its own keys only
  float M = -INFINITY, L_sum = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int base = 0; base < NP; base += 64) {
    const int n = min(base + 64, NP);
    if (base > 0) {
      mine = base + lane < NP ? lses[base + lane] : -INFINITY;
      request(base, n);
    }
    if (base + lane < first) mine = -INFINITY;
    float top = mine;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
    top = fmaxf(top, M);
    if (top == -INFINITY && !__any(mine != mine)) continue;   // nothing seen so far (a NaN LSE, which fmaxf drops, is not that)
    const float keep = __expf(M - top);        // 0 in the first pass that counts
    acc *= keep;
    M = top;
    const float weight = __expf(mine - M);
    float sum = weight;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
    L_sum = L_sum * keep + sum;
    for (int s0 = base; s0 < n; s0 += kAhead * H) {
      if (s0 > base) request(s0, n);
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int s = s0 + k * H + group;
        const float w = __shfl(weight, (s - base) & 63);
        if (s < n && w != 0.f) acc += x[k] * w;
      }
    }
  }
#pragma unroll
  for (int off = L; off < 64; off <<= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], off);
  if (group > 0) return;
  const float inv = L_sum != 0.f ? 1.0f / L_sum : 0.f;
  const int64_t dst = (int64_t)tok * a.so_t + (int64_t)head * a.so_h + col;
  u32x2 w;
  if (out_dtype == FD_BF16)
    w = u32x2{Mma<__bf16>::pack(acc[0] * inv, acc[1] * inv), Mma<__bf16>::pack(acc[2] * inv, acc[3] * inv)};
  else
    w = u32x2{Mma<_Float16>::pack(acc[0] * inv, acc[1] * inv), Mma<_Float16>::pack(acc[2] * inv, acc[3] * inv)};
  *(u32x2*)((uint16_t*)a.out + dst) = w;
  if (a.lse && col == 0) a.lse[row] = L_sum != 0.f ? M + __logf(L_sum) : -INFINITY;
}

}  // namespace

int fd_launch_prefill_merge(hipStream_t stream, const PrefillArgs& a, int head_dim, int out_dtype) {
  const int64_t wgs = ((int64_t)a.total_q * a.Hq + 3) / 4;
  if (wgs >= ((int64_t)1 << 31)) return FD_ERR_TOO_LARGE;
  auto kern = head_dim == 64 ? fd_prefill_merge_kernel<64> : head_dim == 128 ? fd_prefill_merge_kernel<128> : fd_prefill_merge_kernel<256>;
  hipLaunchKernelGGL(kern, dim3((unsigned)wgs), dim3(256), 0, stream, a, out_dtype);
  return hipGetLastError() == hipSuccess ? FD_OK : FD_ERR_LAUNCH;
}
