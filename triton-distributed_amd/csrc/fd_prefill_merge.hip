// Merge of the partials of prompt attention and of a shared-prefix decode step (gfx950).
//
// A row's partials (O_s, LSE_s) of disjoint key ranges merge to out = sum_s w_s O_s / sum_s w_s, w_s = e^{LSE_s - M},
// M = max_s LSE_s, LSE = M + log sum_s w_s.  In a shared-prefix step the ranges of the group's prefix come first and those of
// the sequence's own keys behind them.  D / 4 lanes share a row: each takes one LSE, the weights go round by shuffles, and
// eight partial rows are requested together, 128 bits a lane.  Bound: a launch and its two dependent round trips where there
// are few rows (4.3 us: 1280 rows of 8 partials), the partials' bytes else (9.5 us: 2048 rows of 17, 18 MB).
#include "fd_prefill.h"

namespace {

template <int D>
__global__ void __launch_bounds__(256) fd_prefill_merge_kernel(const PrefillArgs a, int out_dtype) {
  constexpr int L = D / 4;                     // lanes of a row
  constexpr int kAhead = 8;                    // partial rows requested together
  const int64_t row = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  const int sub = threadIdx.x % L, col = sub * 4;
  if (row >= (int64_t)a.total_q * a.Hq) return;      // (all lanes of a row, which are all that exchange anything)
  const int tok = (int)(row / a.Hq), head = (int)(row - (int64_t)tok * a.Hq);
  const int NP = a.splits + a.own_splits;
  const float* lses = a.part_lse + row * NP;
  const float* parts = a.part + row * NP * D + col;
  // the first L LSEs, one a lane, are requested before it is known which of them count
  float mine = sub < NP ? lses[sub] : -INFINITY;
  // the sequence (or group) that holds the token: the last one that starts at or before it
  bool inside = false;
  {
    int lo = 0;                                // sequences that end at or before it, L offsets at a time
    if (a.cu_q) {
      for (int b = sub; b - sub < a.batch; b += L) {
        const int past = b < a.batch && a.cu_q[b + 1] <= tok ? 1 : 0;
        const uint64_t all = __ballot(past);
        lo += __popcll(L == 64 ? all : (all >> ((threadIdx.x & 63) / L * L)) & ((1ull << (L & 63)) - 1));
      }
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
  for (int base = 0; base < NP; base += L) {
    if (base > 0) mine = base + sub < NP ? lses[base + sub] : -INFINITY;
    if (base + sub < first) mine = -INFINITY;
    float top = mine;
#pragma unroll
    for (int off = L / 2; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, L));
    top = fmaxf(top, M);
    if (top == -INFINITY) continue;
    const float keep = __expf(M - top);        // 0 in the first pass that counts
    acc *= keep;
    L_sum *= keep;
    M = top;
    const float weight = __expf(mine - M);
    const int n = min(L, NP - base);
    for (int s0 = 0; s0 < n; s0 += kAhead) {
      f32x4 x[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (s0 + k < n) x[k] = *(const f32x4*)(parts + (int64_t)(base + s0 + k) * D);
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const float w = __shfl(weight, (s0 + k) % L, L);
        if (s0 + k < n) {
          if (w != 0.f) acc += x[k] * w;       // (the row of an empty range may hold anything)
          L_sum += w;
        }
      }
    }
  }
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
  const int per = 256 / (head_dim / 4);
  const int64_t wgs = ((int64_t)a.total_q * a.Hq + per - 1) / per;
  if (wgs >= ((int64_t)1 << 31)) return FD_ERR_TOO_LARGE;
  auto kern = head_dim == 64 ? fd_prefill_merge_kernel<64> : head_dim == 128 ? fd_prefill_merge_kernel<128> : fd_prefill_merge_kernel<256>;
  hipLaunchKernelGGL(kern, dim3((unsigned)wgs), dim3(256), 0, stream, a, out_dtype);
  return hipGetLastError() == hipSuccess ? FD_OK : FD_ERR_LAUNCH;
}
