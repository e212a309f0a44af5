// Merge of the partials of prompt attention and of a shared-prefix decode step (gfx950).
//
// A row's partials (O_s, LSE_s) of disjoint key ranges merge to out = sum_s w_s O_s / sum_s w_s, w_s = e^{LSE_s - M},
// M = max_s LSE_s, LSE = M + log sum_s w_s.  Two lists of partials per row -- the key ranges of the row-tile kernel
// (fd_prefill.h) and, in a shared-prefix step, the ranges of the decode kernel over the sequence's own keys -- so that
// neither kernel needs to know of the other's count.  D / 4 lanes share a row and read 128 bits each; a wave's rows are
// neighbours.  Bound: the partials' bytes, and a launch's latency where there are few.
#include "fd_prefill.h"

namespace {

template <int D>
__global__ void __launch_bounds__(256) fd_prefill_merge_kernel(const PrefillMergeArgs a) {
  constexpr int L = D / 4;                     // lanes of a row
  const int64_t row = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  const int col = (threadIdx.x % L) * 4;
  if (row >= (int64_t)a.rows.total_q * a.rows.Hq) return;
  const int tok = (int)(row / a.rows.Hq), head = (int)(row - (int64_t)tok * a.rows.Hq);
  // the sequence (or group) that holds the token: the last one that starts at or before it
  bool inside = false;
  {
    int lo = 0, hi = a.rows.cu_q ? a.rows.batch : 0;
    while (lo < hi) {                          // first b with cu_q[b + 1] > tok
      const int mid = (lo + hi) >> 1;
      if (a.rows.cu_q[mid + 1] > tok) hi = mid; else lo = mid + 1;
    }
    if (lo < a.rows.batch) {
      int start, count;
      fd_prefill_span(a.rows, lo, start, count);
      inside = tok >= start && tok < start + count;
    }
  }
  if (!inside && !a.part1) return;             // a row behind the last sequence, or padding: left as it is
  const int S0 = inside ? a.rows.splits : 0;
  const float* l0 = a.rows.part_lse + row * a.rows.splits;
  const float* l1 = a.part1_lse + row * a.S1;
  float M = -INFINITY;
  for (int s = 0; s < S0; ++s) M = fmaxf(M, l0[s]);
  for (int s = 0; s < a.S1; ++s) M = fmaxf(M, l1[s]);
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  float L_sum = 0.f;
  auto add = [&](float lse, const float* p) {
    const float w = __expf(lse - M);
    if (w != 0.f) acc += *(const f32x4*)p * w;   // (the row of an empty range may hold anything)
    L_sum += w;
  };
  if (M != -INFINITY) {
    const float* p0 = a.rows.part + row * a.rows.splits * D + col;
    for (int s = 0; s < S0; ++s) add(l0[s], p0 + (int64_t)s * D);
    const float* p1 = a.part1 + row * a.S1 * D + col;
    for (int s = 0; s < a.S1; ++s) add(l1[s], p1 + (int64_t)s * D);
  }
  const float inv = L_sum != 0.f ? 1.0f / L_sum : 0.f;
  const int64_t dst = (int64_t)tok * a.rows.so_t + (int64_t)head * a.rows.so_h + col;
  u32x2 w;
  if (a.out_dtype == FD_BF16)
    w = u32x2{Mma<__bf16>::pack(acc[0] * inv, acc[1] * inv), Mma<__bf16>::pack(acc[2] * inv, acc[3] * inv)};
  else
    w = u32x2{Mma<_Float16>::pack(acc[0] * inv, acc[1] * inv), Mma<_Float16>::pack(acc[2] * inv, acc[3] * inv)};
  *(u32x2*)((uint16_t*)a.rows.out + dst) = w;
  if (a.rows.lse && col == 0) a.rows.lse[row] = L_sum != 0.f ? M + __logf(L_sum) : -INFINITY;
}

}  // namespace

int fd_launch_prefill_merge(hipStream_t stream, const PrefillMergeArgs& a, int head_dim) {
  const int per = 256 / (head_dim / 4);
  const int64_t wgs = ((int64_t)a.rows.total_q * a.rows.Hq + per - 1) / per;
  if (wgs >= ((int64_t)1 << 31)) return FD_ERR_TOO_LARGE;
  auto kern = head_dim == 64 ? fd_prefill_merge_kernel<64> : head_dim == 128 ? fd_prefill_merge_kernel<128> : fd_prefill_merge_kernel<256>;
  hipLaunchKernelGGL(kern, dim3((unsigned)wgs), dim3(256), 0, stream, a);
  return hipGetLastError() == hipSuccess ? FD_OK : FD_ERR_LAUNCH;
}
