// Prompt attention, head_dim 256 (kernel: fd_prefill.h).
#include "fd_prefill.h"

int fd_launch_prefill_d256(hipStream_t stream, const PrefillArgs& a, int q_dtype, bool fp8, int row_groups) {
#define FD_SHAPE(T_, F_)                                                             \
  (row_groups <= 2 ? launch_prefill<T_, F_, 256, 2, 1, 32>(stream, a) : launch_prefill<T_, F_, 256, 4, 1, 32>(stream, a))
  if (q_dtype == FD_BF16) return fp8 ? FD_SHAPE(__bf16, true) : FD_SHAPE(__bf16, false);
  return fp8 ? FD_SHAPE(_Float16, true) : FD_SHAPE(_Float16, false);
#undef FD_SHAPE
}
