// Prompt attention, head_dim 64 (kernel: fd_prefill.h).
#include "fd_prefill.h"

int fd_launch_prefill_d64(hipStream_t stream, const PrefillArgs& a, int q_dtype, bool fp8, bool row_tiles) {
  if (q_dtype == FD_BF16)
    return fp8 ? launch_prefill<__bf16, true, 64>(stream, a, row_tiles) : launch_prefill<__bf16, false, 64>(stream, a, row_tiles);
  return fp8 ? launch_prefill<_Float16, true, 64>(stream, a, row_tiles) : launch_prefill<_Float16, false, 64>(stream, a, row_tiles);
}
