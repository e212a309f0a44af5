// Prompt attention, head_dim 128 (kernel: fd_prefill.h).
#include "fd_prefill.h"

int fd_launch_prefill_d128(hipStream_t stream, const PrefillArgs& a, int q_dtype, bool fp8, bool row_tiles) {
  if (q_dtype == FD_BF16)
    return fp8 ? launch_prefill<__bf16, true, 128>(stream, a, row_tiles) : launch_prefill<__bf16, false, 128>(stream, a, row_tiles);
  return fp8 ? launch_prefill<_Float16, true, 128>(stream, a, row_tiles) : launch_prefill<_Float16, false, 128>(stream, a, row_tiles);
}
