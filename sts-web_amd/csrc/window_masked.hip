// window_masked.hip -- the instances of window_kernel.hpp's kernel behind
// sts_masked_attention.
#include "window_kernel.hpp"

namespace sts {

int launch_window_masked(const WindowParams& p, int row_tiles, bool bf16, dim3 grid,
                       hipStream_t stream) {
  return window::launch_mode<kWindowMasked>(p, row_tiles, bf16, grid, stream);
}

}  // namespace sts
