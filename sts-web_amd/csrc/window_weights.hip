// window_weights.hip -- the instances of window_kernel.hpp's kernel behind
// sts_decode_ring_weights.
#include "window_kernel.hpp"

namespace sts {

int launch_window_weights(const WindowParams& p, int row_tiles, bool bf16, dim3 grid,
                       hipStream_t stream) {
  return window::launch_mode<kWindowWeights>(p, row_tiles, bf16, grid, stream);
}

}  // namespace sts
