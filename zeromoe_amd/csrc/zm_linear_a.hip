// zm_linear_a.hip -- products of the forward pass: x [S][I] by w [O][I], k contiguous in both
#include <hip/hip_runtime.h>

#include "zm_linear.hpp"

namespace zm {

void lin_fwd(int x_type, int w_type, const LinArgs &g, bool vec, int tile, hipStream_t st) {
  if (x_type == LIN_BF16) lin_launch<bf16, 1, true, bf16, 1, true>(g, vec, tile, st);
  else if (x_type == LIN_F16) lin_launch<_Float16, 1, true, _Float16, 1, true>(g, vec, tile, st);
  else if (w_type == LIN_BF16) lin_launch<float, 3, true, bf16, 1, true>(g, vec, tile, st);
  else if (w_type == LIN_F16) lin_launch<float, 3, true, _Float16, 2, true>(g, vec, tile, st);
  else lin_launch<float, 3, true, float, 3, true>(g, vec, tile, st);
}

}  // namespace zm
