// zm_glu_a.hip -- tiles of the gated product: x [S][I] by both weights [F][I], k contiguous in all
#include <hip/hip_runtime.h>

#include "zm_linear.hpp"

namespace zm {

void pair_fwd(int x_type, int w_type, const LinArgs &g, bool vec, int tile, hipStream_t st) {
  if (x_type == LIN_BF16) two_launch<LIN_PAIR, bf16, 1, bf16, 1>(g, vec, tile, st);
  else if (x_type == LIN_F16) two_launch<LIN_PAIR, _Float16, 1, _Float16, 1>(g, vec, tile, st);
  else if (w_type == LIN_BF16) two_launch<LIN_PAIR, float, 3, bf16, 1>(g, vec, tile, st);
  else if (w_type == LIN_F16) two_launch<LIN_PAIR, float, 3, _Float16, 2>(g, vec, tile, st);
  else two_launch<LIN_PAIR, float, 3, float, 3>(g, vec, tile, st);
}

}  // namespace zm
