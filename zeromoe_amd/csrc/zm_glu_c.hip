// zm_glu_c.hip -- the gated product's gradient by x: dg [S][F] by w_gate plus du [S][F] by w_up [F][I], k = F contiguous in
// dg and du, rows in the weights.  dg and du are f32: next to a 16-bit x they enter with 16 bits, as zm_linear's dz does.
#include <hip/hip_runtime.h>

#include "zm_linear.hpp"

namespace zm {

void pair_dx(int x_type, int w_type, const LinArgs &g, bool vec, int tile, hipStream_t st) {
  if (x_type == LIN_BF16) two_launch<LIN_SUM, bf16, 1, bf16, 1>(g, vec, tile, st);
  else if (x_type == LIN_F16) two_launch<LIN_SUM, float, 2, _Float16, 2>(g, vec, tile, st);
  else if (w_type == LIN_BF16) two_launch<LIN_SUM, float, 3, bf16, 1>(g, vec, tile, st);
  else if (w_type == LIN_F16) two_launch<LIN_SUM, float, 3, _Float16, 2>(g, vec, tile, st);
  else two_launch<LIN_SUM, float, 3, float, 3>(g, vec, tile, st);
}

}  // namespace zm
