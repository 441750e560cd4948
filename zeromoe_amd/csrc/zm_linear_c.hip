// zm_linear_c.hip -- products of the gradient by w: dz [S][O] by x [S][I], k = S, rows contiguous in both.
//
// The result is f32, so an f32 dz keeps all its digits: next to bf16 it is three planes of bf16 terms, whose products
// are added (two, 16 bits, left dw of a 2048 x 4096 x 1536 layer 2.8e-6 off, against 8e-7 of an f32 product).
#include <hip/hip_runtime.h>

#include "zm_linear.hpp"

namespace zm {

void lin_dw(int x_type, int dz_type, const LinArgs &g, bool vec, int tile, hipStream_t st) {
  if (x_type == LIN_BF16) {
    lin_launch<bf16, 1, false, bf16, 1, false>(g, vec, tile, st);
  } else if (x_type == LIN_F16) {
    if (dz_type == LIN_F32) lin_launch<float, 3, false, _Float16, 2, false>(g, vec, tile, st);
    else lin_launch<_Float16, 1, false, _Float16, 1, false>(g, vec, tile, st);
  } else {
    lin_launch<float, 3, false, float, 3, false>(g, vec, tile, st);
  }
}

}  // namespace zm
