// zm_linear_b.hip -- products of the gradient by x: dz [S][O] by w [O][I], k = O contiguous in dz, rows in w.
//
// The result has x's type.  Where that is 16 bits and dz is not (behind an activation, or from an f32 result), dz enters
// with two bf16 terms, 16 bits: what they leave out is 2^-16 of |dz w|, next to the result's own rounding of 2^-8 (bf16)
// or 2^-11 (f16).  One term, 2^-8 of |dz w|, would be more than the result's rounding wherever the sum cancels (and one
// f16 term could overflow or lose small gradients).
#include <hip/hip_runtime.h>

#include "zm_linear.hpp"

namespace zm {

void lin_dx(int x_type, int w_type, int dz_type, const LinArgs &g, bool vec, int tile, hipStream_t st) {
  if (x_type == LIN_BF16) {
    lin_launch<bf16, 1, true, bf16, 1, false>(g, vec, tile, st);
  } else if (x_type == LIN_F16) {
    if (dz_type == LIN_F32) lin_launch<float, 2, true, _Float16, 2, false>(g, vec, tile, st);
    else lin_launch<_Float16, 1, true, _Float16, 1, false>(g, vec, tile, st);
  } else if (w_type == LIN_BF16) {
    lin_launch<float, 3, true, bf16, 1, false>(g, vec, tile, st);
  } else if (w_type == LIN_F16) {
    lin_launch<float, 3, true, _Float16, 2, false>(g, vec, tile, st);
  } else {
    lin_launch<float, 3, true, float, 3, false>(g, vec, tile, st);
  }
}

}  // namespace zm
