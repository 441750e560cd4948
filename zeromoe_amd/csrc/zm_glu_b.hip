// zm_glu_b.hip -- the gated product of up to four rows and of up to 128
#include <hip/hip_runtime.h>

#include "zm_linear.hpp"

namespace zm {

void pair_rows(int x_type, int w_type, const LinArgs &g, hipStream_t st) {
  if (x_type == LIN_BF16) pair_rows_of<bf16, bf16>(g, st);
  else if (x_type == LIN_F16) pair_rows_of<_Float16, _Float16>(g, st);
  else if (w_type == LIN_BF16) pair_rows_of<float, bf16>(g, st);
  else if (w_type == LIN_F16) pair_rows_of<float, _Float16>(g, st);
  else pair_rows_of<float, float>(g, st);
}

void pair_few(int x_type, int w_type, const LinArgs &g, hipStream_t st) {
  if (x_type == LIN_BF16) pair_few_of<bf16, 1, bf16, 1>(g, st);
  else if (x_type == LIN_F16) pair_few_of<_Float16, 1, _Float16, 1>(g, st);
  else if (w_type == LIN_BF16) pair_few_of<float, 3, bf16, 1>(g, st);
  else if (w_type == LIN_F16) pair_few_of<float, 3, _Float16, 2>(g, st);
  else pair_few_of<float, 3, float, 3>(g, st);
}

}  // namespace zm
