// zm_linear_d.hip -- the product of up to four rows
#include "zm_linear.hpp"

namespace zm {

void lin_rows(int x_type, int w_type, const LinArgs &g, hipStream_t st) {
  if (x_type == LIN_BF16) lin_rows_of<bf16, bf16>(g, st);
  else if (x_type == LIN_F16) lin_rows_of<_Float16, _Float16>(g, st);
  else if (w_type == LIN_BF16) lin_rows_of<float, bf16>(g, st);
  else if (w_type == LIN_F16) lin_rows_of<float, _Float16>(g, st);
  else lin_rows_of<float, float>(g, st);
}

}  // namespace zm
