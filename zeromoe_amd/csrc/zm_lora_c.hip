// zm_lora_c.hip -- adapters, the gradient by x: dy by B, u by A
#include <hip/hip_runtime.h>

#include "zm_lora.hpp"

namespace zm {

void lora_backward(int dy_type, int w_type, int dx_type, const LoraArgs &g, dim3 grid, hipStream_t st) {
  if (dx_type == LIN_BF16) {
    if (dy_type == LIN_BF16) lora_launch<bf16, bf16, false, bf16>(g, grid, st);
    else lora_launch<float, bf16, false, bf16>(g, grid, st);
  } else if (dx_type == LIN_F16) {
    if (dy_type == LIN_F16) lora_launch<_Float16, _Float16, false, _Float16>(g, grid, st);
    else lora_launch<float, _Float16, false, _Float16>(g, grid, st);
  } else if (w_type == LIN_BF16) {
    lora_launch<float, bf16, false, float>(g, grid, st);
  } else if (w_type == LIN_F16) {
    lora_launch<float, _Float16, false, float>(g, grid, st);
  } else {
    lora_launch<float, float, false, float>(g, grid, st);
  }
}

}  // namespace zm
