// zm_lora_a.hip -- adapters, forward: x by A, v by B
#include <hip/hip_runtime.h>

#include "zm_lora.hpp"

namespace zm {

void lora_forward(int x_type, int w_type, int y_type, const LoraArgs &g, dim3 grid, hipStream_t st) {
  if (x_type == LIN_BF16) {
    if (y_type == LIN_BF16) lora_launch<bf16, bf16, true, bf16>(g, grid, st);
    else lora_launch<bf16, bf16, true, float>(g, grid, st);
  } else if (x_type == LIN_F16) {
    if (y_type == LIN_F16) lora_launch<_Float16, _Float16, true, _Float16>(g, grid, st);
    else lora_launch<_Float16, _Float16, true, float>(g, grid, st);
  } else if (w_type == LIN_BF16) {
    lora_launch<float, bf16, true, float>(g, grid, st);
  } else if (w_type == LIN_F16) {
    lora_launch<float, _Float16, true, float>(g, grid, st);
  } else {
    lora_launch<float, float, true, float>(g, grid, st);
  }
}

}  // namespace zm
