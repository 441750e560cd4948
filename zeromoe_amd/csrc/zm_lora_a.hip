// zm_lora_a.hip -- adapters: the product over the long axis, x by A and (backward) dy by B
#include <hip/hip_runtime.h>

#include "zm_lora.hpp"

namespace zm {
namespace {

template <class TX, class TW, bool KC>
void launch(const LoraArgs &g, int grid, hipStream_t st) {
  switch (lora_r_of(g.R)) {
  case 16: hipLaunchKernelGGL((k_lora_shrink<TX, TW, KC, 1>), dim3(grid), dim3(256), 0, st, g); break;
  case 32: hipLaunchKernelGGL((k_lora_shrink<TX, TW, KC, 2>), dim3(grid), dim3(256), 0, st, g); break;
  default: hipLaunchKernelGGL((k_lora_shrink<TX, TW, KC, 4>), dim3(grid), dim3(256), 0, st, g);
  }
}
template <class TX, class TW>
void of(bool kc, const LoraArgs &g, int grid, hipStream_t st) {
  if (kc) launch<TX, TW, true>(g, grid, st);
  else launch<TX, TW, false>(g, grid, st);
}

}  // namespace

void lora_shrink(int x_type, int w_type, bool kc, const LoraArgs &g, int grid, hipStream_t st) {
  if (x_type == LIN_BF16) of<bf16, bf16>(kc, g, grid, st);
  else if (x_type == LIN_F16) of<_Float16, _Float16>(kc, g, grid, st);
  else if (w_type == LIN_BF16) of<float, bf16>(kc, g, grid, st);
  else if (w_type == LIN_F16) of<float, _Float16>(kc, g, grid, st);
  else of<float, float>(kc, g, grid, st);
}

}  // namespace zm
