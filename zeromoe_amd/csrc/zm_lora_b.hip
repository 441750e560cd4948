// zm_lora_b.hip -- adapters: the sums over an adapter's tokens, and a few tokens at once
#include <hip/hip_runtime.h>

#include <algorithm>

#include "zm_lora.hpp"

namespace zm {
namespace {

template <class TX, class TY>
void sums(const LoraItems &items, const LoraSumArgs &a, unsigned na, const LoraSumArgs &b, unsigned nb, hipStream_t st) {
  // (2^22 workgroups at a time: a launch has less than 2^32 threads)
  constexpr unsigned MOST = 1u << 22;
  for (unsigned first = 0; first < na + nb; first += MOST) {
    const dim3 grid(std::min(MOST, na + nb - first)), wg(64 * LORA_WAVES);
    switch (lora_r_of(a.R)) {
    case 16: hipLaunchKernelGGL((k_lora_sums<TX, TY, 1>), grid, wg, 0, st, items, a, b, na, first); break;
    case 32: hipLaunchKernelGGL((k_lora_sums<TX, TY, 2>), grid, wg, 0, st, items, a, b, na, first); break;
    default: hipLaunchKernelGGL((k_lora_sums<TX, TY, 4>), grid, wg, 0, st, items, a, b, na, first);
    }
  }
}
template <class TX, class TW>
void few(const LoraFewArgs &g, dim3 grid, hipStream_t st) {
  if (g.R <= 16) hipLaunchKernelGGL((k_lora_few<TX, TW, 2>), grid, dim3(512), 0, st, g);
  else hipLaunchKernelGGL((k_lora_few<TX, TW, 4>), grid, dim3(512), 0, st, g);
}

}  // namespace

void lora_sums(int x_type, int dy_type, const LoraItems &items, const LoraSumArgs &a, unsigned na, const LoraSumArgs &b,
               unsigned nb, hipStream_t st) {
  if (x_type == LIN_BF16) {
    if (dy_type == LIN_BF16) sums<bf16, bf16>(items, a, na, b, nb, st);
    else sums<bf16, float>(items, a, na, b, nb, st);
  } else if (x_type == LIN_F16) {
    if (dy_type == LIN_F16) sums<_Float16, _Float16>(items, a, na, b, nb, st);
    else sums<_Float16, float>(items, a, na, b, nb, st);
  } else {
    sums<float, float>(items, a, na, b, nb, st);
  }
}
void lora_few(int x_type, int w_type, const LoraFewArgs &g, dim3 grid, hipStream_t st) {
  if (x_type == LIN_BF16) few<bf16, bf16>(g, grid, st);
  else if (x_type == LIN_F16) few<_Float16, _Float16>(g, grid, st);
  else if (w_type == LIN_BF16) few<float, bf16>(g, grid, st);
  else if (w_type == LIN_F16) few<float, _Float16>(g, grid, st);
  else few<float, float>(g, grid, st);
}

}  // namespace zm
