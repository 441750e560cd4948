// zm_lora_b.hip -- adapters: the product over the short axis, v by B and (backward) u by A; the sums over an adapter's
// tokens; a few tokens at once
#include <hip/hip_runtime.h>

#include "zm_lora.hpp"

namespace zm {
namespace {

template <class TW>
void expand(bool kc, const LoraArgs &g, int grid, hipStream_t st) {
  const size_t n = lora_expand_lds(g.R);
  if (kc) hipLaunchKernelGGL((k_lora_expand<TW, true>), dim3(grid), dim3(256), n, st, g);
  else hipLaunchKernelGGL((k_lora_expand<TW, false>), dim3(grid), dim3(256), n, st, g);
}
template <class TM, bool BY_R>
void sums(const LoraArgs &g, int grid, hipStream_t st) {
  switch (lora_r_of(g.R)) {
  case 16: hipLaunchKernelGGL((k_lora_sums<TM, 1, BY_R>), dim3(grid), dim3(256), 0, st, g); break;
  case 32: hipLaunchKernelGGL((k_lora_sums<TM, 2, BY_R>), dim3(grid), dim3(256), 0, st, g); break;
  default: hipLaunchKernelGGL((k_lora_sums<TM, 4, BY_R>), dim3(grid), dim3(256), 0, st, g);
  }
}
template <class TX, class TW>
void few(const LoraFewArgs &g, dim3 grid, hipStream_t st) {
  hipLaunchKernelGGL((k_lora_few<TX, TW>), grid, dim3(512), 0, st, g);
}

}  // namespace

void lora_expand(int w_type, bool kc, const LoraArgs &g, int grid, hipStream_t st) {
  if (w_type == LIN_BF16) expand<bf16>(kc, g, grid, st);
  else if (w_type == LIN_F16) expand<_Float16>(kc, g, grid, st);
  else expand<float>(kc, g, grid, st);
}
void lora_sums(int m_type, bool by_r, const LoraArgs &g, int grid, hipStream_t st) {
  if (m_type == LIN_BF16) by_r ? sums<bf16, true>(g, grid, st) : sums<bf16, false>(g, grid, st);
  else if (m_type == LIN_F16) by_r ? sums<_Float16, true>(g, grid, st) : sums<_Float16, false>(g, grid, st);
  else by_r ? sums<float, true>(g, grid, st) : sums<float, false>(g, grid, st);
}
void lora_few(int x_type, int w_type, const LoraFewArgs &g, dim3 grid, hipStream_t st) {
  if (x_type == LIN_BF16) few<bf16, bf16>(g, grid, st);
  else if (x_type == LIN_F16) few<_Float16, _Float16>(g, grid, st);
  else if (w_type == LIN_BF16) few<float, bf16>(g, grid, st);
  else if (w_type == LIN_F16) few<float, _Float16>(g, grid, st);
  else few<float, float>(g, grid, st);
}

}  // namespace zm
