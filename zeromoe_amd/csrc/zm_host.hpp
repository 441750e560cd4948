// zm_host.hpp -- host helpers shared by the translation units of
// libzeromoe_hip.so: the thread-local error text behind zm_last_error(), the
// per-device IQ2_XXS grid and the MUL_MAT_ID hook launch counter.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace zm {

// record the reason of a rejected call; returns -1
int fail(const char *fmt, ...) __attribute__((format(printf, 1, 2)));
// the current device's IQ2_XXS grid (256 x u64, device memory), set up on first use
int device_grid(const uint64_t **grid);
// the current device's lookup table of a weight type: the IQ4_XS value table
// (16 x i8) for T_IQ4_XS, the IQ2_XXS grid otherwise
int device_table(int type, const uint64_t **table);
// one more executed MUL_MAT_ID hook launch (zm_mul_mat_id_launches)
void count_mmid_launch();
// S tokens bucketed by ids [S] below E <= 512 (others take no part) by one launch: counts [E], offs [E + 1], pairs [S],
// and items (mmq_item) of up to `tok` tokens of one id, at most S / tok + min(S, E) of them; active [E] and n_active too
void bucket_tokens(const int32_t *ids, int S, int E, int tok, int32_t *counts, int32_t *offs, int32_t *pairs,
                   int32_t *active, int32_t *n_active, int32_t *items, int32_t *n_items, hipStream_t stream);

}  // namespace zm

#define HIP_OK(call)                                                                  \
  do {                                                                                \
    hipError_t e_ = (call);                                                           \
    if (e_ != hipSuccess) return zm::fail("%s: %s", #call, hipGetErrorString(e_));    \
  } while (0)
