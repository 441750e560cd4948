// zm_lora.hip -- C ABI of the adapters that each token names, and of their gradients: checks, workspace layout and the
// choice of kernels, which are in zm_lora.hpp.
#include <hip/hip_runtime.h>

#include "zm_linear_host.hpp"
#include "zm_lora.hpp"

using namespace zm;

namespace {

int check_lora(const zm_lora_desc *d, const char *who) {
  if (!d) return fail("%s: null description", who);
  if (!lin_type(d->x_type) || !lin_type(d->w_type) || !lin_type(d->y_type))
    return fail("%s: types are F32, F16 and BF16", who);
  if (d->x_type != ZM_TYPE_F32 && d->w_type != d->x_type)
    return fail("%s: 16-bit activations need adapters of their own type", who);
  if (d->y_type != ZM_TYPE_F32 && d->y_type != d->x_type)
    return fail("%s: the result is F32 or of the activations' type", who);
  if (d->n <= 0 || d->n > LORA_MOST_N) return fail("%s: 1 to %d adapters, not %d", who, LORA_MOST_N, d->n);
  if (d->R <= 0 || d->R > LORA_MOST_R) return fail("%s: a rank of 1 to %d, not %d", who, LORA_MOST_R, d->R);
  if (d->S < 0 || d->S >= 1 << 24) return fail("%s: S from 0 to 2^24 is needed", who);
  if (d->I <= 0 || d->O <= 0 || d->I >= 1 << 30 || d->O >= 1 << 30) return fail("%s: I and O from 1 to 2^30 are needed", who);
  if (d->x_stride < 0 || d->y_stride < 0 || d->res_stride < 0 || d->a_stride < 0 || d->b_stride < 0 || d->a_adapter < 0 ||
      d->b_adapter < 0)
    return fail("%s: negative stride", who);
  const int64_t most = ((int64_t)1 << 31) / (int64_t)size_of(d->w_type);
  auto large = [&](int64_t rows, int64_t stride, int64_t width) {  // (a stride that large first: the product may pass 64 bits)
    return rows > 1 && (stride >= most || (rows - 1) * stride + width >= most);
  };
  if (d->I >= most || large(d->R, d->a_stride, d->I) || large(d->O, d->b_stride, d->R))
    return fail("%s: an adapter's a and b are below 2^31 bytes", who);
  if ((std::max(d->I, d->O) / 64 + 1) * ((d->R + 15) / 16) * d->n >= 1 << 26) return fail("%s: n x R x I or n x R x O too large", who);
  return 0;
}

// Work items are counted on the device; a launch has as many as there can be.  Items of 16 tokens are worth it where no CU
// gets two of them: that may be so up to 384, with a third of the tokens without an adapter.
int64_t items_of(const zm_lora_desc &d, int T) { return d.S / T + std::min<int64_t>(d.S, d.n); }
bool small_items(const zm_lora_desc &d) { return items_of(d, 16) <= LORA_CUS * 3 / 2; }
int64_t most_items(const zm_lora_desc &d) { return items_of(d, small_items(d) ? 16 : LORA_TOKENS); }

// slices of an axis of K, `unit` at a time, for `want` workgroups where one slice has `n`
int64_t slices_of(int64_t n, int64_t want, int64_t K, int64_t unit, int64_t most) {
  return std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(want / std::max<int64_t>(n, 1), most), K / unit));
}

// slices of an adapter's tokens for its gradient of N columns: both gradients are one launch, of a workgroup for each CU
// where there are tokens for it; the slices' sums take at most 64 MB
int sums_slices(const zm_lora_desc &d, int64_t N) {
  const int64_t groups = ((d.I + 63) / 64 + (d.O + 63) / 64) * ((d.R + lora_r_of(d.R) - 1) / lora_r_of(d.R)) * d.n;
  return (int)slices_of(groups, 256, d.S / d.n, 256, (64 << 20) / (4 * N * d.R * d.n));
}
size_t sums_space(const zm_lora_desc &d, int64_t N) {
  const int z = sums_slices(d, N);
  return z > 1 ? align256((size_t)z * d.n * d.R * N * 4) : 0;
}

// Few items with much to read each are shared by several CUs: the long axis in `slices` of k, the short one in `groups` of
// columns, each a launch.  (116 tokens of three adapters of rank 128, 4516 x 3457: 78 -> 37 us; one token of rank
// 256, 8192 x 8192: 148 -> 32.)
struct Split {
  int slices, groups;
  int64_t kslice;
  size_t part;  // bytes; 0: one launch
};
Split split_of(const zm_lora_desc &d, int64_t K, int64_t N) {
  Split s{1, 1, K, 0};
  const int64_t n = most_items(d), cus = LORA_CUS / n;
  if (cus < 2 || d.R * (K + N) * (int64_t)size_of(d.w_type) < 256 << 10) return s;
  const int64_t z = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(cus, 16), K / 512));
  s.kslice = ((K + z - 1) / z + 511) / 512 * 512;
  s.slices = (int)((K + s.kslice - 1) / s.kslice);
  s.groups = (int)std::max<int64_t>(1, std::min<int64_t>(cus, (N + 511) / 512));
  s.part = align256((size_t)s.slices * d.S * d.R * 4);
  return s;
}

// Workspace: the items | v or u of the slices | (backward) u, and the slices' sums of each gradient.
struct Space {
  size_t items, part, u, total;
};
size_t item_bytes(const zm_lora_desc &d) { return align256((2 * d.n + 2 + (LORA_TOKENS + 1) * most_items(d)) * 4); }
Space space_of(const zm_lora_desc &d, bool backward) {
  Space s{};
  s.items = item_bytes(d);
  s.part = backward ? std::max(split_of(d, d.O, d.I).part, split_of(d, d.O, 0).part) : split_of(d, d.I, d.O).part;
  if (backward) s.u = align256((size_t)d.S * d.R * 4);
  s.total = s.items + s.part + s.u + (backward ? sums_space(d, d.I) + sums_space(d, d.O) : 0);
  return s;
}

// One launch for a few tokens, each computing its v for every 512 columns again: where that is little to read.
bool few_tokens(const zm_lora_desc &d) {
  const int64_t a = d.R * d.I * (int64_t)size_of(d.w_type);
  return d.S <= 4096 && a <= 1 << 20 && d.S * ((d.O + 511) / 512) * a <= 64 << 20;
}

LoraArgs items(const zm_lora_desc &d, const int32_t *ids, const float *scale, uint8_t *ws, hipStream_t st) {
  LoraArgs g{};
  g.R = d.R;
  g.S = (int)d.S;
  g.n = d.n;
  g.ids = ids;
  g.scale = scale;
  int32_t *p = (int32_t *)ws;
  const int64_t most = most_items(d);
  g.rest = (int)((d.S + most - 1) / most);
  g.it.small = small_items(d);
  g.it.tokens = p;
  g.it.item = p + LORA_TOKENS * most;
  g.it.counts = g.it.item + most;
  g.it.first = g.it.counts + d.n;
  g.it.n_items = g.it.first + d.n;
  hipLaunchKernelGGL(k_lora_items, dim3(1), dim3(1024), 0, st, ids, (int)d.S, (int)d.n, g.it);
  return g;
}
template <class F>
void launch(const zm_lora_desc &d, F kernel, int x_type, int y_type, LoraArgs g, float *part, hipStream_t st) {
  const unsigned n = (unsigned)most_items(d);
  const Split s = split_of(d, g.K, g.N);
  if (!s.part) {
    g.phase = LoraArgs::BOTH;
    return kernel(x_type, d.w_type, y_type, g, dim3(n), st);
  }
  g.slices = s.slices;
  g.kslice = s.kslice;
  g.part = part;
  g.phase = LoraArgs::LONG;
  kernel(x_type, d.w_type, y_type, g, dim3(n, s.slices), st);
  g.phase = LoraArgs::SHORT;
  kernel(x_type, d.w_type, y_type, g, dim3(n, s.groups), st);
}
LoraSumArgs sums_args(const zm_lora_desc &d, const float *a, const void *m, int64_t ldm, int64_t N, const float *scale,
                      float *dst, float *space) {
  LoraSumArgs g{};
  g.a = a;
  g.m = m;
  g.ldm = ldm;
  g.N = N;
  g.R = d.R;
  g.n = d.n;
  g.slices = sums_slices(d, N);
  g.chunks = (d.R + lora_r_of(d.R) - 1) / lora_r_of(d.R);
  g.scale = scale;
  g.out = g.slices > 1 ? space : dst;
  return g;
}
unsigned sums_groups(const LoraSumArgs &g) { return (unsigned)((g.N + 63) / 64 * g.chunks * g.slices * g.n); }
void join_sums(const LoraSumArgs &g, const LoraItems &it, float *dst, hipStream_t st) {
  const int64_t all = (int64_t)g.n * g.R * g.N;
  if (g.slices > 1) parts_sum(g.out, g.slices, all, all, dst, nullptr, st, {g.scale, it.counts, g.R * g.N});
}

int check_space(void *ws, size_t size, size_t need, const char *who) {
  if (need && (!ws || size < need || ((uintptr_t)ws & 255)))
    return fail("%s: a 256-byte aligned workspace of %s_workspace_size() bytes is needed", who, who);
  return 0;
}

}  // namespace

extern "C" {

size_t zm_lora_workspace_size(const zm_lora_desc *d) {
  if (check_lora(d, "zm_lora_workspace_size") || !d->S || few_tokens(*d)) return 0;
  return space_of(*d, false).total;
}

int zm_lora(const zm_lora_desc *d, const void *x, const void *a, const void *b, const int32_t *ids, const float *scale,
            const void *residual, void *y, float *v, void *workspace, size_t workspace_size, void *stream) {
  if (check_lora(d, "zm_lora")) return -1;
  if (check_rows(d->S, d->y_stride, d->O, "zm_lora", "y")) return -1;
  if (!d->S) return 0;
  if (!x || !a || !b || !ids || !y) return fail("zm_lora: null pointer");
  if (residual == y && d->S > 1 && d->res_stride != d->y_stride) return fail("zm_lora: a residual in the place of y has y's stride");
  const hipStream_t st = (hipStream_t)stream;
  if (few_tokens(*d)) {
    LoraFewArgs g{x, a, b, d->x_stride, d->a_stride, d->b_stride, d->a_adapter, d->b_adapter, d->I, d->O, d->R, d->n, ids,
                  scale, residual, y, v, d->res_stride, d->y_stride, d->y_type};
    lora_few(d->x_type, d->w_type, g, dim3((unsigned)((d->O + 511) / 512), (unsigned)d->S), st);
    return launched();
  }
  const Space s = space_of(*d, false);
  if (check_space(workspace, workspace_size, s.total, "zm_lora")) return -1;
  LoraArgs g = items(*d, ids, scale, (uint8_t *)workspace, st);
  g.x = x;
  g.ldx = d->x_stride;
  g.m = a;
  g.ldm = d->a_stride;
  g.m_adapter = d->a_adapter;
  g.K = d->I;
  g.l = b;
  g.ldl = d->b_stride;
  g.l_adapter = d->b_adapter;
  g.N = d->O;
  g.res = residual;
  g.ldr = d->res_stride;
  g.y = y;
  g.ldy = d->y_stride;
  g.v = v;
  launch(*d, lora_forward, d->x_type, d->y_type, g, (float *)((uint8_t *)workspace + s.items), st);
  return launched();
}

size_t zm_lora_backward_workspace_size(const zm_lora_desc *d) {
  if (check_lora(d, "zm_lora_backward_workspace_size") || !d->S) return 0;
  return space_of(*d, true).total;
}

int zm_lora_backward(const zm_lora_desc *d, const void *dy, const void *x, const void *a, const void *b, const int32_t *ids,
                     const float *scale, const float *v, void *dx, float *da, float *db, void *workspace,
                     size_t workspace_size, void *stream) {
  if (check_lora(d, "zm_lora_backward")) return -1;
  const hipStream_t st = (hipStream_t)stream;
  if (!d->S) {  // no tokens: the sums over them are zero
    if (da) hipLaunchKernelGGL(k_linear_zero, dim3(256), dim3(256), 0, st, da, d->n * d->R * d->I);
    if (db) hipLaunchKernelGGL(k_linear_zero, dim3(256), dim3(256), 0, st, db, d->n * d->R * d->O);
    return launched();
  }
  if (!dx && !da && !db) return 0;
  if (!dy || !ids || (dx && !a) || ((dx || da) && !b) || (da && !x) || (db && !v)) return fail("zm_lora_backward: null pointer");
  const Space s = space_of(*d, true);
  if (check_space(workspace, workspace_size, s.total, "zm_lora_backward")) return -1;
  uint8_t *ws = (uint8_t *)workspace;
  float *part = (float *)(ws + s.items), *u = part + s.part / 4, *sa = u + s.u / 4, *sb = sa + sums_space(*d, d->I) / 4;
  LoraArgs g = items(*d, ids, scale, ws, st);
  if (dx || da) {
    g.x = dy;
    g.ldx = d->y_stride;
    g.m = b;
    g.ldm = d->b_stride;
    g.m_adapter = d->b_adapter;
    g.K = d->O;
    g.l = a;
    g.ldl = d->a_stride;
    g.l_adapter = d->a_adapter;
    g.N = dx ? d->I : 0;
    g.y = dx;
    g.ldy = d->I;
    g.v = da ? u : nullptr;
    launch(*d, lora_backward, d->y_type, d->x_type, g, part, st);
  }
  if (da || db) {
    const LoraSumArgs ga = sums_args(*d, u, x, d->x_stride, d->I, scale, da, sa);
    const LoraSumArgs gb = sums_args(*d, v, dy, d->y_stride, d->O, scale, db, sb);
    lora_sums(d->x_type, d->y_type, g.it, ga, da ? sums_groups(ga) : 0, gb, db ? sums_groups(gb) : 0, st);
    if (da) join_sums(ga, g.it, da, st);
    if (db) join_sums(gb, g.it, db, st);
  }
  return launched();
}

}  // extern "C"
