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
  if (d->n <= 0 || d->n > BUCKET_MAX_E) return fail("%s: 1 to %d adapters, not %d", who, BUCKET_MAX_E, d->n);
  if (d->R <= 0 || d->R > LORA_MOST_R) return fail("%s: a rank of 1 to %d, not %d", who, LORA_MOST_R, d->R);
  if (d->S < 0 || d->S >= MMQ_MAX_PAIRS) return fail("%s: S from 0 to 2^24 is needed", who);
  if (d->I <= 0 || d->O <= 0 || d->I >= 1 << 30 || d->O >= 1 << 30) return fail("%s: I and O from 1 to 2^30 are needed", who);
  if (d->x_stride < 0 || d->y_stride < 0 || d->res_stride < 0 || d->a_stride < 0 || d->b_stride < 0 || d->a_adapter < 0 ||
      d->b_adapter < 0)
    return fail("%s: negative stride", who);
  if ((d->S / LORA_TOKENS + d->n) * ((std::max(d->I, d->O) + 255) / 256) >= 1 << 26)
    return fail("%s: S x I or S x O too large for one launch", who);
  return 0;
}

// Work items are counted on the device; a launch has as many as there can be.
int64_t most_items(const zm_lora_desc &d) { return d.S / LORA_TOKENS + std::min<int64_t>(d.S, d.n); }

// slices of an axis of K, `unit` at a time, for `want` workgroups where one slice has `n`
int64_t slices_of(int64_t n, int64_t want, int64_t K, int64_t unit, int64_t most) {
  return std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(want / std::max<int64_t>(n, 1), most), K / unit));
}

struct Shrink {
  int slices, chunks;
  int64_t kslice;
  size_t part;  // bytes
};
Shrink shrink_of(const zm_lora_desc &d, int64_t K) {
  Shrink p;
  p.chunks = (d.R + lora_r_of(d.R) - 1) / lora_r_of(d.R);
  const int64_t z = slices_of(most_items(d) * p.chunks, 1024, K, 256, 16);
  p.kslice = ((K + z - 1) / z + 255) / 256 * 256;
  p.slices = (int)((K + p.kslice - 1) / p.kslice);
  p.part = align256((size_t)p.slices * d.S * d.R * 4);
  return p;
}
// slices of an adapter's tokens for its gradient of N columns; their sums take at most 64 MB
int sums_slices(const zm_lora_desc &d, int64_t N) {
  const int64_t groups = (N + 63) / 64 * ((d.R + lora_r_of(d.R) - 1) / lora_r_of(d.R)) * d.n;
  return (int)slices_of(groups, 512, d.S / d.n, 128, (64 << 20) / (4 * N * d.R * d.n));
}
size_t sums_space(const zm_lora_desc &d, int64_t N) {
  const int z = sums_slices(d, N);
  return z > 1 ? align256((size_t)z * d.n * d.R * N * 4) : 0;
}

// Workspace: the buckets | v or u of each slice | (backward) u, and one gradient's sums.
struct Space {
  size_t buckets, part, u, sums, total;
};
size_t bucket_bytes(const zm_lora_desc &d) { return align256((3 * d.n + 3 + d.S + most_items(d)) * 4); }
Space space_of(const zm_lora_desc &d, bool backward) {
  Space s{};
  s.buckets = bucket_bytes(d);
  s.part = shrink_of(d, backward ? d.O : d.I).part;
  if (backward) {
    s.u = align256((size_t)d.S * d.R * 4);
    s.sums = std::max(sums_space(d, d.I), sums_space(d, d.O));
  }
  s.total = s.buckets + s.part + s.u + s.sums;
  return s;
}

// One launch for a few tokens, each computing its v for every 512 columns again: where that is little to read.
bool few_tokens(const zm_lora_desc &d) {
  const int64_t a = d.R * d.I * (int64_t)size_of(d.w_type);
  return d.S <= 4096 && a <= 1 << 20 && d.S * ((d.O + 511) / 512) * a <= 64 << 20;
}

LoraArgs buckets(const zm_lora_desc &d, const int32_t *ids, const float *scale, uint8_t *ws, hipStream_t st) {
  LoraArgs g{};
  g.R = d.R;
  g.S = (int)d.S;
  g.n = d.n;
  g.ids = ids;
  g.scale = scale;
  int32_t *p = (int32_t *)ws;
  int32_t *counts = p, *offs = p + d.n, *active = p + 2 * d.n + 1, *n_active = active + d.n, *n_items = n_active + 1;
  int32_t *pairs = n_items + 1, *items = pairs + d.S;
  bucket_tokens(ids, (int)d.S, d.n, LORA_TOKENS, counts, offs, pairs, active, n_active, items, n_items, st);
  g.counts = counts;
  g.offs = offs;
  g.pairs = pairs;
  g.items = items;
  g.n_items = n_items;
  return g;
}
// x by the matrices m over K, into the slices' parts of v
void shrink(const zm_lora_desc &d, LoraArgs g, const void *x, int x_type, int64_t ldx, const void *m, int64_t ldm,
            int64_t adapter, int64_t K, bool kc, float *part, hipStream_t st) {
  const Shrink p = shrink_of(d, K);
  g.x = x;
  g.ldx = ldx;
  g.m = m;
  g.ldm = ldm;
  g.adapter = adapter;
  g.K = K;
  g.slices = p.slices;
  g.chunks = p.chunks;
  g.kslice = p.kslice;
  g.part = part;
  lora_shrink(x_type, d.w_type, kc, g, (int)(most_items(d) * p.slices * p.chunks), st);
}
// the slices' sums (kept in v, unless null) by the matrices m, N columns of y
void expand(const zm_lora_desc &d, LoraArgs g, const float *part, int slices, float *v, const void *m, int64_t ldm,
            int64_t adapter, int64_t N, bool kc, const void *res, int64_t ldr, void *y, int64_t ldy, int type,
            hipStream_t st) {
  g.part = (float *)part;
  g.slices = slices;
  g.v = v;
  g.m = m;
  g.ldm = ldm;
  g.adapter = adapter;
  g.N = N;
  g.res = res;
  g.ldr = ldr;
  g.y = y;
  g.ldy = ldy;
  g.type = type;
  g.chunks = (int)((N + 255) / 256);
  g.rest = (int)most_items(d);
  lora_expand(d.w_type, kc, g, (int)((g.rest + (d.S + 63) / 64) * g.chunks), st);
}
// dst [n][R][N], or [n][N][R] (by_r): the sums over each adapter's tokens of a's and m's rows
void sums(const zm_lora_desc &d, LoraArgs g, const float *a, const void *m, int m_type, int64_t ldm, int64_t N, bool by_r,
          float *dst, float *space, hipStream_t st) {
  g.v = (float *)a;
  g.x = m;
  g.ldx = ldm;
  g.N = N;
  g.chunks = (d.R + lora_r_of(d.R) - 1) / lora_r_of(d.R);
  g.slices = sums_slices(d, N);
  g.y = g.slices > 1 ? space : dst;
  lora_sums(m_type, by_r, g, (int)((N + 63) / 64 * g.chunks * g.slices * d.n), st);
  const int64_t all = (int64_t)d.n * d.R * N;
  if (g.slices > 1) parts_sum(space, g.slices, all, all, dst, nullptr, st);
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
  const hipStream_t st = (hipStream_t)stream;
  if (few_tokens(*d)) {
    LoraFewArgs g{x, a, b, d->x_stride, d->a_stride, d->b_stride, d->a_adapter, d->b_adapter, d->I, d->O, d->R, d->n, ids,
                  scale, residual, y, v, d->res_stride, d->y_stride, d->y_type};
    lora_few(d->x_type, d->w_type, g, dim3((unsigned)((d->O + 511) / 512), (unsigned)d->S), st);
    return launched();
  }
  const Space s = space_of(*d, false);
  if (check_space(workspace, workspace_size, s.total, "zm_lora")) return -1;
  uint8_t *ws = (uint8_t *)workspace;
  float *part = (float *)(ws + s.buckets);
  const LoraArgs g = buckets(*d, ids, scale, ws, st);
  shrink(*d, g, x, d->x_type, d->x_stride, a, d->a_stride, d->a_adapter, d->I, true, part, st);
  expand(*d, g, part, shrink_of(*d, d->I).slices, v, b, d->b_stride, d->b_adapter, d->O, true, residual, d->res_stride, y,
         d->y_stride, d->y_type, st);
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
  float *part = (float *)(ws + s.buckets), *u = (float *)(ws + s.buckets + s.part), *space = (float *)((uint8_t *)u + s.u);
  const LoraArgs g = buckets(*d, ids, scale, ws, st);
  if (dx || da) {
    const int slices = shrink_of(*d, d->O).slices;
    shrink(*d, g, dy, d->y_type, d->y_stride, b, d->b_stride, d->b_adapter, d->O, false, part, st);
    if (slices == 1) u = part;
    if (dx)
      expand(*d, g, part, slices, da && slices > 1 ? u : nullptr, a, d->a_stride, d->a_adapter, d->I, false, nullptr, 0, dx,
             d->I, d->x_type, st);
    else if (slices > 1) parts_sum(part, slices, d->S * d->R, d->S * d->R, u, nullptr, st);
  }
  if (da) sums(*d, g, u, x, d->x_type, d->x_stride, d->I, false, da, space, st);
  if (db) sums(*d, g, v, dy, d->y_type, d->y_stride, d->O, true, db, space, st);
  return launched();
}

}  // extern "C"
