// zm_linear.hip -- C ABI of the unquantized matrix product with bias, activation and residual, and of its gradients:
// checks of the arguments, workspace layout.  The kernels are in zm_linear.hpp, the choice among them in
// zm_linear_host.hpp; the quantized counterpart is zm_f32_matmul.
#include <hip/hip_runtime.h>

#include "../../include/zeromoe.h"
#include "zm_host.hpp"
#include "zm_linear_host.hpp"

using namespace zm;

namespace {

// ============================================================ dz and the bias gradient

struct DzArgs {
  const void *dy, *pre;  // [S][O] of `type`; pre null without an activation
  int64_t ldy, ldp, S, O;
  int type, act;
  float *dz;         // [S][ldz] f32, or
  bf16 *terms;       // [3][S][ldz], its bf16 terms, or neither (dy is dz)
  int64_t ldz;
  float *part;       // [gridDim.y][O] sums over this chunk of rows, or null
  int64_t chunk;     // rows of a chunk
  int packs, side;   // packs of V columns that a workgroup takes, and rows that it takes at once
};

// dz = dy * act'(pre), and its sums over a chunk of rows in f32.  A thread keeps V columns and takes every side-th row
// of the chunk, four at a time; the rows' sums meet in LDS in order.
template <int V>
__global__ __launch_bounds__(256) void k_linear_dz(DzArgs g) {
  __shared__ float red[256 * V];
  const int c = threadIdx.x % g.packs, r = threadIdx.x / g.packs;
  const int64_t o = ((int64_t)blockIdx.x * g.packs + c) * V;
  const int64_t s0 = blockIdx.y * g.chunk, s1 = min(g.S, s0 + g.chunk);
  v4f sum = {0.f, 0.f, 0.f, 0.f};
  if (o < g.O && r < g.side) {
    for (int64_t s = s0 + r; s < s1; s += 4 * g.side) {
      v4f v[4], p[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t su = s + u * g.side;
        const bool in = su < s1;
        if constexpr (V == 4) {
          v[u] = in ? lin_load4(g.dy, g.type, (size_t)(su * g.ldy + o)) : v4f{0.f, 0.f, 0.f, 0.f};
          if (g.act) p[u] = in ? lin_load4(g.pre, g.type, (size_t)(su * g.ldp + o)) : v4f{0.f, 0.f, 0.f, 0.f};
        } else {
          v[u].x = in ? lin_load(g.dy, g.type, (size_t)(su * g.ldy + o)) : 0.f;
          if (g.act) p[u].x = in ? lin_load(g.pre, g.type, (size_t)(su * g.ldp + o)) : 0.f;
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t su = s + u * g.side;
        if (su >= s1) break;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (g.act) v[u][j] *= lin_act_slope(p[u][j], g.act);
          sum[j] += v[u][j];
        }
        if (g.dz) {
          float *d = g.dz + su * g.ldz + o;
          if constexpr (V == 4) *reinterpret_cast<v4f *>(d) = v[u];
          else *d = v[u].x;
        }
        if (g.terms) {
          v4f r = v[u];
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            bf16 *d = g.terms + (k * g.S + su) * g.ldz + o;
            bf16 e[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
              // an infinity or a NaN is the first term (what follows it is NaN)
              const float most = __builtin_amdgcn_fmed3f(r[j], -BF16_MOST, BF16_MOST);
              e[j] = from_f32<bf16>(k || !(fabsf(r[j]) <= F32_MOST) ? r[j] : most);
              r[j] -= to_f32(e[j]);
            }
            if constexpr (V == 4) __builtin_memcpy(__builtin_assume_aligned(d, 8), e, 8);
            else *d = e[0];
          }
        }
      }
    }
  }
  if (!g.part) return;
#pragma unroll
  for (int j = 0; j < V; ++j) red[(r * g.packs + c) * V + j] = sum[j];  // (threads past side * packs have sums of zero)
  __syncthreads();
  for (int j = threadIdx.x; j < g.packs * V; j += 256) {
    const int64_t k = (int64_t)blockIdx.x * g.packs * V + j;
    if (k >= g.O) break;
    float a = 0.f;
    for (int q = 0; q < g.side; ++q) a += red[q * g.packs * V + j];
    g.part[(size_t)blockIdx.y * g.O + k] = a;
  }
}

// ============================================================ the products

Product forward(const zm_linear_desc &d) {
  return {d.S, d.O, d.I, d.x_type, d.w_type, 1, 0,
          vec_shape(d.x_stride, d.I, d.x_type, true) && vec_shape(d.w_stride, d.I, d.w_type, true), true, true, true, 1};
}
// What the products of the backward pass take for dz: dy itself; behind an activation f32 in the workspace; next to
// bf16, where it is not bf16 itself, three planes of bf16 terms there.
enum DzForm { DZ_DY, DZ_F32, DZ_TERMS };
DzForm dz_form(const zm_linear_desc &d) {
  if (d.x_type == LIN_BF16 && (d.act || d.y_type == LIN_F32)) return DZ_TERMS;
  return d.act ? DZ_F32 : DZ_DY;
}
int dz_type(const zm_linear_desc &d) {
  const DzForm f = dz_form(d);
  return f == DZ_TERMS ? (int)LIN_BF16 : f == DZ_F32 ? (int)LIN_F32 : d.y_type;
}
int64_t dz_ld(const zm_linear_desc &d) { return dz_form(d) == DZ_DY ? d.y_stride : (d.O + 7) / 8 * 8; }
Product by_x(const zm_linear_desc &d) {
  return {d.S, d.I, d.O, dz_type(d), d.w_type, dz_form(d) == DZ_TERMS ? 2 : 1, d.S * dz_ld(d),
          vec_shape(dz_ld(d), d.O, dz_type(d), true) && vec_shape(d.w_stride, d.I, d.w_type, false), true, false, false, 0};
}
Product by_w(const zm_linear_desc &d) {
  return {d.O, d.I, d.S, dz_type(d), d.x_type, dz_form(d) == DZ_TERMS ? 3 : 1, d.S * dz_ld(d),
          vec_shape(dz_ld(d), d.O, dz_type(d), false) && vec_shape(d.x_stride, d.I, d.x_type, false), false, false, false, -1};
}

// Workspace of the backward pass: dz (unless it is dy) | bias partials | the larger product's partials.
struct BackwardSpace {
  size_t dz, bias, part, total;
};
BackwardSpace backward_space(const zm_linear_desc &d) {
  BackwardSpace w{};
  const size_t n = (size_t)d.S * dz_ld(d);
  w.dz = dz_form(d) == DZ_DY ? 0 : align256(dz_form(d) == DZ_F32 ? n * 4 : n * 6);
  w.bias = align256((size_t)dz_chunks(d.S) * d.O * 4);
  w.part = align256(std::max(by_x(d).space(), by_w(d).space()));
  w.total = w.dz + w.bias + w.part;
  return w;
}

}  // namespace

extern "C" {

size_t zm_linear_workspace_size(const zm_linear_desc *d) {
  if (check_desc(d, "zm_linear_workspace_size") || !d->S) return 0;
  return align256(forward(*d).space());
}

int zm_linear(const zm_linear_desc *d, const void *x, const void *w, const float *bias, const void *residual, void *y,
              void *pre, void *workspace, size_t workspace_size, void *stream) {
  if (check_desc(d, "zm_linear")) return -1;
  if (check_rows(d->S, d->y_stride, d->O, "zm_linear", "y")) return -1;
  if (pre && check_rows(d->S, d->pre_stride, d->O, "zm_linear", "pre")) return -1;
  if (!d->S) return 0;
  if (!x || !w || !y) return fail("zm_linear: null pointer");
  const Product q = forward(*d);
  const bool vec = q.shaped && vec_at(x) && vec_at(w);
  const Plan p = q.planned(vec);
  if (p.part && (!workspace || workspace_size < p.part || ((uintptr_t)workspace & 255)))
    return fail("zm_linear: a 256-byte aligned workspace of zm_linear_workspace_size() bytes is needed");
  LinArgs g = product(q, x, d->x_stride, w, d->w_stride, p, (float *)workspace);
  g.e.y = y;
  g.e.res = residual;
  g.e.pre = pre;
  g.e.bias = bias;
  g.e.ldy = d->y_stride;
  g.e.ldr = d->res_stride;
  g.e.ldp = d->pre_stride;
  g.e.type = d->y_type;
  g.e.act = d->act;
  if (p.kind == ROWS) lin_rows(d->x_type, d->w_type, g, (hipStream_t)stream);
  else if (p.kind == FEW) lin_few(d->x_type, d->w_type, g, (hipStream_t)stream);
  else lin_fwd(d->x_type, d->w_type, g, vec, p.tile, (hipStream_t)stream);
  return join(g, (hipStream_t)stream);
}

size_t zm_linear_backward_workspace_size(const zm_linear_desc *d) {
  if (check_desc(d, "zm_linear_backward_workspace_size") || !d->S) return 0;
  return backward_space(*d).total;
}

int zm_linear_backward(const zm_linear_desc *d, const void *dy, const void *x, const void *w, const void *pre, void *dx,
                       float *dw, float *dbias, void *workspace, size_t workspace_size, void *stream) {
  if (check_desc(d, "zm_linear_backward")) return -1;
  const hipStream_t st = (hipStream_t)stream;
  if (!d->S) {  // no rows: the sums over them are zero
    if (dw) hipLaunchKernelGGL(k_linear_zero, dim3(256), dim3(256), 0, st, dw, d->O * d->I);
    if (dbias) hipLaunchKernelGGL(k_linear_zero, dim3(1), dim3(256), 0, st, dbias, d->O);
    return launched();
  }
  if (!dy || (dw && !x) || (dx && !w)) return fail("zm_linear_backward: null pointer");
  if (d->act && !pre) return fail("zm_linear_backward: an activation's gradient needs pre");
  if (!dx && !dw && !dbias) return 0;
  const BackwardSpace s = backward_space(*d);
  if (s.total && (!workspace || workspace_size < s.total || ((uintptr_t)workspace & 255)))
    return fail("zm_linear_backward: a 256-byte aligned workspace of zm_linear_backward_workspace_size() bytes is needed");
  uint8_t *ws = (uint8_t *)workspace;
  float *dz = (float *)ws, *bias_part = (float *)(ws + s.dz), *part = (float *)(ws + s.dz + s.bias);
  const DzForm form = dz_form(*d);
  if (form != DZ_DY || dbias) {
    DzArgs a{};
    a.dy = dy;
    a.pre = pre;
    a.ldy = d->y_stride;
    a.ldp = d->pre_stride;
    a.S = d->S;
    a.O = d->O;
    a.type = d->y_type;
    a.act = d->act;
    a.dz = form == DZ_F32 ? dz : nullptr;
    a.terms = form == DZ_TERMS ? (bf16 *)dz : nullptr;
    a.ldz = dz_ld(*d);
    a.part = dbias ? bias_part : nullptr;
    const int64_t n = dz_chunks(d->S);
    a.chunk = (d->S + n - 1) / n;
    const bool v = !(d->O & 3);
    const int64_t packs = v ? d->O / 4 : d->O;
    a.packs = (int)std::min<int64_t>(packs, 64);
    a.side = 256 / a.packs;
    const dim3 grid((unsigned)((packs + a.packs - 1) / a.packs), (unsigned)n);
    if (v) hipLaunchKernelGGL((k_linear_dz<4>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_linear_dz<1>), grid, dim3(256), 0, st, a);
    if (dbias) parts_sum(bias_part, (int)n, d->O, d->O, dbias, nullptr, st);
  }
  const void *z = form == DZ_DY ? dy : (const void *)dz;
  const int z_type = dz_type(*d);
  if (dx) {
    const Product q = by_x(*d);
    const bool vec = q.shaped && vec_at(z) && vec_at(w);
    const Plan p = q.planned(vec);
    LinArgs g = product(q, z, dz_ld(*d), w, d->w_stride, p, part);
    g.e.y = dx;
    g.e.ldy = d->I;
    g.e.type = d->x_type;
    lin_dx(d->x_type, d->w_type, z_type, g, vec, p.tile, st);
    if (join(g, st)) return -1;
  }
  if (dw) {
    const Product q = by_w(*d);
    const bool vec = q.shaped && vec_at(z) && vec_at(x);
    const Plan p = q.planned(vec);
    LinArgs g = product(q, z, dz_ld(*d), x, d->x_stride, p, part);
    g.e.y = dw;
    g.e.ldy = d->I;
    g.e.type = LIN_F32;
    lin_dw(d->x_type, z_type, g, vec, p.tile, st);
    if (join(g, st)) return -1;
  }
  return launched();
}

}  // extern "C"
