// zm_glu.hip -- C ABI of the gated product y = act(x w_gate^T + b_gate) (x w_up^T + b_up) and of its gradients: checks,
// workspace layout, and the gradients by both factors.  The products are those of zm_linear.hpp, with two weights.
#include <hip/hip_runtime.h>

#include "zm_linear_host.hpp"

using namespace zm;

namespace {

// ============================================================ gradients by the factors

struct FactorArgs {
  const void *dy, *gate, *up;  // [S][F] of `type`
  int64_t ldy, ldg, ldu, S, F;
  int type, act, count;  // count: terms
  float *dz;             // [S][ldz] f32: dg at column 0, du at column F; or
  bf16 *terms;           // [count][S][ldz], their bf16 terms; or neither
  int64_t ldz;
  float *part;           // [gridDim.y][2 F] sums over this chunk of rows, or null
  int64_t chunk;         // rows of a chunk
  int packs, side;       // packs of V columns that a workgroup takes, and rows that it takes at once
};

// V values of one row into dz or into its terms (an infinity or a NaN is the first term; what follows it is NaN)
template <int V>
__device__ __forceinline__ void put_factor(const FactorArgs &g, int64_t s, int64_t col, v4f v) {
  if (g.dz) {
    float *d = g.dz + s * g.ldz + col;
    if constexpr (V == 4) *reinterpret_cast<v4f *>(d) = v;
    else *d = v.x;
  }
  if (g.terms) {
    for (int k = 0; k < g.count; ++k) {
      bf16 *d = g.terms + (k * g.S + s) * g.ldz + col;
      bf16 e[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float most = __builtin_amdgcn_fmed3f(v[j], -BF16_MOST, BF16_MOST);
        e[j] = from_f32<bf16>(k || !(fabsf(v[j]) <= F32_MOST) ? v[j] : most);
        v[j] -= to_f32(e[j]);
      }
      if constexpr (V == 4) __builtin_memcpy(__builtin_assume_aligned(d, 8), e, 8);
      else *d = e[0];
    }
  }
}

// dg = dy up act'(gate) and du = dy act(gate), with their sums over a chunk of rows in f32.  A thread keeps V columns of
// both and takes every side-th row of the chunk, two at a time; the rows' sums meet in LDS in order.
template <int V>
__global__ __launch_bounds__(256) void k_glu_factors(FactorArgs g) {
  __shared__ float red[2][256 * V];
  constexpr int U = 2;
  const int c = threadIdx.x % g.packs, r = threadIdx.x / g.packs;
  const int64_t f = ((int64_t)blockIdx.x * g.packs + c) * V;
  const int64_t s0 = blockIdx.y * g.chunk, s1 = min(g.S, s0 + g.chunk);
  v4f sg = {0.f, 0.f, 0.f, 0.f}, su = {0.f, 0.f, 0.f, 0.f};
  if (f < g.F && r < g.side) {
    for (int64_t s = s0 + r; s < s1; s += U * g.side) {
      v4f d[U], z[U], u[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int64_t sk = s + k * g.side;
        d[k] = z[k] = u[k] = v4f{0.f, 0.f, 0.f, 0.f};
        if (sk >= s1) continue;
        if constexpr (V == 4) {
          d[k] = lin_load4(g.dy, g.type, (size_t)(sk * g.ldy + f));
          z[k] = lin_load4(g.gate, g.type, (size_t)(sk * g.ldg + f));
          u[k] = lin_load4(g.up, g.type, (size_t)(sk * g.ldu + f));
        } else {
          d[k].x = lin_load(g.dy, g.type, (size_t)(sk * g.ldy + f));
          z[k].x = lin_load(g.gate, g.type, (size_t)(sk * g.ldg + f));
          u[k].x = lin_load(g.up, g.type, (size_t)(sk * g.ldu + f));
        }
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int64_t sk = s + k * g.side;
        if (sk >= s1) break;
        v4f dg = {0.f, 0.f, 0.f, 0.f}, du = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float a, slope;
          factor_and_slope(z[k][j], g.act, a, slope);
          dg[j] = d[k][j] * u[k][j] * slope;
          du[j] = d[k][j] * a;
          sg[j] += dg[j];
          su[j] += du[j];
        }
        put_factor<V>(g, sk, f, dg);
        put_factor<V>(g, sk, g.F + f, du);
      }
    }
  }
  if (!g.part) return;
#pragma unroll
  for (int j = 0; j < V; ++j) {  // (threads past side * packs have sums of zero)
    red[0][(r * g.packs + c) * V + j] = sg[j];
    red[1][(r * g.packs + c) * V + j] = su[j];
  }
  __syncthreads();
  for (int j = threadIdx.x; j < g.packs * V; j += 256) {
    const int64_t k = (int64_t)blockIdx.x * g.packs * V + j;
    if (k >= g.F) break;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float a = 0.f;
      for (int q = 0; q < g.side; ++q) a += red[h][q * g.packs * V + j];
      g.part[(size_t)blockIdx.y * 2 * g.F + h * g.F + k] = a;
    }
  }
}

// ============================================================ the products

// the checks and choices of zm_linear go by this: both weights are one of 2 F rows
zm_linear_desc as_linear(const zm_glu_desc &d) {
  return {d.x_type, d.w_type, d.y_type, d.act, d.S, d.I, 2 * ((d.F + 15) / 16 * 16), d.x_stride, d.w_stride, d.y_stride,
          d.gate_stride, d.up_stride};
}
int check_glu(const zm_glu_desc *d, const char *who) {
  if (!d) return fail("%s: null description", who);
  if (d->F <= 0 || d->F >= (int64_t)1 << 30) return fail("%s: F from 1 to 2^30 is needed", who);
  const zm_linear_desc l = as_linear(*d);
  return check_desc(&l, who);
}
Product forward(const zm_glu_desc &d) {
  const zm_linear_desc l = as_linear(d);
  Product q = {d.S, l.O, d.I, d.x_type, d.w_type, 1, 0,
               vec_shape(d.x_stride, d.I, d.x_type, true) && vec_shape(d.w_stride, d.I, d.w_type, true), true, true, true, 1};
  q.form = LIN_PAIR;
  return q;
}
// The gradients by the factors lie side by side, in rows of 2 F values: f32, or next to bf16 planes of bf16 terms, of
// which dx (16 bits) takes two and dw (f32) three.
int dz_type(const zm_glu_desc &d) { return d.x_type == LIN_BF16 ? LIN_BF16 : LIN_F32; }
int64_t dz_ld(const zm_glu_desc &d) { return (2 * d.F + 7) / 8 * 8; }
Product by_x(const zm_glu_desc &d) {
  const int t = dz_type(d);
  Product q = {d.S, d.I, d.F, t, d.w_type, t == LIN_BF16 ? 4 : 2, d.S * dz_ld(d),
               vec_shape(dz_ld(d), d.F, t, true) && vec_shape(d.w_stride, d.I, d.w_type, false), true, false, false, 0};
  q.form = LIN_SUM;
  return q;
}
Product by_w(const zm_glu_desc &d) {
  const int t = dz_type(d);
  return {2 * d.F, d.I, d.S, t, d.x_type, t == LIN_BF16 ? 3 : 1, d.S * dz_ld(d),
          vec_shape(dz_ld(d), 2 * d.F, t, false) && vec_shape(d.x_stride, d.I, d.x_type, false), false, false, false, -1};
}

// chunks of rows of the factors' gradients: 8 rows each, at most 512, so that a thread has its few rows on their way at
// once (2048 x 1536 in bf16, chunks of 32: 34 us)
int64_t factor_chunks(int64_t S) { return std::min<int64_t>((S + 7) / 8, 512); }

// Workspace of the backward pass: both factors' gradients | bias partials | the larger product's partials.
struct BackwardSpace {
  size_t dz, bias, part, total;
};
BackwardSpace backward_space(const zm_glu_desc &d) {
  BackwardSpace w{};
  w.dz = align256((size_t)d.S * dz_ld(d) * (dz_type(d) == LIN_BF16 ? 6 : 4));
  w.bias = align256((size_t)factor_chunks(d.S) * 2 * d.F * 4);
  w.part = align256(std::max(by_x(d).space(), by_w(d).space()));
  w.total = w.dz + w.bias + w.part;
  return w;
}

}  // namespace

extern "C" {

size_t zm_glu_workspace_size(const zm_glu_desc *d) {
  if (check_glu(d, "zm_glu_workspace_size") || !d->S) return 0;
  return align256(forward(*d).space());
}

int zm_glu(const zm_glu_desc *d, const void *x, const void *w_gate, const void *w_up, const float *b_gate, const float *b_up,
           void *y, void *gate, void *up, void *workspace, size_t workspace_size, void *stream) {
  if (check_glu(d, "zm_glu")) return -1;
  if (check_rows(d->S, d->y_stride, d->F, "zm_glu", "y")) return -1;
  if (!gate != !up) return fail("zm_glu: gate and up are kept together");
  if (gate && (check_rows(d->S, d->gate_stride, d->F, "zm_glu", "gate") || check_rows(d->S, d->up_stride, d->F, "zm_glu", "up")))
    return -1;
  if (!d->S) return 0;
  if (!x || !w_gate || !w_up || !y) return fail("zm_glu: null pointer");
  const Product q = forward(*d);
  const bool vec = q.shaped && vec_at(x) && vec_at(w_gate) && vec_at(w_up);
  const Plan p = q.planned(vec);
  if (p.part && (!workspace || workspace_size < p.part || ((uintptr_t)workspace & 255)))
    return fail("zm_glu: a 256-byte aligned workspace of zm_glu_workspace_size() bytes is needed");
  LinArgs g = product(q, x, d->x_stride, w_gate, d->w_stride, p, (float *)workspace);
  g.b2 = w_up;
  g.F = d->F;
  g.e.y = y;
  g.e.pre = gate;
  g.e.up = up;
  g.e.bias = b_gate;
  g.e.bias2 = b_up;
  g.e.ldy = d->y_stride;
  g.e.ldp = d->gate_stride;
  g.e.ldr = d->up_stride;
  g.e.type = d->y_type;
  g.e.act = d->act;
  const hipStream_t st = (hipStream_t)stream;
  if (p.kind == ROWS) pair_rows(d->x_type, d->w_type, g, st);
  else if (p.kind == FEW) pair_few(d->x_type, d->w_type, g, st);
  else pair_fwd(d->x_type, d->w_type, g, vec, p.tile, st);
  if (g.slices > 1) pair_join(g, st);
  return launched();
}

size_t zm_glu_backward_workspace_size(const zm_glu_desc *d) {
  if (check_glu(d, "zm_glu_backward_workspace_size") || !d->S) return 0;
  return backward_space(*d).total;
}

int zm_glu_backward(const zm_glu_desc *d, const void *dy, const void *x, const void *w_gate, const void *w_up,
                    const void *gate, const void *up, void *dx, float *dw, float *db, void *workspace,
                    size_t workspace_size, void *stream) {
  if (check_glu(d, "zm_glu_backward")) return -1;
  const hipStream_t st = (hipStream_t)stream;
  if (!d->S) {  // no rows: the sums over them are zero
    if (dw) hipLaunchKernelGGL(k_linear_zero, dim3(256), dim3(256), 0, st, dw, 2 * d->F * d->I);
    if (db) hipLaunchKernelGGL(k_linear_zero, dim3(1), dim3(256), 0, st, db, 2 * d->F);
    return launched();
  }
  if (!dx && !dw && !db) return 0;
  if (!dy || !gate || !up || (dw && !x) || (dx && (!w_gate || !w_up))) return fail("zm_glu_backward: null pointer");
  const BackwardSpace s = backward_space(*d);
  if (!workspace || workspace_size < s.total || ((uintptr_t)workspace & 255))
    return fail("zm_glu_backward: a 256-byte aligned workspace of zm_glu_backward_workspace_size() bytes is needed");
  uint8_t *ws = (uint8_t *)workspace;
  float *dz = (float *)ws, *bias_part = (float *)(ws + s.dz), *part = (float *)(ws + s.dz + s.bias);
  const int z_type = dz_type(*d);
  const int64_t ldz = dz_ld(*d);
  FactorArgs a{};
  a.dy = dy;
  a.gate = gate;
  a.up = up;
  a.ldy = d->y_stride;
  a.ldg = d->gate_stride;
  a.ldu = d->up_stride;
  a.S = d->S;
  a.F = d->F;
  a.type = d->y_type;
  a.act = d->act;
  a.count = dw ? 3 : 2;
  if (dx || dw) {
    a.dz = z_type == LIN_F32 ? dz : nullptr;
    a.terms = z_type == LIN_F32 ? nullptr : (bf16 *)dz;
  }
  a.ldz = ldz;
  a.part = db ? bias_part : nullptr;
  const int64_t n = factor_chunks(d->S);
  a.chunk = (d->S + n - 1) / n;
  const bool v = !(d->F & 3);
  const int64_t packs = v ? d->F / 4 : d->F;
  a.packs = (int)std::min<int64_t>(packs, 64);
  a.side = 256 / a.packs;
  const dim3 grid((unsigned)((packs + a.packs - 1) / a.packs), (unsigned)n);
  if (v) hipLaunchKernelGGL((k_glu_factors<4>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((k_glu_factors<1>), grid, dim3(256), 0, st, a);
  if (db) parts_sum(bias_part, (int)n, 2 * d->F, 2 * d->F, db, nullptr, st);
  if (dx) {
    const Product q = by_x(*d);
    const bool vec = q.shaped && vec_at(w_gate) && vec_at(w_up);
    const Plan p = q.planned(vec);
    LinArgs g = product(q, dz, ldz, w_gate, d->w_stride, p, part);
    g.b2 = w_up;
    g.half = q.planes / 2;
    g.b_skip = ((intptr_t)w_up - (intptr_t)w_gate) / (intptr_t)size_of(d->w_type);
    g.e.y = dx;
    g.e.ldy = d->I;
    g.e.type = d->x_type;
    pair_dx(d->x_type, d->w_type, g, vec, p.tile, st);
    if (join(g, st)) return -1;
  }
  if (dw) {
    const Product q = by_w(*d);
    const bool vec = q.shaped && vec_at(x);
    const Plan p = q.planned(vec);
    LinArgs g = product(q, dz, ldz, x, d->x_stride, p, part);
    g.e.y = dw;
    g.e.ldy = d->I;
    g.e.type = LIN_F32;
    lin_dw(d->x_type, z_type, g, vec, p.tile, st);
    if (join(g, st)) return -1;
  }
  return launched();
}

}  // extern "C"
