// zm_linear.hip -- C ABI of the unquantized matrix product with bias, activation and residual, and of its gradients:
// checks of the arguments, choice of tiles and k slices, workspace layout.  The kernels are in zm_linear.hpp; the
// quantized counterpart is zm_f32_matmul.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/zeromoe.h"
#include "zm_host.hpp"
#include "zm_linear.hpp"

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

__global__ __launch_bounds__(256) void k_linear_zero(float *__restrict__ dst, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) dst[i] = 0.f;
}

// ============================================================ choices

struct Plan {
  int kind, tile, tiles_m, tiles_n, slices;
  int64_t kslice;
  size_t part;  // bytes of the slices' partial results
};

// the kernels of a product, by its rows and by whether its operands can be read 16 bytes at a time
enum Kind { ROWS, FEW, TILES };

// `products`: of terms, for each product of values; 1: 16-bit operands of one type, which go straight into LDS;
// `side`: Product's
Plan plan(Kind kind, int64_t M, int64_t N, int64_t K, int planes, int products, int side, bool vec, size_t most) {
  const bool dma = products == 1;
  const int step = dma ? DMA_BK : 32;
  Plan p{};
  p.kind = kind;
  int64_t z = 1, bk = 64;
  if (kind == FEW) {
    // slices of k until there is a workgroup of 8 waves, or two of 4, per CU
    const int cols = few_columns(M, N);
    p.tiles_m = (int)((M + FEW_ROWS - 1) / FEW_ROWS);
    p.tiles_n = (int)((N + cols - 1) / cols);
    bk = FEW_UNIT;
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n, want = cols == 64 ? 512 : 256;
    z = std::min<int64_t>((want - 1 + tiles) / tiles, (K + bk - 1) / bk);
  } else if (kind == TILES) {
    const int64_t steps = planes * ((K + step - 1) / step);
    const size_t plane = (size_t)M * N * 4;
    p.tile = M <= 64;
    int bm = p.tile ? 32 : 128, bn = 128;
    if (p.tile) {
      // 32 x 128 for up to 64 rows; k in as many slices as give two workgroups per CU, at least 256 of it each
      const int64_t tiles = ((M + bm - 1) / bm) * ((N + bn - 1) / bn);
      z = std::min<int64_t>(512 / std::max<int64_t>(tiles, 1), planes * K / 256);
      z = std::max<int64_t>(1, std::min<int64_t>(z, (int64_t)(most / plane)));
    } else {
      // The cheapest tile and number of slices by what they measured: us of a step with one tile a CU and, where two
      // fit, with two; us to start and end a tile (half more for two together); and a join of the slices at 5 TB/s
      // with 4 us to start.
      struct Tile {
        int kind, bm, bn;
        double one, two, start;
      };
      static const Tile dma_tiles[] = {
          {2, 256, 256, 1.9, 0, 0}, {3, 256, 128, 1.04, 0, 0}, {0, 128, 128, 0.75, 1.09, 0}};
      static const Tile term_tiles[] = {
          {0, 128, 128, 1.0, 1.5, 0}, {0, 128, 128, 1.2, 2.1, 0}, {0, 128, 128, 1.3, 0, 0}};
      // w's side of a product may be narrow, as a router's is: 160 rows fill one tile of 160, and 62% of two of 128
      // (4095 rows by w of 160 x 5120: 74 -> 56 us, its gradient by w 84 -> 67; w of 288 x 2048 89 -> 72 and 99 -> 83)
      static const Tile wide_m[] = {{0, 128, 128, 1.43, 0, 5.5}, {4, 160, 128, 1.8, 0, 8}};
      // with one buffer two tiles share a CU, and one's start and end lie under the other's products: short k and more
      // tiles than CUs (gradient by x of 4095 x 5120 with k = 160: 70 -> 57 us, of 2048 x 4096 with k = 512 58 -> 54;
      // alone on its CU it takes 111 us where two buffers take 98, 2048^3)
      static const Tile wide_n[] = {
          {0, 128, 128, 1.43, 0, 5.5}, {5, 128, 128, 1.65, 2.88, 5.5}, {4, 128, 160, 1.8, 0, 8}};
      const bool lds = dma && vec;  // (without 16-byte loads 16-bit operands go through registers too)
      const Tile *first = lds ? dma_tiles : term_tiles + (products <= 3 ? 0 : products <= 5 ? 1 : 2);
      int tiles_of = lds ? 3 : 1;
      if (products == 6 && vec) first = side < 0 ? wide_m : wide_n, tiles_of = side > 0 ? 3 : 2;
      double best = 1e30;
      for (const Tile *t = first; t < first + tiles_of; ++t) {
        const int64_t tiles = ((M + t->bm - 1) / t->bm) * ((N + t->bn - 1) / t->bn);
        for (int64_t s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
          if (s > 1 && (s * plane > most || steps < 4 * s || tiles * s > 1024)) break;
          const int64_t n = tiles * s;
          const double k = (double)((steps + s - 1) / s), one = t->one * k + t->start, two = t->two * k + 1.5 * t->start;
          double us = t->two ? n / 512 * two + (n % 512 > 256 ? two : n % 512 ? one : 0.0) : (n + 255) / 256 * one;
          us += s > 1 ? 4.0 + s * plane * 2 / 5e6 : 0.0;
          if (us < best) {
            best = us;
            z = s;
            p.tile = t->kind;
            bm = t->bm;
            bn = t->bn;
          }
        }
      }
    }
    p.tiles_m = (int)((M + bm - 1) / bm);
    p.tiles_n = (int)((N + bn - 1) / bn);
    p.kslice = (steps + z - 1) / z;
    p.slices = (int)((steps + p.kslice - 1) / p.kslice);
    p.part = p.slices > 1 ? (size_t)p.slices * plane : 0;
    return p;
  }
  z = std::max<int64_t>(1, std::min<int64_t>(z, (int64_t)(most / ((size_t)M * N * 4))));
  p.kslice = ((K + z - 1) / z + bk - 1) / bk * bk;
  p.slices = (int)((K + p.kslice - 1) / p.kslice);
  p.part = p.slices > 1 ? (size_t)p.slices * M * N * 4 : 0;
  return p;
}

size_t size_of(int type) { return type == LIN_F32 ? 4 : 2; }
bool lin_type(int t) { return t == LIN_F32 || t == LIN_F16 || t == LIN_BF16; }
size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// Whether an operand can be read 16 bytes at a time: `row` values contiguous in memory, taken 8 at a time where they
// are k (kc), else in 16 bytes.  By its shape, and by where it lies.
bool vec_shape(int64_t ld, int64_t row, int type, bool kc) {
  const size_t e = size_of(type);
  return !((size_t)ld * e & 15) && ld < BUF_ROW / (int64_t)e && !(kc ? row & 7 : (int64_t)((size_t)row * e & 15));
}
bool vec_at(const void *p) { return !((uintptr_t)p & 15); }

// One of a call's products: its shape decides the workspace; where the pointers then forbid 16-byte loads the plan has
// to do with that.
struct Product {
  int64_t M, N, K;
  int a_type, b_type, planes;
  int64_t plane;    // values from one plane of a to the next
  bool shaped;      // strides and widths allow 16-byte loads
  bool a_kc, b_kc;  // k contiguous in a and in b, else rows
  bool forward;     // the product has kernels for few rows
  int side;         // w's rows are columns (1) or rows (-1) of the result, or neither (0)
  Kind kind(bool vec) const {
    if (!forward || N >= (1 << 26) || K >= (1 << 30)) return TILES;
    return M <= LIN_ROWS ? ROWS : vec && lin_few_rows(M, N) ? FEW : TILES;
  }
  Plan plan_for(bool vec, size_t most) const {
    const int f32_by = b_type == LIN_BF16 ? 3 : b_type == LIN_F16 ? 5 : 6;
    return plan(kind(vec), M, N, K, planes, a_type == LIN_F32 ? f32_by : 1, side, vec, most);
  }
  // partial sums of at most 64 MB
  size_t space() const { return plan_for(shaped, 64 << 20).part; }
  Plan planned(bool vec) const { return plan_for(vec, vec == shaped ? 64 << 20 : space()); }
};
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

// chunks of rows of the bias gradient: 32 rows each, at most 256
int64_t dz_chunks(int64_t S) { return std::min<int64_t>((S + 31) / 32, 256); }

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

int check_desc(const zm_linear_desc *d, const char *who) {
  if (!d) return fail("%s: null description", who);
  if (!lin_type(d->x_type) || !lin_type(d->w_type) || !lin_type(d->y_type))
    return fail("%s: types are F32, F16 and BF16", who);
  if (d->x_type != ZM_TYPE_F32 && d->w_type != d->x_type)
    return fail("%s: 16-bit activations need weights of their own type", who);
  if (d->y_type != ZM_TYPE_F32 && d->y_type != d->x_type)
    return fail("%s: the result is F32 or of the activations' type", who);
  if (d->act < 0 || d->act >= ACT_COUNT) return fail("%s: unknown activation %d", who, d->act);
  if (d->S < 0 || d->I <= 0 || d->O <= 0) return fail("%s: S >= 0, I > 0 and O > 0 are needed", who);
  const int64_t most = (int64_t)1 << 31;
  if (d->S >= most || d->I >= most || d->O >= most) return fail("%s: S, I and O are below 2^31", who);
  if (d->x_stride < 0 || d->w_stride < 0 || d->y_stride < 0 || d->res_stride < 0 || d->pre_stride < 0)
    return fail("%s: negative stride", who);
  if (((d->S + 31) / 32) * ((d->O + 127) / 128) > 0x3fffff || ((d->S + 31) / 32) * ((d->I + 127) / 128) > 0x3fffff ||
      ((d->O + 31) / 32) * ((d->I + 127) / 128) > 0x3fffff)
    return fail("%s: S x O, S x I or O x I too large for one launch", who);
  return 0;
}

// the rows of a written matrix must not overlap
int check_rows(int64_t rows, int64_t stride, int64_t width, const char *who, const char *what) {
  if (rows > 1 && stride < width) return fail("%s: rows of %s overlap", who, what);
  return 0;
}

int launched() {
  HIP_OK(hipGetLastError());
  return 0;
}

LinArgs product(const Product &q, const void *a, int64_t lda, const void *b, int64_t ldb, const Plan &p, float *part) {
  LinArgs g{};
  g.a = a;
  g.b = b;
  g.lda = lda;
  g.ldb = ldb;
  g.M = q.M;
  g.N = q.N;
  g.K = q.K;
  g.planes = q.planes;
  g.plane = q.plane;
  g.tiles_m = p.tiles_m;
  g.tiles_n = p.tiles_n;
  g.slices = p.slices;
  g.kslice = p.kslice;
  g.part = part;
  g.terms = q.a_type == LIN_F32 || q.planes > 1;
  g.a_kc = q.a_kc;
  g.b_kc = q.b_kc;
  g.a_type = q.a_type;
  g.b_type = q.b_type;
  return g;
}

int join(const LinArgs &g, hipStream_t st) {
  if (g.slices > 1) lin_join(g, st);
  return launched();
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
