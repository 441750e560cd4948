// zm_linear_host.hpp -- host side of the unquantized products: which kernel, tile and number of k slices a product takes,
// the checks that the calls share, and the launch's arguments.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/zeromoe.h"
#include "zm_host.hpp"
#include "zm_linear.hpp"

namespace zm {
namespace {

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
Plan plan(Kind kind, int64_t M, int64_t N, int64_t K, int planes, int products, int side, bool pair, bool vec,
          size_t most) {
  const bool dma = products == 1;
  const int step = dma ? DMA_BK : 32;
  Plan p{};
  p.kind = kind;
  int64_t z = 1, bk = 64;
  if (kind == FEW) {
    // slices of k until there is a workgroup of 8 waves, or two of 4, per CU
    const int cols = pair ? few_pair_columns(M, N) : few_columns(M, N);
    p.tiles_m = (int)((M + FEW_ROWS - 1) / FEW_ROWS);
    p.tiles_n = (int)((N + cols - 1) / cols);
    bk = FEW_UNIT;
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n, want = cols == (pair ? 128 : 64) ? 512 : 256;
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
      // 16-bit operands: a tile alone on its CU starts and ends with nothing beside it, two of 128 x 128 hide each other's
      // (gradients by x of 8192 x 8192 with k = 1024: 256 x 256 304 us, 256 x 128 297, 128 x 128 181; of 8192 x 7168 with
      // k = 2048: 387, 398, 277; 8192^3: 971, 1115, 1051).  Two weights end a tile with twice the sums and the activation
      // (8192 x 7168 by two of 2048: 437, 450, 428 on one set of operands, 448, 558, 476 on three in turn).  In slices a 256 x 128 tile starts and ends in less, since CUs have one each (512 rows by w of 4096 x
      // 4096 in four slices 31 us, tiles of 128 x 128 in two 34; 130 rows in eight 19 and 20; 2048 x 2048 with k = 16384 in
      // two 180 and 161).  Over 389 products of 130 to 16384 rows the choice takes 0.7% more than the best one.
      const double more = pair ? 8.0 : 0.0;
      const Tile dma_tiles[] = {{2, 256, 256, 1.72, 0, 27 + more}, {3, 256, 128, 1.0, 0, 12}, {0, 128, 128, 0.76, 1.0, 3.3}};
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
      if (products == 6 && vec) first = side < 0 ? wide_m : wide_n, tiles_of = side > 0 && !pair ? 3 : 2;
      double best = 1e30;
      for (const Tile *t = first; t < first + tiles_of; ++t) {
        const int64_t tiles = ((M + t->bm - 1) / t->bm) * ((N + t->bn - 1) / t->bn);
        for (int64_t s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
          if (s > 1 && (s * plane > most || steps < 4 * s || tiles * s > 1024)) break;
          const int64_t n = tiles * s;
          const double k = (double)((steps + s - 1) / s), two = t->two * k + 1.5 * t->start;
          const double one = lds && t->kind == 3 && s > 1 ? 1.1 * k + 3 : t->one * k + t->start;
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
  int form = LIN_ONE;
  Kind kind(bool vec) const {
    if (!forward || N >= (1 << 26) || K >= (1 << 30)) return TILES;
    return M <= LIN_ROWS ? ROWS : vec && lin_few_rows(M, N) ? FEW : TILES;
  }
  Plan plan_for(bool vec, size_t most) const {
    const int f32_by = b_type == LIN_BF16 ? 3 : b_type == LIN_F16 ? 5 : 6;
    return plan(kind(vec), M, N, K, planes, a_type == LIN_F32 ? f32_by : 1, side, form == LIN_PAIR, vec,
                most);
  }
  // partial sums of at most 64 MB
  size_t space() const { return plan_for(shaped, 64 << 20).part; }
  Plan planned(bool vec) const { return plan_for(vec, vec == shaped ? 64 << 20 : space()); }
};
// chunks of rows of the bias gradient: 32 rows each, at most 256
int64_t dz_chunks(int64_t S) { return std::min<int64_t>((S + 31) / 32, 256); }

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
  g.form = q.form;
  return g;
}

int join(const LinArgs &g, hipStream_t st) {
  if (g.slices > 1) lin_join(g, st);
  return launched();
}

}  // namespace
}  // namespace zm
