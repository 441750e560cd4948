// zm_linear.hpp -- matrix products of unquantized operands on the matrix cores:
// C[m][n] = sum_k A(m, k) B(n, k) with an epilogue (bias, activation,
// residual), and its gradients.
//
// f32 operands have no fast matrix instruction (the f32 forms run at 1/16 of the
// bf16 rate), so an f32 value enters as a sum of bf16 terms
//   v = t0 + t1 + t2,  t0 = bf16(v), t1 = bf16(v - t0), t2 = bf16(v - t0 - t1)
// (3 x 8 significant bits cover the 24 of f32; the differences are exact), an f16
// value as two (11 bits), a bf16 value as one.  A product of two sums keeps the
// term pairs (i, j) with i + j <= 2: 6 bf16 products for f32 x f32, 5 for
// f32 x f16, 3 for f32 x bf16, accumulated in f32.  A term is at most 2^-8 of the
// one before it, so the pairs left out, (1, 2) and (2, 1), are at most 2^-23 of
// |a||b| (2^-24.2 in 2e7 products of values from [1, 2)).
// bf16 x bf16 and f16 x f16 are one product in their own type.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "zm_device.hpp"

namespace zm {

struct bf16 {
  uint16_t u;
};
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

enum { LIN_F32 = 0, LIN_F16 = 1, LIN_BF16 = 30 };
enum { ACT_NONE = 0, ACT_RELU, ACT_GELU, ACT_GELU_TANH, ACT_SILU, ACT_SIGMOID, ACT_COUNT };

template <class T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<_Float16>(_Float16 v) { return (float)v; }
template <>
__device__ __forceinline__ float to_f32<bf16>(bf16 v) { return __uint_as_float((uint32_t)v.u << 16); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ _Float16 from_f32<_Float16>(float v) { return (_Float16)v; }
template <>
__device__ __forceinline__ bf16 from_f32<bf16>(float v) { return bf16{__builtin_bit_cast(uint16_t, (__bf16)v)}; }

__device__ __forceinline__ float lin_load(const void *p, int type, size_t i) {
  if (type == LIN_F32) return ((const float *)p)[i];
  if (type == LIN_F16) return (float)((const _Float16 *)p)[i];
  return to_f32(((const bf16 *)p)[i]);
}
__device__ __forceinline__ void lin_store(void *p, int type, size_t i, float v) {
  if (type == LIN_F32) ((float *)p)[i] = v;
  else if (type == LIN_F16) ((_Float16 *)p)[i] = (_Float16)v;
  else ((bf16 *)p)[i] = from_f32<bf16>(v);
}
// four neighbouring values, at any address that their type allows (memory takes whole accesses at any alignment)
typedef v4f v4fu __attribute__((aligned(4)));
__device__ __forceinline__ v4f lin_load4(const void *p, int type, size_t i) {
  if (type == LIN_F32) return *reinterpret_cast<const v4fu *>((const float *)p + i);
  uint2 r;
  __builtin_memcpy(&r, (const uint16_t *)p + i, 8);
  if (type == LIN_F16) {
    typedef _Float16 v4h __attribute__((ext_vector_type(4)));
    const v4h h = __builtin_bit_cast(v4h, r);
    return v4f{(float)h.x, (float)h.y, (float)h.z, (float)h.w};
  }
  return v4f{__uint_as_float(r.x << 16), __uint_as_float(r.x & 0xffff0000u), __uint_as_float(r.y << 16),
             __uint_as_float(r.y & 0xffff0000u)};
}
__device__ __forceinline__ void lin_store4(void *p, int type, size_t i, v4f v) {
  if (type == LIN_F32) {
    *reinterpret_cast<v4fu *>((float *)p + i) = v;
  } else if (type == LIN_F16) {
    typedef _Float16 v4h __attribute__((ext_vector_type(4)));
    const v4h h = {(_Float16)v.x, (_Float16)v.y, (_Float16)v.z, (_Float16)v.w};
    __builtin_memcpy((_Float16 *)p + i, &h, 8);
  } else {
    typedef __bf16 v4b __attribute__((ext_vector_type(4)));
    const v4b h = {(__bf16)v.x, (__bf16)v.y, (__bf16)v.z, (__bf16)v.w};
    __builtin_memcpy((bf16 *)p + i, &h, 8);
  }
}

// act(z) and its slope; gelu by erf, gelu_tanh by its tanh form
__device__ __forceinline__ float lin_act(float z, int act) {
  switch (act) {
  case ACT_RELU: return z > 0.f ? z : (z != z ? z : 0.f);
  case ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
  case ACT_GELU_TANH: return 0.5f * z * (1.0f + tanhf(0.79788456080286536f * (z + 0.044715f * z * z * z)));
  case ACT_SILU: return z / (1.0f + expf(-z));
  case ACT_SIGMOID: return 1.0f / (1.0f + expf(-z));
  default: return z;
  }
}
__device__ __forceinline__ float lin_slope_of_number(float z, int act) {
  switch (act) {
  case ACT_RELU: return z > 0.f ? 1.0f : 0.0f;
  case ACT_GELU: {
    const float zc = fminf(fmaxf(z, -20.f), 20.f);  // exp(-z^2/2) is 0 there; z * exp() has no inf * 0
    return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) + zc * expf(-0.5f * zc * zc) * 0.39894228040143268f;
  }
  case ACT_GELU_TANH: {
    const float zc = fminf(fmaxf(z, -20.f), 20.f);  // tanh is +-1 there: slope 0 or 1
    const float t = tanhf(0.79788456080286536f * (zc + 0.044715f * zc * zc * zc));
    return 0.5f * (1.0f + t) + 0.5f * zc * (1.0f - t * t) * 0.79788456080286536f * (1.0f + 0.134145f * zc * zc);
  }
  case ACT_SILU: {
    const float zc = fminf(fmaxf(z, -120.f), 120.f);  // the sigmoid is 0 or 1 there
    const float g = 1.0f / (1.0f + expf(-zc));
    return g * (1.0f + zc * (1.0f - g));
  }
  case ACT_SIGMOID: {
    const float e = expf(-fabsf(z)), r = 1.0f / (1.0f + e);
    return e * r * r;  // sigmoid(z) sigmoid(-z): g (1 - g) has no digits left where g is near 1
  }
  default: return 1.0f;
  }
}
// (the clamps and comparisons above would make a number of a NaN)
__device__ __forceinline__ float lin_act_slope(float z, int act) {
  const float s = lin_slope_of_number(z, act);
  return z == z ? s : z;
}

// ============================================================ terms

constexpr float BF16_MOST = 3.38953139e38f;  // largest finite bf16
constexpr float F32_MOST = 3.40282347e38f;   // largest finite f32

// v[8] as NT bf16 terms, without a branch.  T is what the values came from: an f32 past bf16's largest is cut to that
// for its first term (it would round to infinity and leave inf - inf behind); an infinity ends as a NaN term.
template <class T, int NT>
__device__ __forceinline__ void split_terms(const float (&v)[8], v8bf (&t)[NT]) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    t[0][i] = (__bf16)(NT > 1 && sizeof(T) == 4 ? __builtin_amdgcn_fmed3f(v[i], -BF16_MOST, BF16_MOST) : v[i]);
    if (NT > 1) r[i] = v[i] - (float)t[0][i];
  }
#pragma unroll
  for (int k = 1; k < NT; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      t[k][i] = (__bf16)r[i];
      if (k + 1 < NT) r[i] -= (float)t[k][i];
    }
}

// 16 bytes from a buffer resource; an offset of OOR reads as zeros and touches no memory.  Bases move along k with the
// loop, so offsets stay within the tile: rows shorter than 8 MB.
__device__ __forceinline__ v4u buf16(rsrc_t r, int vo, int so) { return __builtin_bit_cast(v4u, bld16(r, vo, so)); }
__device__ __forceinline__ rsrc_t buf_at(const void *p) { return make_rsrc(p, 0x7ffffff0u); }
constexpr int64_t BUF_ROW = 1 << 23;  // bytes of a row, less than: 256 rows of a tile stay below 2^31

// ============================================================ sums over partial rows

// dst0[i] (i < n0) and dst1[i - n0] (n0 <= i < n) = sum over p < parts of part[p][i], either null: not wanted.  A
// workgroup takes 16 packs of V columns; its 16 groups of 16 threads take every 16th part, eight loads in flight, and
// their sums meet in LDS, all in a fixed order.  512 parts of 14336 columns (29 MB): 9 us, against 123 us with a
// thread per column going through all parts.
template <int V>
static __global__ __launch_bounds__(256) void k_parts_sum(const float *__restrict__ part, int parts, int64_t n, int64_t n0,
                                                          float *__restrict__ dst0, float *__restrict__ dst1) {
  __shared__ float red[16][16 * V];
  const int c = threadIdx.x & 15, g = threadIdx.x >> 4;
  const int64_t i = ((int64_t)blockIdx.x * 16 + c) * V;
  float v[V] = {};
  if (i < n) {
    for (int p0 = g; p0 < parts; p0 += 128) {
      float t[8][V];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int p = p0 + 16 * u;
        if constexpr (V == 4) {
          const v4f r = p < parts ? *reinterpret_cast<const v4f *>(part + (size_t)p * n + i) : v4f{0.f, 0.f, 0.f, 0.f};
          t[u][0] = r.x, t[u][1] = r.y, t[u][2] = r.z, t[u][3] = r.w;
        } else {
          t[u][0] = p < parts ? part[(size_t)p * n + i] : 0.f;
        }
      }
#pragma unroll
      for (int u = 0; u < 8; ++u)
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] += t[u][j];
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) red[g][c * V + j] = v[j];
  __syncthreads();
  for (int j = threadIdx.x; j < 16 * V; j += 256) {
    const int64_t k = (int64_t)blockIdx.x * 16 * V + j;
    if (k >= n) break;
    float a = 0.f;
#pragma unroll
    for (int q = 0; q < 16; ++q) a += red[q][j];
    float *dst = k < n0 ? dst0 : dst1;
    if (dst) dst[k < n0 ? k : k - n0] = a;
  }
}
static inline void parts_sum(const float *part, int parts, int64_t n, int64_t n0, float *dst0, float *dst1,
                             hipStream_t st) {
  if (!(n & 3) && !((uintptr_t)part & 15))
    hipLaunchKernelGGL((k_parts_sum<4>), dim3((unsigned)((n + 63) / 64)), dim3(256), 0, st, part, parts, n, n0, dst0, dst1);
  else
    hipLaunchKernelGGL((k_parts_sum<1>), dim3((unsigned)((n + 15) / 16)), dim3(256), 0, st, part, parts, n, n0, dst0, dst1);
}

// ============================================================ operands
//
// A tile of ROWS rows (m or n) x BK columns (k) goes from global memory through registers into LDS, one plane per term:
// plane[row][BK] of 16-bit values.  LDS has 64 banks of 4 bytes, and 16 lanes read 16 bytes each at once: the 16-byte
// chunks of a row are permuted by the row so that one chunk of 16 neighbouring rows (a fragment) covers all banks; rows
// eight apart, which a row-contiguous operand writes together, fall apart too.
//
// A unit is one thread's part: 8 consecutive k of one row where k is contiguous
// in memory (KC), else 4 bytes of rows (one f32, two 16-bit) for each of 8 consecutive k, transposed in registers:
// small enough for every thread to have its share of the splitting into terms.
template <int BK>
__device__ __forceinline__ int chunk_at(int row, int c) {
  if (BK == 128) return c ^ (row & 15);
  if (BK == 64) return c ^ (((row >> 1) ^ (row >> 4)) & 7);
  return c ^ (((row >> 2) ^ (row >> 4)) & 3);
}

template <class T, int NT, bool KC, int ROWS, int BK, int NTHR, bool VEC>
struct Operand {
  static constexpr int R = KC ? 1 : 4 / (int)sizeof(T);  // rows of a unit
  static constexpr int CH = BK / 8;
  static constexpr int UNITS = ROWS / R * CH;
  static constexpr int UPT = (UNITS + NTHR - 1) / NTHR;
  static constexpr int NW = KC ? 2 * (int)sizeof(T) : 8;  // words of a unit
  static constexpr int PLANE = ROWS * BK;                 // 16-bit values of a term plane

  const T *base;  // the tile's first row
  int64_t ld;
  int rows;       // of the matrix, from the tile's first row
  int first;      // the thread (where units and threads do not match some units are loaded and stored twice)
  int off[UPT];   // bytes from the tile's first row and column (16-byte loads)
  struct Raw {    // a step of the tile as it came from memory: the thread's units
    uint32_t r[UPT][NW];
  };

  // `row0`: the tile's first row; `total`: rows of the matrix
  __device__ __forceinline__ void init(const void *p, int64_t ld_, int64_t row0, int64_t total, int t) {
    ld = ld_;
    base = (const T *)p + (KC ? row0 * ld : row0);
    rows = (int)(total - row0 < ROWS ? total - row0 : ROWS);
    first = t;
#pragma unroll
    for (int i = 0; i < UPT; ++i) {
      int row, c;
      place(first + i * NTHR, row, c);
      if (KC) off[i] = (min(row, rows - 1) * (int)ld + 8 * c) * (int)sizeof(T);
      else off[i] = (8 * c * (int)ld + min(row, rows - R)) * (int)sizeof(T);
    }
  }
  __device__ __forceinline__ static void place(int u, int &row, int &c) {
    if (UNITS % NTHR) u %= UNITS;
    if (KC) {
      row = u / CH;
      c = u % CH;
    } else {
      row = u % (ROWS / R) * R;
      c = u / (ROWS / R);
    }
  }
  // columns [k, k + left) of the tile, `skip` values on, and zeros; rows past the matrix
  // repeat its last ones (their results are not stored)
  __device__ __forceinline__ void load(Raw &to, int64_t k, int left, int64_t skip) const {
    const T *at = base + skip + (KC ? k : k * ld);
    const rsrc_t r = buf_at(at);
#pragma unroll
    for (int i = 0; i < UPT; ++i) {
      int row, c;
      place(first + i * NTHR, row, c);
      if constexpr (VEC && KC) {
        const int vo = 8 * c < left ? off[i] : OOR;
#pragma unroll
        for (int q = 0; q < NW / 4; ++q) {
          const v4u v = buf16(r, vo, 16 * q);
#pragma unroll
          for (int j = 0; j < 4; ++j) to.r[i][4 * q + j] = v[j];
        }
      } else if constexpr (VEC) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          to.r[i][j] = bld4(r, 8 * c + j < left ? off[i] : OOR, j * (int)ld * (int)sizeof(T));
      } else if (left == BK && (KC || rows >= R)) {
        // any alignment: memory takes it, the whole step exists
        if constexpr (KC) {
          __builtin_memcpy(to.r[i], at + (int64_t)min(row, rows - 1) * ld + 8 * c, sizeof(to.r[i]));
        } else {
          const T *p = at + (int64_t)8 * c * ld + min(row, rows - R);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            __builtin_memcpy(&to.r[i][j], p + j * ld, 4);
            if (R == 2 && row > rows - R) to.r[i][j] >>= 16;  // the last row of an odd number of them
          }
        }
      } else if constexpr (KC) {
        const T *p = at + (int64_t)min(row, rows - 1) * ld + 8 * c;
        T e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = 8 * c + j < left ? p[j] : from_f32<T>(0.f);
        __builtin_memcpy(to.r[i], e, sizeof(e));
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const T *p = at + (int64_t)(8 * c + j) * ld;
          T e[R];
#pragma unroll
          for (int q = 0; q < R; ++q) e[q] = 8 * c + j < left ? p[min(row + q, rows - 1)] : from_f32<T>(0.f);
          __builtin_memcpy(&to.r[i][j], e, 4);
        }
      }
    }
  }
  __device__ __forceinline__ void store(uint16_t *lds, const Raw &from) const {
#pragma unroll
    for (int i = 0; i < UPT; ++i) {
      int row, c;
      place(first + i * NTHR, row, c);
      if constexpr (KC) {
        put8(lds, row, c, from.r[i]);
      } else if constexpr (sizeof(T) == 4) {
        put8(lds, row, c, from.r[i]);
      } else {
        // word j holds rows 0 and 1 at column j
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t o[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            o[j] = __builtin_amdgcn_perm(from.r[i][2 * j + 1], from.r[i][2 * j], h ? 0x07060302u : 0x05040100u);
          put8(lds, row + h, c, o);
        }
      }
    }
  }
  // 8 values of one row, as they came, into the planes
  __device__ __forceinline__ void put8(uint16_t *lds, int row, int c, const uint32_t *w) const {
    uint16_t *at = lds + row * BK + chunk_at<BK>(row, c) * 8;
    if constexpr (NT == 1 && sizeof(T) == 2) {
      *reinterpret_cast<v4u *>(at) = v4u{w[0], w[1], w[2], w[3]};
    } else {
      T e[8];
      float v[8];
      __builtin_memcpy(e, w, sizeof(e));
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = to_f32(e[j]);
      v8bf t[NT];
      split_terms<T, NT>(v, t);
#pragma unroll
      for (int n = 0; n < NT; ++n) *reinterpret_cast<v8bf *>(at + n * PLANE) = t[n];
    }
  }
};

// ============================================================ the product

struct LinEpilogue {
  void *y;             // [M][N], row stride ldy, of type `type`
  const void *res;     // [M][N] of the same type, or null
  void *pre;           // [M][N] of the same type: z = sum + bias before the activation, or null
  const float *bias;   // [N] or null
  int64_t ldy, ldr, ldp;
  int type, act;
};

struct LinArgs {
  const void *a, *b;
  int64_t lda, ldb;
  int64_t M, N, K;
  int tiles_m, tiles_n;
  int planes;      // of a, to be added: each `plane` values after the last, all times the same b
  int64_t plane;
  int slices;      // of k
  int64_t kslice;  // k of a slice; k_linear, k_linear_dma: steps of a slice
  float *part;     // [slices][M][N] when slices > 1
  LinEpilogue e;
  bool terms;      // values enter as sums of terms: what follows says how they lie, for lin_again()
  bool a_kc, b_kc; // k contiguous, else rows
  int a_type, b_type;
};

__device__ __forceinline__ float lin_finish1(const LinEpilogue &e, int64_t m, int64_t n, float z) {
  if (e.bias) z += e.bias[n];
  if (e.pre) lin_store(e.pre, e.type, (size_t)(m * e.ldp + n), z);
  float y = lin_act(z, e.act);
  if (e.res) y += lin_load(e.res, e.type, (size_t)(m * e.ldr + n));
  return y;
}
// four results of one row, columns n .. n + 3 of which those below N exist
__device__ __forceinline__ void lin_finish4(const LinEpilogue &e, int64_t m, int64_t n, int64_t N, v4f z) {
  if (n + 4 <= N) {
    if (e.bias) z += *reinterpret_cast<const v4fu *>(e.bias + n);
    if (e.pre) lin_store4(e.pre, e.type, (size_t)(m * e.ldp + n), z);
    if (e.act) {
#pragma unroll
      for (int j = 0; j < 4; ++j) z[j] = lin_act(z[j], e.act);
    }
    if (e.res) z += lin_load4(e.res, e.type, (size_t)(m * e.ldr + n));
    lin_store4(e.y, e.type, (size_t)(m * e.ldy + n), z);
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (n + j < N) lin_store(e.y, e.type, (size_t)(m * e.ldy + n + j), lin_finish1(e, m, n + j, z[j]));
}

__device__ __forceinline__ bool lin_finite(float v) { return fabsf(v) <= F32_MOST; }
// One sum again from the values themselves.  An infinity times a sum of terms is a sum of infinities of both signs or of
// zero times one, so NaN stands where the formula may have an infinity, and terms' products may pass f32's largest where
// their sum does not.  A sum that is not finite is taken again in f32, value by value: what an infinity gives does not go
// by the number of rows or by the kernel.  Finite sums cost a check (2048^3 in f32: 108 us with and without it); with an
// infinity in every row all of them are taken again, 16 ms (512 x 4096 x 4096, f32 by bf16: 32); behind a NaN, where the
// sum stays one, 0.14 ms.
__device__ __forceinline__ float lin_again(const LinArgs &g, int64_t m, int64_t n) {
  const int64_t ak = g.a_kc ? 1 : g.lda, bk = g.b_kc ? 1 : g.ldb;
  size_t ia = (size_t)(g.a_kc ? m * g.lda : m), ib = (size_t)(g.b_kc ? n * g.ldb : n);
  float s = 0.f;
  for (int64_t k = 0; k < g.K && s == s; k += 4, ia += 4 * ak, ib += 4 * bk) {
    float a[4], b[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bool in = k + u < g.K;
      a[u] = in ? lin_load(g.a, g.a_type, ia + u * ak) : 0.f;
      for (int p = 1; p < g.planes && lin_finite(a[u]); ++p)  // (an infinity or a NaN is its first term)
        a[u] += in ? lin_load(g.a, g.a_type, ia + u * ak + p * g.plane) : 0.f;
      b[u] = in ? lin_load(g.b, g.b_type, ib + u * bk) : 0.f;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) s = __builtin_fmaf(a[u], b[u], s);
  }
  return s;
}
// sums of row m, columns n .. n + 3: those that are not finite again
__device__ __forceinline__ void lin_repair(const LinArgs &g, int64_t m, int64_t n, v4f &v) {
  if (m >= g.M || lin_finite((fabsf(v.x) + fabsf(v.y)) + (fabsf(v.z) + fabsf(v.w)))) return;
#pragma unroll 1
  for (int q = 0; q < 4; ++q) {
    const float x = q == 0 ? v.x : q == 1 ? v.y : q == 2 ? v.z : v.w;
    if (lin_finite(x) || n + q >= g.N) continue;
    const float y = lin_again(g, m, n + q);
    v.x = q == 0 ? y : v.x;
    v.y = q == 1 ? y : v.y;
    v.z = q == 2 ? y : v.z;
    v.w = q == 3 ? y : v.w;
  }
}
// the same for a wave's fragments, where there is one slice (else the slices' join does it); at(i, 0), at(j, 1): their m
// and n; TERMS: whether the kernel's operands may come as terms
template <bool TERMS, int FM, int FN, class At>
__device__ __forceinline__ void lin_repair_all(const LinArgs &g, v4f (&acc)[FM][FN], const At &at) {
  if (!TERMS || !g.terms || g.slices > 1) return;
  float most = 0.f;  // (a sum past f32's largest is looked at again value by value)
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) most += fabsf(acc[i][j][q]);
  if (__ballot(!lin_finite(most)) == 0) return;
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) lin_repair(g, at(i, 0), at(j, 1), acc[i][j]);
}

// four sums of slice z: into its plane, or finished where there is one slice
__device__ __forceinline__ void lin_result(const LinArgs &g, int z, int64_t m, int64_t n, v4f v) {
  if (m >= g.M || n >= g.N) return;
  if (g.slices == 1) return lin_finish4(g.e, m, n, g.N, v);
  float *p = g.part + ((size_t)z * g.M + m) * g.N + n;
  if (n + 4 <= g.N) {
    *reinterpret_cast<v4fu *>(p) = v;
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (n + q < g.N) p[q] = v[q];
  }
}

// Workgroup -> tile.  Workgroups go to the 8 XCDs in turn; each XCD takes a run
// of neighbouring tiles instead, so that the operands they share meet in its L2.
__device__ __forceinline__ int xcd_order(int b, int n) {
  const int q = n / 8, r = n % 8, x = b % 8;
  return x * q + min(x, r) + b / 8;
}

// The steps of one slice: BK of k each, through the planes of `a` one after the other.
struct LinSteps {
  int64_t k, left, per;  // where the step is; steps left; steps of a plane
  int p;
  __device__ __forceinline__ LinSteps(const LinArgs &g, int z, int bk) {
    per = (g.K + bk - 1) / bk;
    const int64_t first = z * g.kslice;
    left = min(g.planes * per - first, g.kslice);
    p = g.planes > 1 ? (int)(first / per) : 0;
    k = (first - p * per) * bk;
  }
  __device__ __forceinline__ bool next(int bk) {
    k += bk;
    if (k >= per * bk) k = 0, ++p;
    return --left > 0;
  }
};

// The term pairs (i, j) of a product: (0, 0) first, then those 2^-8 and 2^-16 smaller, up to this i + j
constexpr int PAIRS_MOST = 2;

// One workgroup: BM x BN results over one slice of k; WM x WN waves of 16 x 16 matrix instructions.  Two steps of BK
// deep in LDS: while one is multiplied, the next one, in registers, is split into terms and stored, and the one after
// that is on its way from memory; one barrier a step.  The instruction's rows are the results' columns n, so that a
// lane ends with 4 neighbouring n of one row m.  f32 by f32, 2048^3: 95 us, 181 TFLOP/s of f32 products (1085 of bf16
// ones).  With one buffer (BUFS) the splitting follows the products, one step is on its way, and two workgroups of f32
// by f32 share a CU (where there are two: 4096 x 5120 by k = 64 42 -> 35 us; alone 98 -> 111, 2048^3).
template <class TA, int NA, bool KCA, class TB, int NB, bool KCB, int BM, int BN, int WM, int WN, bool VEC,
          int BUFS = 2>
__global__ __launch_bounds__(64 * WM * WN, BUFS == 1 ? 4 : 1) void k_linear(LinArgs g) {
  constexpr bool F16 = std::is_same<TA, _Float16>::value && std::is_same<TB, _Float16>::value && NA == 1 && NB == 1;
  constexpr int BK = NA * NB == 1 ? 64 : 32;
  constexpr int NTHR = 64 * WM * WN;
  constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  typedef Operand<TA, NA, KCA, BM, BK, NTHR, VEC> OA;
  typedef Operand<TB, NB, KCB, BN, BK, NTHR, VEC> OB;
  constexpr int LA = NA * BM * BK, LDS = LA + NB * BN * BK;
  __shared__ __attribute__((aligned(16))) uint16_t lds[BUFS][LDS];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int tile = xcd_order(blockIdx.x, gridDim.x);
  const int per = g.tiles_m * g.tiles_n;
  const int z = tile / per, tt = tile - z * per;
  const int64_t m0 = (int64_t)(tt / g.tiles_n) * BM, n0 = (int64_t)(tt % g.tiles_n) * BN;
  OA a;
  OB b;
  a.init(g.a, g.lda, m0, g.M, tid);
  b.init(g.b, g.ldb, n0, g.N, tid);
  v4f acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
  const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
  const int fr = lane & 15, fc = lane >> 4;
  LinSteps at(g, z, BK);  // the step to be asked for
  const int64_t steps = at.left;
  struct Raw {
    typename OA::Raw a;
    typename OB::Raw b;
  };
  auto load = [&](Raw &to) {  // zeros behind the last step
    const int left = at.left > 0 ? (int)min(g.K - at.k, (int64_t)BK) : 0;
    a.load(to.a, at.k, left, at.p * g.plane);
    b.load(to.b, at.k, left, 0);
    at.next(BK);
  };
  auto step = [&](const uint16_t *from, uint16_t *to, const Raw &next, Raw &after) {
    load(after);
#pragma unroll
    for (int s = 0; s < BK / 32; ++s) {
      v8bf fa[FM][NA], fb[FN][NB];
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int r = wm + 16 * i + fr;
#pragma unroll
        for (int t = 0; t < NA; ++t)
          fa[i][t] = *reinterpret_cast<const v8bf *>(from + t * BM * BK + r * BK + chunk_at<BK>(r, 4 * s + fc) * 8);
      }
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const int r = wn + 16 * j + fr;
#pragma unroll
        for (int t = 0; t < NB; ++t)
          fb[j][t] = *reinterpret_cast<const v8bf *>(from + LA + t * BN * BK + r * BK + chunk_at<BK>(r, 4 * s + fc) * 8);
      }
      if (BUFS == 2 && s == BK / 32 - 1) {
        a.store(to, next.a);
        b.store(to + LA, next.b);
      }
#pragma unroll
      for (int ta = 0; ta < NA; ++ta)
#pragma unroll
        for (int tb = 0; tb < NB; ++tb) {
          if (ta + tb > PAIRS_MOST) continue;
#pragma unroll
          for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) {
              if constexpr (F16)
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, fb[j][tb]),
                                                                  __builtin_bit_cast(v8h, fa[i][ta]), acc[i][j], 0, 0, 0);
              else
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[j][tb], fa[i][ta], acc[i][j], 0, 0, 0);
            }
        }
    }

    if (BUFS == 1) {
      __syncthreads();
      a.store(to, next.a);
      b.store(to + LA, next.b);
    } else if (NA * NB > 1) {
      // the splitting into terms goes between the products, which leave the vector units three of four issues
#pragma unroll
      for (int i = 0; i < FM * FN * NA * NB; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x2, 2, 0);
      }
    }
    __syncthreads();
  };
  Raw p, q;
  load(p);
  if (BUFS == 2) load(q);
  a.store(lds[0], p.a);
  b.store(lds[0] + LA, p.b);
  __syncthreads();
  for (int64_t t = 0; t < steps; t += 2) {
    step(lds[0], lds[BUFS - 1], BUFS == 2 ? q : p, p);
    if (t + 1 >= steps) break;
    step(lds[BUFS - 1], lds[0], p, BUFS == 2 ? q : p);
  }
  lin_repair_all<(NA * NB > 1 || !KCB), FM, FN>(
      g, acc, [&](int i, int n) { return n ? n0 + wn + 16 * i + 4 * fc : m0 + wm + 16 * i + fr; });
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) lin_result(g, z, m0 + wm + 16 * i + fr, n0 + wn + 16 * j + 4 * fc, acc[i][j]);
}

// ============================================================ 16-bit operands, large
//
// The same product for 16-bit operands of one type, bound by the matrix cores.  Tiles go from global memory straight
// into LDS (16 bytes a lane, whole cache lines of 64 k), two steps deep; fragments are read into registers half a step
// ahead; one barrier a step.  8192^3 in bf16: 945 us, 1160 TFLOP/s (without its loads the loop does 1460; with them
// answered by L2 alone 1290; reading them where a step of 32 k is four deep, in half lines, 780).
//
// An operand whose k is contiguous lies in LDS in rows of 64 k, its 16-byte chunks permuted by the row so that 16 rows
// of a fragment cover all banks.  A row-contiguous one lies as it is in memory, a row of LDS for each k, and is turned
// by the transposing reads (16 lanes read 4 k of 16 rows and get 4 k of one row each); its 32-byte pieces are permuted
// by k so that the 8 k that 32 lanes read fall into different banks.  LDS is written in the lanes' order, so the
// permutation is in what each lane asks for.
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
constexpr int DMA_BK = 64;

template <bool KC, int ROWS, int NTHR, int FR>
struct DmaOperand {
  static constexpr int BK = DMA_BK;
  static constexpr int PER = ROWS * BK / 8 / NTHR, WIDE = ROWS / 8;  // 16-byte chunks of a thread; of a row of k
  static constexpr int BYTES = ROWS * BK * 2;
  const uint16_t *base;
  int64_t ld;
  int off[PER];
  uint32_t at[KC ? 2 : FR];  // where the lane's part of each fragment is (KC: of each half of the step)
  __device__ __forceinline__ static int turn(int k) { return (k & 3) | ((k >> 3) & 1) << 2; }
  __device__ __forceinline__ static void place(int i, int &r, int &c) {  // KC: row, chunk; else k, first row
    const int s = i * NTHR + (int)threadIdx.x;
    if (KC) {
      r = s / 8;
      c = s % 8 ^ (r >> 1 & 7);
    } else {
      r = s / WIDE;
      const int q = s % WIDE;
      c = 8 * ((((q >> 1) ^ turn(r)) << 1) | (q & 1));
    }
  }
  // `w0`: the wave's first row of the tile
  __device__ __forceinline__ void init(const void *p, int64_t ld_, int64_t row0, int64_t total, int w0) {
    ld = ld_;
    base = (const uint16_t *)p + (KC ? row0 * ld : row0);
    const int rows = (int)(total - row0 < ROWS ? total - row0 : ROWS);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      int r, c;
      place(i, r, c);
      off[i] = 2 * (KC ? min(r, rows - 1) * (int)ld + 8 * c : r * (int)ld + min(c, rows - 8));
    }
    const int lane = threadIdx.x & 63, fr = lane & 15, fc = lane >> 4;
    if constexpr (KC) {
#pragma unroll
      for (int s = 0; s < 2; ++s) at[s] = 2 * ((w0 + fr) * BK + ((4 * s + fc) ^ (fr >> 1)) * 8);  // (w0: 16 n)
    } else {
      const int k = 8 * fc + (fr >> 2);
#pragma unroll
      for (int i = 0; i < FR; ++i) at[i] = 2 * (k * ROWS + (((w0 >> 4) + i ^ turn(k)) << 4) + 4 * (fr & 3));
    }
  }
  __device__ __forceinline__ v4u_t source(int64_t k, int64_t skip) const {
    return dma_rsrc(base + skip + (KC ? k : k * ld), 0x7ffffff0u);
  }
  // the i-th request of a step into the buffer at `lds`; `left`: k of the step that exist (zeros past them)
  __device__ __forceinline__ void ask(v4u_t rs, uint32_t lds, int i, int left) const {
    int r, c;
    place(i, r, c);
    dma_lds16(rs, lds + (threadIdx.x >> 6) * 1024u + i * NTHR * 16u, (KC ? 8 * c : r) < left ? off[i] : OOR, 0);
  }
  // fragment i of the wave, half s of the step, from the buffer at `lds`
  __device__ __forceinline__ v8bf frag(uint32_t lds, int i, int s) const {
    if constexpr (KC) {
      typedef __attribute__((address_space(3))) v8s *lp;
      return __builtin_bit_cast(v8bf, *(lp)(lds + at[s] + 2 * 16 * BK * i));
    } else {
      typedef __attribute__((address_space(3))) v4s *lp;
      const uint32_t q = lds + at[i] + 64 * ROWS * s;
      const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)q),
                hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(q + 8 * ROWS));
      return __builtin_bit_cast(v8bf, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

template <bool F16, bool KCA, bool KCB, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void k_linear_dma(LinArgs g) {
  constexpr int NTHR = 64 * WM * WN, FM = BM / WM / 16, FN = BN / WN / 16;
  typedef DmaOperand<KCA, BM, NTHR, FM> OA;
  typedef DmaOperand<KCB, BN, NTHR, FN> OB;
  constexpr int BYTES = OA::BYTES + OB::BYTES;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * BYTES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int tile = xcd_order(blockIdx.x, gridDim.x);
  const int per = g.tiles_m * g.tiles_n;
  const int z = tile / per, tt = tile - z * per;
  // four rows of tiles at a time, so that the 32 tiles of an XCD read about 4 x 8 tiles' operands
  const int band = tt / (4 * g.tiles_n), in = tt - band * 4 * g.tiles_n, hi = min(4, g.tiles_m - 4 * band);
  const int64_t m0 = (int64_t)(4 * band + in % hi) * BM, n0 = (int64_t)(in / hi) * BN;
  const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
  OA a;
  OB b;
  a.init(g.a, g.lda, m0, g.M, wm);
  b.init(g.b, g.ldb, n0, g.N, wn);
  v4f acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
  LinSteps at(g, z, DMA_BK);  // the step to be asked for
  const uint32_t l0 = lds_addr(lds);
  const int64_t steps = at.left;
  int left = (int)min(g.K - at.k, (int64_t)DMA_BK);
  auto next = [&] {
    at.next(DMA_BK);
    left = at.left > 0 ? (int)min(g.K - at.k, (int64_t)DMA_BK) : 0;
  };
  auto load = [&](uint32_t to) {
    const v4u_t ra = a.source(at.k, at.p * g.plane), rb = b.source(at.k, 0);
#pragma unroll
    for (int i = 0; i < OA::PER; ++i) a.ask(ra, to, i, left);
#pragma unroll
    for (int i = 0; i < OB::PER; ++i) b.ask(rb, to + OA::BYTES, i, left);
    next();
  };
  auto row = [&](int i, const v8bf &fa, const v8bf (&fb)[FN]) {
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      if constexpr (F16)
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, fb[j]), __builtin_bit_cast(v8h, fa),
                                                          acc[i][j], 0, 0, 0);
      else
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[j], fa, acc[i][j], 0, 0, 0);
    }
  };
  // Step t lies in one buffer, step t + 1 lands in the other.  While the step's first half is multiplied its second
  // half is read; then all waves have read the buffer and step t + 1 has landed, and while the second half is multiplied
  // the first half of step t + 1 is read and step t + 2 asked for, into the buffer that is free.
  load(l0);
  wait_barrier<0>();
  load(l0 + BYTES);
  v8bf a0[FM], b0[FN], a1[FM], b1[FN];
#pragma unroll
  for (int j = 0; j < FN; ++j) b0[j] = b.frag(l0 + OA::BYTES, j, 0);
#pragma unroll
  for (int i = 0; i < FM; ++i) a0[i] = a.frag(l0, i, 0);
  uint32_t cur = l0, other = l0 + BYTES;
  // the fragments of half s in the buffer at `from`, a few behind each row of products, the first ones needed first
  auto read = [&](int i, v8bf (&fa)[FM], v8bf (&fb)[FN], uint32_t from, int s) {
    constexpr int EACH = (FM + FN + FM / 2 - 1) / (FM / 2);
#pragma unroll
    for (int q = i * EACH; q < (i + 1) * EACH && q < FM + FN; ++q) {
      if (q < FN) fb[q] = b.frag(from + OA::BYTES, q, s);
      else fa[q - FN] = a.frag(from, q - FN, s);
    }
  };
  for (int64_t t = 0; t < steps; ++t) {
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      row(i, a0[i], b0);
      __builtin_amdgcn_sched_barrier(0);
      read(i, a1, b1, cur, 1);
      __builtin_amdgcn_sched_barrier(0);
    }
    wait_barrier<0>();
    const v4u_t ra = a.source(at.k, at.p * g.plane), rb = b.source(at.k, 0);
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      row(i, a1[i], b1);
      __builtin_amdgcn_sched_barrier(0);
      read(i, a0, b0, other, 0);
#pragma unroll
      for (int q = i * OA::PER / FM; q < (i + 1) * OA::PER / FM; ++q) a.ask(ra, cur, q, left);
#pragma unroll
      for (int q = i * OB::PER / FM; q < (i + 1) * OB::PER / FM; ++q) b.ask(rb, cur + OA::BYTES, q, left);
      __builtin_amdgcn_sched_barrier(0);
    }
    next();
    const uint32_t swap = cur;
    cur = other;
    other = swap;
  }
  wait_vm<0>();  // (what was asked for past the end writes zeros: not into another workgroup's LDS)
  const int fr = lane & 15, fc = lane >> 4;
  lin_repair_all<!KCB, FM, FN>(
      g, acc, [&](int i, int n) { return n ? n0 + wn + 16 * i + 4 * fc : m0 + wm + 16 * i + fr; });
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) lin_result(g, z, m0 + wm + 16 * i + fr, n0 + wn + 16 * j + 4 * fc, acc[i][j]);
}

// Results of the k slices added in order (the same bits on every call), then the epilogue.  G threads share four
// results where there are many slices: each adds every G-th, four loads in flight, and their sums meet in LDS.
template <int G>
static __global__ __launch_bounds__(256) void k_linear_join(LinArgs g) {
  constexpr int Q = 256 / G;  // quads of results of a workgroup
  __shared__ v4f red[G][Q];
  const int64_t nq = (g.N + 3) / 4, q = (int64_t)blockIdx.x * Q + threadIdx.x % Q;
  const int first = threadIdx.x / Q;
  const bool in = q < g.M * nq;
  const int64_t m = q / nq, n = (q - m * nq) * 4;
  v4f v = {0.f, 0.f, 0.f, 0.f};
  const size_t plane = (size_t)g.M * g.N;
  const float *p = g.part + (size_t)m * g.N + n;
  if (in) {
    for (int z0 = first; z0 < g.slices; z0 += 4 * G) {
      v4f t[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int z = z0 + u * G;
        t[u] = v4f{0.f, 0.f, 0.f, 0.f};
        if (z < g.slices) {
          if (n + 4 <= g.N) {
            t[u] = *reinterpret_cast<const v4fu *>(p + z * plane);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (n + j < g.N) t[u][j] = p[z * plane + j];
          }
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) v += t[u];
    }
  }
  if (G > 1) {
    red[first][threadIdx.x % Q] = v;
    __syncthreads();
    if (first) return;
#pragma unroll
    for (int k = 1; k < G; ++k) v += red[k][threadIdx.x];
  }
  if (!in) return;
  if (g.terms) lin_repair(g, m, n, v);
  lin_finish4(g.e, m, n, g.N, v);
}
static inline void lin_join(const LinArgs &g, hipStream_t st) {
  const int64_t quads = g.M * ((g.N + 3) / 4);
  if (g.slices > 8 && quads < (1 << 26))
    hipLaunchKernelGGL((k_linear_join<16>), dim3((unsigned)((quads + 15) / 16)), dim3(256), 0, st, g);
  else hipLaunchKernelGGL((k_linear_join<1>), dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, st, g);
}

// ============================================================ few rows
//
// Up to four rows of x: bound by reading w once.  WPR waves share a row of w (one wave a row, or four where there are
// few rows); a lane multiplies 16 bytes of it at a time by the same columns of each row of x, in f32, eight such loads
// in flight before the first product.  x comes from L2 (it is short).
constexpr int LIN_ROWS = 4;
template <class TX, class TW, int S, int WPR>
__global__ __launch_bounds__(256) void k_linear_rows(LinArgs g) {
  constexpr int V = 16 / (int)sizeof(TW), U = 8;
  __shared__ float red[4][S];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t o = WPR == 1 ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x;
  if (WPR == 1 && o >= g.N) return;
  const TW *w = (const TW *)g.b + o * g.ldb;
  const TX *x = (const TX *)g.a;
  float acc[S] = {};
  const int K = (int)g.K, first = ((WPR == 1 ? 0 : wave * 64) + lane) * V, step = 64 * WPR * V;
  typedef v4u v4uu __attribute__((aligned(2)));
  for (int k0 = first; k0 + V <= K; k0 += U * step) {
    v4u rw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * step;
      rw[u] = k + V <= K ? __builtin_nontemporal_load(reinterpret_cast<const v4uu *>(w + k)) : v4u{0, 0, 0, 0};
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * step;
      if (k + V > K) break;
      TW e[V];
      __builtin_memcpy(e, &rw[u], 16);
#pragma unroll
      for (int s = 0; s < S; ++s) {
        TX f[V];
        __builtin_memcpy(f, x + s * g.lda + k, sizeof(f));
#pragma unroll
        for (int j = 0; j < V; ++j) acc[s] = __builtin_fmaf(to_f32(e[j]), to_f32(f[j]), acc[s]);
      }
    }
  }
  // the last, partial pack: a value a lane
  const int last = K / V * V + lane;
  if (last < K && (WPR == 1 || wave == 0))
#pragma unroll
    for (int s = 0; s < S; ++s) acc[s] = __builtin_fmaf(to_f32(w[last]), to_f32(x[s * g.lda + last]), acc[s]);
#pragma unroll
  for (int s = 0; s < S; ++s) acc[s] = group_sum<64>(acc[s]);
  if (WPR > 1) {
    if (!lane)
#pragma unroll
      for (int s = 0; s < S; ++s) red[wave][s] = acc[s];
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int s = 0; s < S; ++s) acc[s] = (red[0][s] + red[1][s]) + (red[2][s] + red[3][s]);
  }
  float z = acc[0];
#pragma unroll
  for (int s = 1; s < S; ++s) z = lane == s ? acc[s] : z;
  if (lane < S) lin_store(g.e.y, g.e.type, (size_t)(lane * g.e.ldy + o), lin_finish1(g.e, lane, o, z));
}

template <class TX, class TW, int S>
void lin_rows_launch(const LinArgs &g, hipStream_t st) {
  // one wave a row from 2048 rows on, else four
  if (g.N >= 2048) hipLaunchKernelGGL((k_linear_rows<TX, TW, S, 1>), dim3((unsigned)((g.N + 3) / 4)), dim3(256), 0, st, g);
  else hipLaunchKernelGGL((k_linear_rows<TX, TW, S, 4>), dim3((unsigned)g.N), dim3(256), 0, st, g);
}
template <class TX, class TW>
void lin_rows_of(const LinArgs &g, hipStream_t st) {
  switch (g.M) {
  case 1: lin_rows_launch<TX, TW, 1>(g, st); break;
  case 2: lin_rows_launch<TX, TW, 2>(g, st); break;
  case 3: lin_rows_launch<TX, TW, 3>(g, st); break;
  default: lin_rows_launch<TX, TW, 4>(g, st); break;
  }
}

// A few dozen rows of x: bound by reading w once, multiplied on the matrix cores.  A workgroup takes 128 NF columns of
// the result, 16 MT rows and a slice of k in units of KS.  Each of its 8 waves reads its rows of w straight from global
// memory into the instruction's operands (a lane's 16 or 32 bytes: no other wave needs them); x's part of a unit goes
// into LDS as terms, once for all waves.  The next unit's loads are in flight while one is multiplied; x's are asked
// for before w's, since loads are waited for in order.
template <class T>
struct Eight {  // 8 consecutive values as they lie in memory
  v4u r[sizeof(T) / 2];
};
template <class T>
__device__ __forceinline__ Eight<T> load8(rsrc_t r, int vo) {
  Eight<T> e;
#pragma unroll
  for (int q = 0; q < (int)sizeof(T) / 2; ++q) e.r[q] = buf16(r, vo, 16 * q);
  return e;
}
template <class T, int NT>
__device__ __forceinline__ void terms_of(const Eight<T> &e, v8bf (&t)[NT]) {
  if constexpr (sizeof(T) == 2 && NT == 1) {
    t[0] = __builtin_bit_cast(v8bf, e.r[0]);
  } else {
    T f[8];
    float v[8];
    __builtin_memcpy(f, &e, sizeof(f));
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_f32(f[j]);
    split_terms<T, NT>(v, t);
  }
}

constexpr int FEW_ROWS = 64;
// where it is the faster one (us, tiles -> this): w of 256 x 7168 f32, 192 rows 25.1 -> 16.6, 384 rows 28.7 -> 22.3,
// 1024 rows 35.5 -> 36.9; w of 4096 x 4096 bf16, 128 rows 23.4 -> 25.3, 192 rows 26.7 -> 37.7; w of 1536 x 4096 bf16
// under f32 rows, 128 rows 27.1 -> 24.5, 256 rows 31.8 -> 31.1
inline bool lin_few_rows(int64_t M, int64_t N) { return M <= 128 || (M <= 384 && N <= 512); }
constexpr int FEW_UNIT = 128;  // a slice is a multiple of it: one unit of a 16-bit w, two of an f32 one
template <class TX, int NX, class TW, int NW, int MT, int NF, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_linear_few(LinArgs g) {
  constexpr bool F16 = std::is_same<TX, _Float16>::value && NX == 1;
  constexpr int KS = sizeof(TW) == 2 ? FEW_UNIT : FEW_UNIT / 2, CH = KS / 8, ROWS = 16 * MT;
  constexpr int THREADS = 64 * WAVES, UX = (ROWS * CH + THREADS - 1) / THREADS, PLANE = ROWS * KS;
  __shared__ __attribute__((aligned(16))) uint16_t lds[2][NX * PLANE];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int fr = lane & 15, fc = lane >> 4;
  const int per = g.tiles_m * g.tiles_n;
  const int z = blockIdx.x / per, tile = blockIdx.x - z * per;
  const int64_t m0 = (int64_t)(tile % g.tiles_m) * ROWS, n0 = (int64_t)(tile / g.tiles_m) * (16 * NF * WAVES);
  const int64_t n1 = n0 + wave * 16 * NF;
  const int64_t kb = z * g.kslice, ke = min(g.K, kb + g.kslice);
  const int rows = (int)min(g.M - m0, (int64_t)ROWS);
  // bytes from the workgroup's first column, and from its first row of x
  const TW *w = (const TW *)g.b + n0 * g.ldb;
  const TX *x = (const TX *)g.a + m0 * g.lda;
  int wo[NF], xo[UX];
#pragma unroll
  for (int j = 0; j < NF; ++j) wo[j] = (int)((min(n1 + 16 * j + fr, g.N - 1) - n0) * g.ldb + 8 * fc) * (int)sizeof(TW);
#pragma unroll
  for (int u = 0; u < UX; ++u) {
    const int q = threadIdx.x + THREADS * u, r = q / CH, c = q % CH;
    xo[u] = r < rows ? (r * (int)g.lda + 8 * c) * (int)sizeof(TX) : OOR;
  }
  v4f acc[MT][NF];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
  struct Unit {
    Eight<TX> x[UX];
    Eight<TW> w[KS / 32][NF];
  };
  auto load = [&](Unit &t, int64_t k) {
    const int left = (int)min(ke - k, (int64_t)KS);
    const rsrc_t rx = buf_at(x + k), rw = buf_at(w + k);
#pragma unroll
    for (int u = 0; u < UX; ++u) t.x[u] = load8<TX>(rx, 8 * ((threadIdx.x + THREADS * u) % CH) < left ? xo[u] : OOR);
#pragma unroll
    for (int h = 0; h < KS / 32; ++h)
#pragma unroll
      for (int j = 0; j < NF; ++j)
        t.w[h][j] = load8<TW>(rw, 32 * h + 8 * fc < left ? wo[j] + 32 * h * (int)sizeof(TW) : OOR);
  };
  // x's terms into `to` (which the waves have left behind a barrier ago), then the unit's products
  auto step = [&](Unit &t, uint16_t *to) {
#pragma unroll
    for (int u = 0; u < UX; ++u) {
      const int q = threadIdx.x + THREADS * u, r = q / CH, c = q % CH;
      if (r >= ROWS) break;
      v8bf e[NX];
      terms_of<TX, NX>(t.x[u], e);
#pragma unroll
      for (int a = 0; a < NX; ++a) *reinterpret_cast<v8bf *>(to + a * PLANE + r * KS + chunk_at<KS>(r, c) * 8) = e[a];
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < KS / 32; ++h) {
      v8bf tw[NF][NW];
#pragma unroll
      for (int j = 0; j < NF; ++j) terms_of<TW, NW>(t.w[h][j], tw[j]);
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int a = 0; a < NX; ++a) {
          const int r = 16 * i + fr;
          const v8bf tx = *reinterpret_cast<const v8bf *>(to + a * PLANE + r * KS + chunk_at<KS>(r, 4 * h + fc) * 8);
#pragma unroll
          for (int b = 0; b < NW; ++b) {
            if (a + b > PAIRS_MOST) continue;
#pragma unroll
            for (int j = 0; j < NF; ++j) {
              if constexpr (F16)
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, tw[j][b]),
                                                                  __builtin_bit_cast(v8h, tx), acc[i][j], 0, 0, 0);
              else
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(tw[j][b], tx, acc[i][j], 0, 0, 0);
            }
          }
        }
    }
  };
  Unit p, q;
  load(p, kb);
  for (int64_t k = kb; k < ke; k += 2 * KS) {
    if (k + KS < ke) load(q, k + KS);
    step(p, lds[0]);
    if (k + KS >= ke) break;
    if (k + 2 * KS < ke) load(p, k + 2 * KS);
    step(q, lds[1]);
  }
  lin_repair_all<(NX * NW > 1), MT, NF>(g, acc, [&](int i, int n) { return n ? n1 + 16 * i + 4 * fc : m0 + 16 * i + fr; });
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) lin_result(g, z, m0 + 16 * i + fr, n1 + 16 * j + 4 * fc, acc[i][j]);
}

// columns of a workgroup (one wave each 16 of them): 64 where w is narrow, so that more of them share its reading, else
// 128; 32 for each wave where the rows are many too
inline int few_columns(int64_t M, int64_t N) { return M <= 32 ? (N < 2048 ? 64 : 128) : (N < 4096 ? 128 : 256); }
template <class TX, int NX, class TW, int NW, int MT>
void lin_few_launch(const LinArgs &g, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)g.tiles_m * g.tiles_n * g.slices));
  switch (few_columns(g.M, g.N)) {
  case 64: hipLaunchKernelGGL((k_linear_few<TX, NX, TW, NW, MT, 1, 4>), grid, dim3(256), 0, st, g); break;
  case 128: hipLaunchKernelGGL((k_linear_few<TX, NX, TW, NW, MT, 1, 8>), grid, dim3(512), 0, st, g); break;
  default: hipLaunchKernelGGL((k_linear_few<TX, NX, TW, NW, MT, 2, 8>), grid, dim3(512), 0, st, g);
  }
}
template <class TX, int NX, class TW, int NW>
void lin_few_of(const LinArgs &g, hipStream_t st) {
  if (g.M <= 16) lin_few_launch<TX, NX, TW, NW, 1>(g, st);
  else if (g.M <= 32) lin_few_launch<TX, NX, TW, NW, 2>(g, st);
  else lin_few_launch<TX, NX, TW, NW, 4>(g, st);
}

// The launch of one kernel instance.  `tile`: 0 = 128 x 128, 1 = 32 x 128, for 16-bit operands with 16-byte loads
// (`vec`) 2 = 256 x 256 and 3 = 256 x 128; for f32 by f32 4 = 160 x 128 (gradient by w) or 128 x 160 (forward)
// and 5 = 128 x 128 with one buffer (forward, gradient by x).
template <class TA, int NA, bool KCA, class TB, int NB, bool KCB>
void lin_launch(const LinArgs &g, bool vec, int tile, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)g.tiles_m * g.tiles_n * g.slices)), b(512);
  if (tile == 1) {
    if (vec) hipLaunchKernelGGL((k_linear<TA, NA, KCA, TB, NB, KCB, 32, 128, 1, 8, true>), grid, b, 0, st, g);
    else hipLaunchKernelGGL((k_linear<TA, NA, KCA, TB, NB, KCB, 32, 128, 1, 8, false>), grid, b, 0, st, g);
  } else if (!vec) {
    hipLaunchKernelGGL((k_linear<TA, NA, KCA, TB, NB, KCB, 128, 128, 2, 4, false>), grid, b, 0, st, g);
  } else if constexpr (std::is_same<TA, TB>::value && sizeof(TA) == 2) {
    constexpr bool F16 = std::is_same<TA, _Float16>::value;
    if (tile == 2) hipLaunchKernelGGL((k_linear_dma<F16, KCA, KCB, 256, 256, 2, 4>), grid, b, 0, st, g);
    else if (tile == 3) hipLaunchKernelGGL((k_linear_dma<F16, KCA, KCB, 256, 128, 4, 2>), grid, b, 0, st, g);
    else hipLaunchKernelGGL((k_linear_dma<F16, KCA, KCB, 128, 128, 2, 4>), grid, b, 0, st, g);
  } else {
    if constexpr (NA * NB == 9 && KCA) {
      if (tile == 5) {
        hipLaunchKernelGGL((k_linear<TA, NA, KCA, TB, NB, KCB, 128, 128, 2, 4, true, 1>), grid, b, 0, st, g);
        return;
      }
    }
    if constexpr (NA * NB == 9 && KCA == KCB) {
      if (tile == 4) {
        constexpr int BM = KCA ? 128 : 160, BN = KCA ? 160 : 128, WM = KCA ? 4 : 2;
        hipLaunchKernelGGL((k_linear<TA, NA, KCA, TB, NB, KCB, BM, BN, WM, 8 / WM, true>), grid, b, 0, st, g);
        return;
      }
    }
    hipLaunchKernelGGL((k_linear<TA, NA, KCA, TB, NB, KCB, 128, 128, 2, 4, true>), grid, b, 0, st, g);
  }
}

// the products by what their operands are: forward (x, w), dx (dz, w), dw (dz, x)
void lin_rows(int x_type, int w_type, const LinArgs &g, hipStream_t st);  // M <= LIN_ROWS, any alignment
void lin_few(int x_type, int w_type, const LinArgs &g, hipStream_t st);   // where lin_few_rows(), by 16-byte loads
void lin_fwd(int x_type, int w_type, const LinArgs &g, bool vec, int tile, hipStream_t st);
void lin_dx(int x_type, int w_type, int dz_type, const LinArgs &g, bool vec, int tile, hipStream_t st);
void lin_dw(int x_type, int dz_type, const LinArgs &g, bool vec, int tile, hipStream_t st);

}  // namespace zm
