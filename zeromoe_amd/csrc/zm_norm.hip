// zm_norm.hip -- layer norm over the rows of a matrix, forward and backward, with the reduction of the gradients of
// its weight and bias.
//
//   mean_r = sum_i x_ri / n,  rstd_r = 1 / sqrt(sum_i (x_ri - mean_r)^2 / n + eps)
//   h = (x - mean) rstd,  y = h weight + bias
//   g = dy weight,  dx = rstd (g - sum_i g_i / n - h sum_i (g_i h_i) / n)
//   dweight_i = sum_r dy_ri h_ri,  dbias_i = sum_r dy_ri
//
// Bound by memory: x in and y out; x and dy in and dx out.  A row sits in the registers of one workgroup (or one
// wave), so it is read once; the variance is taken around the mean, not from the sum of squares, so a mean far from
// zero costs no digits.  All sums are f32.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/zeromoe.h"
#include "zm_host.hpp"
#include "zm_linear.hpp"

using namespace zm;

namespace {

struct NormArgs {
  const void *x, *dy;
  const float *weight, *bias;  // or null: 1, 0
  void *y;                     // or dx
  float *mean, *rstd;          // [rows]; optional in the forward pass
  float *part;                 // backward: [gridDim.x][2][n], or null
  int64_t rows, ldx, ldg, ldy; // ldg: rows of dy
  int n;
  float eps;
};

// sum over the TPR threads of a row (64 or 256); every one of them gets it
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float *red) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  if (TPR > 64) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();  // the last sum has been read
    if (!(threadIdx.x & 63)) red[wave] = v;
    __syncthreads();
    v = (red[0] + red[1]) + (red[2] + red[3]);
  }
  return v;
}

// 16 bytes of T as floats
template <class T>
struct Pack {
  static constexpr int V = 16 / (int)sizeof(T);
};
template <class T>
__device__ __forceinline__ void unpack(v4u r, float (&v)[Pack<T>::V]) {
  T e[Pack<T>::V];
  __builtin_memcpy(e, &r, 16);
#pragma unroll
  for (int i = 0; i < Pack<T>::V; ++i) v[i] = to_f32(e[i]);
}
template <class T>
__device__ __forceinline__ v4u pack(const float (&v)[Pack<T>::V]) {
  T e[Pack<T>::V];
#pragma unroll
  for (int i = 0; i < Pack<T>::V; ++i) e[i] = from_f32<T>(v[i]);
  v4u r;
  __builtin_memcpy(&r, e, 16);
  return r;
}
__device__ __forceinline__ void load_vec(const float *p, int i, bool on, int V, float other, float *v) {
  for (int j = 0; j < V; j += 4) {
    const v4f f = p && on ? *reinterpret_cast<const v4f *>(p + i + j) : v4f{other, other, other, other};
    v[j] = f.x, v[j + 1] = f.y, v[j + 2] = f.z, v[j + 3] = f.w;
  }
}

// TPR threads keep one row in C packs of 16 bytes each; 256 / TPR rows per workgroup.
template <class T, int TPR, int C>
__global__ __launch_bounds__(256) void k_norm(NormArgs g) {
  constexpr int V = Pack<T>::V;
  __shared__ float red[4];
  const int t = threadIdx.x & (TPR - 1);
  const int64_t row = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  if (TPR == 64 && row >= g.rows) return;
  const T *x = (const T *)g.x + row * g.ldx;
  float v[C][V];
  float sum = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = (t + TPR * c) * V;
    unpack<T>(i < g.n ? *reinterpret_cast<const v4u *>(x + i) : v4u{0, 0, 0, 0}, v[c]);
  }
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int j = 0; j < V; ++j) sum += v[c][j];
  const float mean = row_sum<TPR>(sum, red) / (float)g.n;
  float sq = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const bool in = (t + TPR * c) * V < g.n;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      v[c][j] = in ? v[c][j] - mean : 0.f;
      sq += v[c][j] * v[c][j];
    }
  }
  const float rstd = 1.0f / sqrtf(row_sum<TPR>(sq, red) / (float)g.n + g.eps);
  T *y = (T *)g.y + row * g.ldy;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = (t + TPR * c) * V;
    if (i >= g.n) continue;
    float w[V], b[V];
    load_vec(g.weight, i, true, V, 1.0f, w);
    load_vec(g.bias, i, true, V, 0.0f, b);
#pragma unroll
    for (int j = 0; j < V; ++j) v[c][j] = v[c][j] * rstd * w[j] + b[j];
    *reinterpret_cast<v4u *>(y + i) = pack<T>(v[c]);
  }
  if (!t) {
    if (g.mean) g.mean[row] = mean;
    if (g.rstd) g.rstd[row] = rstd;
  }
}

// Any width and alignment: a row is read three times (the later ones from L2).
template <class T>
__global__ __launch_bounds__(256) void k_norm_any(NormArgs g) {
  __shared__ float red[4];
  const int64_t row = blockIdx.x;
  const T *x = (const T *)g.x + row * g.ldx;
  float sum = 0.f;
  for (int i = threadIdx.x; i < g.n; i += 256) sum += to_f32(x[i]);
  const float mean = row_sum<256>(sum, red) / (float)g.n;
  float sq = 0.f;
  for (int i = threadIdx.x; i < g.n; i += 256) {
    const float d = to_f32(x[i]) - mean;
    sq += d * d;
  }
  const float rstd = 1.0f / sqrtf(row_sum<256>(sq, red) / (float)g.n + g.eps);
  T *y = (T *)g.y + row * g.ldy;
  for (int i = threadIdx.x; i < g.n; i += 256) {
    const float h = (to_f32(x[i]) - mean) * rstd;
    y[i] = from_f32<T>(h * (g.weight ? g.weight[i] : 1.0f) + (g.bias ? g.bias[i] : 0.0f));
  }
  if (!threadIdx.x) {
    if (g.mean) g.mean[row] = mean;
    if (g.rstd) g.rstd[row] = rstd;
  }
}

// Workgroup b takes rows b, b + gridDim.x, ...: each thread keeps the same columns throughout, so the sums over the
// rows stay in its registers until the end.
template <class T, int C>
__global__ __launch_bounds__(256) void k_norm_backward(NormArgs g) {
  constexpr int V = Pack<T>::V;
  __shared__ float red[4];
  const int t = threadIdx.x;
  float dw[C][V], db[C][V];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int j = 0; j < V; ++j) dw[c][j] = db[c][j] = 0.f;
  for (int64_t row = blockIdx.x; row < g.rows; row += gridDim.x) {
    const T *x = (const T *)g.x + row * g.ldx, *dy = (const T *)g.dy + row * g.ldg;
    const float mean = g.mean[row], rstd = g.rstd[row];
    v4u rx[C], rg[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int i = (t + 256 * c) * V;
      rx[c] = i < g.n ? *reinterpret_cast<const v4u *>(x + i) : v4u{0, 0, 0, 0};
      rg[c] = i < g.n ? *reinterpret_cast<const v4u *>(dy + i) : v4u{0, 0, 0, 0};
    }
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int i = (t + 256 * c) * V;
      float xv[V], gv[V], w[V];
      unpack<T>(rx[c], xv);
      unpack<T>(rg[c], gv);
      load_vec(g.weight, i, i < g.n, V, 1.0f, w);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float h = (xv[j] - mean) * rstd;  // past n: dy is 0, so nothing is added
        dw[c][j] += gv[j] * h;
        db[c][j] += gv[j];
        s1 += gv[j] * w[j];
        s2 += gv[j] * w[j] * h;
      }
    }
    s1 = row_sum<256>(s1, red) / (float)g.n;
    s2 = row_sum<256>(s2, red) / (float)g.n;
    if (g.y) {
      T *dx = (T *)g.y + row * g.ldy;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int i = (t + 256 * c) * V;
        if (i >= g.n) continue;
        float xv[V], gv[V], w[V];
        unpack<T>(rx[c], xv);
        unpack<T>(rg[c], gv);
        load_vec(g.weight, i, true, V, 1.0f, w);
#pragma unroll
        for (int j = 0; j < V; ++j) xv[j] = rstd * (gv[j] * w[j] - s1 - (xv[j] - mean) * rstd * s2);
        *reinterpret_cast<v4u *>(dx + i) = pack<T>(xv);
      }
    }
  }
  if (!g.part) return;
  float *pw = g.part + (size_t)blockIdx.x * 2 * g.n, *pb = pw + g.n;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = (t + 256 * c) * V;
    if (i >= g.n) continue;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      pw[i + j] = dw[c][j];
      pb[i + j] = db[c][j];
    }
  }
}

// Any width and alignment; the sums over the rows are kept in the workgroup's part of the workspace, which thread t
// alone touches at columns t, t + 256, ...
template <class T>
__global__ __launch_bounds__(256) void k_norm_backward_any(NormArgs g) {
  __shared__ float red[4];
  float *pw = g.part ? g.part + (size_t)blockIdx.x * 2 * g.n : nullptr, *pb = pw + g.n;
  if (pw)
    for (int i = threadIdx.x; i < g.n; i += 256) pw[i] = pb[i] = 0.f;
  for (int64_t row = blockIdx.x; row < g.rows; row += gridDim.x) {
    const T *x = (const T *)g.x + row * g.ldx, *dy = (const T *)g.dy + row * g.ldg;
    const float mean = g.mean[row], rstd = g.rstd[row];
    float s1 = 0.f, s2 = 0.f;
    for (int i = threadIdx.x; i < g.n; i += 256) {
      const float h = (to_f32(x[i]) - mean) * rstd, d = to_f32(dy[i]), w = d * (g.weight ? g.weight[i] : 1.0f);
      if (pw) {
        pw[i] += d * h;
        pb[i] += d;
      }
      s1 += w;
      s2 += w * h;
    }
    s1 = row_sum<256>(s1, red) / (float)g.n;
    s2 = row_sum<256>(s2, red) / (float)g.n;
    if (g.y) {
      T *dx = (T *)g.y + row * g.ldy;
      for (int i = threadIdx.x; i < g.n; i += 256) {
        const float h = (to_f32(x[i]) - mean) * rstd;
        dx[i] = from_f32<T>(rstd * (to_f32(dy[i]) * (g.weight ? g.weight[i] : 1.0f) - s1 - h * s2));
      }
    }
  }
}

// dweight and dbias: the workgroups' sums added in order
__global__ __launch_bounds__(256) void k_norm_sum(const float *__restrict__ part, int parts, int n,
                                                  float *__restrict__ dweight, float *__restrict__ dbias) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= 2 * n) return;
  float v = 0.f;
  for (int p = 0; p < parts; ++p) v += part[(size_t)p * 2 * n + i];
  float *dst = i < n ? dweight : dbias;
  if (dst) dst[i < n ? i : i - n] = v;
}

// rows' worth of workgroups of the backward pass: two per CU
int norm_parts(int64_t rows) { return (int)std::min<int64_t>(rows, 512); }

bool aligned(const void *p, int64_t ld, size_t e) { return !p || (!((uintptr_t)p & 15) && !((size_t)ld * e & 15)); }

int check(const char *who, int type, int64_t rows, int64_t n) {
  if (type != LIN_F32 && type != LIN_F16 && type != LIN_BF16) return fail("%s: types are F32, F16 and BF16", who);
  if (rows < 0 || rows >= (1 << 24)) return fail("%s: rows out of range", who);
  if (n <= 0 || n > (1 << 24)) return fail("%s: n is 1 to 2^24", who);
  return 0;
}

template <class T>
void norm(const NormArgs &g, bool vec, hipStream_t st) {
  constexpr int V = Pack<T>::V;
  const unsigned rows = (unsigned)g.rows, quads = (unsigned)((g.rows + 3) / 4);
  const int packs = (g.n + V - 1) / V;
  const dim3 b(256);
  if (!vec || packs > 8 * 256) hipLaunchKernelGGL((k_norm_any<T>), dim3(rows), b, 0, st, g);
  else if (packs <= 64) hipLaunchKernelGGL((k_norm<T, 64, 1>), dim3(quads), b, 0, st, g);
  else if (packs <= 128) hipLaunchKernelGGL((k_norm<T, 64, 2>), dim3(quads), b, 0, st, g);
  else if (packs <= 256) hipLaunchKernelGGL((k_norm<T, 256, 1>), dim3(rows), b, 0, st, g);
  else if (packs <= 512) hipLaunchKernelGGL((k_norm<T, 256, 2>), dim3(rows), b, 0, st, g);
  else if (packs <= 1024) hipLaunchKernelGGL((k_norm<T, 256, 4>), dim3(rows), b, 0, st, g);
  else hipLaunchKernelGGL((k_norm<T, 256, 8>), dim3(rows), b, 0, st, g);
}

template <class T>
void norm_backward(const NormArgs &g, bool vec, unsigned parts, hipStream_t st) {
  constexpr int V = Pack<T>::V;
  const int packs = (g.n + V - 1) / V;
  const dim3 b(256);
  if (!vec || packs > 4 * 256) hipLaunchKernelGGL((k_norm_backward_any<T>), dim3(parts), b, 0, st, g);
  else if (packs <= 256) hipLaunchKernelGGL((k_norm_backward<T, 1>), dim3(parts), b, 0, st, g);
  else if (packs <= 512) hipLaunchKernelGGL((k_norm_backward<T, 2>), dim3(parts), b, 0, st, g);
  else hipLaunchKernelGGL((k_norm_backward<T, 4>), dim3(parts), b, 0, st, g);
}

__global__ __launch_bounds__(256) void k_norm_zero(float *dweight, float *dbias, int n) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  if (dweight) dweight[i] = 0.f;
  if (dbias) dbias[i] = 0.f;
}

}  // namespace

extern "C" {

int zm_layer_norm(int type, const void *x, int64_t x_stride, const float *weight, const float *bias, float eps,
                  int64_t rows, int64_t n, void *y, int64_t y_stride, float *mean, float *rstd, void *stream) {
  if (check("zm_layer_norm", type, rows, n)) return -1;
  if (!rows) return 0;
  if (!x || !y) return fail("zm_layer_norm: null pointer");
  if (x_stride < 0 || (rows > 1 && y_stride < n)) return fail("zm_layer_norm: bad stride");
  if (!(eps >= 0.f)) return fail("zm_layer_norm: eps is not negative");
  NormArgs g{};
  g.x = x;
  g.y = y;
  g.weight = weight;
  g.bias = bias;
  g.mean = mean;
  g.rstd = rstd;
  g.rows = rows;
  g.n = (int)n;
  g.eps = eps;
  g.ldx = x_stride;
  g.ldy = y_stride;
  const size_t e = type == LIN_F32 ? 4 : 2;
  const bool vec = !(n * e & 15) && aligned(x, x_stride, e) && aligned(y, y_stride, e) && aligned(weight, 0, 4) &&
                   aligned(bias, 0, 4);
  if (type == LIN_F32) norm<float>(g, vec, (hipStream_t)stream);
  else if (type == LIN_F16) norm<_Float16>(g, vec, (hipStream_t)stream);
  else norm<bf16>(g, vec, (hipStream_t)stream);
  HIP_OK(hipGetLastError());
  return 0;
}

size_t zm_layer_norm_backward_workspace_size(int64_t rows, int64_t n) {
  return rows <= 0 || n <= 0 ? 0 : (size_t)norm_parts(rows) * 2 * (size_t)n * 4;
}

int zm_layer_norm_backward(int type, const void *dy, int64_t dy_stride, const void *x, int64_t x_stride,
                           const float *weight, const float *mean, const float *rstd, int64_t rows, int64_t n, void *dx,
                           int64_t dx_stride, float *dweight, float *dbias, void *workspace, size_t workspace_size,
                           void *stream) {
  if (check("zm_layer_norm_backward", type, rows, n)) return -1;
  const hipStream_t st = (hipStream_t)stream;
  if (!rows) {  // no rows: the sums over them are zero
    if (dweight || dbias)
      hipLaunchKernelGGL(k_norm_zero, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, dweight, dbias, (int)n);
    HIP_OK(hipGetLastError());
    return 0;
  }
  if (!dy || !x || !mean || !rstd) return fail("zm_layer_norm_backward: null pointer");
  if (x_stride < 0 || dy_stride < 0 || (dx && rows > 1 && dx_stride < n)) return fail("zm_layer_norm_backward: bad stride");
  const bool sums = dweight || dbias;
  if (sums && (!workspace || ((uintptr_t)workspace & 15) || workspace_size < zm_layer_norm_backward_workspace_size(rows, n)))
    return fail("zm_layer_norm_backward: a 16-byte aligned workspace of zm_layer_norm_backward_workspace_size() bytes is needed");
  if (!dx && !sums) return 0;
  NormArgs g{};
  g.x = x;
  g.dy = dy;
  g.y = dx;
  g.weight = weight;
  g.mean = const_cast<float *>(mean);
  g.rstd = const_cast<float *>(rstd);
  g.part = sums ? (float *)workspace : nullptr;
  g.rows = rows;
  g.n = (int)n;
  g.ldx = x_stride;
  g.ldg = dy_stride;
  g.ldy = dx_stride;
  const size_t e = type == LIN_F32 ? 4 : 2;
  const bool vec = !(n * e & 15) && aligned(x, x_stride, e) && aligned(dy, dy_stride, e) && aligned(dx, dx_stride, e) &&
                   aligned(weight, 0, 4);
  const unsigned parts = (unsigned)norm_parts(rows);
  if (type == LIN_F32) norm_backward<float>(g, vec, parts, st);
  else if (type == LIN_F16) norm_backward<_Float16>(g, vec, parts, st);
  else norm_backward<bf16>(g, vec, parts, st);
  if (sums)
    hipLaunchKernelGGL(k_norm_sum, dim3((unsigned)((2 * n + 255) / 256)), dim3(256), 0, st, (const float *)workspace,
                       (int)parts, (int)n, dweight, dbias);
  HIP_OK(hipGetLastError());
  return 0;
}

}  // extern "C"
