// zm_norm.hip -- layer norm over the rows of a matrix, forward and backward, with the reduction of the gradients of
// its weight and bias.
//
//   mean_r = sum_i x_ri / n,  rstd_r = 1 / sqrt(sum_i (x_ri - mean_r)^2 / n + eps)
//   h = (x - mean) rstd,  y = h weight + bias
//   g = dy weight,  dx = rstd (g - sum_i g_i / n - h sum_i (g_i h_i) / n)
//   dweight_i = sum_r dy_ri h_ri,  dbias_i = sum_r dy_ri
//
// Bound by memory: x in and y out; x and dy in and dx out.  A row sits in the registers of one workgroup (or one
// wave), so it is read once.  All sums are f32.  The sum's rounding leaves a first mean off by some 2^-24 of the values'
// size, which is many standard deviations where a row's mean is far larger than its spread; so the differences from
// it are summed too (next to their squares): their mean corrects the differences and the variance.  What is left of the
// error is 2^-24 of the differences.  The saved mean is rounded to f32 once.
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

// sums over the TPR threads of a row (64 and more); every one of them gets them.  `red`: one entry for each wave of
// the workgroup, not in use by another sum; all threads of the workgroup call together where TPR > 64.
template <int TPR, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*red)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = group_sum<64>(v[k]);
  if (TPR > 64) {
    const int wave = threadIdx.x >> 6, first = wave / (TPR / 64) * (TPR / 64);
    if (!(threadIdx.x & 63))
#pragma unroll
      for (int k = 0; k < N; ++k) red[wave][k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
      v[k] = red[first][k];
#pragma unroll
      for (int w = 1; w < TPR / 64; ++w) v[k] += red[first + w][k];
    }
  }
}
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float (*red)[1]) {
  float a[1] = {v};
  row_sums<TPR, 1>(a, red);
  return a[0];
}
// d[0] = sum of d and d[1] = sum of d^2 over a row, d the differences from a first mean: what is to be taken off them,
// and 1 / sqrt(variance + eps)
__device__ __forceinline__ void row_stats(const float (&d)[2], float n, float eps, float &delta, float &rstd) {
  delta = d[0] / n;
  const float var = d[1] / n - delta * delta;
  rstd = 1.0f / sqrtf((var < 0.f ? 0.f : var) + eps);  // (a NaN stays one)
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
// V values from i on of a row of n (zeros past it); ALIGNED: n and the addresses allow whole packs, else memory takes
// whole packs where they lie and the last one goes value by value
template <class T, bool ALIGNED>
__device__ __forceinline__ v4u load_pack(const T *p, int i, int n) {
  constexpr int V = Pack<T>::V;
  if (ALIGNED) return i < n ? *reinterpret_cast<const v4u *>(p + i) : v4u{0, 0, 0, 0};
  v4u r = {0, 0, 0, 0};
  if (i + V <= n) {
    __builtin_memcpy(&r, p + i, 16);
  } else if (i < n) {
    T e[V];
#pragma unroll
    for (int j = 0; j < V; ++j) e[j] = i + j < n ? p[i + j] : from_f32<T>(0.f);
    __builtin_memcpy(&r, e, 16);
  }
  return r;
}
template <class T, bool ALIGNED>
__device__ __forceinline__ void store_pack(T *p, int i, int n, const float (&v)[Pack<T>::V]) {
  constexpr int V = Pack<T>::V;
  const v4u r = pack<T>(v);
  if (ALIGNED) {
    if (i < n) __builtin_nontemporal_store(r, reinterpret_cast<v4u *>(p + i));
  } else if (i + V <= n) {
    __builtin_memcpy(p + i, &r, 16);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (i + j < n) p[i + j] = from_f32<T>(v[j]);
  }
}
// V floats of a vector of n, `other` where it is null or past its end
template <int V, bool ALIGNED>
__device__ __forceinline__ void load_vec(const float *p, int i, int n, float other, float (&v)[V]) {
#pragma unroll
  for (int j = 0; j < V; j += 4) {
    if (ALIGNED) {
      const v4f f = p && i < n ? *reinterpret_cast<const v4f *>(p + i + j) : v4f{other, other, other, other};
      v[j] = f.x, v[j + 1] = f.y, v[j + 2] = f.z, v[j + 3] = f.w;
    } else {
#pragma unroll
      for (int q = j; q < j + 4; ++q) v[q] = p && i + q < n ? p[i + q] : other;
    }
  }
}

// Workgroups of NT threads go over the rows; TPR = 64 or NT threads keep one row in C packs of 16 bytes each.  Weight
// and bias stay in registers (from L2 they are 8 bytes a value next to 4 of a 16-bit row), and the next row's loads are
// in flight while this one's sums are taken.  Buffers of the sums alternate, so that one barrier a sum is enough.
template <class T, int NT, int TPR, int C, bool ALIGNED>
__global__ __launch_bounds__(NT) void k_norm(NormArgs g) {
  constexpr int V = Pack<T>::V, RPB = NT / TPR;
  __shared__ float red[2][NT / 64][1], red2[2][NT / 64][2];
  const int t = threadIdx.x & (TPR - 1);
  float w[C][V], b[C][V];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = (t + TPR * c) * V;
    load_vec<V, ALIGNED>(g.weight, i, g.n, 1.0f, w[c]);
    load_vec<V, ALIGNED>(g.bias, i, g.n, 0.0f, b[c]);
  }
  const float n = (float)g.n;
  v4u next[C];
  int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
  const int64_t step = (int64_t)gridDim.x * RPB;
  auto fetch = [&](int64_t r) {
    const T *x = (const T *)g.x + r * g.ldx;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int i = (t + TPR * c) * V;
      next[c] = r < g.rows ? load_pack<T, ALIGNED>(x, i, g.n) : v4u{0, 0, 0, 0};
    }
  };
  fetch(row);
  // (with one row per workgroup all threads leave the loop together)
  for (int par = 0; row < g.rows; row += step, par ^= 1) {
    float v[C][V];
#pragma unroll
    for (int c = 0; c < C; ++c) unpack<T>(next[c], v[c]);
    fetch(row + step);
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j) sum += v[c][j];
    const float mean = row_sum<TPR>(sum, red[par]) / n;
    float d[2] = {0.f, 0.f}, delta, rstd;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int i = (t + TPR * c) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[c][j] = (ALIGNED ? i : i + j) < g.n ? v[c][j] - mean : 0.f;
        d[0] += v[c][j];
        d[1] = __builtin_fmaf(v[c][j], v[c][j], d[1]);
      }
    }
    row_sums<TPR, 2>(d, red2[par]);
    row_stats(d, n, g.eps, delta, rstd);
    T *y = (T *)g.y + row * g.ldy;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int i = (t + TPR * c) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) v[c][j] = __builtin_fmaf((v[c][j] - delta) * rstd, w[c][j], b[c][j]);
      store_pack<T, ALIGNED>(y, i, g.n, v[c]);
    }
    if (!t) {
      if (g.mean) g.mean[row] = mean + delta;
      if (g.rstd) g.rstd[row] = rstd;
    }
  }
}

// Rows too long for registers: read three times (the later ones from L2).
template <class T>
__global__ __launch_bounds__(256) void k_norm_any(NormArgs g) {
  __shared__ float red[4][1], red2[4][2];
  const int64_t row = blockIdx.x;
  const T *x = (const T *)g.x + row * g.ldx;
  float sum = 0.f;
  for (int i = threadIdx.x; i < g.n; i += 256) sum += to_f32(x[i]);
  const float mean = row_sum<256>(sum, red) / (float)g.n;
  float s[2] = {0.f, 0.f}, delta, rstd;
  for (int i = threadIdx.x; i < g.n; i += 256) {
    const float d = to_f32(x[i]) - mean;
    s[0] += d;
    s[1] += d * d;
  }
  row_sums<256, 2>(s, red2);
  row_stats(s, (float)g.n, g.eps, delta, rstd);
  T *y = (T *)g.y + row * g.ldy;
  for (int i = threadIdx.x; i < g.n; i += 256) {
    const float h = (to_f32(x[i]) - mean - delta) * rstd;
    y[i] = from_f32<T>(h * (g.weight ? g.weight[i] : 1.0f) + (g.bias ? g.bias[i] : 0.0f));
  }
  if (!threadIdx.x) {
    if (g.mean) g.mean[row] = mean + delta;
    if (g.rstd) g.rstd[row] = rstd;
  }
}

// NT threads, TPR of them for a row: a workgroup goes over rows b * NT / TPR + ..., and each thread keeps the same
// columns throughout, so the sums over the rows stay in its registers until the end, and the weight too.  The next
// rows' loads are in flight while this one's sums are taken.
template <class T, int NT, int TPR, int C, bool ALIGNED>
__global__ __launch_bounds__(NT) void k_norm_backward(NormArgs g) {
  constexpr int V = Pack<T>::V, RPB = NT / TPR;
  __shared__ float red[2][NT / 64][2];
  __shared__ __attribute__((aligned(16))) float meet[RPB > 1 ? 2 * TPR * C * V : 4];
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
  float dw[C][V], db[C][V], w[C][V];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = (t + TPR * c) * V;
    load_vec<V, ALIGNED>(g.weight, i, g.n, 1.0f, w[c]);
#pragma unroll
    for (int j = 0; j < V; ++j) dw[c][j] = db[c][j] = 0.f;
  }
  v4u nx[C], ng[C];
  float nm, nr;
  auto fetch = [&](int64_t r) {
    const T *x = (const T *)g.x + r * g.ldx, *dy = (const T *)g.dy + r * g.ldg;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int i = (t + TPR * c) * V;
      nx[c] = r < g.rows ? load_pack<T, ALIGNED>(x, i, g.n) : v4u{0, 0, 0, 0};
      ng[c] = r < g.rows ? load_pack<T, ALIGNED>(dy, i, g.n) : v4u{0, 0, 0, 0};
    }
    nm = r < g.rows ? g.mean[r] : 0.f;
    nr = r < g.rows ? g.rstd[r] : 0.f;
  };
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t first = (int64_t)blockIdx.x * RPB;
  fetch(first + group);
  int par = 0;
  for (; first < g.rows; first += step, par ^= 1) {  // the same for the whole workgroup: a row past the end adds zeros
    const int64_t row = first + group;
    const float mean = nm, rstd = nr;
    v4u rx[C], rg[C];
#pragma unroll
    for (int c = 0; c < C; ++c) rx[c] = nx[c], rg[c] = ng[c];
    fetch(row + step);
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float xv[V], gv[V];
      unpack<T>(rx[c], xv);
      unpack<T>(rg[c], gv);
      const int i = (t + TPR * c) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        // past n dy is 0, and h too: mean rstd may be past f32's largest where the row's own h are not
        const float h = (xv[j] - mean) * ((ALIGNED ? i : i + j) < g.n ? rstd : 0.f);
        const float gw = gv[j] * w[c][j];
        dw[c][j] = __builtin_fmaf(gv[j], h, dw[c][j]);
        db[c][j] += gv[j];
        s[0] += gw;
        s[1] = __builtin_fmaf(gw, h, s[1]);
      }
    }
    row_sums<TPR, 2>(s, red[par]);
    if (!g.y || row >= g.rows) continue;
    const float s1 = s[0] / (float)g.n, rs2 = s[1] / (float)g.n * rstd;
    T *dx = (T *)g.y + row * g.ldy;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int i = (t + TPR * c) * V;
      float xv[V], gv[V];
      unpack<T>(rx[c], xv);
      unpack<T>(rg[c], gv);
#pragma unroll
      for (int j = 0; j < V; ++j) xv[j] = rstd * __builtin_fmaf(mean - xv[j], rs2, __builtin_fmaf(gv[j], w[c][j], -s1));
      store_pack<T, ALIGNED>(dx, i, g.n, xv);
    }
  }
  if (!g.part) return;
  if (RPB > 1) {  // the groups' sums, one group after the other
    for (int q = 0; q < RPB; ++q) {
      if (group == q) {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            float *m = meet + (c * V + j) * TPR + t;
            m[0] = q ? m[0] + dw[c][j] : dw[c][j];
            m[TPR * C * V] = q ? m[TPR * C * V] + db[c][j] : db[c][j];
          }
      }
      __syncthreads();
    }
    if (group) return;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        dw[c][j] = meet[(c * V + j) * TPR + t];
        db[c][j] = meet[(C * V + c * V + j) * TPR + t];
      }
  }
  float *pw = g.part + (size_t)blockIdx.x * 2 * g.n, *pb = pw + g.n;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = (t + TPR * c) * V;
    if (i >= g.n) continue;
    if (ALIGNED) {
#pragma unroll
      for (int j = 0; j < V; j += 4) {
        *reinterpret_cast<v4f *>(pw + i + j) = v4f{dw[c][j], dw[c][j + 1], dw[c][j + 2], dw[c][j + 3]};
        *reinterpret_cast<v4f *>(pb + i + j) = v4f{db[c][j], db[c][j + 1], db[c][j + 2], db[c][j + 3]};
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (i + j < g.n) {
          pw[i + j] = dw[c][j];
          pb[i + j] = db[c][j];
        }
    }
  }
}

// Rows too long for registers; the sums over the rows are kept in the workgroup's part of the workspace, which thread t
// alone touches at columns t, t + 256, ...
template <class T>
__global__ __launch_bounds__(256) void k_norm_backward_any(NormArgs g) {
  __shared__ float red[2][4][2];
  int par = 0;
  float *pw = g.part ? g.part + (size_t)blockIdx.x * 2 * g.n : nullptr, *pb = pw + g.n;
  if (pw)
    for (int i = threadIdx.x; i < g.n; i += 256) pw[i] = pb[i] = 0.f;
  for (int64_t row = blockIdx.x; row < g.rows; row += gridDim.x, par ^= 1) {
    const T *x = (const T *)g.x + row * g.ldx, *dy = (const T *)g.dy + row * g.ldg;
    const float mean = g.mean[row], rstd = g.rstd[row];
    float s[2] = {0.f, 0.f};
    for (int i = threadIdx.x; i < g.n; i += 256) {
      const float h = (to_f32(x[i]) - mean) * rstd, d = to_f32(dy[i]), w = d * (g.weight ? g.weight[i] : 1.0f);
      if (pw) {
        pw[i] += d * h;
        pb[i] += d;
      }
      s[0] += w;
      s[1] += w * h;
    }
    row_sums<256, 2>(s, red[par]);
    const float s1 = s[0] / (float)g.n, s2 = s[1] / (float)g.n;
    if (g.y) {
      T *dx = (T *)g.y + row * g.ldy;
      for (int i = threadIdx.x; i < g.n; i += 256) {
        const float h = (to_f32(x[i]) - mean) * rstd;
        dx[i] = from_f32<T>(rstd * (to_f32(dy[i]) * (g.weight ? g.weight[i] : 1.0f) - s1 - h * s2));
      }
    }
  }
}

// Workgroups of the backward pass: every one leaves a row of sums behind (8 n bytes written and read again), so not
// more than two a CU, and as few as go over the rows in as many rounds.
constexpr int NORM_PARTS = 512;
int norm_parts(int64_t rows) {
  const int64_t rounds = (rows + NORM_PARTS - 1) / NORM_PARTS;
  return (int)((rows + rounds - 1) / rounds);
}

bool aligned(const void *p, int64_t ld, size_t e) { return !p || (!((uintptr_t)p & 15) && !((size_t)ld * e & 15)); }

int check(const char *who, int type, int64_t rows, int64_t n) {
  if (type != LIN_F32 && type != LIN_F16 && type != LIN_BF16) return fail("%s: types are F32, F16 and BF16", who);
  if (rows < 0 || rows >= (1 << 24)) return fail("%s: rows out of range", who);
  if (n <= 0 || n > (1 << 24)) return fail("%s: n is 1 to 2^24", who);
  return 0;
}

template <class T, bool ALIGNED>
void norm_rows(const NormArgs &g, int packs, hipStream_t st) {
  const int64_t quads = (g.rows + 3) / 4;
  // as many workgroups as fit the chip at once (`most`), or as few as take as many rounds
  auto grid = [](int64_t n, int64_t most) {
    const int64_t rounds = (n + most - 1) / most;
    return dim3((unsigned)((n + rounds - 1) / rounds));
  };
  if (packs <= 64) hipLaunchKernelGGL((k_norm<T, 256, 64, 1, ALIGNED>), grid(quads, 2048), dim3(256), 0, st, g);
  else if (packs <= 128) hipLaunchKernelGGL((k_norm<T, 256, 64, 2, ALIGNED>), grid(quads, 1536), dim3(256), 0, st, g);
  else if (packs <= 256) hipLaunchKernelGGL((k_norm<T, 256, 256, 1, ALIGNED>), grid(g.rows, 2048), dim3(256), 0, st, g);
  else if (packs <= 512) hipLaunchKernelGGL((k_norm<T, 512, 512, 1, ALIGNED>), grid(g.rows, 1024), dim3(512), 0, st, g);
  else if (packs <= 1024) hipLaunchKernelGGL((k_norm<T, 512, 512, 2, ALIGNED>), grid(g.rows, 1024), dim3(512), 0, st, g);
  else hipLaunchKernelGGL((k_norm<T, 512, 512, 4, ALIGNED>), grid(g.rows, 512), dim3(512), 0, st, g);
}
template <class T>
void norm(const NormArgs &g, bool vec, hipStream_t st) {
  const int packs = (g.n + Pack<T>::V - 1) / Pack<T>::V;
  if (packs > 4 * 512) hipLaunchKernelGGL((k_norm_any<T>), dim3((unsigned)g.rows), dim3(256), 0, st, g);
  else if (vec) norm_rows<T, true>(g, packs, st);
  else norm_rows<T, false>(g, packs, st);
}

template <class T, bool ALIGNED>
void norm_backward_rows(const NormArgs &g, int packs, unsigned parts, hipStream_t st) {
  const dim3 grid(parts), b(512);
  if (packs <= 64) hipLaunchKernelGGL((k_norm_backward<T, 512, 64, 1, ALIGNED>), grid, b, 0, st, g);
  else if (packs <= 128) hipLaunchKernelGGL((k_norm_backward<T, 512, 128, 1, ALIGNED>), grid, b, 0, st, g);
  else if (packs <= 256) hipLaunchKernelGGL((k_norm_backward<T, 512, 256, 1, ALIGNED>), grid, b, 0, st, g);
  else if (packs <= 512) hipLaunchKernelGGL((k_norm_backward<T, 512, 512, 1, ALIGNED>), grid, b, 0, st, g);
  else if (packs <= 1024) hipLaunchKernelGGL((k_norm_backward<T, 512, 512, 2, ALIGNED>), grid, b, 0, st, g);
  else hipLaunchKernelGGL((k_norm_backward<T, 512, 512, 4, ALIGNED>), grid, b, 0, st, g);
}
template <class T>
void norm_backward(const NormArgs &g, bool vec, unsigned parts, hipStream_t st) {
  const int packs = (g.n + Pack<T>::V - 1) / Pack<T>::V;
  if (packs > 4 * 512) hipLaunchKernelGGL((k_norm_backward_any<T>), dim3(parts), dim3(256), 0, st, g);
  else if (vec) norm_backward_rows<T, true>(g, packs, parts, st);
  else norm_backward_rows<T, false>(g, packs, parts, st);
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
  if (x_stride < 0 || dy_stride < 0 || (dx && rows > 1 && dx_stride < n))
    return fail("zm_layer_norm_backward: bad stride");
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
  if (sums) parts_sum((const float *)workspace, (int)parts, 2 * n, n, dweight, dbias, st);
  HIP_OK(hipGetLastError());
  return 0;
}

}  // extern "C"
