// zm_grads.hip -- the norm of many gradients together, and the gradients scaled down to a largest norm.
//
//   norm = sqrt(sum of all g^2),  c = min(1, max_norm / (norm + eps)),  out = c g
//
// Bound by memory: every gradient is read for the norm, and read again and written where c < 1.  All tensors of a list
// are one space of units of 4096 values, cut into one contiguous run of units for each workgroup; the list comes as a
// kernel argument, 120 tensors a launch.  Squares are exact in f64 (an f32 has 24 bits) and cannot leave its range, so
// the norm of finite gradients is right wherever f32 holds it; per workgroup one f64 sum, added in a fixed order by every
// workgroup that needs the norm: no atomics, no launch in between.  The second pass takes the runs from their ends, which
// the caches still hold.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <vector>

#include "../../include/zeromoe.h"
#include "zm_host.hpp"
#include "zm_linear.hpp"

using namespace zm;

namespace {

constexpr int MOST_TENSORS = 120;  // of a launch: 32 bytes each, below 4 KB of arguments
constexpr int UNIT = 4096;         // values: 16 a thread
constexpr int MOST_GROUPS = 2048;  // of all launches of a pass (and one more for each launch): 8 a CU

struct Entry {
  const void *g;
  void *out;
  int64_t n;
  uint32_t first;  // unit of the launch
  uint8_t type, out_type;
};
struct Table {
  Entry e[MOST_TENSORS];
  int count;
  uint32_t units;
};

// the run of units of workgroup b of n
__device__ __forceinline__ uint32_t run_start(uint32_t units, uint32_t b, uint32_t n) {
  return (uint32_t)((uint64_t)units * b / n);
}
// the tensor that unit u lies in
__device__ __forceinline__ int entry_of(const Table &t, uint32_t u) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.e[mid].first <= u) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// 16 values of a thread: four packs of four, 1024 apart, so that a wave reads whole lines.  As they lie in memory, so that
// nothing waits for a load before all are asked for.
template <class T>
struct Unit {
  typedef uint32_t Pack __attribute__((ext_vector_type(sizeof(T))));  // (four values: sizeof(T) words)
  typedef Pack PackU __attribute__((aligned(2)));
  Pack p[4];
  __device__ __forceinline__ void load(const T *at) {
#pragma unroll
    for (int q = 0; q < 4; ++q) p[q] = *reinterpret_cast<const PackU *>(at + 1024 * q);
  }
  __device__ __forceinline__ void load_part(const T *at, int64_t left) {  // left: values from `at` on
    T e[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
#pragma unroll
      for (int j = 0; j < 4; ++j) e[j] = 1024 * q + j < left ? at[1024 * q + j] : from_f32<T>(0.f);
      __builtin_memcpy(&p[q], e, sizeof(e));
    }
  }
  __device__ __forceinline__ float get(int q, int j) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(p[q][j]);
    else return to_f32(__builtin_bit_cast(T, (uint16_t)(p[q][j / 2] >> 16 * (j & 1))));
  }
};

// Units u0 .. u1 - 1 of a tensor, this thread's values
template <class T>
__device__ __forceinline__ void add_squares(const Entry &e, uint32_t u0, uint32_t u1, double (&s)[4]) {
  const T *at = (const T *)e.g + (int64_t)u0 * UNIT + 4 * threadIdx.x;
  int64_t left = e.n - (int64_t)u0 * UNIT;
  auto add = [&](const Unit<T> &v) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] = __builtin_fma((double)v.get(q, j), (double)v.get(q, j), s[j]);
  };
  constexpr int N = 8 / (int)sizeof(T);  // units on their way: 128 bytes a thread
  for (; u0 + N <= u1 && left >= N * UNIT; u0 += N, left -= N * UNIT, at += N * UNIT) {
    Unit<T> v[N];
#pragma unroll
    for (int k = 0; k < N; ++k) v[k].load(at + k * UNIT);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int k = 0; k < N; ++k) add(v[k]);
  }
  for (; u0 < u1; ++u0, left -= UNIT, at += UNIT) {
    Unit<T> v;
    if (left >= UNIT) v.load(at);
    else v.load_part(at, left - 4 * (int)threadIdx.x);
    add(v);
  }
}

__global__ __launch_bounds__(256) void k_grad_squares(Table t, double *__restrict__ part) {
  __shared__ double red[4];
  const uint32_t u0 = run_start(t.units, blockIdx.x, gridDim.x), u1 = run_start(t.units, blockIdx.x + 1, gridDim.x);
  double s[4] = {0.0, 0.0, 0.0, 0.0};
  if (u0 < u1) {
    int at = entry_of(t, u0);
    for (uint32_t u = u0; u < u1; ++at) {
      const Entry &e = t.e[at];
      const uint32_t end = min(u1, at + 1 < t.count ? t.e[at + 1].first : t.units);
      if (e.type == LIN_F32) add_squares<float>(e, u - e.first, end - e.first, s);
      else if (e.type == LIN_F16) add_squares<_Float16>(e, u - e.first, end - e.first, s);
      else add_squares<bf16>(e, u - e.first, end - e.first, s);
      u = end;
    }
  }
  const double w = wave_sum_f64((s[0] + s[1]) + (s[2] + s[3]));
  if (!(threadIdx.x & 63)) red[threadIdx.x >> 6] = w;
  __syncthreads();
  if (!threadIdx.x) part[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// the sums of all workgroups added, in the same order by every one
__device__ __forceinline__ double grad_norm(const double *__restrict__ part, int parts) {
  __shared__ double red[4];
  double s = 0.0;
  for (int p0 = threadIdx.x; p0 < parts; p0 += 8 * 256) {
    double v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = p0 + 256 * u < parts ? part[p0 + 256 * u] : 0.0;
#pragma unroll
    for (int u = 0; u < 8; ++u) s += v[u];
  }
  const double w = wave_sum_f64(s);
  if (!(threadIdx.x & 63)) red[threadIdx.x >> 6] = w;
  __syncthreads();
  return sqrt((red[0] + red[1]) + (red[2] + red[3]));
}

__global__ __launch_bounds__(256) void k_grad_norm(const double *__restrict__ part, int parts, float *__restrict__ norm) {
  const double n = grad_norm(part, parts);
  if (!threadIdx.x) *norm = (float)n;
}

// out = c g, rounded to f32 and from there to its type (c in f64: it may lie below f32's range where the gradients are
// huge).  A c of 1 leaves gradients that are scaled in place as they are, unread.
template <class T, class O>
__device__ __forceinline__ void scale_units(const Entry &e, uint32_t u0, uint32_t u1, double c) {  // from the last one down
  for (uint32_t u = u1; u-- > u0;) {
    const int64_t i = (int64_t)u * UNIT + 4 * threadIdx.x, left = e.n - i;
    const T *at = (const T *)e.g + i;
    O *to = (O *)e.out + i;
    Unit<T> v;
    const bool whole = e.n - (int64_t)u * UNIT >= UNIT;
    if (whole) v.load(at);
    else v.load_part(at, left);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      v4f f;
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = (float)((double)v.get(q, j) * c);
      constexpr int type = std::is_same<O, float>::value ? LIN_F32 : std::is_same<O, bf16>::value ? LIN_BF16 : LIN_F16;
      if (whole) {
        lin_store4(to, type, 1024 * q, f);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (1024 * q + j < left) lin_store(to, type, 1024 * q + j, f[j]);
      }
    }
  }
}
template <class T>
__device__ __forceinline__ void scale_to(const Entry &e, uint32_t u0, uint32_t u1, double c) {
  if (e.out_type == LIN_F32) scale_units<T, float>(e, u0, u1, c);
  else if (e.out_type == LIN_F16) scale_units<T, _Float16>(e, u0, u1, c);
  else scale_units<T, bf16>(e, u0, u1, c);
}
__global__ __launch_bounds__(256) void k_grad_scale(Table t, const double *__restrict__ part, int parts, double max_norm,
                                                    double eps, float *norm) {
  const double n = grad_norm(part, parts);
  double c = max_norm / (n + eps);
  if (c > 1.0) c = 1.0;  // (a NaN stays one)
  if (norm && !blockIdx.x && !threadIdx.x) *norm = (float)n;
  const uint32_t u0 = run_start(t.units, blockIdx.x, gridDim.x), u1 = run_start(t.units, blockIdx.x + 1, gridDim.x);
  if (u0 >= u1) return;
  uint32_t end = u1;
  for (int at = entry_of(t, u1 - 1); end > u0; --at) {
    const Entry &e = t.e[at];
    const uint32_t from = max(u0, e.first);
    if (!(c == 1.0 && e.out == e.g)) {
      if (e.type == LIN_F32) scale_to<float>(e, from - e.first, end - e.first, c);
      else if (e.type == LIN_F16) scale_to<_Float16>(e, from - e.first, end - e.first, c);
      else scale_to<bf16>(e, from - e.first, end - e.first, c);
    }
    end = from;
  }
}

// ============================================================ host

size_t size_of(int type) { return type == LIN_F32 ? 4 : 2; }
bool type_ok(int t) { return t == LIN_F32 || t == LIN_F16 || t == LIN_BF16; }
int64_t units_of(const zm_grad &g) { return (g.n + UNIT - 1) / UNIT; }
int64_t launches_of(int64_t count) { return (count + MOST_TENSORS - 1) / MOST_TENSORS; }

int check_list(const zm_grad *g, int64_t count, const char *who, bool writes) {
  if (count < 0 || count >= (int64_t)1 << 24 || (count && !g)) return fail("%s: a list of 0 to 2^24 gradients is needed", who);
  int64_t units = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (!type_ok(g[i].type) || (writes && !type_ok(g[i].out_type))) return fail("%s: types are F32, F16 and BF16", who);
    if (g[i].n < 0 || g[i].n >= (int64_t)1 << 42) return fail("%s: gradient %lld has no possible size", who, (long long)i);
    if (g[i].n && (!g[i].data || (writes && !g[i].out))) return fail("%s: null pointer", who);
    if (writes && g[i].n && g[i].out == g[i].data && g[i].out_type != g[i].type)
      return fail("%s: a gradient scaled in place keeps its type", who);
    units += units_of(g[i]);
  }
  if (units >= (int64_t)1 << 31) return fail("%s: too many values", who);
  return 0;
}

// What is written overlaps nothing else: not another gradient, nor one of its own that is not scaled in place.
int check_overlap(const zm_grad *g, int64_t count, const char *who) {
  struct Range {
    uintptr_t from, to;
    bool written;
  };
  try {
    std::vector<Range> r;
    r.reserve(2 * count);
    for (int64_t i = 0; i < count; ++i) {
      if (!g[i].n) continue;
      const uintptr_t d = (uintptr_t)g[i].data, o = (uintptr_t)g[i].out;
      if (d != o) r.push_back({d, d + g[i].n * size_of(g[i].type), false});
      r.push_back({o, o + g[i].n * size_of(g[i].out_type), true});
    }
    std::sort(r.begin(), r.end(), [](const Range &a, const Range &b) { return a.from < b.from; });
    uintptr_t any = 0, written = 0;
    for (const Range &a : r) {
      if (a.from < (a.written ? any : written)) return fail("%s: a result overlaps a gradient or another result", who);
      any = std::max(any, a.to);
      if (a.written) written = std::max(written, a.to);
    }
  } catch (...) {
    return fail("%s: out of host memory", who);
  }
  return 0;
}

// the norm is written while gradients are still read
int check_norm(const zm_grad *g, int64_t count, const float *norm, const char *who) {
  const uintptr_t at = (uintptr_t)norm;
  auto overlaps = [&](const void *p, size_t bytes) { return at < (uintptr_t)p + bytes && (uintptr_t)p < at + sizeof(float); };
  for (int64_t i = 0; norm && i < count; ++i)
    if (g[i].n && (overlaps(g[i].data, g[i].n * size_of(g[i].type)) || overlaps(g[i].out, g[i].n * size_of(g[i].out_type))))
      return fail("%s: norm overlaps gradient %lld or its result", who, (long long)i);
  return 0;
}

// the workgroups of each launch, by its share of all units
int groups_of(int64_t units, int64_t all) {
  return (int)std::min<int64_t>(units, units * MOST_GROUPS / std::max<int64_t>(all, 1) + 1);
}
int64_t all_units(const zm_grad *g, int64_t count) {
  int64_t n = 0;
  for (int64_t i = 0; i < count; ++i) n += units_of(g[i]);
  return n;
}
Table table_of(const zm_grad *g, int64_t count) {
  Table t{};
  for (int64_t i = 0; i < count; ++i) {
    if (!g[i].n) continue;
    Entry &e = t.e[t.count++];
    e = {g[i].data, g[i].out, g[i].n, t.units, (uint8_t)g[i].type, (uint8_t)g[i].out_type};
    t.units += (uint32_t)units_of(g[i]);
  }
  return t;
}

int squares(const zm_grad *g, int64_t count, int64_t all, double *part, hipStream_t st) {
  int parts = 0;
  for (int64_t i = 0; i < count; i += MOST_TENSORS) {
    const Table t = table_of(g + i, std::min<int64_t>(MOST_TENSORS, count - i));
    const int n = groups_of(t.units, all);
    if (!n) continue;
    hipLaunchKernelGGL(k_grad_squares, dim3(n), dim3(256), 0, st, t, part + parts);
    parts += n;
  }
  return parts;
}

int check_space(void *ws, size_t size, int64_t count, const char *who) {
  if (!ws || size < zm_grad_norm_workspace_size(count) || ((uintptr_t)ws & 255))
    return fail("%s: a 256-byte aligned workspace of zm_grad_norm_workspace_size() bytes is needed", who);
  return 0;
}

}  // namespace

extern "C" {

size_t zm_grad_norm_workspace_size(int64_t count) {
  if (count < 0 || count >= (int64_t)1 << 24) return 0;
  return ((MOST_GROUPS + launches_of(count)) * sizeof(double) + 255) & ~(size_t)255;
}

int zm_grad_norm(const zm_grad *g, int64_t count, float *norm, void *workspace, size_t workspace_size, void *stream) {
  if (check_list(g, count, "zm_grad_norm", false)) return -1;
  if (!norm) return fail("zm_grad_norm: null pointer");
  if (check_space(workspace, workspace_size, count, "zm_grad_norm")) return -1;
  const hipStream_t st = (hipStream_t)stream;
  const int parts = squares(g, count, all_units(g, count), (double *)workspace, st);
  hipLaunchKernelGGL(k_grad_norm, dim3(1), dim3(256), 0, st, (const double *)workspace, parts, norm);
  HIP_OK(hipGetLastError());
  return 0;
}

int zm_grad_clip(const zm_grad *g, int64_t count, double max_norm, double eps, float *norm, void *workspace,
                 size_t workspace_size, void *stream) {
  if (check_list(g, count, "zm_grad_clip", true)) return -1;
  if (!(max_norm >= 0.0) || !(eps >= 0.0) || std::isinf(eps))
    return fail("zm_grad_clip: max_norm >= 0 and a finite eps >= 0 are needed");
  if (check_overlap(g, count, "zm_grad_clip")) return -1;
  if (check_space(workspace, workspace_size, count, "zm_grad_clip")) return -1;
  if (check_norm(g, count, norm, "zm_grad_clip")) return -1;
  const hipStream_t st = (hipStream_t)stream;
  double *part = (double *)workspace;
  const int64_t all = all_units(g, count);
  const int parts = squares(g, count, all, part, st);
  bool told = !norm;
  for (int64_t i = 0; i < count; i += MOST_TENSORS) {
    const Table t = table_of(g + i, std::min<int64_t>(MOST_TENSORS, count - i));
    const int n = groups_of(t.units, all);
    if (!n) continue;
    hipLaunchKernelGGL(k_grad_scale, dim3(n), dim3(256), 0, st, t, (const double *)part, parts, max_norm, eps,
                       told ? nullptr : norm);
    told = true;
  }
  if (!told) hipLaunchKernelGGL(k_grad_norm, dim3(1), dim3(256), 0, st, (const double *)part, parts, norm);
  HIP_OK(hipGetLastError());
  return 0;
}

}  // extern "C"
