// zm_lora.hpp -- low-rank adapters, one named by each token:
//
//   y[s] = residual[s] + c[e] (x[s] A[e]^T) B[e]^T,  e = ids[s],  A [n][R][I], B [n][O][R]
//
// and the gradients by x, A and B.  R is small (16 of thousands), so all of it is bound by reading x and the named
// adapters and by reading and writing y: 2 R operations a value.  Two products of one shape each carry both directions:
//
//   shrink  v[s][r] = sum_k x[s][k] M(r, k)            M = A, k contiguous; backward x = dy, M(r, k) = B[k][r]
//   expand  y[s][o] = residual + c sum_r v[s][r] M(o, r)  M = B, r contiguous; backward M(o, r) = A[r][o]
//
// and the adapters' gradients are one of a third: sum over an adapter's tokens of c a[s][r] m[s][j] (a = u, m = x for dA,
// a = v, m = dy for dB).  Tokens are bucketed by adapter first (k_bucket: a stable order, so sums have a fixed order);
// an item is up to 64 tokens of one adapter.  v stays f32, and enters products as three bf16 terms (zm_linear.hpp).
//
// The matrix instructions (16 x 16, 32 of the summed index) take 8 consecutive values of that index a lane: lane (fr, fc)
// row fr, values 8 fc ..  Where memory has the rows contiguous instead (B in the backward pass, and all operands of a sum
// over tokens), a lane loads NF neighbouring rows of each of its 8 values at once and takes one of each fragment: rows
// NF fr + h belong to fragment h.
#pragma once

#include "zm_kernels.hpp"
#include "zm_linear.hpp"

namespace zm {

constexpr int LORA_TOKENS = 64;  // of an item
constexpr int LORA_MOST_R = 256;

struct LoraArgs {
  const void *x, *m;       // shrink: rows and matrices; expand: matrices; sums: rows
  int64_t ldx, ldm, adapter;  // strides of x's rows, of m's rows and from one adapter to the next
  int64_t K, N;            // shrink: the summed index; expand, sums: columns of the result
  int R, S, n;
  const int32_t *counts, *offs, *pairs, *items, *n_items, *ids;
  int slices, chunks;      // shrink: slices of k and chunks of r; expand: chunks of columns; sums: slices of tokens
  int64_t kslice;
  float *part;             // shrink writes, expand adds [slices][S][R]
  float *v;                // expand: the sums of the slices, or null; sums: a [S][R]
  const float *scale;      // [n] or null
  const void *res;         // expand: [S][ldr] of `type`, or null
  void *y;
  int64_t ldr, ldy;
  int type;
  int rest;                // expand: the first workgroup that looks for tokens without an adapter
};

struct LoraItem {
  int e, count;
  const int32_t *tokens;
};
__device__ __forceinline__ bool lora_item(const LoraArgs &g, int i, LoraItem &it) {
  if (i >= *g.n_items) return false;
  const int32_t w = g.items[i];
  it.e = mmq_item_expert(w);
  const int first = mmq_item_first(w);
  it.count = min(LORA_TOKENS, g.counts[it.e] - first);
  it.tokens = g.pairs + g.offs[it.e] + first;
  return true;
}

// ============================================================ fragments

template <class T>
struct Pack8 {
  T v[8];
};
// 8 consecutive values, of which the first `left` exist (zeros past them); any alignment
template <class T>
__device__ __forceinline__ void load_k(Pack8<T> &p, const T *at, int left) {
  if (left >= 8) {
    __builtin_memcpy(&p, at, sizeof(p));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) p.v[j] = j < left ? at[j] : from_f32<T>(0.f);
  }
}
template <class T, int NT>
__device__ __forceinline__ void frag_of(const Pack8<T> &p, v8bf (&t)[NT]) {
  if constexpr (sizeof(T) == 2 && NT == 1) {
    t[0] = __builtin_bit_cast(v8bf, p);
  } else {
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = to_f32(p.v[j]);
    split_terms<T, NT>(f, t);
  }
}
// NF neighbouring values at `at`, of which `left` exist
template <class T, int NF>
__device__ __forceinline__ void load_rows(T (&p)[NF], const T *at, int left) {
  if (left >= NF) {
    __builtin_memcpy(p, at, sizeof(p));
  } else {
#pragma unroll
    for (int h = 0; h < NF; ++h) p[h] = h < left ? at[h] : from_f32<T>(0.f);
  }
}
template <class T, int NF>
__device__ __forceinline__ Pack8<T> column_of(const T (&p)[8][NF], int h) {
  Pack8<T> r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r.v[j] = p[j][h];
  return r;
}
// acc += all wanted products of the terms of a (rows of the result's lanes) and b (its columns)
template <bool F16, int NA, int NB>
__device__ __forceinline__ void mul_terms(v4f &acc, const v8bf (&a)[NA], const v8bf (&b)[NB]) {
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      if (i + j > PAIRS_MOST) continue;
      if constexpr (F16)
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a[i]), __builtin_bit_cast(v8h, b[j]), acc, 0, 0, 0);
      else
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[j], acc, 0, 0, 0);
    }
}
// terms of a value of type T beside one of type O (see zm_linear.hpp)
template <class T, class O>
constexpr int terms_beside() {
  return std::is_same<T, float>::value ? 3 : std::is_same<T, O>::value ? 1 : std::is_same<T, bf16>::value ? 1 : 2;
}

// ============================================================ shrink
//
// A workgroup takes an item, 16 NF of r and a slice of k; its four waves take 64 k of it in turn (whole lines of x) for
// all 64 tokens, so each value of M is read once a workgroup, and their sums meet in LDS.
template <class TX, class TW, bool KC, int NF>
struct LoraShrink {
  static constexpr int NX = terms_beside<TX, TW>(), NW = terms_beside<TW, TX>();
  static constexpr bool F16 = std::is_same<TX, _Float16>::value && std::is_same<TW, _Float16>::value;
  // the sums of MT tiles of 16 tokens over this wave's part of [k0, k1)
  template <int MT>
  __device__ __forceinline__ static void sums(const LoraArgs &g, const LoraItem &it, int r0, int64_t k0, int64_t k1,
                                              v4f (&acc)[MT][NF]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, fc = lane >> 4;
    const TW *m = (const TW *)g.m + it.e * g.adapter;
    const TX *x[MT];  // (tokens past the item's last repeat it, rows past R others: what they give is not stored)
#pragma unroll
    for (int i = 0; i < MT; ++i) x[i] = (const TX *)g.x + (int64_t)it.tokens[min(16 * i + fr, it.count - 1)] * g.ldx;
    const int rc = NF * fr + r0 < g.R ? NF * fr + r0 : 0, rl = min(g.R - rc, NF);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int h = 0; h < NF; ++h) acc[i][h] = v4f{0.f, 0.f, 0.f, 0.f};
    auto step = [&](int64_t k, auto whole) {
      Pack8<TX> px[2][MT];
      Pack8<TW> pk[2][NF];
      TW pr[2][8][NF];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int64_t ks = k + 32 * s + 8 * fc;
        const int left = decltype(whole)::value ? 8 : (int)min(k1 - ks, (int64_t)8);
#pragma unroll
        for (int i = 0; i < MT; ++i) load_k(px[s][i], x[i] + ks, left);
        if constexpr (KC) {
#pragma unroll
          for (int h = 0; h < NF; ++h) load_k(pk[s][h], m + (int64_t)min(r0 + 16 * h + fr, g.R - 1) * g.ldm + ks, left);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) load_rows<TW, NF>(pr[s][j], m + (ks + j) * g.ldm + rc, j < left ? rl : 0);
        }
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        v8bf fw[NF][NW];
#pragma unroll
        for (int h = 0; h < NF; ++h) {
          if constexpr (KC) frag_of<TW, NW>(pk[s][h], fw[h]);
          else frag_of<TW, NW>(column_of<TW, NF>(pr[s], h), fw[h]);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          v8bf fx[NX];
          frag_of<TX, NX>(px[s][i], fx);
#pragma unroll
          for (int h = 0; h < NF; ++h) mul_terms<F16, NW, NX>(acc[i][h], fw[h], fx);
        }
      }
    };
    int64_t k = k0 + 64 * wave;
    for (; k + 64 <= k1; k += 256) step(k, std::true_type());
    if (k < k1) step(k, std::false_type());
  }
  // and those of all waves, to the slice's part of v
  template <int MT>
  __device__ __forceinline__ static void run(const LoraArgs &g, const LoraItem &it, int z, int r0,
                                             float (&red)[4][16][16 * NF + 4]) {
    constexpr int NR = 16 * NF;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, fc = lane >> 4;
    v4f acc[MT][NF];
    const int64_t k0 = z * g.kslice;
    sums<MT>(g, it, r0, k0, min(g.K, k0 + g.kslice), acc);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      if (16 * i >= it.count) break;
      if (i) __syncthreads();
#pragma unroll
      for (int h = 0; h < NF; ++h)
#pragma unroll
        for (int q = 0; q < 4; ++q) red[wave][fr][KC ? 16 * h + 4 * fc + q : NF * (4 * fc + q) + h] = acc[i][h][q];
      __syncthreads();
      for (int t = threadIdx.x; t < 16 * NR; t += 256) {
        const int s = t / NR, r = t % NR;
        if (16 * i + s >= it.count || r0 + r >= g.R) continue;
        g.part[((size_t)z * g.S + it.tokens[16 * i + s]) * g.R + r0 + r] =
            (red[0][s][r] + red[1][s][r]) + (red[2][s][r] + red[3][s][r]);
      }
    }
  }
};
template <class TX, class TW, bool KC, int NF>
__global__ __launch_bounds__(256) void k_lora_shrink(LoraArgs g) {
  const int per = g.slices * g.chunks, b = blockIdx.x % per, z = b % g.slices, r0 = b / g.slices * 16 * NF;
  __shared__ float red[4][16][16 * NF + 4];
  LoraItem it;
  if (!lora_item(g, blockIdx.x / per, it)) return;
  if (it.count <= 16) LoraShrink<TX, TW, KC, NF>::template run<1>(g, it, z, r0, red);
  else LoraShrink<TX, TW, KC, NF>::template run<LORA_TOKENS / 16>(g, it, z, r0, red);
}

// ============================================================ expand
//
// A workgroup takes an item and 256 columns, 64 a wave.  The slices of v are added, scaled and split into terms in LDS
// once; matrices come straight from memory.  Columns are given to fragments so that a lane ends with 16 neighbouring
// ones of a row: residual and result go in whole lines.  Workgroups from g.rest on look through 64 tokens each for those
// without an adapter: their rows are the residual (or zeros), and NaN where the id names none.
// r whose terms lie in LDS at a time: all up to 128 (52 KB)
__host__ __device__ __forceinline__ int lora_r_step(int R) { return R < 128 ? (R + 31) & ~31 : 128; }
__device__ __forceinline__ void load16(v4f (&v)[4], const void *p, int type, size_t i, int left) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if (4 * q + 4 <= left) {
      v[q] = lin_load4(p, type, i + 4 * q);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[q][j] = 4 * q + j < left ? lin_load(p, type, i + 4 * q + j) : 0.f;
    }
  }
}
template <class TW, bool KC>
__global__ __launch_bounds__(256) void k_lora_expand(LoraArgs g) {
  constexpr int NW = terms_beside<TW, float>(), NF = 4, MT = LORA_TOKENS / 16;
  extern __shared__ __attribute__((aligned(16))) uint16_t lds[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, fc = lane >> 4;
  const int chunk = blockIdx.x % g.chunks, item = blockIdx.x / g.chunks;
  const int64_t o0 = (int64_t)chunk * 256 + 64 * wave;
  if (item >= g.rest) {
    const int s0 = (item - g.rest) * 64;
    const int e = s0 + lane < g.S ? g.ids[s0 + lane] : 0;
    uint64_t todo = __ballot((unsigned)e >= (unsigned)g.n);
    while (todo) {
      const int k = __builtin_ctzll(todo);
      todo &= todo - 1;
      const int s = s0 + k, ek = __builtin_amdgcn_readlane(e, k);
      const float fill = ek < 0 ? 0.f : __builtin_nanf("");
      const int64_t o = o0 + lane;
      if (o < g.N) {
        float y = fill;
        if (ek < 0 && g.res) y = lin_load(g.res, g.type, (size_t)(s * g.ldr + o));
        lin_store(g.y, g.type, (size_t)(s * g.ldy + o), y);
      }
      if (g.v && !chunk)
        for (int r = threadIdx.x; r < g.R; r += 256) g.v[(size_t)s * g.R + r] = fill;
    }
    return;
  }
  LoraItem it;
  if (!lora_item(g, item, it)) return;
  const int mt = (it.count + 15) >> 4;
  const int RP = lora_r_step(g.R), LD = RP + 8, PLANE = LORA_TOKENS * LD;  // (8 more: 16 rows cover all banks)
  const float c = g.scale ? g.scale[it.e] : 1.f;
  const TW *m = (const TW *)g.m + it.e * g.adapter;
  v4f acc[MT][NF];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int h = 0; h < NF; ++h) acc[i][h] = v4f{0.f, 0.f, 0.f, 0.f};
  for (int rb = 0; rb < g.R; rb += RP) {
    if (rb) __syncthreads();
    for (int t = threadIdx.x; t < 16 * mt * RP; t += 256) {  // v: added, scaled, split
      const int s = t / RP, r = t - s * RP;
      float f = 0.f;
      if (s < it.count && rb + r < g.R) {
        const size_t at = (size_t)it.tokens[s] * g.R + rb + r;
        for (int z = 0; z < g.slices; ++z) f += g.part[(size_t)z * g.S * g.R + at];
        if (g.v && !chunk) g.v[at] = f;
        f *= c;
      }
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        const bf16 e = from_f32<bf16>(k ? f : __builtin_amdgcn_fmed3f(f, -BF16_MOST, BF16_MOST));
        lds[k * PLANE + s * LD + r] = e.u;
        f -= to_f32(e);
      }
    }
    __syncthreads();
    if (o0 >= g.N) continue;
    for (int rk = 0; rk < RP && rb + rk < g.R; rk += 32) {
      const int r = rb + rk + 8 * fc, left = min(g.R - r, 8);
      v8bf fw[NF][NW];
      if constexpr (KC) {
#pragma unroll
        for (int h = 0; h < NF; ++h) {
          Pack8<TW> p;
          load_k(p, m + min(o0 + 16 * (fr >> 2) + 4 * h + (fr & 3), g.N - 1) * g.ldm + r, left);
          frag_of<TW, NW>(p, fw[h]);
        }
      } else {
        TW p[8][NF];
        const int64_t o = min(o0 + NF * fr, g.N - 1);
        const int cols = (int)min(g.N - o, (int64_t)NF);
#pragma unroll
        for (int j = 0; j < 8; ++j) load_rows<TW, NF>(p[j], m + (r + j) * g.ldm + o, j < left ? cols : 0);
#pragma unroll
        for (int h = 0; h < NF; ++h) frag_of<TW, NW>(column_of<TW, NF>(p, h), fw[h]);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        if (i >= mt) break;
        v8bf fv[3];
#pragma unroll
        for (int k = 0; k < 3; ++k)
          fv[k] = *reinterpret_cast<const v8bf *>(lds + k * PLANE + (16 * i + fr) * LD + rk + 8 * fc);
#pragma unroll
        for (int h = 0; h < NF; ++h) mul_terms<false, NW, 3>(acc[i][h], fw[h], fv);
      }
    }
  }
  if (o0 < g.N) {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      if (16 * i + fr >= it.count) continue;
      const int64_t s = it.tokens[16 * i + fr], o = o0 + 16 * fc;
      const int left = (int)min(g.N - o, (int64_t)16);
      v4f y[4];
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int j = 0; j < 4; ++j) y[q][j] = KC ? acc[i][q][j] : acc[i][j][q];
      if (g.res) {
        v4f z[4];
        load16(z, g.res, g.type, (size_t)(s * g.ldr + o), left);
#pragma unroll
        for (int q = 0; q < 4; ++q) y[q] += z[q];
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (4 * q + 4 <= left) {
          lin_store4(g.y, g.type, (size_t)(s * g.ldy + o + 4 * q), y[q]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (4 * q + j < left) lin_store(g.y, g.type, (size_t)(s * g.ldy + o + 4 * q + j), y[q][j]);
        }
      }
    }
  }
}
inline size_t lora_expand_lds(int R) { return (size_t)3 * LORA_TOKENS * (lora_r_step(R) + 8) * 2; }

// ============================================================ sums over an adapter's tokens
//
// result[e][r][j] = c[e] sum over its tokens of a[s][r] m[s][j], or with r and j changed (BY_R, dB's order).  A workgroup
// takes an adapter, 64 columns j, 16 NR of r and a slice of its tokens; its waves take 32 tokens in turn, and their sums
// meet in LDS.  Both operands are summed over their rows in memory.
template <class TM, int NR, bool BY_R>
__global__ __launch_bounds__(256) void k_lora_sums(LoraArgs g) {
  constexpr int NM = terms_beside<TM, float>(), NF = 4;
  __shared__ float red[4][NF][256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, fc = lane >> 4;
  const int64_t cols = (g.N + 63) / 64;
  int64_t b = blockIdx.x;
  const int64_t j0 = b % cols * 64;
  b /= cols;
  const int r0 = (int)(b % g.chunks) * 16 * NR;
  b /= g.chunks;
  const int z = (int)(b % g.slices), e = (int)(b / g.slices);
  const int count = g.counts[e], per = ((count + g.slices - 1) / g.slices + 31) & ~31;
  const int t0 = min(z * per, count), t1 = min(t0 + per, count);
  const int32_t *tokens = g.pairs + g.offs[e];
  v4f acc[NR][NF];
#pragma unroll
  for (int h = 0; h < NR; ++h)
#pragma unroll
    for (int f = 0; f < NF; ++f) acc[h][f] = v4f{0.f, 0.f, 0.f, 0.f};
  const int64_t j = min(j0 + NF * fr, g.N - 1);
  const int jl = (int)min(g.N - j, (int64_t)NF);
  const int r = min(r0 + NR * fr, g.R - 1), rl = min(g.R - r, NR);
  for (int t = t0 + 32 * wave; t < t1; t += 128) {
    float pa[8][NR];
    TM pm[8][NF];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int at = t + 8 * fc + k;
      const bool in = at < t1;
      const int64_t s = tokens[in ? at : t0];
      load_rows<float, NR>(pa[k], g.v + s * g.R + r, in ? rl : 0);
      load_rows<TM, NF>(pm[k], (const TM *)g.x + s * g.ldx + j, in ? jl : 0);
    }
    v8bf fm[NF][NM];
#pragma unroll
    for (int f = 0; f < NF; ++f) frag_of<TM, NM>(column_of<TM, NF>(pm, f), fm[f]);
#pragma unroll
    for (int h = 0; h < NR; ++h) {
      v8bf fa[3];
      frag_of<float, 3>(column_of<float, NR>(pa, h), fa);
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        if constexpr (BY_R) mul_terms<false, 3, NM>(acc[h][f], fa, fm[f]);
        else mul_terms<false, NM, 3>(acc[h][f], fm[f], fa);
      }
    }
  }
  const float c = g.scale ? g.scale[e] : 1.f;
  float *out = (float *)g.y + ((size_t)z * g.n + e) * g.R * g.N;
#pragma unroll
  for (int h = 0; h < NR; ++h) {
    if (h) __syncthreads();
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
      for (int q = 0; q < 4; ++q) red[wave][f][64 * q + lane] = acc[h][f][q];
    __syncthreads();
    // value (f, lane, q): index 4 fc + q of the operand that gives the rows, fr of the other; neighbours of the result
    // go to neighbouring threads
    for (int t = threadIdx.x; t < NF * 256; t += 256) {
      const int jr = BY_R ? t >> 4 : t & 63, ri = BY_R ? t & 15 : t >> 6;  // j - j0, and r = r0 + NR ri + h
      const int f = jr & 3, row = BY_R ? ri : jr >> 2, col = BY_R ? jr >> 2 : ri;
      const int k = 64 * (row & 3) + 16 * (row >> 2) + col;
      const int64_t jj = j0 + jr;
      const int rr = r0 + NR * ri + h;
      if (jj >= g.N || rr >= g.R) continue;
      const float v = c * ((red[0][f][k] + red[1][f][k]) + (red[2][f][k] + red[3][f][k]));
      out[BY_R ? (size_t)jj * g.R + rr : (size_t)rr * g.N + jj] = v;
    }
  }
}

// ============================================================ few tokens
//
// A workgroup takes a token and 512 columns: it computes all of the token's v (a wave a row of A at a time, two in flight),
// which costs reading A once for each 512 columns but no second launch, then a column a thread.
struct LoraFewArgs {
  const void *x, *a, *b;
  int64_t ldx, lda, ldb, a_adapter, b_adapter, I, O;
  int R, n;
  const int32_t *ids;
  const float *scale;
  const void *res;
  void *y;
  float *v;
  int64_t ldr, ldy;
  int type;
};
template <class TX, class TW>
__global__ __launch_bounds__(512) void k_lora_few(LoraFewArgs g) {
  constexpr int V = 16 / (int)sizeof(TW), U = 4;
  __shared__ float vs[LORA_MOST_R];
  typedef v4u v4uu __attribute__((aligned(2)));
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t s = blockIdx.y, o = (int64_t)blockIdx.x * 512 + threadIdx.x;
  const int e = g.ids[s];
  float y = 0.f;
  if (o < g.O && g.res) y = lin_load(g.res, g.type, (size_t)(s * g.ldr + o));
  if ((unsigned)e >= (unsigned)g.n) {
    if (e >= 0) y = __builtin_nanf("");
    if (o < g.O) lin_store(g.y, g.type, (size_t)(s * g.ldy + o), y);
    if (g.v && !blockIdx.x && threadIdx.x < g.R) g.v[(size_t)s * g.R + threadIdx.x] = e < 0 ? 0.f : __builtin_nanf("");
    return;
  }
  const TX *x = (const TX *)g.x + s * g.ldx;
  const TW *a = (const TW *)g.a + e * g.a_adapter, *b = (const TW *)g.b + e * g.b_adapter;
  const int K = (int)g.I;
  for (int r = 2 * wave; r < g.R; r += 16) {
    const TW *w[2] = {a + r * g.lda, a + min(r + 1, g.R - 1) * g.lda};
    float acc[2] = {0.f, 0.f};
    for (int k0 = lane * V; k0 + V <= K; k0 += U * 64 * V) {
      v4u rw[2][U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = k0 + u * 64 * V;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          rw[h][u] = k + V <= K ? *reinterpret_cast<const v4uu *>(w[h] + k) : v4u{0, 0, 0, 0};
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = k0 + u * 64 * V;
        if (k + V > K) break;
        TX f[V];
        __builtin_memcpy(f, x + k, sizeof(f));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          TW t[V];
          __builtin_memcpy(t, &rw[h][u], 16);
#pragma unroll
          for (int j = 0; j < V; ++j) acc[h] = __builtin_fmaf(to_f32(t[j]), to_f32(f[j]), acc[h]);
        }
      }
    }
    const int last = K / V * V + lane;
    if (last < K)
#pragma unroll
      for (int h = 0; h < 2; ++h) acc[h] = __builtin_fmaf(to_f32(w[h][last]), to_f32(x[last]), acc[h]);
#pragma unroll
    for (int h = 0; h < 2; ++h) acc[h] = group_sum<64>(acc[h]);
    if (lane < 2 && r + lane < g.R) vs[r + lane] = lane ? acc[1] : acc[0];
  }
  __syncthreads();
  if (g.v && !blockIdx.x && threadIdx.x < g.R) g.v[(size_t)s * g.R + threadIdx.x] = vs[threadIdx.x];
  if (o >= g.O) return;
  const TW *w = b + o * g.ldb;
  float sum = 0.f;
  int r = 0;
  for (; r + V <= g.R; r += V) {
    TW t[V];
    __builtin_memcpy(t, w + r, 16);
#pragma unroll
    for (int j = 0; j < V; ++j) sum = __builtin_fmaf(to_f32(t[j]), vs[r + j], sum);
  }
  for (; r < g.R; ++r) sum = __builtin_fmaf(to_f32(w[r]), vs[r], sum);
  y += (g.scale ? g.scale[e] : 1.f) * sum;
  lin_store(g.y, g.type, (size_t)(s * g.ldy + o), y);
}

// the products by their operands' types; `kc`: the forward pass's order of the matrices
void lora_shrink(int x_type, int w_type, bool kc, const LoraArgs &g, int grid, hipStream_t st);
void lora_expand(int w_type, bool kc, const LoraArgs &g, int grid, hipStream_t st);
void lora_sums(int m_type, bool by_r, const LoraArgs &g, int grid, hipStream_t st);
void lora_few(int x_type, int w_type, const LoraFewArgs &g, dim3 grid, hipStream_t st);
// r of a workgroup: 16, 32 or 64
inline int lora_r_of(int R) { return R <= 16 ? 16 : R <= 32 ? 32 : 64; }

}  // namespace zm
