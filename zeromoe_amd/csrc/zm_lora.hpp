// zm_lora.hpp -- low-rank adapters, one named by each token:
//
//   y[s] = residual[s] + c[e] (x[s] A[e]^T) B[e]^T,  e = ids[s],  A [n][R][I], B [n][O][R]
//
// and the gradients by x, A and B.  R is small (16 of thousands), so all of it is bound by reading x and the named
// adapters and by reading and writing y: 2 R operations a value.  One kernel carries both directions, a product over the
// long axis and one over the short axis with v between them in LDS, where it stays f32 and enters as three bf16 terms
// (zm_linear.hpp):
//
//   v[s][r] = sum_k x[s][k] M(r, k)                 M = A, k contiguous; backward x = dy, M(r, k) = B[k][r]
//   y[s][o] = residual + c sum_r v[s][r] L(o, r)    L = B, r contiguous; backward L(o, r) = A[r][o]
//
// and the adapters' gradients are sums over an adapter's tokens of c a[s][r] m[s][j] (a = u, m = x for dA, a = v, m = dy
// for dB).  Tokens are sorted by adapter first (a stable order, so sums have a fixed order) into items of up to 32 tokens
// of one adapter.  (Two kernels with v in memory, the long axis in slices, took 50 + 58 us where the one takes 60:
// 8192 x 7168 x 2048, R 64, bf16.  Where items are few and have much to read, each axis is a launch of its own after all.)
//
// The matrix instructions (16 x 16, 32 of the summed index) take 8 consecutive values of that index a lane: lane (fr, fc)
// row fr, values 8 fc ..  Where memory has the rows contiguous instead (B in the backward pass, and all operands of a sum
// over tokens), a lane loads NF neighbouring rows of each of its 8 values at once and takes one of each fragment: rows
// NF fr + h belong to fragment h.
#pragma once

#include "zm_linear.hpp"

namespace zm {

constexpr int LORA_TOKENS = 32;  // of an item, at most (16 or 32)
constexpr int LORA_CUS = 256;
constexpr int LORA_MOST_R = 256, LORA_MOST_N = 512;

// The items, of up to T tokens: item i's tokens lie at tokens[T i ..], in ascending order, and item[i] is its
// adapter and (from bit 16 on) how many there are.  Adapter e has counts[e] tokens, in the items from first[e] on.
//
// A CU runs one item at a time, so T is 16 where no CU gets a second one then, else 32: dx alone of 4095 tokens of four
// adapters, 4096 x 1536, R 16: 51 us a call in 258 items of 16, 39 in 130 of 32; 4060 tokens in 256 of 16: 34.  How
// many there are depends on the ids, so that is decided on the device.
struct LoraItems {
  int32_t *counts, *first, *item, *tokens, *n_items;  // [n], [n], [items], [items][T], items and log2 T
  int small;  // whether T may be 16
};
struct LoraArgs {
  const void *x, *m, *l;  // rows, the matrices of the long axis and those of the short one
  int64_t ldx, ldm, ldl;  // strides of their rows
  int64_t m_adapter, l_adapter;
  int64_t K, N;           // the long axis, and columns of the result (0: v alone)
  int R, S, n;
  LoraItems it;
  const int32_t *ids;
  float *v;               // [S][R], or null
  const float *scale;     // [n] or null
  const void *res;        // [S][ldr] or null
  void *y;
  int64_t ldr, ldy;
  int rest;               // tokens that a workgroup looks through for those without an adapter, at most 32
  // both axes in one launch, or (few items) each in its own, the long one in slices of k, the short one in groups of columns
  enum { BOTH, LONG, SHORT };
  int phase, slices;
  int64_t kslice;
  float *part;            // [slices][S][R]
};

// ============================================================ items
//
// One workgroup; each of its 16 waves takes a run of tokens, 64 at a time.  The lanes of one id find each other by a
// ballot for each bit of it; their first one counts them in the wave's own counters, so no atomic is needed and a token's
// place among its wave's is known at once; it is kept in registers for the first 16 chunks (16384 tokens of the call) and
// found again for the others.  8192 tokens of 8 adapters: 7.6 us.
constexpr int LORA_CHUNKS = 16;
static __global__ __launch_bounds__(1024) void k_lora_items(const int32_t *__restrict__ ids, int S, int n, LoraItems o) {
  __shared__ int cnt[16][LORA_MOST_N], first[LORA_MOST_N], total[LORA_MOST_N], sums[16];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int seg = (S + 1023) / 1024 * 64, p0 = w * seg, p1 = min(p0 + seg, S);
  const int bits = n > 1 ? 32 - __builtin_clz((unsigned)(n - 1)) : 0;
  auto load = [&](int p) {
    const int e = p < p1 ? ids[p] : -1;
    return (unsigned)e < (unsigned)n ? e : -1;
  };
  int e[LORA_CHUNKS], at[LORA_CHUNKS];
  // all asked for before the first is waited for (a condition on the load would wait for each: 1 us a chunk)
#pragma unroll
  for (int c = 0; c < LORA_CHUNKS; ++c)
    if (64 * c < seg) e[c] = ids[min(p0 + 64 * c + lane, S - 1)];
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int c = 0; c < LORA_CHUNKS; ++c)
    e[c] = 64 * c < seg && p0 + 64 * c + lane < p1 && (unsigned)e[c] < (unsigned)n ? e[c] : -1;
  for (int k = lane; k < n; k += 64) cnt[w][k] = 0;
  stage_sync();
  // the place of a token among those of its adapter in its wave
  auto place = [&](int e) {
    uint64_t same = __ballot(e >= 0);
    for (int j = 0; j < bits; ++j) {
      const uint64_t b = __ballot(e >= 0 && ((e >> j) & 1));
      same &= ((e >> j) & 1) ? b : ~b;
    }
    const int rank = __builtin_popcountll(same & ((1ull << lane) - 1));
    int at = 0;
    if (e >= 0) at = cnt[w][e];
    stage_sync();
    if (e >= 0 && !rank) cnt[w][e] = at + __builtin_popcountll(same);
    stage_sync();
    return at + rank;
  };
#pragma unroll
  for (int c = 0; c < LORA_CHUNKS; ++c)
    if (64 * c < seg) at[c] = place(e[c]);
  for (int p = p0 + 64 * LORA_CHUNKS; p < p1; p += 64) place(load(p + lane));
  __syncthreads();
  // by adapter: tokens of the waves before, all of them, and their items (small: of 16 tokens in the low half, of 32 in the
  // other; there are 384 at most)
  int mine = 0;
  if (tid < n) {
    int run = 0;
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      const int k = cnt[v][tid];
      cnt[v][tid] = run;
      run += k;
    }
    total[tid] = run;
    mine = (run + 31) >> 5;
    if (o.small) mine = mine << 16 | (run + 15) >> 4;
  }
  int incl = mine;  // (adapters are below 512: waves 0 to 7 hold them)
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int up = __shfl_up(incl, m, 64);
    if (lane >= m) incl += up;
  }
  if (lane == 63) sums[w] = incl;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int v = 0; v < 8; ++v) {
    if (v < w) before += sums[v];
    all += sums[v];
  }
  const int lg = o.small && (all & 0xffff) <= LORA_CUS ? 4 : 5, T = 1 << lg;
  auto items = [&](int k) { return !o.small ? k : lg == 4 ? k & 0xffff : k >> 16; };
  if (tid < n) {
    first[tid] = items(before + incl - mine);
    o.first[tid] = first[tid];
    o.counts[tid] = total[tid];
  }
  if (!tid) {
    o.n_items[0] = items(all);
    o.n_items[1] = lg;
  }
  __syncthreads();
  auto put = [&](int p, int e, int at) {  // token p, `at` among e's
    o.tokens[((size_t)first[e] << lg) + at] = p;
    if (!(at & (T - 1))) o.item[first[e] + (at >> lg)] = e | min(T, total[e] - at) << 16;
  };
#pragma unroll
  for (int c = 0; c < LORA_CHUNKS; ++c)
    if (64 * c < seg && e[c] >= 0) put(p0 + 64 * c + lane, e[c], at[c] + cnt[w][e[c]]);
  if (seg <= 64 * LORA_CHUNKS) return;
  // the chunks past the registers: their places again, on from those of the chunks before
  stage_sync();
  for (int c = 0; c < LORA_CHUNKS; ++c) {
    const int k = load(p0 + 64 * c + lane);
    if (k >= 0) atomicAdd(&cnt[w][k], 1);
  }
  stage_sync();
  for (int p = p0 + 64 * LORA_CHUNKS; p < p1; p += 64) {
    const int k = load(p + lane);
    const int a = place(k);
    if (k >= 0) put(p + lane, k, a);
  }
}

// This wave's view of item i: its adapter, its tokens and how many there are.  All are asked for before any is waited for.
struct LoraItem {
  int e, count, lanes;  // lanes: token lane % 32 of the item
  // token t of the item; those past the last are its first (all lanes of the wave take part)
  __device__ __forceinline__ int64_t token(int t) const { return __shfl(lanes, t < count ? t : 0, 64); }
};
__device__ __forceinline__ bool lora_item(const LoraArgs &g, int i, LoraItem &it) {
  // (its place follows from T: both are read)
  const int32_t *at = g.it.tokens + threadIdx.x % LORA_TOKENS;
  int item = g.it.item[i], n = g.it.n_items[0], lg = g.it.n_items[1], t16 = at[16 * (size_t)i], t32 = at[32 * (size_t)i];
  asm volatile("" : "+v"(item), "+v"(n), "+v"(lg), "+v"(t16), "+v"(t32));  // (else some are asked for past the branch)
  if (i >= uniform(n)) return false;  // (before item is used)
  it.e = uniform(item & 0xffff);
  it.count = uniform(item >> 16);
  it.lanes = uniform(lg) == 4 ? t16 : t32;
  return true;
}

// ============================================================ fragments

template <class T>
__device__ __forceinline__ uint32_t bits_of(T v) {
  if constexpr (sizeof(T) == 4) return __builtin_bit_cast(uint32_t, v);
  else return __builtin_bit_cast(uint16_t, v);
}
template <class T>
__device__ __forceinline__ float f32_of_bits(uint32_t w) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(w);
  else return to_f32(__builtin_bit_cast(T, (uint16_t)w));
}
// N neighbouring values as words (two of 16 bits a word, a single one by itself)
template <class T, int N>
struct Words {
  static constexpr int W = (N * (int)sizeof(T) + 3) / 4;
  uint32_t w[W];
  __device__ __forceinline__ float get(int j) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[j]);
    else return f32_of_bits<T>(j & 1 ? w[j / 2] >> 16 : w[j / 2] & 0xffffu);
  }
};
// N values at `at` of which the first `left` exist (zeros past them), at any alignment; `safe`: a value that exists
template <class T, int N>
__device__ __forceinline__ void load_words(Words<T, N> &p, const T *at, int left, const T *safe) {
  if (left >= N) {
    if constexpr (N * sizeof(T) < 4) p.w[0] = bits_of(*at);
    else __builtin_memcpy(p.w, at, N * sizeof(T));
  } else {
    uint32_t e[N];
#pragma unroll
    for (int j = 0; j < N; ++j) e[j] = bits_of(*(j < left ? at + j : safe));
#pragma unroll
    for (int j = 0; j < N; ++j) e[j] = j < left ? e[j] : 0u;
#pragma unroll
    for (int k = 0; k < Words<T, N>::W; ++k) {
      if constexpr (sizeof(T) == 4) p.w[k] = e[k];
      else p.w[k] = 2 * k + 1 < N ? e[2 * k] | e[2 * k + 1] << 16 : e[2 * k];
    }
  }
}
// 8 values of the summed index as terms
template <class T, int NT>
__device__ __forceinline__ void frag_of(const Words<T, 8> &p, v8bf (&t)[NT]) {
  if constexpr (sizeof(T) == 2 && NT == 1) {
    t[0] = __builtin_bit_cast(v8bf, v4u{p.w[0], p.w[1], p.w[2], p.w[3]});
  } else {
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = p.get(j);
    split_terms<T, NT>(f, t);
  }
}
// the same from 8 groups of NF neighbouring rows: row h of each
template <class T, int NT, int NF>
__device__ __forceinline__ void frag_of_rows(const Words<T, NF> (&p)[8], int h, v8bf (&t)[NT]) {
  if constexpr (sizeof(T) == 2 && NT == 1) {
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      o[j] = __builtin_amdgcn_perm(p[2 * j + 1].w[h / 2], p[2 * j].w[h / 2], h & 1 ? 0x07060302u : 0x05040100u);
    t[0] = __builtin_bit_cast(v8bf, v4u{o[0], o[1], o[2], o[3]});
  } else {
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = p[j].get(h);
    split_terms<T, NT>(f, t);
  }
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

// ============================================================ both products
//
// A workgroup takes an item.  Over the long axis its eight waves take a line of x (64 k of 16 bits, 32 of f32) in turn for
// all of its tokens and 16 NF of r, so each value of M is read once a workgroup, from L2 as a rule; the next line or two
// are on their way while one is multiplied.  The waves' sums meet in LDS as v and become terms there.  Over the short axis a
// wave takes 64 columns at a time, the next ones on their way.
//
// A fragment's 16 neighbouring lanes hold 16 rows, and a load that follows that asks for 16 lines for each 16 lanes: the
// address units take one a cycle, 16 bytes (such a kernel read 35 GB/s a CU, whatever was on its way).  So rows come in
// whole lines, 8 neighbouring lanes each, and go to fragments through LDS of the wave's own (no barrier), and results go
// back the same way.  RL: values of r whose terms LDS has room for.
//
// Every workgroup also looks through g.rest tokens for those without an adapter: their rows are the residual (or zeros),
// and NaN where the id names none.  (Workgroups of their own waited for a CU behind the items: 68.6 us for 65.)
//
// Sums of terms have NaN where the formula may have an infinity (zm_linear.hpp, lin_again).  A value of v or of the result
// that is not finite is taken again value by value in f32, so that what an infinity gives does not go by the number of
// tokens; v stays without the scale, which multiplies the sums, as k_lora_few has it.
constexpr int LORA_WAVES = 8;

// ROWS rows of PIECES x 16 bytes by way of registers into LDS, rows 128 bytes apart, their pieces permuted so that 16 rows
// of a fragment cover all banks
template <class T, int ROWS, int PIECES>
struct Stage {
  static constexpr int V = 16 / (int)sizeof(T), PER = ROWS * PIECES / 64;
  Words<T, V> reg[PER];
  __device__ __forceinline__ static int row(int i) { return (i * 64 + ((int)threadIdx.x & 63)) / PIECES; }
  __device__ __forceinline__ static int piece() { return (int)threadIdx.x % PIECES; }
  __device__ __forceinline__ static uint32_t at(int row, int piece) { return row * 128 + ((piece ^ (row >> 1)) & 7) * 16; }
  // `left`: values that exist of the row's part, for this lane's piece at(i) = its row's first value
  template <class At>
  __device__ __forceinline__ void load(const At &at, int left, const T *safe) {
    if (left >= PIECES * V) {
#pragma unroll
      for (int i = 0; i < PER; ++i) load_words(reg[i], at(i) + V * piece(), V, safe);
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) load_words(reg[i], at(i) + V * piece(), left - V * piece(), safe);
    }
  }
  __device__ __forceinline__ void store(uint8_t *lds) const {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      *reinterpret_cast<v4u *>(lds + at(row(i), piece())) = v4u{reg[i].w[0], reg[i].w[1], reg[i].w[2], reg[i].w[3]};
  }
  // values 32 s + 8 fc .. of row `row`
  __device__ __forceinline__ static Words<T, 8> frag(const uint8_t *lds, int row, int s) {
    const int fc = ((int)threadIdx.x & 63) >> 4;
    Words<T, 8> p;
#pragma unroll
    for (int q = 0; q < (int)sizeof(T) / 2; ++q) {
      const v4u v = *reinterpret_cast<const v4u *>(lds + at(row, (4 * s + fc) * ((int)sizeof(T) / 2) + q));
#pragma unroll
      for (int j = 0; j < 4; ++j) p.w[4 * q + j] = v[j];
    }
    return p;
  }
};

template <class TX, class TW, bool KC, int NF, int RL, class TY>
struct Lora {
  static constexpr int NX = terms_beside<TX, TW>(), NM = terms_beside<TW, TX>(), NL = terms_beside<TW, float>();
  static constexpr bool F16 = std::is_same<TX, _Float16>::value && std::is_same<TW, _Float16>::value;
  static constexpr int H = 4 / (int)sizeof(TX), LINE = 32 * H;  // matrix instructions and k of a step
  static constexpr int NR = 16 * NF, LD = RL + 8;               // (8 more: 16 rows cover all banks)
  static constexpr int C = 4;                                   // fragments of 16 columns of a wave
  static constexpr int DEPTH = (KC ? sizeof(TW) == 2 : NF <= 2) ? 2 : 1;  // lines on their way (as registers allow)
  static constexpr int BUF = 128 * (LORA_TOKENS + (NR < 32 ? 32 : NR));  // bytes of a wave: a line; 64 rows of L
  struct Lds {
    union {
      uint8_t wave[LORA_WAVES][BUF];
      float sums[LORA_WAVES][16][NR + 4];
    };
    uint16_t terms[3][LORA_TOKENS][LD];
  };

  // the sums of MT tiles of 16 tokens over this wave's lines, r from r0 on
  template <int MT>
  __device__ __forceinline__ static void long_axis(const LoraArgs &g, const LoraItem &it, int r0, int64_t k0, int64_t k1,
                                                   uint8_t *buf, v4f (&acc)[MT][NF]) {
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), fr = lane & 15, fc = lane >> 4;
    constexpr int STEP = LINE * LORA_WAVES;
    typedef Stage<TX, 16 * MT, 8> SX;
    typedef Stage<TW, NR, LINE * (int)sizeof(TW) / 16> SM;  // KC
    const TW *m = (const TW *)g.m + it.e * g.m_adapter;
    const TX *x[SX::PER];  // (tokens past the item's last, and rows past R, repeat others: what they give is not used)
#pragma unroll
    for (int i = 0; i < SX::PER; ++i) x[i] = (const TX *)g.x + it.token(SX::row(i)) * g.ldx;
    uint32_t row[SM::PER];  // bytes (zm_lora admits adapters of less than 2^31)
#pragma unroll
    for (int i = 0; i < SM::PER; ++i) row[i] = (uint32_t)min(r0 + SM::row(i), g.R - 1) * (uint32_t)(g.ldm * sizeof(TW));
    const int rc = NF * fr + r0 < g.R ? NF * fr + r0 : 0, rl = min(g.R - rc, NF);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int h = 0; h < NF; ++h) acc[i][h] = v4f{0.f, 0.f, 0.f, 0.f};
    struct Line {
      SX x;
      SM m;                        // KC
      Words<TW, NF> r[KC ? 1 : H][8];  // else
    };
    int64_t k = k0 + LINE * wave;
    if (k >= k1) return;
    const int64_t last = k + (k1 - 1 - k) / STEP * STEP;
    auto load = [&](Line &to, int64_t k) {
      // (past the end the last line again: a load under a condition would be waited for where its paths meet)
      k = min(k, last);
      const int left = (int)min(k1 - k, (int64_t)LINE);
      to.x.load([&](int i) { return x[i] + k; }, left, (const TX *)g.x);
      if constexpr (KC) {
        to.m.load([&](int i) { return (const TW *)((const uint8_t *)(m + k) + row[i]); }, left, m);
      } else if (left == LINE && g.R % NF == 0) {
#pragma unroll
        for (int s = 0; s < H; ++s)
#pragma unroll
          for (int j = 0; j < 8; ++j) load_words(to.r[s][j], m + (k + 32 * s + 8 * fc + j) * g.ldm + rc, NF, m);
      } else {
#pragma unroll
        for (int s = 0; s < H; ++s)
#pragma unroll
          for (int j = 0; j < 8; ++j)
            load_words(to.r[s][j], m + (k + 32 * s + 8 * fc + j) * g.ldm + rc, 32 * s + 8 * fc + j < left ? rl : 0, m);
      }
    };
    uint8_t *bx = buf, *bm = buf + 128 * 16 * MT;
    auto step = [&](Line &line, int64_t k) {
      line.x.store(bx);
      v8bf fr_m[KC ? 1 : H][NF][NM];
      if constexpr (KC) {
        line.m.store(bm);
      } else {
#pragma unroll
        for (int s = 0; s < H; ++s)
#pragma unroll
          for (int h = 0; h < NF; ++h) frag_of_rows(line.r[s], h, fr_m[s][h]);
      }
      load(line, k + DEPTH * STEP);
      stage_sync();
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int s = 0; s < H; ++s) {
        v8bf fm[NF][NM];
        if constexpr (KC) {
#pragma unroll
          for (int h = 0; h < NF; ++h) frag_of(SM::frag(bm, 16 * h + fr, s), fm[h]);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          v8bf fx[NX];
          frag_of(SX::frag(bx, 16 * i + fr, s), fx);
#pragma unroll
          for (int h = 0; h < NF; ++h) {
            if constexpr (KC) mul_terms<F16, NM, NX>(acc[i][h], fm[h], fx);
            else mul_terms<F16, NM, NX>(acc[i][h], fr_m[s][h], fx);
          }
        }
      }
      stage_sync();
    };
    Line a, b;
    load(a, k);
    if constexpr (DEPTH == 2) load(b, k + STEP);
    for (; k < k1; k += DEPTH * STEP) {
      step(a, k);
      if constexpr (DEPTH == 2) {
        if (k + STEP >= k1) break;
        step(b, k + STEP);
      }
    }
  }

  // v of a token again
  __device__ __forceinline__ static float long_again(const LoraArgs &g, const LoraItem &it, int64_t token, int r) {
    const TX *x = (const TX *)g.x + token * g.ldx;
    const int64_t step = KC ? 1 : g.ldm;
    const TW *m = (const TW *)g.m + it.e * g.m_adapter + (KC ? r * g.ldm : r);
    float v = 0.f;
    for (int64_t k = 0; k < g.K && v == v; k += 4) {
      float a[4], b[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        a[u] = k + u < g.K ? to_f32(x[k + u]) : 0.f;
        b[u] = k + u < g.K ? to_f32(m[(k + u) * step]) : 0.f;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) v = __builtin_fmaf(a[u], b[u], v);
    }
    return v;
  }
  // the sum of the item's token s in column o again, without the scale
  __device__ __forceinline__ static float short_again(const LoraArgs &g, const LoraItem &it, const Lds &lds, int s, int64_t o) {
    const int64_t step = KC ? 1 : g.ldl;
    const TW *l = (const TW *)g.l + it.e * g.l_adapter + (KC ? o * g.ldl : o);
    float sum = 0.f;
    for (int r = 0; r < g.R && sum == sum; ++r) {
      float t[3];
#pragma unroll
      for (int k = 0; k < 3; ++k) t[k] = to_f32(bf16{lds.terms[k][s][r]});
      sum = __builtin_fmaf(t[0] + (t[1] + t[2]), to_f32(l[r * step]), sum);  // (the terms' sum is v, in every bit)
    }
    return sum;
  }

  template <int MT>
  __device__ __forceinline__ static void run(const LoraArgs &g, const LoraItem &it, Lds &lds) {
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), fr = lane & 15, fc = lane >> 4;
    const float c = g.scale ? g.scale[it.e] : 1.f;
    auto put_terms = [&](int s, int r, float v) {  // (an infinity or a NaN is the first one, zeros follow)
      const bool number = lin_finite(v);
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        const bf16 e = from_f32<bf16>(k || !number ? v : __builtin_amdgcn_fmed3f(v, -BF16_MOST, BF16_MOST));
        lds.terms[k][s][r] = e.u;
        v = number ? v - to_f32(e) : 0.f;
      }
    };
    if (g.phase == LoraArgs::SHORT) {
      const int RP = (g.R + 31) & ~31;
      for (int t = threadIdx.x; t < 16 * MT * RP; t += 64 * LORA_WAVES) {
        const int s = t / RP, r = t - s * RP;
        float v = 0.f;
        if (s < it.count && r < g.R) {
          const int token = g.it.tokens[((size_t)blockIdx.x << g.it.n_items[1]) + s];
          const size_t at = (size_t)token * g.R + r;
          for (int z = 0; z < g.slices; ++z) v += g.part[(size_t)z * g.S * g.R + at];
          if (NX * NM > 1 && !lin_finite(v)) v = long_again(g, it, token, r);
          if (g.v && !blockIdx.y) g.v[at] = v;
        }
        put_terms(s, r, v);
      }
      __syncthreads();
      return short_axis<MT>(g, it, c, lds);
    }
    const int64_t k0 = g.phase == LoraArgs::LONG ? blockIdx.y * g.kslice : 0;
    const int64_t k1 = g.phase == LoraArgs::LONG ? min(g.K, k0 + g.kslice) : g.K;
    float *part = g.phase == LoraArgs::LONG ? g.part + (size_t)blockIdx.y * g.S * g.R : g.v;
    for (int r0 = 0; r0 < g.R; r0 += NR) {
      v4f acc[MT][NF];
      long_axis<MT>(g, it, r0, k0, k1, lds.wave[wave], acc);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        __syncthreads();
#pragma unroll
        for (int h = 0; h < NF; ++h) {
          if constexpr (KC) {
            *reinterpret_cast<v4f *>(&lds.sums[wave][fr][16 * h + 4 * fc]) = acc[i][h];
          } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) lds.sums[wave][fr][NF * (4 * fc + q) + h] = acc[i][h][q];
          }
        }
        __syncthreads();
        constexpr int WIDE = NR < 32 ? 32 : NR;  // (zeros up to the 32 of a matrix instruction)
        for (int t = threadIdx.x; t < 16 * WIDE; t += 64 * LORA_WAVES) {
          const int s = t / WIDE, r = t % WIDE;
          const int64_t to = part || NX * NM > 1 ? it.token(16 * i + s) : 0;  // (by all lanes of the wave)
          float v = 0.f;
          if (r < NR && r0 + r < g.R) {
#pragma unroll
            for (int u = 0; u < LORA_WAVES; ++u) v += lds.sums[u][s][r];
            if (NX * NM > 1 && g.phase == LoraArgs::BOTH && !lin_finite(v)) v = long_again(g, it, to, r0 + r);
            if (part && 16 * i + s < it.count) part[(size_t)to * g.R + r0 + r] = v;
          }
          put_terms(16 * i + s, r0 + r, v);
        }
      }
      __syncthreads();
    }
    if (g.phase == LoraArgs::BOTH) short_axis<MT>(g, it, c, lds);
  }

  template <int MT>
  __device__ __forceinline__ static void short_axis(const LoraArgs &g, const LoraItem &it, float c, Lds &lds) {
    const int STEP = 64 * LORA_WAVES * gridDim.y;  // (groups of columns)
    constexpr bool STAGED = KC && RL > 32;                   // (shorter rows of L are several to a line)
    constexpr int RS = STAGED ? 128 / (int)sizeof(TW) : 32;  // r of a step
    typedef Stage<TW, 64, 8> SL;
    // the result: a row of 64 columns in VY-value pieces, PY of them
    constexpr int VY = 16 / (int)sizeof(TY), PY = 64 / VY, OUT = 16 * PY / 64;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), fr = lane & 15, fc = lane >> 4;
    uint8_t *buf = lds.wave[wave];
    const TW *l = (const TW *)g.l + it.e * g.l_adapter;
    const int yr = lane / PY, yc = lane % PY * VY;  // the lane's row (of 64 / PY at once) and its first column
    auto out_row = [&](int i, int q) { return 16 * i + yr + 64 / PY * q; };
    int token[MT][OUT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int q = 0; q < OUT; ++q) token[i][q] = (int)it.token(out_row(i, q));
    struct Part {  // of the matrix: 64 columns, RS of r
      SL s;                     // STAGED
      Words<TW, 8> k[C];        // KC
      Words<TW, C> r[8];        // else
    };
    struct Columns {
      Words<TY, VY> z[MT][OUT];
      Part l;
    };
    auto load_part = [&](Part &to, int64_t o0, int r) {
      const bool whole = o0 + 64 <= g.N;
      if constexpr (STAGED) {
        to.s.load([&](int i) {
          const uint32_t o = (uint32_t)(whole ? o0 + SL::row(i) : min(o0 + SL::row(i), g.N - 1));
          return (const TW *)((const uint8_t *)(l + r) + o * (uint32_t)(g.ldl * sizeof(TW)));
        }, min(g.R - r, RS), l);
      } else if constexpr (KC) {
        const int left = min(g.R - (r + 8 * fc), 8);
#pragma unroll
        for (int h = 0; h < C; ++h) {
          const TW *at = l + min(o0 + 16 * h + fr, g.N - 1) * g.ldl;
          if (g.R % 8 == 0) {  // a pack is whole or none: no condition on the load
            load_words(to.k[h], at + (left > 0 ? r + 8 * fc : 0), 8, at);
#pragma unroll
            for (int k = 0; k < Words<TW, 8>::W; ++k) to.k[h].w[k] = left > 0 ? to.k[h].w[k] : 0u;
          } else {
            load_words(to.k[h], at + r + 8 * fc, left, at);
          }
        }
      } else {
        const int64_t o = min(o0 + C * fr, g.N - 1);
        const int n = (int)min(g.N - o, (int64_t)C);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int rj = r + 8 * fc + j;  // (past R v has zeros, but what lies there may be no number)
          load_words(to.r[j], l + min(rj, g.R - 1) * g.ldl + o, whole ? C : n, l);
#pragma unroll
          for (int k = 0; k < Words<TW, C>::W; ++k) to.r[j].w[k] = rj < g.R ? to.r[j].w[k] : 0u;
        }
      }
    };
    int64_t o0 = 64 * (LORA_WAVES * blockIdx.y + wave);
    if (o0 >= g.N) return;
    const int64_t last = o0 + (g.N - 1 - o0) / STEP * STEP;
    auto load = [&](Columns &to, int64_t o0) {
      o0 = min(o0, last);
      const int cols = (int)min(g.N - (o0 + yc), (int64_t)VY);
      if (g.res) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int q = 0; q < OUT; ++q) {
            const TY *at = (const TY *)g.res + token[i][q] * g.ldr + o0 + yc;
            load_words(to.z[i][q], at, o0 + 64 <= g.N ? VY : cols, (const TY *)g.res);
          }
      }
      load_part(to.l, o0, 0);
    };
    auto columns = [&](Columns &now, Columns &next, int64_t o0) {
      const int cols = (int)min(g.N - (o0 + yc), (int64_t)VY);
      v4f acc[MT][C];
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int h = 0; h < C; ++h) acc[i][h] = v4f{0.f, 0.f, 0.f, 0.f};
      auto multiply = [&](const v8bf (&fl)[C][NL], int r) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          v8bf fv[3];
#pragma unroll
          for (int k = 0; k < 3; ++k) fv[k] = *reinterpret_cast<const v8bf *>(&lds.terms[k][16 * i + fr][r + 8 * fc]);
#pragma unroll
          for (int h = 0; h < C; ++h) mul_terms<false, NL, 3>(acc[i][h], fl[h], fv);
        }
      };
      auto part = [&](const Part &p, int r) {
        v8bf fl[C][NL];
        if constexpr (STAGED) {
          p.s.store(buf);
          stage_sync();
#pragma unroll
          for (int s = 0; s < RS / 32; ++s) {
            if (r + 32 * s >= g.R) break;
#pragma unroll
            for (int h = 0; h < C; ++h) frag_of(SL::frag(buf, 16 * h + fr, s), fl[h]);
            multiply(fl, r + 32 * s);
          }
          stage_sync();
        } else {
#pragma unroll
          for (int h = 0; h < C; ++h) {
            if constexpr (KC) frag_of(p.k[h], fl[h]);
            else frag_of_rows(p.r, h, fl[h]);
          }
          multiply(fl, r);
        }
      };
      load(next, o0 + STEP);
      __builtin_amdgcn_sched_barrier(0);
      part(now.l, 0);
      if constexpr (RL > RS) {
#pragma unroll 1
        for (int r = RS; r < g.R; r += RS) {
          load_part(now.l, o0, r);
          part(now.l, r);
        }
      }
      // (a product that is infinite or no number has a factor that is)
      float most = 0.f;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int h = 0; h < C; ++h)
#pragma unroll
          for (int q = 0; q < 4; q += 2) most = __builtin_fmaf(acc[i][h][q], acc[i][h][q + 1], most);
      const bool again = __ballot(!lin_finite(most));
      // a tile of 16 tokens at a time, rows of 64 columns and 4 more
      float *rows = (float *)buf;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        if (16 * i >= it.count) break;
#pragma unroll
        for (int h = 0; h < C; ++h) {
          if constexpr (KC) {
            *reinterpret_cast<v4f *>(rows + fr * 68 + 16 * h + 4 * fc) = acc[i][h];
          } else {
            // columns 4 (4 fc + q) + h
            *reinterpret_cast<v4f *>(rows + fr * 68 + 16 * fc + 4 * h) = v4f{acc[i][0][h], acc[i][1][h], acc[i][2][h], acc[i][3][h]};
          }
        }
        stage_sync();
        if (again) {
#pragma unroll 1
          for (int s = 0; s < 16 && 16 * i + s < it.count; ++s) {
            float &at = rows[s * 68 + lane];
            if (o0 + lane < g.N && !lin_finite(at)) at = short_again(g, it, lds, 16 * i + s, o0 + lane);
          }
          stage_sync();
        }
#pragma unroll
        for (int q = 0; q < OUT; ++q) {
          const int s = out_row(i, q);
          float f[VY];
#pragma unroll
          for (int j = 0; j < VY; j += 4) {
            const v4f v = *reinterpret_cast<const v4f *>(rows + (s - 16 * i) * 68 + yc + j);
#pragma unroll
            for (int k = 0; k < 4; ++k) f[j + k] = __builtin_fmaf(c, v[k], g.res ? now.z[i][q].get(j + k) : 0.f);
          }
          if (s >= it.count) continue;
          TY *at = (TY *)g.y + token[i][q] * g.ldy + o0 + yc;
          if (cols >= VY) {
            Words<TY, VY> out;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if constexpr (sizeof(TY) == 4) out.w[k] = bits_of(f[k]);
              else out.w[k] = bits_of(from_f32<TY>(f[2 * k])) | bits_of(from_f32<TY>(f[2 * k + 1])) << 16;
            }
            __builtin_memcpy(at, out.w, 16);
          } else {
#pragma unroll
            for (int j = 0; j < VY; ++j)
              if (j < cols) at[j] = from_f32<TY>(f[j]);
          }
        }
        stage_sync();
      }
    };
    Columns a, b;
    load(a, o0);
    for (;;) {
      columns(a, b, o0);
      if ((o0 += STEP) >= g.N) break;
      columns(b, a, o0);
      if ((o0 += STEP) >= g.N) break;
    }
  }

  // tokens without an adapter among the 64 from s0 on, e: this lane's id (any id behind the last token)
  __device__ __forceinline__ static void rest(const LoraArgs &g, int s0, int e) {
    constexpr int U = 8, STEP = 64 * LORA_WAVES;
    uint64_t todo = __ballot((unsigned)e >= (unsigned)g.n);
    while (todo) {
      const int k = __builtin_ctzll(todo);
      todo &= todo - 1;
      const int64_t s = s0 + k;
      const bool none = __builtin_amdgcn_readlane(e, k) < 0;
      const float fill = none ? 0.f : __builtin_nanf("");
      for (int64_t o0 = threadIdx.x; o0 < g.N; o0 += U * STEP) {
        TY v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = from_f32<TY>(fill);
        if (none && g.res) {  // (all asked for before the first is waited for)
#pragma unroll
          for (int u = 0; u < U; ++u) v[u] = ((const TY *)g.res)[s * g.ldr + min(o0 + u * STEP, g.N - 1)];
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (o0 + u * STEP < g.N) ((TY *)g.y)[s * g.ldy + o0 + u * STEP] = v[u];
      }
      if (g.v)
        for (int r = threadIdx.x; r < g.R; r += STEP) g.v[(size_t)s * g.R + r] = fill;
    }
  }
};
template <class TX, class TW, bool KC, int NF, int RL, class TY>
__global__ __launch_bounds__(64 * LORA_WAVES) void k_lora(LoraArgs g) {
  typedef Lora<TX, TW, KC, NF, RL, TY> L;
  __shared__ __attribute__((aligned(16))) typename L::Lds lds;
  const int lane = threadIdx.x & 63;
  const int s0 = min((int)blockIdx.x * g.rest, g.S), s = s0 + lane;
  const int e = lane < g.rest && s < g.S ? g.ids[s] : 0;  // (asked for here already)
  LoraItem it;
  if (lora_item(g, blockIdx.x, it)) {
    if (it.count <= 16) L::template run<1>(g, it, lds);
    else L::template run<2>(g, it, lds);
  }
  if (g.phase == LoraArgs::LONG || blockIdx.y) return;
  L::rest(g, s0, e);
}

// ============================================================ sums over an adapter's tokens
//
// result[e][r][j] = c[e] sum over its tokens of a[s][r] m[s][j], or with r and j changed (BY_R, dB's order).  A workgroup
// takes an adapter, 64 columns j, 16 NR of r and a slice of its tokens; its waves take 32 tokens in turn, and their sums
// meet in LDS.  Both operands are summed over their rows in memory; a step's rows are on their way while the one before it
// is multiplied.
struct LoraSumArgs {
  const float *a;        // [S][R]
  const void *m;
  int64_t ldm, N;
  int R, n, slices, chunks;  // slices of tokens, chunks of r
  const float *scale;
  float *out;            // [slices][n][R][N], or [slices][n][N][R]
};
template <class TM, int NR, bool BY_R>
__device__ __forceinline__ void lora_sums_wg(const LoraSumArgs &g, const LoraItems &items, unsigned b,
                                             float (&red)[LORA_WAVES][4][256]) {
  constexpr int NM = terms_beside<TM, float>(), NF = 4, STEP = 32 * LORA_WAVES;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), fr = lane & 15, fc = lane >> 4;
  const unsigned cols = (unsigned)((g.N + 63) / 64);
  const int64_t j0 = (int64_t)(b % cols) * 64;
  b /= cols;
  const int r0 = (int)(b % g.chunks) * 16 * NR;
  b /= g.chunks;
  const int z = (int)(b % g.slices), e = (int)(b / g.slices);
  const int count = items.counts[e], per = ((count + g.slices - 1) / g.slices + 31) & ~31;
  const int t0 = min(z * per, count), t1 = min(t0 + per, count);
  const int32_t *tokens = items.tokens + ((size_t)items.first[e] << items.n_items[1]);
  // (the scale of an adapter without tokens may be no number: its sums are zero all the same; slices are joined before it;
  // asked for beside the count)
  const float by = g.scale && g.slices == 1 ? g.scale[e] : 1.f, c = count ? by : 1.f;
  v4f acc[NR][NF];
#pragma unroll
  for (int h = 0; h < NR; ++h)
#pragma unroll
    for (int f = 0; f < NF; ++f) acc[h][f] = v4f{0.f, 0.f, 0.f, 0.f};
  const int64_t j = min(j0 + NF * fr, g.N - 1);
  const int jl = (int)min(g.N - j, (int64_t)NF);
  const int r = min(r0 + NR * fr, g.R - 1), rl = min(g.R - r, NR);
  const float *a = g.a + r;
  const TM *m = (const TM *)g.m + j;
  struct Step {
    Words<float, NR> a[8];
    Words<TM, NF> m[8];
  };
  // the 32 tokens at t (of those past t1, which take no part, the last one's)
  auto load = [&](Step &p, int t, auto whole) {
    constexpr bool WHOLE = decltype(whole)::value;
    int s[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) s[k] = tokens[min(t + 8 * fc + k, t1 - 1)];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const bool in = WHOLE || t + 8 * fc + k < t1;
      load_words(p.a[k], a + (int64_t)s[k] * g.R, WHOLE ? NR : in ? rl : 0, g.a);
      load_words(p.m[k], m + (int64_t)s[k] * g.ldm, WHOLE ? NF : in ? jl : 0, (const TM *)g.m);
    }
  };
  auto multiply = [&](const Step &p) {
    v8bf fm[NF][NM];
#pragma unroll
    for (int f = 0; f < NF; ++f) frag_of_rows(p.m, f, fm[f]);
#pragma unroll
    for (int h = 0; h < NR; ++h) {
      v8bf fa[3];
      frag_of_rows(p.a, h, fa);
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        if constexpr (BY_R) mul_terms<false, 3, NM>(acc[h][f], fa, fm[f]);
        else mul_terms<false, NM, 3>(acc[h][f], fm[f], fa);
      }
    }
  };
  int t = t0 + 32 * wave;
  Step p, q;
  if (j0 + 64 <= g.N && r0 + 16 * NR <= g.R && t + 32 <= t1) {  // whole steps, the next one on its way
    load(p, t, std::true_type());
    for (;;) {
      load(q, t + STEP, std::true_type());
      __builtin_amdgcn_sched_barrier(0);
      multiply(p);
      if ((t += STEP) + 32 > t1) break;
      load(p, t + STEP, std::true_type());
      __builtin_amdgcn_sched_barrier(0);
      multiply(q);
      if ((t += STEP) + 32 > t1) break;
    }
  }
  for (; t < t1; t += STEP) {
    load(p, t, std::false_type());
    multiply(p);
  }
  float *out = g.out + ((size_t)z * g.n + e) * g.R * g.N;
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
    auto result = [&](int t, auto again) {  // whether it is finite
      const int jr = BY_R ? t >> 4 : t & 63, ri = BY_R ? t & 15 : t >> 6;  // j - j0, and r = r0 + NR ri + h
      const int f = jr & 3, row = BY_R ? ri : jr >> 2, col = BY_R ? jr >> 2 : ri;
      const int k = 64 * (row & 3) + 16 * (row >> 2) + col;
      const int64_t jj = j0 + jr;
      const int rr = r0 + NR * ri + h;
      if (jj >= g.N || rr >= g.R) return true;
      float v = 0.f;
#pragma unroll
      for (int u = 0; u < LORA_WAVES; ++u) v += red[u][f][k];
      const bool finite = lin_finite(v);
      if (decltype(again)::value) {
        if (finite) return true;
        v = 0.f;
        for (int t = t0; t < t1 && v == v; ++t) {
          const int64_t s = tokens[t];
          v = __builtin_fmaf(g.a[s * g.R + rr], to_f32(((const TM *)g.m)[s * g.ldm + jj]), v);
        }
      }
      out[BY_R ? (size_t)jj * g.R + rr : (size_t)rr * g.N + jj] = c * v;
      return finite;
    };
    bool finite = true;
    for (int t = threadIdx.x; t < NF * 256; t += 64 * LORA_WAVES) finite &= result(t, std::false_type());
    if (__ballot(!finite)) {  // those that are not, value by value, as in the products
#pragma unroll 1
      for (int t = threadIdx.x; t < NF * 256; t += 64 * LORA_WAVES) result(t, std::true_type());
    }
  }
}
// dA by the first `na` workgroups, dB by the others: what they wait for is the same.  `first`: of this launch
template <class TX, class TY, int NR>
__global__ __launch_bounds__(64 * LORA_WAVES) void k_lora_sums(LoraItems items, LoraSumArgs a, LoraSumArgs b, unsigned na,
                                                               unsigned first) {
  __shared__ float red[LORA_WAVES][4][256];
  const unsigned wg = first + blockIdx.x;
  if (wg < na) lora_sums_wg<TX, NR, false>(a, items, wg, red);
  else lora_sums_wg<TY, NR, true>(b, items, wg - na, red);
}

// ============================================================ few tokens
//
// A workgroup takes a token and 512 columns: it computes all of the token's v (a wave NR rows of A at a time, 16 loads of
// them in flight), which costs reading A once for each 512 columns but no second launch, then a column a thread.
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
template <class TX, class TW, int NR>
__global__ __launch_bounds__(512) void k_lora_few(LoraFewArgs g) {
  constexpr int V = 16 / (int)sizeof(TW), U = 16 / NR;
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
  for (int r = NR * wave; r < g.R; r += 8 * NR) {
    const TW *w[NR];
#pragma unroll
    for (int h = 0; h < NR; ++h) w[h] = a + min(r + h, g.R - 1) * g.lda;
    float acc[NR] = {};
    for (int k0 = lane * V; k0 + V <= K; k0 += U * 64 * V) {
      v4u rw[U][NR];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = k0 + u * 64 * V;
#pragma unroll
        for (int h = 0; h < NR; ++h)
          rw[u][h] = k + V <= K ? *reinterpret_cast<const v4uu *>(w[h] + k) : v4u{0, 0, 0, 0};
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = k0 + u * 64 * V;
        if (k + V > K) break;
        TX f[V];
        __builtin_memcpy(f, x + k, sizeof(f));
#pragma unroll
        for (int h = 0; h < NR; ++h) {
          TW t[V];
          __builtin_memcpy(t, &rw[u][h], 16);
#pragma unroll
          for (int j = 0; j < V; ++j) acc[h] = __builtin_fmaf(to_f32(t[j]), to_f32(f[j]), acc[h]);
        }
      }
    }
    const int last = K / V * V + lane;
    if (last < K)
#pragma unroll
      for (int h = 0; h < NR; ++h) acc[h] = __builtin_fmaf(to_f32(w[h][last]), to_f32(x[last]), acc[h]);
    float v = 0.f;
#pragma unroll
    for (int h = 0; h < NR; ++h) {
      const float s = group_sum<64>(acc[h]);
      v = lane == h ? s : v;
    }
    if (lane < NR && r + lane < g.R) vs[r + lane] = v;
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

// the kernels by their operands' types: of the rows, the adapters and the result
void lora_forward(int x_type, int w_type, int y_type, const LoraArgs &g, dim3 grid, hipStream_t st);
void lora_backward(int x_type, int w_type, int y_type, const LoraArgs &g, dim3 grid, hipStream_t st);
void lora_sums(int x_type, int dy_type, const LoraItems &items, const LoraSumArgs &a, unsigned na, const LoraSumArgs &b,
               unsigned nb, hipStream_t st);
void lora_few(int x_type, int w_type, const LoraFewArgs &g, dim3 grid, hipStream_t st);
template <class TX, class TW, bool KC, class TY>
void lora_launch(const LoraArgs &g, dim3 n, hipStream_t st) {
  const dim3 wg(64 * LORA_WAVES);
  if (g.R <= 16) hipLaunchKernelGGL((k_lora<TX, TW, KC, 1, 32, TY>), n, wg, 0, st, g);
  else if (g.R <= 32) hipLaunchKernelGGL((k_lora<TX, TW, KC, 2, 32, TY>), n, wg, 0, st, g);
  else if (g.R <= 64) hipLaunchKernelGGL((k_lora<TX, TW, KC, 4, 64, TY>), n, wg, 0, st, g);
  else hipLaunchKernelGGL((k_lora<TX, TW, KC, 4, 256, TY>), n, wg, 0, st, g);
}
// r of a workgroup of sums: 16, 32 or 64
inline int lora_r_of(int R) { return R <= 16 ? 16 : R <= 32 ? 32 : 64; }

}  // namespace zm
