// Attention of a ragged batch's new rows over a paged KV cache.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = e^(scale q.k_j - m),  max(0, pos - window + 1) <= j <= pos,
//
// one pass over the keys with a running maximum m and sum, cut into spans of keys whose
// results are merged.
//
//  k_paged_tile   up to 32 (row, head) pairs of a kv head: single tokens, or a few
//                 (item_by_tile).  Bound by memory: 48 tokens over up to 4096 keys, 14B class, bf16,
//                 458 MB in 92 to 97 us; 32 tokens over up to 4096 keys in fp32, 8 kv heads of 128
//                 dims, 5.1 TB/s, 2 of 512 dims, 5.6 TB/s (a large copy: 4.6 TB/s).  8-bit pools: the 48 tokens'
//                 237 MB in 44 us (5.4 TB/s); one token over 131065 keys, 2 kv heads of 128 dims, capped, 69 MB in 21 us.
//  k_paged_block  longer chunks, and single tokens beside them (item_by_block, item_by_tile).
//                 Bound by the matrix cores: 4096 rows over 16384 keys, 14B class, bf16 (three
//                 products a multiplication): 2.7 to 2.9 ms among other calls (2.9 to 3.1 in ten
//                 passes under the profiler), 1.3 PFLOP/s of bf16 products, MFMA busy 56% of the time
//                 at 2.1 GHz (a large bf16 matrix product: 1.2 PFLOP/s).  8-bit pools (two products): e4m3 2.29 to
//                 2.33 ms, int8 2.36, with a cap 3.27 and 3.38 ms; capped over bf16 3.3 ms, fp16 2.45, fp32 5.6.
//  k_paged_merge  the spans' results (k_paged_merge_cols: of many spans a row, over 8-bit pools or capped).
#pragma once
#include <cmath>
#include <type_traits>

#include "devutil.h"
#include "paged.h"

namespace ms {

constexpr int kTile = 32;  // keys of a tile

struct PagedAttnArgs {
  const float *q;
  float *out;
  size_t q_ld, out_ld;
  const void *k, *v;
  const int32_t *pages;
  int stride;             // pages per sequence of the table
  const PagedItem *items;
  int n_kv, G, window, page_size, page_rows;
  FastDiv by_page, by_g;  // n / page_size, n / G
  // The scores' scale, log2(e) in it (capped scores: over the cap), is q_scale (0.5 to 1 in size) times s_scale (a power
  // of two).
  float q_scale, s_scale;
  float *part_o, *part_ml;  // [part][kv head][part_rows][head dim], [part][kv head][part_rows][2]
  int part_rows;          // (row, head) pairs of the longest item
  const float *k_scale, *v_scale;  // 8-bit pools: [page][kv head][slot]
  int hp_log;             // 8-bit pools, item_by_tile: log2 of the kv heads of a block
  // Capped scores: log2(e) times the cap is cap_p[0] (0.5 to 1) times cap_to (a power of two; 0: not
  // capped); cap_p[1..5] the coefficients of tanh's near form, times cap_p[0]; cap_2 is
  // 2 cap_p[0] in log2, inv_2 its inverse (cap_args).
  float cap_to, cap_p[6], cap_2, inv_2;
};

// The split of the batch's work for a shape of layers (made anew after each set).  tail: a last turn of whole spans that
// does not fill the blocks is cut; count: the plan says whether sequences share pages.
int plan_for(ms_paged_batch *b, int G, int rows, bool block, int n_kv, int window, int blocks,
             int tile_cost, int merge_cost, bool tail, bool count, PagedPlan **out);

// The launches of pools of 8 bits (dtype MS_KV_E4M3, MS_KV_I8; scores capped or not) and of the other pools
// with capped scores: each in a source of its own.
int launch_attn_e4m3(PagedAttnArgs &a, ms_paged_batch *b, int hd, int most, hipStream_t st);
int launch_attn_i8(PagedAttnArgs &a, ms_paged_batch *b, int hd, int most, hipStream_t st);
int launch_attn_capped(PagedAttnArgs &a, ms_paged_batch *b, int dtype, int hd, int most, hipStream_t st);

namespace {

template <int DT>
__device__ inline float load_kv(const void *pool, size_t at) {
  if constexpr (DT == MS_KV_F32)
    return ldg<float>(static_cast<const float *>(pool) + at);
  else if constexpr (DT == MS_KV_BF16)
    return __uint_as_float((uint32_t)ldg<uint16_t>(static_cast<const uint16_t *>(pool) + at) << 16);
  else if constexpr (DT == MS_KV_F16)
    return (float)ldg<_Float16>(static_cast<const _Float16 *>(pool) + at);
  else if constexpr (DT == MS_KV_E4M3)
    return __builtin_amdgcn_cvt_f32_fp8(ldg<uint8_t>(static_cast<const uint8_t *>(pool) + at), 0);
  else
    return (float)ldg<int8_t>(static_cast<const int8_t *>(pool) + at);
}

typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr float kLow = -0x1.fffffep+127f;  // running maximum before the first key
// The maximum that scores are taken against may lag behind by this much (log2): a
// probability is at most 2^kLag.
constexpr float kLag = 8.0f;

// How a pool's type is multiplied.  Operands are 16-bit MFMA parts: part b of a pool's value
// times part a of q or of a probability, for a + b less than the parts of these.
//   bf16  q and p in three bf16 parts (all 24 bits), the pool's value as it is
//   fp32  three bf16 parts each, six products (what is dropped is below 2^-25)
//   fp16  q and p in two fp16 parts (22 bits): q scaled by a power of two to below 2^15, p by
//         2^kLift, so that what falls below fp16's smallest step is below 2^-32 of the largest
//   8-bit the codes, which fp16 holds exactly, and two fp16 parts of q and of p times the values'
//         scales, in 2^-7 of a power of two that is at most twice the largest of these products so far
//         (a scale's head has a code of full size, so that what is lost is below 2^-31 of that too; a large scale of a key
//         that weighs nothing takes no bits from the others).  The keys' scales multiply the scores.  (Three bf16 parts of p times the scales as they are: the chunk of 4096 rows over 16384
//         keys 2.60 ms, so 2.53, before its last spans were cut and its keys loaded earlier)
template <int DT>
struct Form {
  static constexpr bool E8 = DT == MS_KV_E4M3 || DT == MS_KV_I8;
  static constexpr int ES = DT == MS_KV_F32 ? 4 : E8 ? 1 : 2;  // bytes of a pool's value
  static constexpr bool F16 = DT == MS_KV_F16 || E8;           // fp16 parts
  static constexpr bool LIFT = DT == MS_KV_F16;                // the sum of p too is lifted
  static constexpr int QP = F16 ? 2 : 3, KP = DT == MS_KV_F32 ? 3 : 1;
};
constexpr float kLift = 7.0f;
constexpr float kRoom = 0x1p8f;  // 2^(7 + 8) is below fp16's largest

template <bool F16>
__device__ inline uint32_t pack2(float a, float b) {
  if constexpr (F16)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), half2_t));
  else
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), bf2));
}
template <bool F16>
__device__ inline f2 unpack2(uint32_t x) {
  if constexpr (F16)
    return __builtin_convertvector(__builtin_bit_cast(half2_t, x), f2);
  else
    return f2{__uint_as_float(x << 16), __uint_as_float(x & 0xFFFF0000u)};
}
// Two values in N parts, rounded to nearest: part i to p[i * step].
template <bool F16, int N>
__device__ inline void split2(float a, float b, uint32_t *p, int step) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    p[i * step] = pack2<F16>(a, b);
    if (i + 1 < N) {
      const f2 u = unpack2<F16>(p[i * step]);
      a -= u.x;
      b -= u.y;
    }
  }
}
// Four 8-bit codes as fp16: those of bytes 0 and 1 to lo, 2 and 3 to hi.
template <int DT>
__device__ inline void codes4(uint32_t w, uint32_t *lo, uint32_t *hi) {
  if constexpr (DT == MS_KV_E4M3) {
    *lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false));
    *hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true));
  } else {
    // 1024 + (c + 128) has c + 128 in fp16's low bits
    constexpr half2_t off = {(_Float16)1152.f, (_Float16)1152.f};
    w ^= 0x80808080u;
    *lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - off);
    *hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - off);
  }
}
template <bool F16>
__device__ inline f4 mfma(u4 a, u4 b, f4 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a),
                                                  __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a),
                                                   __builtin_bit_cast(bf8, b), c, 0, 0, 0);
}
// Over the lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ inline float max_groups(float v) {
  unsigned x = __float_as_uint(v);
  auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  x = __float_as_uint(v);
  r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float sum_groups(float v) {
  unsigned x = __float_as_uint(v);
  auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  x = __float_as_uint(v);
  r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Capped scores: c tanh(z), c = cap_p[0].  To |z| = 0.6, z2 < kNear, c z (1 + z^2 P(z^2)), P a polynomial fitted here
// by least squares, reweighted until its largest relative error (3e-9) is least: scores far below the cap keep
// all their bits.  Past it c - 2 c t / (1 + t), t = e^(-2 z); scores near the cap are told apart by the second term: as
// 32-bit numbers of the cap's size (50: 72 in log2) each would be off by up to 4e-6.
constexpr float kNear = 0.36f;
inline void cap_args(PagedAttnArgs *a, float cap) {
  constexpr double p[6] = {1, -0.333332986, 0.133319244, -0.0537838228, 0.0207959525, -0.00589513639};
  int e = 0;
  const double c = cap * 1.4426950408889634, part = std::frexp(c, &e);
  a->cap_to = (float)std::ldexp(1.0, e);
  for (int i = 0; i < 6; ++i) a->cap_p[i] = (float)(part * p[i]);
  a->cap_2 = (float)std::log2(2 * part);
  a->inv_2 = (float)(0.5 / part);
}
// Both less h.
__device__ inline float cap_near(const PagedAttnArgs &a, float z, float h) {
  const float z2 = z * z;
  float p = a.cap_p[5];
#pragma unroll
  for (int i = 4; i > 0; --i) p = __builtin_fmaf(p, z2, a.cap_p[i]);
  return __builtin_fmaf(z * z2, p, __builtin_fmaf(z, a.cap_p[0], -h));
}
__device__ inline float cap_any(const PagedAttnArgs &a, float z, float h) {
  // (2 c t; 2^100: the second term is 2 c)
  const float t = __builtin_amdgcn_exp2f(fminf(__builtin_fmaf(z, -2.f * 1.44269504f, a.cap_2), 100.f));
  const float far = __builtin_fmaf(-t, __builtin_amdgcn_rcpf(__builtin_fmaf(t, a.inv_2, 1.f)), a.cap_p[0] - h);
  return z * z >= kNear ? far : cap_near(a, z, h);
}

// Of an 8-bit pool's scales: where that of a page's slot is.
__device__ inline size_t scale_at(const PagedAttnArgs &a, int page, int slot, int kvh) {
  return ((size_t)page * a.n_kv + kvh) * a.page_rows + slot;
}

// The item's rows one after the other, key by key, with NT threads: a key that a row does
// not attend to is not multiplied by anything.
template <int HD, int DT, int NT, bool CAP>
__device__ __forceinline__ void item_by_key(const PagedAttnArgs &a, const PagedItem &it, int kvh,
                                         int most, float *lds) {
  constexpr int ND = (HD + NT - 1) / NT, NW = NT / 64;
  float *p_of = lds, *red = lds + NT;  // probabilities of NT keys (-1: not attended); 2 NW
  const int tid = threadIdx.x;
  const int nrows = min(most, it.n_new * a.G - it.r0);
  for (int r = 0; r < nrows; ++r) {
    const int t = (it.r0 + r) / a.G, h = (it.r0 + r) % a.G;
    const int pos = it.len - it.n_new + t;
    const int lo = a.window && pos - a.window + 1 > 0 ? pos - a.window + 1 : 0;
    const float *q = a.q + (size_t)(it.row + t) * a.q_ld + (size_t)(kvh * a.G + h) * HD;
    float m = -INFINITY, l = 0.f, o[ND] = {};
    for (int k0 = it.k0; k0 < it.k1; k0 += NT) {
      const int key = k0 + tid;
      const bool on = key < it.k1 && key >= lo && key <= pos;
      float s = 0.f;
      if (on) {
        const uint32_t pg = div_by(key, a.by_page);
        const size_t row = (size_t)a.pages[(size_t)it.seq * a.stride + pg] * a.page_rows +
                           (key - pg * a.page_size);
        const size_t at = (row * a.n_kv + kvh) * HD;
        for (int d = 0; d < HD; ++d) s += q[d] * a.q_scale * load_kv<DT>(a.k, at + d);
        if constexpr (Form<DT>::E8)
          s *= ldg<float>(a.k_scale + scale_at(a, a.pages[(size_t)it.seq * a.stride + pg], key - pg * a.page_size, kvh));
        s *= a.s_scale;
        if constexpr (CAP) s = a.cap_to * cap_any(a, s, 0.f);
      }
      float mx = on ? s : -INFINITY;
      for (int off = 1; off < 64; off <<= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
      if ((tid & 63) == 0) red[tid >> 6] = mx;
      __syncthreads();
      mx = red[0];
      for (int w = 1; w < NW; ++w) mx = fmaxf(mx, red[w]);
      const float mn = fmaxf(m, mx), base = mn == -INFINITY ? 0.f : mn;
      // (lifted like the tiles' probabilities: parts of both kinds are merged)
      const float p = on ? __builtin_amdgcn_exp2f(Form<DT>::LIFT ? s - base + kLift : s - base) : 0.f;
      p_of[tid] = on ? p : -1.f;
      float sum = p;
      for (int off = 1; off < 64; off <<= 1) sum += __shfl_xor(sum, off, 64);
      if ((tid & 63) == 0) red[NW + (tid >> 6)] = sum;
      __syncthreads();
      const float al = __builtin_amdgcn_exp2f(m - base);
      l *= al;
      for (int w = 0; w < NW; ++w) l += red[NW + w];
#pragma unroll
      for (int i = 0; i < ND; ++i) o[i] *= al;
      m = mn;
      for (int j = 0; j < NT && k0 + j < it.k1; ++j) {
        float pj = p_of[j];
        if (pj == -1.f) continue;
        const uint32_t pg = div_by(k0 + j, a.by_page);
        const size_t row = (size_t)a.pages[(size_t)it.seq * a.stride + pg] * a.page_rows +
                           (k0 + j - pg * a.page_size);
        const size_t at = (row * a.n_kv + kvh) * HD;
        if constexpr (Form<DT>::E8)
          pj *= ldg<float>(a.v_scale + scale_at(a, a.pages[(size_t)it.seq * a.stride + pg], k0 + j - pg * a.page_size, kvh));
#pragma unroll
        for (int i = 0; i < ND; ++i)
          if (tid + NT * i < HD) o[i] += pj * load_kv<DT>(a.v, at + tid + NT * i);
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      const int d = tid + NT * i;
      if (d >= HD) continue;
      if (it.part < 0) {
        a.out[(size_t)(it.row + t) * a.out_ld + (size_t)(kvh * a.G + h) * HD + d] = o[i] / l;
      } else {
        const size_t pr = ((size_t)it.part * a.n_kv + kvh) * a.part_rows + r;
        a.part_o[pr * HD + d] = o[i];
        if (d == 0) {
          a.part_ml[pr * 2] = m;
          a.part_ml[pr * 2 + 1] = l;
        }
      }
    }
  }
}

// A tile's probabilities as the operand of the second product, from its scores: t = s sc - m,
// m the running maximum, in log2; p = 2^t.  `edge`: some row does not attend to some key.
// m serves all of a query's keys and may lag behind by kLag, so that a tile needs neither a
// cross-lane maximum nor a rescaling of the sums, unless a score exceeds it.  sc is a power of two, so
// that s sc is exact: t of the key that m was raised to is 0 whatever the scores' size.  (With a rounded
// product in m and not in t it was off by up to half of m's last place: from 2^29 on rows came out
// as 0 or NaN.)
// span(n, &low, &high): the keys that the lane's query of query tile n attends to.
// ks, vs: an 8-bit pool's scales of keys 4 g .. 4 g + 3 of both half tiles; vtop: the power of two that the query's probabilities
// times these are taken in; none is above kRoom of it.  CAP: the scores are capped.  l_far: 8-bit pools and
// capped scores, the sums of the tiles but for the last sixteen (fold).
template <int DT, bool CAP, int NQ, int ND, class Span>
__device__ __forceinline__ void probabilities(const PagedAttnArgs &a, f4 (&s)[2][NQ], int kb, bool edge,
                                              const float (&scale)[NQ], const f4 (&ks)[2], const f4 (&vs)[2],
                                              const Span &span, float (&vtop)[NQ], float (&m)[NQ], float (&l)[NQ], float (&l_far)[NQ],
                                              f4 (&o)[NQ][ND], uint32_t (&pf)[NQ][Form<DT>::QP][4]) {
  constexpr bool F16 = Form<DT>::F16, E8 = Form<DT>::E8;
  float sc[NQ], z2 = 0.f;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    sc[n] = CAP ? a.cap_to : scale[n];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (E8) s[i][n] *= ks[i];
      if constexpr (CAP) {
        s[i][n] *= scale[n];
#pragma unroll
        for (int e = 0; e < 4; ++e) z2 = fmaxf(z2, s[i][n][e] * s[i][n][e]);
      }
    }
  }
  // A lane that has a score of query n past kNear takes all eight in their distance to the cap, `from`: cap - m is exact
  // where m is near it, and t then has an error of its own size.  (The lane's smaller scores are off by up to 2^-25 of the
  // cap, what those at half of it are in any case; the smaller the less they weigh beside the one past it.)
  float from[NQ] = {};
  const int g = (threadIdx.x & 63) >> 4;
  // (both forms for each score of every tile: 4096 rows over 16384 keys, 14B class, i8, 3.5 ms; the near one alone
  // where a tile's scores allow it, 3.2 ms; uncapped 2.5 ms, all before the values' unit went by the products)
  if constexpr (CAP) {
    if (__any(z2 >= kNear)) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        float most = 0.f;
        if (edge) {  // (of keys that the query attends to)
          int low, high;
          span(n, &low, &high);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int key = kb + 16 * (j >> 2) + 4 * g + (j & 3);
            most = fmaxf(most, key > high || key < low ? 0.f : s[j >> 2][n][j & 3]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) most = fmaxf(most, s[j >> 2][n][j & 3]);
        }
        const float h = most * most >= kNear ? a.cap_p[0] : 0.f;
        from[n] = h * a.cap_to;
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j >> 2][n][j & 3] = cap_any(a, s[j >> 2][n][j & 3], h);
      }
    } else {
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j >> 2][n][j & 3] = cap_near(a, s[j >> 2][n][j & 3], 0.f);
    }
  }
  float t[NQ][8], top = -INFINITY;
#pragma unroll
  for (int n = 0; n < NQ; ++n)
#pragma unroll
    for (int j = 0; j < 8; ++j) t[n][j] = __builtin_fmaf(s[j >> 2][n][j & 3], sc[n], CAP ? from[n] - m[n] : -m[n]);
  if (edge) {
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      int low, high;
      span(n, &low, &high);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = kb + 16 * (j >> 2) + 4 * g + (j & 3);
        if (key > high || key < low) t[n][j] = -INFINITY;
      }
    }
  }
#pragma unroll
  for (int n = 0; n < NQ; ++n)
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, t[n][j]);
  if (__any(top > kLag)) {
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      // (from the scores: beside kLow they are lost in t)
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        mx = fmaxf(mx, t[n][j] == -INFINITY ? -INFINITY
                       : CAP                ? __builtin_fmaf(s[j >> 2][n][j & 3], sc[n], from[n])
                                            : s[j >> 2][n][j & 3] * sc[n]);
      const float mn = fmaxf(m[n], max_groups(mx)), al = __builtin_amdgcn_exp2f(m[n] - mn);
      m[n] = mn;
      l[n] *= al;
      if constexpr (E8 || CAP) l_far[n] *= al;
      float by = al;
      if constexpr (E8) {  // (vtop falls with the products: what is left of al is 1 to 2)
        const float now = vtop[n] * al;
        const uint32_t u = __float_as_uint(now);
        by = now < 0x1p-119f ? now * 0x1p119f : __uint_as_float((u & 0x7FFFFFu) | 0x3F800000u);
        vtop[n] = fmaxf(0x1p-119f, __uint_as_float(u & 0x7F800000u));
      }
#pragma unroll
      for (int d = 0; d < ND; ++d) o[n][d] *= by;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (t[n][j] != -INFINITY) t[n][j] = __builtin_fmaf(s[j >> 2][n][j & 3], sc[n], CAP ? from[n] - mn : -mn);
    }
  }
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    float *p = t[n];
#pragma unroll
    for (int j = 0; j < 8; ++j) p[j] = __builtin_amdgcn_exp2f(Form<DT>::LIFT ? p[j] + kLift : p[j]);
    l[n] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
    if constexpr (E8)
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] *= vs[j >> 2][j & 3];
  }
  if constexpr (E8) {
    float big[NQ];
    bool more = false;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      big[n] = 0.f;  // (a key that is masked: 0, or NaN, which is no maximum)
#pragma unroll
      for (int j = 0; j < 8; ++j) big[n] = fmaxf(big[n], t[n][j]);
      more |= big[n] > kRoom * vtop[n];
    }
    if (__any(more))
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const uint32_t up = (__float_as_uint(max_groups(big[n])) + 0x7FFFFFu) & 0x7F800000u;
        const float to = fmaxf(vtop[n], __uint_as_float(up)), f = vtop[n] / to;
        vtop[n] = to;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[n][d] *= f;
      }
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const float by = __uint_as_float(((254u + (int)kLift) << 23) - __float_as_uint(vtop[n]));  // 2^kLift / vtop
#pragma unroll
      for (int j = 0; j < 8; ++j) t[n][j] *= by;
    }
  }
#pragma unroll
  for (int n = 0; n < NQ; ++n)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      split2<F16, Form<DT>::QP>(t[n][2 * j], t[n][2 * j + 1], &pf[n][0][j], 4);
}

// Every sixteenth of a wave's tiles.  One key may weigh as much as all others: added one after the other to a sum of its
// size the tiles lost up to half of its last place each (16,000 rows over 65,536 keys: 2.8e-6 of the result, so 0.7e-6; where
// all keys but the first are alike 8e-5, so below 1e-5).  (The plain calls add them up as they come, and keep their results to
// the last bit.)
template <int DT, bool CAP, int NQ>
__device__ __forceinline__ void fold(int nth, float (&l)[NQ], float (&l_far)[NQ]) {
  if (!(Form<DT>::E8 || CAP) || (nth & 15) != 0) return;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    l_far[n] += l[n];
    l[n] = 0.f;
  }
}

// 2^k that brings the largest of fp16 queries' values below 2^15, and its inverse.
__device__ inline void lift_of(float big, float *up, float *down) {
  int e = big > 0.f && big < INFINITY ? 14 + 127 - (int)((__float_as_uint(big) >> 23) & 255) : 0;
  e = max(-126, min(126, e));
  *up = __uint_as_float((uint32_t)(127 + e) << 23);
  *down = __uint_as_float((uint32_t)(127 - e) << 23);
}

// What a query's products are multiplied by (waves that share its dims have them brought down already).  Capped: finite, so
// that a score of 0 stays 0 however far q is from the cap; and a value of its own: the compiler else moves the
// kernel's arguments about it to LDS (1890 rows of 256 dims, bf16: 41 to 52 us).
template <int DT, bool CAP, int SP>
__device__ inline float score_scale(float s_scale, float down) {
  constexpr bool OWN = Form<DT>::F16 && SP == 1;  // a lane's query's
  float s = OWN ? s_scale * down : s_scale;
  if constexpr (CAP && OWN) {
    s = fminf(s, 0x1p127f);
    asm volatile("" : "+v"(s));
  } else if constexpr (CAP) {
    asm volatile("" : "+s"(s));
  }
  return s;
}

// KS 32-dim steps of a query's dims from qp on (that lane's eight of each; WIDE: its sixteen of two), times `scale` (0.5 to 1 in
// size; one rounding), in parts, as the first product's operand; 0 where the query is not real.  What
// their product has to be multiplied by, a power of two: *down.
template <int DT, int KS, bool WIDE = false>
__device__ __forceinline__ void load_q(const float *qp, bool real, float scale,
                                       u4 (&q)[KS][Form<DT>::QP], float *down) {
  constexpr bool F16 = Form<DT>::F16;
  constexpr int QP = Form<DT>::QP;
  f4 x[KS][2];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int at = WIDE ? 64 * (ks / 2) + 8 * (ks % 2) : 32 * ks;
    x[ks][0] = ldg<f4>(qp + at);
    x[ks][1] = ldg<f4>(qp + at + 4);
  }
  __builtin_amdgcn_sched_barrier(0);
  float up = 1.f;
  *down = 1.f;
  if constexpr (F16) {
    float big = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int j = 0; j < 8; ++j) big = fmaxf(big, fabsf(x[ks][j >> 2][j & 3]));
    lift_of(max_groups(big), &up, down);
  }
  // (a factor of 0 in place of a choice for each value: an item beside a row whose q is not finite may
  // then be done again key by key)
  up = real ? up * scale : 0.f;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    uint32_t p[QP][4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      split2<F16, QP>(x[ks][j >> 1][2 * (j & 1)] * up, x[ks][j >> 1][2 * (j & 1) + 1] * up, &p[0][j], 4);
#pragma unroll
    for (int i = 0; i < QP; ++i) q[ks][i] = u4{p[i][0], p[i][1], p[i][2], p[i][3]};
  }
}

// Waves that share a tile in item_by_tile: 128 dims each at most, so that a wave's registers hold its
// whole tile.
template <int HD>
constexpr int tile_split() {
  return HD <= 128 ? 1 : HD / 128;
}
// Dims of a value row that a lane of item_by_tile loads at once: 16 bytes, 8 at head dim 64 (8-bit pools: half
// of that, so that 16 lanes have a row).
template <int HD, int DT>
__host__ __device__ constexpr int v_dims() {
  return DT == MS_KV_F32 || HD == 64 ? 4 : 8;
}

// The attention of one item of at most 16 NQ (row, head) pairs: the block's W waves, in groups of
// SP that divide the head's dims, take its 32-key tiles in turn, each with sums of its own that are
// joined at the end.  K and V come from the pages straight into the registers that the
// MFMAs take them from; LDS carries only the groups' scores.
//
// v_mfma_f32_16x16x32: lane l holds A[l % 16][8 (l / 16) + j], B[8 (l / 16) + j][l % 16] and
// D[4 (l / 16) + e][l % 16].
//   S^T = K Q^T     A: lane l loads 8 dims of key l % 16 of a half tile (16 bytes of bf16; of 8-bit codes
//                   the 16 dims of two steps: which dims a step takes is free, q's are taken alike).
//                   D: lane l has the scores of query l % 16 with keys 4 (l / 16) + e.
//   O^T = V^T P^T   B is those probabilities as they are: k index 8 (l / 16) + j stands for
//                   key 4 (l / 16) + j of the first half tile (j < 4) or key
//                   4 (l / 16) + j - 4 of the second.  A: lane l loads VD dims of its eight keys
//                   and turns them in its registers: MFMA t of a chunk of 16 VD dims takes
//                   dim VD (l % 16) + t.  D: dims VD (4 (l / 16) + e) + t of query l % 16.
// A value that is not finite makes the sums it is multiplied into not finite, with the
// zeros of masked keys too; where the end finds such a sum the item is done again key by
// key.
template <int HD, int DT, int NQ, int W, bool CAP, bool ONCE>
__device__ __forceinline__ void item_by_tile(const PagedAttnArgs &a, const PagedItem &it, int kvh0,
                                             int hp_log, char *lds) {
  using F = Form<DT>;
  constexpr bool F16 = F::F16;
  constexpr int SP = tile_split<HD>(), HW = HD / SP;
  constexpr bool E8 = F::E8;
  constexpr int QP = F::QP, KP = F::KP, KS = HW / 32, ES = F::ES;
  constexpr int KL = E8 ? KS / 2 : KS, KB = E8 ? 64 : 32 * ES;  // loads of 16 or 32 bytes of a key, bytes between them
  constexpr int VD = v_dims<HD, DT>(), CD = 16 * VD, NC = HW / CD;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c16 = lane & 15, g = lane >> 4;
  // kv head, group of the waves of its head, part of the head's dims
  const int hp = E8 && SP == 1 ? hp_log : 0, NG = W / SP >> hp;
  const int kvh = kvh0 + (wave & ((1 << hp) - 1)), grp = wave / SP >> hp, part = wave % SP;
  const int nrows = min(16 * NQ, it.n_new * a.G - it.r0), base = it.len - it.n_new;
  const int t_first = (int)div_by(it.r0, a.by_g), t_last = (int)div_by(it.r0 + nrows - 1, a.by_g);
  const int low_key = a.window ? max(it.k0, base + t_first - a.window + 1) : it.k0;
  const int n_tiles = (it.k1 - it.k0 + kTile - 1) / kTile;

  // row of key kb + (lane & 31), never one outside the attended keys
  const int32_t *pages = a.pages + (size_t)it.seq * a.stride;
  auto find = [&](int tile, int *page, int *slot) {
    const int key = min(max(it.k0 + min(tile, n_tiles - 1) * kTile + (lane & 31), low_key), it.k1 - 1);
    const int pg = (int)div_by((uint32_t)key, a.by_page);
    *slot = key - pg * a.page_size;
    *page = ldg<int32_t>(pages + pg);
  };
  int page, slot;
  find(grp, &page, &slot);
  const uint32_t row_bytes = (uint32_t)a.n_kv * HD * ES;
  constexpr int LD8 = E8 ? 16 : 8;  // dims of a key's load
  const char *kb0 = static_cast<const char *>(a.k) + ((size_t)kvh * HD + HW * part + LD8 * g) * ES;
  const char *vb0 = static_cast<const char *>(a.v) + ((size_t)kvh * HD + HW * part + VD * c16) * ES;
  // The next tile's keys are loaded once this one's are multiplied, its values once these are, where
  // there are registers for it (not for fp32 pools and one query tile: 160 us with spills, 118 us with
  // the tile's own loads in it; 32 tokens over 4096 keys, 8 kv heads of 128 dims).  Of those the compiler
  // issues four of a tile's keys at a time, between the products, and most of the values behind them:
  // where a block has one tile that chain is most of its time.
  constexpr bool AHEAD = E8 || (F16 ? NQ == 1 : ES == 2 || NQ == 2);
  u4 kr[2][KL][ES == 4 ? 2 : 1];
  std::conditional_t<E8, u2, u4> vr[8][NC];
  auto load_k = [&](int row) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const char *p = kb0 + (uint64_t)(uint32_t)__shfl(row, 16 * i + c16, 64) * row_bytes;
#pragma unroll
      for (int ks = 0; ks < KL; ++ks)
#pragma unroll
        for (int j = 0; j < (ES == 4 ? 2 : 1); ++j) kr[i][ks][j] = ldg<u4>(p + ks * KB + 16 * j);
    }
  };
  // 8-bit values that no other item reads are not kept in the caches, where those that are still to come are looked
  // for; 14B class, 48 tokens over up to 4096 and 16384 keys, e4m3, not in the caches before: 56 to 52 and 190 to 175 us (two
  // heads of 256 dims that are: 28 to 30 us; the keys too: 56 and 185; rows of 64 bytes: 36 to 37).  Where sequences share
  // pages they are kept (PagedPlan::shared): 48 tokens over 4096 keys, the first of them the same pages for all, 29% of these
  // read again 80 us past the caches and 83 kept, 49% 77 and 77, 73% 72 and 70, 93% 68 and 62; the first the same for two or
  // four sequences, 25% 85 and 84, 45% 83 to 85 and 80; 15,000 shared by 48, 244 and 198.
  auto get_v = [&](const char *p) {
    if constexpr (ONCE)
      return __builtin_nontemporal_load(reinterpret_cast<const u2 *>(p));
    else
      return ldg<u2>(p);
  };
  auto load_v = [&](int row) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const char *p = vb0 + (uint64_t)(uint32_t)__shfl(row, 16 * (j >> 2) + 4 * g + (j & 3), 64) * row_bytes;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if constexpr (E8 && VD == 8) {
          vr[j][c] = get_v(p + c * CD);
        } else if constexpr (E8) {
          vr[j][c] = u2{ldg<uint32_t>(p + c * CD), 0};
        } else if constexpr (VD * ES == 16) {
          vr[j][c] = ldg<u4>(p + c * CD * ES);
        } else {
          const u2 y = ldg<u2>(p);
          vr[j][0] = u4{y[0], y[1], 0, 0};
        }
      }
    }
  };
  int ahead = grp;
  float scl = 0.f;  // the scale of key lane of the next tile, of value lane - 32
  auto next = [&]() {  // pool row of the lane's key of the next tile
    const int row = page * a.page_rows + slot;
    if constexpr (E8) scl = ldg<float>((lane < 32 ? a.k_scale : a.v_scale) + scale_at(a, page, slot, kvh));
    find(ahead += NG, &page, &slot);
    return row;
  };
  int row;
  if (AHEAD && grp < n_tiles) {
    row = next();
    load_k(row);
    load_v(row);
  }

  // ---- q
  float sc[NQ], down[NQ];
  u4 q[NQ][KS][QP];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int r = 16 * n + c16;
    const bool real = r < nrows;
    const int t = real ? (int)div_by(it.r0 + r, a.by_g) : t_first, h = real ? it.r0 + r - t * a.G : 0;
    const float *qp = a.q + (size_t)(it.row + t) * a.q_ld + (size_t)(kvh * a.G + h) * HD + LD8 * g;
    load_q<DT, KS, E8>(qp + HW * part, real, a.q_scale, q[n], &down[n]);
    sc[n] = score_scale<DT, CAP, SP>(a.s_scale, down[n]);
  }

  f4 o[NQ][NC * VD] = {};
  float m[NQ], l[NQ], l_far[NQ], vtop[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    m[n] = kLow;
    l[n] = l_far[n] = 0.f;
    vtop[n] = 0x1p-119f;
  }
  auto span = [&](int n, int *low, int *high) {
    const int pos = base + (int)div_by(it.r0 + min(16 * n + c16, nrows - 1), a.by_g);
    *high = min(it.k1 - 1, pos);
    *low = a.window ? max(low_key, pos - a.window + 1) : low_key;
  };
  // keys that every row attends to
  const int all_lo = a.window ? max(low_key, base + t_last - a.window + 1) : low_key;
  const int all_hi = min(it.k1 - 1, base + t_first);
  f4 *xs = reinterpret_cast<f4 *>(lds);  // [2][wave][half][nq][64]
  for (int step = 0; step * NG < n_tiles; ++step) {
    const int tile = step * NG + grp, kb = it.k0 + tile * kTile;
    const bool work = SP == 1 || tile < n_tiles, more = tile + NG < n_tiles;
    if (SP == 1 && tile >= n_tiles) break;
    fold<DT, CAP, NQ>(step, l, l_far);
    f4 s[2][NQ] = {}, ks8[2] = {}, vs8[2] = {};
    if (work) {
      if (!AHEAD) {
        row = next();
        load_k(row);
        load_v(row);
      }
      if constexpr (E8)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          ks8[j >> 2][j & 3] = __shfl(scl, 16 * (j >> 2) + 4 * g + (j & 3), 64);
          vs8[j >> 2][j & 3] = __shfl(scl, 32 + 16 * (j >> 2) + 4 * g + (j & 3), 64);
        }
      // ---- scores (the products of the leading parts have a sum of their own: a running sum
      // that takes the small ones too rounds as often as there are products)
      f4 s_low[2][NQ] = {};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t kf[KP][4];
          if constexpr (E8) {
            codes4<DT>(kr[i][ks / 2][0][2 * (ks & 1)], &kf[0][0], &kf[0][1]);
            codes4<DT>(kr[i][ks / 2][0][2 * (ks & 1) + 1], &kf[0][2], &kf[0][3]);
          } else if constexpr (ES == 2) {
#pragma unroll
            for (int j = 0; j < 4; ++j) kf[0][j] = kr[i][ks][0][j];
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              split2<false, KP>(__uint_as_float(kr[i][ks][j / 2][2 * (j & 1)]),
                                __uint_as_float(kr[i][ks][j / 2][2 * (j & 1) + 1]), &kf[0][j], 4);
          }
#pragma unroll
          for (int pb = KP - 1; pb >= 0; --pb)
#pragma unroll
            for (int pa = QP - 1; pa >= 0; --pa) {
              if (pa + pb >= QP) continue;
#pragma unroll
              for (int n = 0; n < NQ; ++n) {
                f4 &d = (pa + pb ? s_low : s)[i][n];
                d = mfma<F16>(u4{kf[pb][0], kf[pb][1], kf[pb][2], kf[pb][3]}, q[n][ks][pa], d);
              }
            }
        }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int n = 0; n < NQ; ++n) s[i][n] += s_low[i][n];
      if (AHEAD && more) {
        row = next();
        load_k(row);
      }
    }
    if constexpr (SP > 1) {
      // (two buffers: the next step's scores do not wait for this one's readers)
      f4 *x = xs + (step & 1) * W * 2 * NQ * 64 + lane;
      if (work)
#pragma unroll
        for (int i = 0; i < 2 * NQ; ++i) x[(wave * 2 * NQ + i) * 64] = s[i / NQ][i % NQ] * down[i % NQ];
      __syncthreads();
      if (work)
#pragma unroll
        for (int i = 0; i < 2 * NQ; ++i) {
          f4 z = x[(grp * SP * 2 * NQ + i) * 64];
#pragma unroll
          for (int w = 1; w < SP; ++w) z += x[((grp * SP + w) * 2 * NQ + i) * 64];
          s[i / NQ][i % NQ] = z;
        }
    }
    if (!work) continue;
    uint32_t pf[NQ][QP][4];
    probabilities<DT, CAP, NQ>(a, s, kb, kb < all_lo || kb + kTile - 1 > all_hi, sc, ks8, vs8, span, vtop, m, l, l_far, o, pf);

    // ---- values
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      uint32_t vf[VD][KP][4];
      if constexpr (E8)
#pragma unroll
        for (int t = 0; t < VD; t += 2)
#pragma unroll
          for (int d = 0; d < 4; ++d)  // dims t and t + 1 of both keys, then each dim's pair
            codes4<DT>(__builtin_amdgcn_perm(vr[2 * d + 1][c][t / 4], vr[2 * d][c][t / 4],
                                                    t & 2 ? 0x07030602u : 0x05010400u),
                              &vf[t][0][d], &vf[t + 1][0][d]);
#pragma unroll
      for (int t = 0; t < (E8 ? 0 : VD); ++t)
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          if constexpr (ES == 2)
            vf[t][0][d] = __builtin_amdgcn_perm(vr[2 * d + 1][c][t / 2], vr[2 * d][c][t / 2],
                                                t & 1 ? 0x07060302u : 0x05040100u);
          else
            split2<false, KP>(__uint_as_float(vr[2 * d][c][t]), __uint_as_float(vr[2 * d + 1][c][t]),
                              &vf[t][0][d], 4);
        }
#pragma unroll
      for (int pa = QP - 1; pa >= 0; --pa)
#pragma unroll
        for (int pb = KP - 1; pb >= 0; --pb) {
          if (pa + pb >= QP) continue;
#pragma unroll
          for (int t = 0; t < VD; ++t)
#pragma unroll
            for (int n = 0; n < NQ; ++n)
              o[n][c * VD + t] = mfma<F16>(u4{vf[t][pb][0], vf[t][pb][1], vf[t][pb][2], vf[t][pb][3]},
                                           u4{pf[n][pa][0], pf[n][pa][1], pf[n][pa][2], pf[n][pa][3]},
                                           o[n][c * VD + t]);
        }
    }
    if (AHEAD && more) load_v(row);
  }

  // ---- the groups' sums joined
  int bad = 0;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    l[n] = sum_groups(E8 || CAP ? l[n] + l_far[n] : l[n]);
    bad |= !(fabsf(l[n]) < INFINITY);
    if constexpr (E8)
#pragma unroll
      for (int d = 0; d < NC * VD; ++d) o[n][d] *= vtop[n] * 0x1p-7f;
#pragma unroll
    for (int d = 0; d < NC * VD; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) bad |= !(fabsf(o[n][d][e]) < INFINITY);
  }
  // (also: every wave is done with xs)
  if (__syncthreads_or(bad)) {
    for (int h = 0; h < 1 << hp; ++h)
      item_by_key<HD, DT, 64 * W, CAP>(a, it, kvh0 + h, 16 * NQ, reinterpret_cast<float *>(lds));
    return;
  }
  float *ml = reinterpret_cast<float *>(lds);  // [2][group][head][16 NQ]
  constexpr int NS = W / SP;                   // groups by heads
  const int sub = wave & ((1 << hp) - 1);
  constexpr int LD = CD + 4, ROWS = 16 * NQ;
  float *os = ml + 2 * NS * ROWS;              // [wave][16][LD]
  if (g == 0 && part == 0)
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      ml[((grp << hp) + sub) * ROWS + 16 * n + c16] = m[n];
      ml[(NS + (grp << hp) + sub) * ROWS + 16 * n + c16] = l[n];
    }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    if (16 * n >= nrows) break;
    float top = kLow;
#pragma unroll
    for (int w = 0; w < NG; ++w) top = fmaxf(top, ml[((w << hp) + sub) * ROWS + 16 * n + c16]);
    const float f = __builtin_amdgcn_exp2f(m[n] - top);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (n + c) __syncthreads();
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int t = 0; t < VD; t += 4) {
          f4 x;
#pragma unroll
          for (int u = 0; u < 4; ++u) x[u] = o[n][c * VD + t + u][e] * f;
          *reinterpret_cast<f4 *>(os + (wave * 16 + c16) * LD + VD * (4 * g + e) + t) = x;
        }
      __syncthreads();
      for (int i0 = tid; i0 < 16 * SP * (CD / 4) << hp; i0 += 64 * W) {
        const int h_of = i0 & ((1 << hp) - 1), i = i0 >> hp;
        const int d = i % (CD / 4) * 4, pt = i / (CD / 4) % SP, r16 = i / (CD / 4 * SP), r = 16 * n + r16;
        if (r >= nrows) break;
        float mt = kLow, ls = 0.f;
#pragma unroll
        for (int w = 0; w < NG; ++w) mt = fmaxf(mt, ml[((w << hp) + h_of) * ROWS + r]);
        f4 x = {};
#pragma unroll
        for (int w = 0; w < NG; ++w) {
          const int at = (w << hp) + h_of;
          ls += ml[(NS + at) * ROWS + r] * __builtin_amdgcn_exp2f(ml[at * ROWS + r] - mt);
          x += *reinterpret_cast<const f4 *>(os + ((at * SP + pt) * 16 + r16) * LD + d);
        }
        const int dim = pt * HW + c * CD + d;
        if (it.part < 0) {
          const int t = (int)div_by(it.r0 + r, a.by_g), h = it.r0 + r - t * a.G;
          *reinterpret_cast<f4 *>(a.out + (size_t)(it.row + t) * a.out_ld + (size_t)((kvh0 + h_of) * a.G + h) * HD + dim) =
              x / ls;
        } else {
          const size_t pr = ((size_t)it.part * a.n_kv + kvh0 + h_of) * a.part_rows + r;
          *reinterpret_cast<f4 *>(a.part_o + pr * HD + dim) = x;
          if (dim == 0) {
            a.part_ml[pr * 2] = mt;
            a.part_ml[pr * 2 + 1] = ls;
          }
        }
      }
    }
  }
}

// How a block of item_by_block divides an item: W waves in groups of SP, a group having 16 NQ
// (row, head) pairs, each of its waves HD / SP dims of them.  A wave's share of q in parts and of
// the sums then stays in its registers (two waves a SIMD).
template <int HD, int DT>
struct Shape {
  // two query tiles a wave where the registers hold them: a fragment then serves six products
  static constexpr int NQ = HD == 64 || (HD == 128 && DT != MS_KV_F32) ? 2 : 1;
  // the fragments of K and V take turns in one buffer where LDS has no room for both (fp32, 512 dims:
  // 96 KB each; 1024 rows over 4096 keys, 8 heads: 0.57 ms, by item_by_tile 0.70 ms, with two waves a
  // group, whose registers spill, 1.0 ms)
  static constexpr bool ONE = HD == 512 && DT == MS_KV_F32;
  static constexpr int W = NQ == 2 ? 4 : 8, SP = ONE ? 4 : HD == 512 ? 2 : 1;
  static constexpr int PAIRS = 16 * NQ * W / SP;
  // dims of a value row a lane loads: 8-bit codes four at a time, and where that leaves waves without any, a
  // wave has half of a tile's keys
  static constexpr int VD = Form<DT>::E8 ? 4 : HD / (16 * W) < 2 ? 2 : HD / (16 * W);
  static constexpr int VH = Form<DT>::E8 && HD / (16 * VD) <= W / 2 ? 2 : 1;
  static constexpr int FRAG = kTile * HD * 2 * Form<DT>::KP;        // bytes of K's or V's fragments
  static constexpr int XS_AT = FRAG * (ONE ? 1 : 2), XS = SP > 1 ? W * NQ * 2 * 64 * 16 : 0;
  static constexpr int ROWS_AT = XS_AT + XS, SCL_AT = ROWS_AT + 2 * kTile * 4;
  static constexpr int USED = SCL_AT + (Form<DT>::E8 ? 4 * kTile * 4 : 0);
  static constexpr int OUT = W * 16 * (16 * VD + 4) * 4;
  static constexpr int LDS = USED > OUT ? USED : OUT;
};

// The attention of one item of a longer chunk.  The waves go over the item's 32-key tiles
// together: a tile's keys and values are loaded once for the block, in whole rows, and put
// into LDS as MFMA fragments (those of fp32 pools in parts): K as the rows lie, V turned in
// registers; the waves read both without bank conflicts.  (item_by_tile's loads of K take 16
// bytes of 16 rows a quarter wave, sixteen cache accesses where a row's take one or two; with
// many queries these accesses bound it.)  The next tile's rows are loaded beside the second
// product of this one and wait in registers; where its pages lie the first wave finds before its own
// first product, a load that it waits for.  Where a group has several waves each computes the scores over
// its dims, and all take the sum, in the same order.
template <int HD, int DT, bool CAP>
__device__ __forceinline__ void item_by_block(const PagedAttnArgs &a, const PagedItem &it, int kvh,
                                              char *lds) {
  using F = Form<DT>;
  using B = Shape<HD, DT>;
  constexpr bool F16 = F::F16;
  constexpr int NQ = B::NQ, W = B::W, SP = B::SP;
  constexpr bool E8 = F::E8;
  constexpr int QP = F::QP, KP = F::KP, KS = HD / 32, ES = F::ES;
  constexpr int VD = B::VD, CD = 16 * VD, NC = HD / CD;
  constexpr int KW = KS / SP, CW = NC / SP;  // a wave's 32-dim steps and chunks of CD dims
  constexpr int D8 = HD / 8, UK = kTile * D8 / (64 * W);  // K units of 8 dims a thread
  constexpr bool STRICT = KW * KP >= 8;
  constexpr int RING = 3;
  // 8-bit keys, few registers, are loaded from the time on that the last tile's are in LDS, so that the first
  // product and the softmax too lie before their use; their rows are then found two tiles ahead.
  // (4096 rows over 16384 keys, 14B class, e4m3: 2.48 -> 2.44 ms; 16-bit keys of 256 dims: no gain)
  constexpr bool EARLY = E8;
  static_assert(CW >= 1 && UK >= 1 && 64 * W / D8 * UK == kTile, "shape");
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c16 = lane & 15, g = lane >> 4;
  const int grp = wave / SP, part = wave % SP;
  const int nrows = min(B::PAIRS, it.n_new * a.G - it.r0), base = it.len - it.n_new;
  u4 *kf = reinterpret_cast<u4 *>(lds);                        // [half][ks][part][64], slots turned by (ks, g)
  u4 *vf = B::ONE ? kf : kf + B::FRAG / 16;                    // [c][t][part][64]
  f4 *xs = reinterpret_cast<f4 *>(lds + B::XS_AT);             // [wave][nq][half][64]
  uint32_t *rows = reinterpret_cast<uint32_t *>(lds + B::ROWS_AT);  // [2][32]
  float *scl = reinterpret_cast<float *>(lds + B::SCL_AT);     // [2][keys', values'][32]

  float sc[NQ], down[NQ], m[NQ], l[NQ], l_far[NQ], vtop[NQ];
  const int t_first = (int)div_by(it.r0, a.by_g), r_wave = 16 * NQ * grp;
  const int low_key = a.window ? max(it.k0, base + t_first - a.window + 1) : it.k0;
  const bool busy = r_wave < nrows;
  // the keys that all of this wave's rows attend to, and that any of them does
  const int tw0 = (int)div_by(it.r0 + r_wave, a.by_g);
  const int tw1 = (int)div_by(it.r0 + min(nrows, r_wave + 16 * NQ) - 1, a.by_g);
  const int all_lo = a.window ? max(low_key, base + tw1 - a.window + 1) : low_key;
  const int all_hi = min(it.k1 - 1, base + tw0), any_hi = min(it.k1 - 1, base + tw1);
  const int any_lo = a.window ? max(low_key, base + tw0 - a.window + 1) : low_key;
  const int n_tiles = (it.k1 - it.k0 + kTile - 1) / kTile;
  auto span = [&](int n, int *low, int *high) {
    const int r = min(r_wave + 16 * n + c16, nrows - 1), pos = base + (int)div_by(it.r0 + r, a.by_g);
    *high = min(it.k1 - 1, pos);
    *low = a.window ? max(low_key, pos - a.window + 1) : low_key;
  };
  const uint32_t row_bytes = (uint32_t)a.n_kv * HD * ES;
  const char *kb0 = static_cast<const char *>(a.k) + ((size_t)kvh * HD + 8 * (tid % D8)) * ES;
  const int v_chunk = wave / B::VH, v_half = wave % B::VH;
  const char *vb0 = static_cast<const char *>(a.v) + ((size_t)kvh * HD + v_chunk * CD + VD * c16) * ES;
  // Pool row of a tile's key `tid`, never one outside the attended keys; two tiles' rows in LDS.
  // Those of the next (EARLY: of the one behind it, in place of this one's) are written between the two barriers of a
  // tile, in place of the last's, whose readers are past the first of them.
  float k_scl = 0.f, v_scl = 0.f;  // of the next tile's key `tid`
  size_t scl_from = 0;
  auto find = [&](int tile) {
    const int key = min(max(it.k0 + tile * kTile + tid, low_key), it.k1 - 1);
    const int pg = (int)div_by((uint32_t)key, a.by_page);
    const int page = ldg<int32_t>(a.pages + (size_t)it.seq * a.stride + pg);
    if constexpr (E8) scl_from = scale_at(a, page, key - pg * a.page_size, kvh);
    return page * a.page_rows + key - pg * a.page_size;
  };
  auto load_scales = [&]() {
    k_scl = ldg<float>(a.k_scale + scl_from);
    v_scl = ldg<float>(a.v_scale + scl_from);
  };
  uint32_t kr[UK][ES * 2];      // 8 dims of a key
  uint32_t vr[8 / B::VH][VD * ES / 4];  // VD dims of eight keys (or four)
  auto load_k = [&](int tile) {
    const uint32_t *row = rows + (tile & 1) * kTile + tid / D8;
#pragma unroll
    for (int u = 0; u < UK; ++u) {
      const char *p = kb0 + (uint64_t)row[64 * W / D8 * u] * row_bytes;
      if constexpr (E8) {
        const u2 x = ldg<u2>(p);
        kr[u][0] = x[0];
        kr[u][1] = x[1];
      }
#pragma unroll
      for (int j = 0; j < ES / 2; ++j) {
        const u4 x = ldg<u4>(p + 16 * j);
#pragma unroll
        for (int e = 0; e < 4; ++e) kr[u][4 * j + e] = x[e];
      }
    }
  };
  auto load_v = [&](int tile) {
    const u4 *row = reinterpret_cast<const u4 *>(rows + (tile & 1) * kTile) + g;
    const u4 r0 = row[B::VH == 2 ? 4 * v_half : 0], r1 = row[4];
#pragma unroll
    for (int j = 0; j < 8 / B::VH; ++j) {
      const char *p = vb0 + (uint64_t)(j < 4 ? r0[j & 3] : r1[j & 3]) * row_bytes;
      if constexpr (VD * ES == 4) {
        vr[j][0] = ldg<uint32_t>(p);
      } else if constexpr (VD * ES == 8) {
        const u2 x = ldg<u2>(p);
        vr[j][0] = x[0];
        vr[j][1] = x[1];
      } else {
#pragma unroll
        for (int i = 0; i < VD * ES / 16; ++i) {
          const u4 x = ldg<u4>(p + 16 * i);
#pragma unroll
          for (int e = 0; e < 4; ++e) vr[j][4 * i + e] = x[e];
        }
      }
    }
  };
  const bool v_busy = v_chunk < NC;
  if (tid < kTile) {
    rows[tid] = find(0);
    if constexpr (E8) load_scales();
    if constexpr (EARLY) rows[kTile + tid] = find(min(1, n_tiles - 1));
  }
  __syncthreads();
  load_k(0);
  if (v_busy) load_v(0);

  // ---- q, beside the first tile's loads
  u4 q[NQ][KW][QP];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int r = r_wave + 16 * n + c16;
    const bool real = r < nrows;
    const int t = real ? (int)div_by(it.r0 + r, a.by_g) : t_first, h = real ? (it.r0 + r) - t * a.G : 0;
    m[n] = kLow;
    l[n] = l_far[n] = 0.f;
    vtop[n] = 0x1p-119f;
    const float *qp = a.q + (size_t)(it.row + t) * a.q_ld + (size_t)(kvh * a.G + h) * HD + 8 * g;
    load_q<DT, KW>(qp + 32 * KW * part, real, a.q_scale, q[n], &down[n]);
    sc[n] = score_scale<DT, CAP, SP>(a.s_scale, down[n]);
  }
  f4 o[NQ][CW * VD] = {};
  for (int tile = 0; tile < n_tiles; ++tile) {
    const int kb = it.k0 + tile * kTile;
    if (B::ONE && tile) __syncthreads();
    fold<DT, CAP, NQ>(tile, l, l_far);
#pragma unroll
    for (int u = 0; u < UK; ++u) {
      const int key = (tid + 64 * W * u) / D8, d8 = tid % D8;
      u4 *dst = kf + (((key >> 4) * KS + (d8 >> 2)) * KP) * 64 + (d8 & 3) * 16 + ((key ^ d8) & 15);
      if constexpr (E8) {
        u4 x;
        uint32_t lo, hi;
        codes4<DT>(kr[u][0], &lo, &hi);
        x[0] = lo;
        x[1] = hi;
        codes4<DT>(kr[u][1], &lo, &hi);
        x[2] = lo;
        x[3] = hi;
        dst[0] = x;
      } else if constexpr (ES == 2) {
        dst[0] = u4{kr[u][0], kr[u][1], kr[u][2], kr[u][3]};
      } else {
        uint32_t p[KP][4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          split2<false, KP>(__uint_as_float(kr[u][2 * j]), __uint_as_float(kr[u][2 * j + 1]), &p[0][j], 4);
#pragma unroll
        for (int i = 0; i < KP; ++i) dst[64 * i] = u4{p[i][0], p[i][1], p[i][2], p[i][3]};
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (E8 && tid < kTile) {
      // (two tiles' in turn: the scales of the last one are read until its barriers' end)
      scl[(tile & 1) * 2 * kTile + tid] = k_scl;
      scl[(tile & 1) * 2 * kTile + kTile + tid] = v_scl;
    }
    __syncthreads();
    int next = 0;
    if (tid < kTile) {
      if constexpr (EARLY) load_scales();
      next = find(min(tile + (EARLY ? 2 : 1), n_tiles - 1));
    }
    if (EARLY && tile + 1 < n_tiles) load_k(tile + 1);
    uint32_t pf[NQ][QP][4];
    f4 ks8[2] = {}, vs8[2] = {};
    if constexpr (E8)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        ks8[i] = *reinterpret_cast<const f4 *>(scl + (tile & 1) * 2 * kTile + 16 * i + 4 * g);
        vs8[i] = *reinterpret_cast<const f4 *>(scl + (tile & 1) * 2 * kTile + kTile + 16 * i + 4 * g);
      }
    f4 s[2][NQ] = {};
    const bool work = busy && kb <= any_hi && kb + kTile - 1 >= any_lo;
    const bool edge = kb < all_lo || kb + kTile - 1 > all_hi;
    if (work) {
      // (fragment by fragment, read RING - 1 ahead: over many of them the compiler, left to
      // itself, reads as far ahead as it can and runs out of registers)
      f4 s_low[NQ] = {};
      u4 x[RING];
      auto read = [&](int f) {
        const int i = f / (KW * KP), ks = KW * part + f / KP % KW, pb = KP - 1 - f % KP;
        x[f % RING] = kf[((i * KS + ks) * KP + pb) * 64 + g * 16 + ((c16 ^ (4 * ks + g)) & 15)];
      };
#pragma unroll
      for (int f = 0; f < RING - 1; ++f) read(f);
#pragma unroll
      for (int f = 0; f < 2 * KW * KP; ++f) {
        const int i = f / (KW * KP), ks = f / KP % KW, pb = KP - 1 - f % KP;
        if (f + RING - 1 < 2 * KW * KP) read(f + RING - 1);
#pragma unroll
        for (int pa = QP - 1; pa >= 0; --pa) {
          if (pa + pb >= QP) continue;
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            f4 &d = pa + pb ? s_low[n] : s[i][n];
            d = mfma<F16>(x[f % RING], q[n][ks][pa], d);
          }
        }
        if (ks == KW - 1 && pb == 0) {
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            s[i][n] += s_low[n];
            s_low[n] = f4{};
            if constexpr (SP > 1) xs[((wave * NQ + n) * 2 + i) * 64 + lane] = s[i][n] * down[n];
          }
        }
        if constexpr (STRICT) __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (SP == 1) probabilities<DT, CAP, NQ>(a, s, kb, edge, sc, ks8, vs8, span, vtop, m, l, l_far, o, pf);
    }
    if (B::ONE) __syncthreads();
    if (tid < kTile) rows[((tile + (EARLY ? 0 : 1)) & 1) * kTile + tid] = next;
    if (E8 && v_busy) {
#pragma unroll
      for (int t = 0; t < VD; t += 2) {
        uint32_t p[2][4 / B::VH];
#pragma unroll
        for (int d = 0; d < 4 / B::VH; ++d)
          codes4<DT>(__builtin_amdgcn_perm(vr[2 * d + 1][t / 4], vr[2 * d][t / 4],
                                                  t & 2 ? 0x07030602u : 0x05010400u), &p[0][d], &p[1][d]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          u4 *dst = vf + (v_chunk * VD + t + i) * 64 + lane;
          if constexpr (B::VH == 2)
            reinterpret_cast<u2 *>(dst)[v_half] = u2{p[i][0], p[i][1]};
          else
            *dst = u4{p[i][0], p[i][1], p[i][2], p[i][3]};
        }
      }
    }
    if (!E8 && v_busy) {
#pragma unroll
      for (int t = 0; t < VD; ++t) {
        uint32_t p[KP][4];
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          if constexpr (ES == 2)
            p[0][d] = __builtin_amdgcn_perm(vr[2 * d + 1][t / 2], vr[2 * d][t / 2],
                                            t & 1 ? 0x07060302u : 0x05040100u);
          else
            split2<false, KP>(__uint_as_float(vr[2 * d][t]), __uint_as_float(vr[2 * d + 1][t]), &p[0][d], 4);
        }
#pragma unroll
        for (int i = 0; i < KP; ++i)
          vf[((wave * VD + t) * KP + i) * 64 + lane] = u4{p[i][0], p[i][1], p[i][2], p[i][3]};
        if constexpr (ES == 4) __builtin_amdgcn_sched_barrier(0);
      }
    }
    __syncthreads();
    if (tile + 1 < n_tiles) {
      if constexpr (!EARLY) load_k(tile + 1);
      if (v_busy) load_v(tile + 1);
    }
    if (work) {
      if constexpr (SP > 1) {
#pragma unroll
        for (int w = 0; w < SP; ++w) {
#pragma unroll
          for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const f4 x = xs[(((grp * SP + w) * NQ + n) * 2 + i) * 64 + lane];
              s[i][n] = w ? s[i][n] + x : x;
            }
          __builtin_amdgcn_sched_barrier(0);
        }
        probabilities<DT, CAP, NQ>(a, s, kb, edge, sc, ks8, vs8, span, vtop, m, l, l_far, o, pf);
      }
      u4 x[RING];
      auto read = [&](int f) {
        x[f % RING] = vf[((CW * VD * part + f / KP) * KP + KP - 1 - f % KP) * 64 + lane];
      };
#pragma unroll
      for (int f = 0; f < RING - 1; ++f) read(f);
#pragma unroll
      for (int f = 0; f < CW * VD * KP; ++f) {
        const int d = f / KP, pb = KP - 1 - f % KP;
        if (f + RING - 1 < CW * VD * KP) read(f + RING - 1);
#pragma unroll
        for (int pa = QP - 1; pa >= 0; --pa) {
          if (pa + pb >= QP) continue;
#pragma unroll
          for (int n = 0; n < NQ; ++n)
            o[n][d] = mfma<F16>(x[f % RING], u4{pf[n][pa][0], pf[n][pa][1], pf[n][pa][2], pf[n][pa][3]}, o[n][d]);
        }
        if constexpr (STRICT) __builtin_amdgcn_sched_barrier(0);
      }
    }
  }

  // ---- every wave has its rows' sums
  int bad = 0;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    l[n] = sum_groups(E8 || CAP ? l[n] + l_far[n] : l[n]);
    bad |= !(fabsf(l[n]) < INFINITY);
    if constexpr (E8)
#pragma unroll
      for (int d = 0; d < CW * VD; ++d) o[n][d] *= vtop[n] * 0x1p-7f;
#pragma unroll
    for (int d = 0; d < CW * VD; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) bad |= !(fabsf(o[n][d][e]) < INFINITY);
  }
  if (__syncthreads_or(bad)) {
    item_by_key<HD, DT, 64 * W, CAP>(a, it, kvh, B::PAIRS, reinterpret_cast<float *>(lds));
    return;
  }
  // Through LDS, a wave's own part of it, so that rows are stored whole: a lane's dims are 16 bytes of
  // sixteen rows a quarter wave.
  constexpr int LD = CD + 4, C4 = CD / 4;
  static_assert(W * 16 * LD * 4 <= B::LDS, "LDS");
  int ln = lane;  // (an opaque copy: the addresses below are not made ahead of the loop)
  asm volatile("" : "+v"(ln));
  float *own = reinterpret_cast<float *>(lds) + wave * 16 * LD;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const float f = it.part < 0 ? 1.f / l[n] : 1.f;
#pragma unroll
    for (int c = 0; c < CW; ++c) {
#pragma unroll
      for (int e = 0; e < 4 * VD; e += 4) {  // dims VD (4 g + e / VD) + e % VD of the chunk
        f4 x;
#pragma unroll
        for (int u = 0; u < 4; ++u) x[u] = o[n][c * VD + (e + u) % VD][(e + u) / VD] * f;
        *reinterpret_cast<f4 *>(own + (ln & 15) * LD + 4 * VD * (ln >> 4) + e) = x;
      }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int j = 0; j < 16 * C4 / 64; ++j) {
        const int i = 64 * j + ln, r = r_wave + 16 * n + i / C4, d = CD * (CW * part + c) + i % C4 * 4;
        const f4 x = *reinterpret_cast<const f4 *>(own + i / C4 * LD + i % C4 * 4);
        if (r >= nrows) continue;
        const int t = (int)div_by(it.r0 + r, a.by_g), h = (it.r0 + r) - t * a.G;
        float *dst = it.part < 0 ? a.out + (size_t)(it.row + t) * a.out_ld + (size_t)(kvh * a.G + h) * HD
                                 : a.part_o + (((size_t)it.part * a.n_kv + kvh) * a.part_rows + r) * HD;
        *reinterpret_cast<f4 *>(dst + d) = x;
      }
      __builtin_amdgcn_wave_barrier();
    }
    const int r = r_wave + 16 * n + ln;
    if (it.part >= 0 && ln < 16 && part == 0 && r < nrows) {
      const size_t pr = ((size_t)it.part * a.n_kv + kvh) * a.part_rows + r;
      a.part_ml[pr * 2] = m[n];
      a.part_ml[pr * 2 + 1] = l[n];
    }
  }
}

template <int HD, int DT, int NQ, int W>
constexpr int tile_lds() {
  constexpr int x = tile_split<HD>() > 1 ? 2 * W * 2 * NQ * 64 * 16 : 0;
  constexpr int e = (32 * NQ * (W / tile_split<HD>()) + W * 16 * (16 * v_dims<HD, DT>() + 4)) * 4;
  return x > e ? x : e;
}

// Blocks go to the eight dies in turn: those of an item's heads to one die, whose cache then finds the rows of a page
// whole (8 heads of 64 dims in 8 bits, 48 tokens: 83 us where a die has one head of all items, 50 us; the items of the last
// groups of eight that are not whole as they come).
struct BlockOf {
  int item, head;
};
__device__ inline BlockOf block_of(int block, int n_blocks, int heads) {
  const int per = 8 * heads;
  if (block >= n_blocks / per * per) return {block / heads, block % heads};
  return {block / per * 8 + block % 8, block % per / 8};
}

// Items of at most 16 NQ pairs: single tokens, or a few of them.  (Two query tiles of three parts do
// not fit the registers of two waves a SIMD: with spills 110 us where one wave takes 72 us.)
template <int HD, int DT, int NQ, bool CAP, bool ONCE>
__global__ __launch_bounds__(256, NQ == 2 && DT != MS_KV_F16 ? 1 : 2) void k_paged_tile(PagedAttnArgs a) {
  __shared__ __align__(16) char lds[tile_lds<HD, DT, NQ, 4>()];
  if constexpr (Form<DT>::E8) {
    const BlockOf b = block_of(blockIdx.x, gridDim.x, a.n_kv >> a.hp_log);
    item_by_tile<HD, DT, NQ, 4, CAP, ONCE>(a, a.items[b.item], b.head << a.hp_log, a.hp_log, lds);
  } else {
    item_by_tile<HD, DT, NQ, 4, CAP, false>(a, a.items[blockIdx.x / a.n_kv], blockIdx.x % a.n_kv, 0, lds);
  }
}

// Items of longer chunks, and single tokens beside them: 47 of these over 4096 keys and a chunk of 128 rows, e4m3, 114 us,
// with their values kept in the caches 118.  (A chunk's last few rows, whose values its other items read: 129 rows of 8
// heads of 512 dims, 20 times, 590 us either way.)
template <int HD, int DT, bool CAP, int NT = 64 * Shape<HD, DT>::W>
__global__ __launch_bounds__(NT, 2) void k_paged_block(PagedAttnArgs a) {
  constexpr int A = tile_lds<HD, DT, 1, Shape<HD, DT>::W>(), B = Shape<HD, DT>::LDS;
  __shared__ __align__(16) char lds[A > B ? A : B];
  const PagedItem it = a.items[blockIdx.x / a.n_kv];
  if (it.n_new * a.G - it.r0 <= 16)
    item_by_tile<HD, DT, 1, Shape<HD, DT>::W, CAP, Form<DT>::E8>(a, it, blockIdx.x % a.n_kv, 0, lds);
  else
    item_by_block<HD, DT, CAP>(a, it, blockIdx.x % a.n_kv, lds);
}

// The parts of one result, weighted by e^(their maximum - the largest).  A block takes RPB rows,
// its NT threads being HD / 4 columns of RPB rows by GRP groups of parts: many rows of a few parts
// (chunks) or one row of many (a single token over a long context).  Bound by the launch and a chain of
// three loads: 3.5 to 4.2 us for a few parts, 5.9 us for 256 of a row, 9.2 us for 46 MB of them.
template <int HD, int NT>
__global__ __launch_bounds__(NT) void k_paged_merge(PagedAttnArgs a, const PagedMerge *merge, int rpb) {
  constexpr int COLS = HD / 4, ALL = NT / COLS;
  constexpr int AHEAD = 4;
  __shared__ f4 os[ALL][COLS];
  __shared__ f2 ls[ALL];
  const int tid = threadIdx.x, kvh = blockIdx.x % a.n_kv, col = tid % COLS, at = tid / COLS;
  const int gpr = ALL / rpb, row = at / gpr, grp = at % gpr, r = blockIdx.y * rpb + row;
  const PagedMerge g = merge[blockIdx.x / a.n_kv];
  const bool real = r < g.n_new * a.G - g.r0 && r < a.part_rows;
  const size_t step = (size_t)a.n_kv * a.part_rows;
  const size_t pr = ((size_t)g.part * a.n_kv + kvh) * a.part_rows + (real ? r : 0);
  const int n = real ? g.n : 0;
  // (maxima and sums come in the same round of loads: both are written by other dies)
  float m = kLow, l = 0.f;
  f4 o = {};
  const float *po = a.part_o + pr * HD + 4 * col;
  for (int p0 = grp; p0 < n; p0 += AHEAD * gpr) {
    f2 ml[AHEAD];
    f4 x[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int p = min(p0 + i * gpr, n - 1);
      ml[i] = ldg<f2>(a.part_ml + (pr + p * step) * 2);
      x[i] = ldg<f4>(po + p * step * HD);
      if (p0 + i * gpr >= n) ml[i].x = -INFINITY;
    }
    float mn = m;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) mn = fmaxf(mn, ml[i].x);
    const float f = __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    l *= f;
    o *= f;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (p0 + i * gpr >= n) continue;
      const float w = __builtin_amdgcn_exp2f(ml[i].x - mn);
      l += w * ml[i].y;
      o += w * x[i];
    }
  }
  if (gpr > 1) {
    os[at][col] = o;
    if (col == 0) ls[at] = f2{m, l};
    __syncthreads();
    if (grp) return;
    float top = m;
    for (int i = 1; i < gpr; ++i) top = fmaxf(top, ls[at + i].x);
    const float f = __builtin_amdgcn_exp2f(m - top);
    l *= f;
    o *= f;
    for (int i = 1; i < gpr; ++i) {
      const float w = __builtin_amdgcn_exp2f(ls[at + i].x - top);
      l += w * ls[at + i].y;
      o += w * os[at + i][col];
    }
  }
  if (!real) return;
  const int t = (int)div_by(g.r0 + r, a.by_g), h = g.r0 + r - t * a.G;
  *reinterpret_cast<f4 *>(a.out + (size_t)(g.row + t) * a.out_ld + (size_t)(kvh * a.G + h) * HD + 4 * col) =
      o / l;
}

// The same where a row has many parts: a block takes 32 dims of one row, its threads being 8 columns by 128
// groups of parts.  A block per row (k_paged_merge) reads all of the row's parts through one CU: 512 parts of 8 rows
// of 128 dims, 2 MB, 8.4 us; by four blocks each 5.5 us.
template <int HD>
__global__ __launch_bounds__(1024) void k_paged_merge_cols(PagedAttnArgs a, const PagedMerge *merge) {
  constexpr int W = 16, GRP = 128, AHEAD = 4;
  __shared__ f4 os[W][8];
  __shared__ f2 ls[W];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, kvh = blockIdx.x % a.n_kv;
  const int col = 8 * blockIdx.z + (tid & 7), r = blockIdx.y;
  const PagedMerge g = merge[blockIdx.x / a.n_kv];
  if (r >= g.n_new * a.G - g.r0 || r >= a.part_rows) return;
  const size_t step = (size_t)a.n_kv * a.part_rows;
  const size_t pr = ((size_t)g.part * a.n_kv + kvh) * a.part_rows + r;
  float m = kLow, l = 0.f;
  f4 o = {};
  // (weights are of what both have: a part that is not there has kLow, and 0 of everything)
  auto join = [&](float m2, float l2, f4 o2) {
    const float mn = fmaxf(m, m2), f = __builtin_amdgcn_exp2f(m - mn), w = __builtin_amdgcn_exp2f(m2 - mn);
    m = mn;
    l = l * f + l2 * w;
    o = o * f + o2 * w;
  };
  const float *po = a.part_o + pr * HD + 4 * col;
  for (int p0 = tid / 8; p0 < g.n; p0 += AHEAD * GRP) {
    f2 ml[AHEAD];
    f4 x[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int p = min(p0 + i * GRP, g.n - 1);
      ml[i] = ldg<f2>(a.part_ml + (pr + p * step) * 2);
      x[i] = ldg<f4>(po + p * step * HD);
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (p0 + i * GRP < g.n) join(ml[i].x, ml[i].y, x[i]);
  }
#pragma unroll
  for (int off = 8; off < 64; off <<= 1) {
    f4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = __shfl_xor(o[e], off, 64);
    join(__shfl_xor(m, off, 64), __shfl_xor(l, off, 64), y);
  }
  if (lane < 8) os[wave][lane] = o;
  if (lane == 0) ls[wave] = f2{m, l};
  __syncthreads();
  if (tid >= 8) return;
#pragma unroll
  for (int w = 1; w < W; ++w) join(ls[w].x, ls[w].y, os[w][tid]);
  const int t = (int)div_by(g.r0 + r, a.by_g), h = g.r0 + r - t * a.G;
  *reinterpret_cast<f4 *>(a.out + (size_t)(g.row + t) * a.out_ld + (size_t)(kvh * a.G + h) * HD + 4 * col) = o / l;
}

template <int HD, int DT, bool CAP>
int launch(PagedAttnArgs &a, ms_paged_batch *b, int most, hipStream_t st) {
  using B = Shape<HD, DT>;
  // Few pairs: tiles by a wave each, two query tiles of them to head dim 128 (32 sequences of 8 rows x
  // 4 heads over 4096 keys, bf16: 72 us against 104 us of the block's 128 pairs), 16 pairs an item
  // at larger ones, whose second item finds its keys in the caches (head dim 256: 44 us, 52 us with two
  // query tiles, 64 us by blocks).
  constexpr bool TWO = HD <= 128;
  const bool block = most > 32;
  const int rows = block ? B::PAIRS : most > 16 && TWO ? 32 : 16;
  PagedPlan *p = nullptr;
  // blocks that run at once; a step of single tokens takes a tile for every group of waves
  const int w = block ? B::W : 4;
  // 8-bit pools: a block's waves share two heads of 128 dims, four of 64, so that 256 bytes of a row are read about
  // at once
  if constexpr (Form<DT>::E8)
    if (!block)
      while (HD << a.hp_log < 256 && a.n_kv % (2 << a.hp_log) == 0) ++a.hp_log;
  const int cost = std::max(1, (4 << a.hp_log) * tile_split<HD>() / w);
  // A merge's launch takes 3.4 us; a step of a single token (4 in the plan's measure) 0.7 us at head dim 64,
  // 1.15 at 128 and 1.4 to 1.6 at 256 and 512 over 16-bit pools, 1.7 to 5 us over fp32 ones: one token over 250
  // keys of 64 dims (bf16) 5.4 us in one block a head, 9.0 us cut and merged; over 1500 keys 12.4 and 9.1 us.
  const int merge = block ? 8 : DT == MS_KV_F32 ? 4 : HD == 64 ? 20 : HD == 128 ? 12 : 8;
  // (pools and scores that the plain calls take keep their split, and so their results to the last bit)
  const bool tail = block && (Form<DT>::E8 || CAP);
  constexpr bool ONCE = Form<DT>::E8 && v_dims<HD, DT>() == 8;
  const bool count = ONCE && !block && (TWO || most <= 16);  // (of 17 to 32 pairs two items have the same keys)
  if (int rc = plan_for(b, a.G, rows, block, a.n_kv >> a.hp_log, a.window, 8 / w * ctx().n_cu, cost, merge, tail, count, &p))
    return rc;
  const bool once = count && !p->shared;
  a.part_rows = p->most;
  if (const size_t n = (size_t)p->n_parts * a.n_kv * a.part_rows) {
    void *buf = nullptr;
    if (int rc = scratch(n * (HD + 2) * 4, &buf)) return rc;
    a.part_o = static_cast<float *>(buf);
    a.part_ml = a.part_o + n * HD;
  }
  a.items = reinterpret_cast<const PagedItem *>(p->up.d);
  // (a launch has fewer than 2^32 threads)
  MS_CHECK_ARG((int64_t)p->n_items * a.n_kv * 64 * w < ((int64_t)1 << 32),
               "paged_attention: too many rows for one call");
  const dim3 grid(p->n_items * (a.n_kv >> a.hp_log));
  if (block) {
    hipLaunchKernelGGL((k_paged_block<HD, DT, CAP>), grid, dim3(64 * B::W), 0, st, a);
  } else if (rows == 16) {
    if (once)
      hipLaunchKernelGGL((k_paged_tile<HD, DT, 1, CAP, ONCE>), grid, dim3(256), 0, st, a);
    else
      hipLaunchKernelGGL((k_paged_tile<HD, DT, 1, CAP, false>), grid, dim3(256), 0, st, a);
  } else {
    if constexpr (TWO) {
      if (once)
        hipLaunchKernelGGL((k_paged_tile<HD, DT, 2, CAP, ONCE>), grid, dim3(256), 0, st, a);
      else
        hipLaunchKernelGGL((k_paged_tile<HD, DT, 2, CAP, false>), grid, dim3(256), 0, st, a);
    }
  }
  if (p->n_merge) {
    // about four parts a thread, more of them in a larger block
    const PagedMerge *merge = reinterpret_cast<const PagedMerge *>(p->up.d + p->merge_at);
    int rpb = 1024 / HD;
    while (rpb > 1 && 1024 / HD / rpb * 4 < p->most_parts) rpb /= 2;
    const dim3 mg(p->n_merge * a.n_kv, cdiv(p->most, rpb));
    // many parts of few rows: by several blocks a row where these are no more than compute units in all (48
    // sequences, 14B class, one of 131072 keys and 47 of 3000, int8: 131 us, with every row's so 143).  (The plain calls
    // keep their order of sums, and so their results to the last bit.)
    constexpr bool COLS = Form<DT>::E8 || CAP;
    if (1024 / HD * 4 >= p->most_parts) {
      hipLaunchKernelGGL((k_paged_merge<HD, 256>), mg, dim3(256), 0, st, a, merge, rpb);
    } else if (COLS && (int64_t)p->n_merge * a.n_kv * p->most <= ctx().n_cu) {
      if constexpr (COLS)
        hipLaunchKernelGGL(k_paged_merge_cols<HD>, dim3(p->n_merge * a.n_kv, p->most, HD / 32), dim3(1024), 0, st, a, merge);
    } else {
      hipLaunchKernelGGL((k_paged_merge<HD, 1024>), mg, dim3(1024), 0, st, a, merge, rpb);
    }
  }
  MS_HIP_TRY(hipGetLastError());
  return MS_OK;
}
template <int DT, bool CAP>
int launch_dims(PagedAttnArgs &a, ms_paged_batch *b, int hd, int most, hipStream_t st) {
  switch (hd) {
    case 64: return launch<64, DT, CAP>(a, b, most, st);
    case 128: return launch<128, DT, CAP>(a, b, most, st);
    case 256: return launch<256, DT, CAP>(a, b, most, st);
    default: return launch<512, DT, CAP>(a, b, most, st);
  }
}

}  // namespace
}  // namespace ms
