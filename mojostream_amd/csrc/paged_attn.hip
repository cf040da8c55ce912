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
//                 dims, 5.1 TB/s, 2 of 512 dims, 5.6 TB/s (a large copy: 4.6 TB/s).
//  k_paged_block  longer chunks, and single tokens beside them (item_by_block, item_by_tile).
//                 Bound by the matrix cores: 4096 rows over 16384 keys, 14B class, bf16 (three
//                 products a multiplication): 2.7 to 2.9 ms among other calls (2.9 to 3.1 in ten
//                 passes under the profiler), 1.3 PFLOP/s of bf16 products, MFMA busy 56% of the time
//                 at 2.1 GHz (a large bf16 matrix product: 1.2 PFLOP/s).
//  k_paged_merge  the spans' results.
#include <algorithm>
#include <cmath>
#include <exception>

#include "devutil.h"
#include "paged.h"

namespace ms {
namespace {

constexpr int kTile = 32;  // keys of a tile
constexpr int kMaxParts = 1024;  // about the most parts of one result

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
  // The scores' scale, log2(e) in it, is q_scale (0.5 to 1 in size) times s_scale (a power of two).
  float q_scale, s_scale;
  float *part_o, *part_ml;  // [part][kv head][part_rows][head dim], [part][kv head][part_rows][2]
  int part_rows;          // (row, head) pairs of the longest item
};

template <int DT>
__device__ inline float load_kv(const void *pool, size_t at) {
  if constexpr (DT == MS_KV_F32)
    return ldg<float>(static_cast<const float *>(pool) + at);
  else if constexpr (DT == MS_KV_BF16)
    return __uint_as_float((uint32_t)ldg<uint16_t>(static_cast<const uint16_t *>(pool) + at) << 16);
  else
    return (float)ldg<_Float16>(static_cast<const _Float16 *>(pool) + at);
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
// times part a of q or of a probability, for a + b < TERMS.
//   bf16  q and p in three bf16 parts (all 24 bits), the pool's value as it is
//   fp32  three bf16 parts each, six products (what is dropped is below 2^-25)
//   fp16  q and p in two fp16 parts (22 bits): q scaled by a power of two to below 2^15, p by
//         2^kLift, so that what falls below fp16's smallest step is below 2^-32 of the largest
template <int DT>
struct Form {
  static constexpr bool F16 = DT == MS_KV_F16;
  static constexpr int QP = F16 ? 2 : 3, KP = DT == MS_KV_F32 ? 3 : 1, TERMS = QP;
};
constexpr float kLift = 7.0f;

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

// The item's rows one after the other, key by key, with NT threads: a key that a row does
// not attend to is not multiplied by anything.
template <int HD, int DT, int NT>
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
        s *= a.s_scale;
      }
      float mx = on ? s : -INFINITY;
      for (int off = 1; off < 64; off <<= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
      if ((tid & 63) == 0) red[tid >> 6] = mx;
      __syncthreads();
      mx = red[0];
      for (int w = 1; w < NW; ++w) mx = fmaxf(mx, red[w]);
      const float mn = fmaxf(m, mx), base = mn == -INFINITY ? 0.f : mn;
      // (lifted like the tiles' probabilities: parts of both kinds are merged)
      const float p = on ? __builtin_amdgcn_exp2f(Form<DT>::F16 ? s - base + kLift : s - base) : 0.f;
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
        const float pj = p_of[j];
        if (pj == -1.f) continue;
        const uint32_t pg = div_by(k0 + j, a.by_page);
        const size_t row = (size_t)a.pages[(size_t)it.seq * a.stride + pg] * a.page_rows +
                           (k0 + j - pg * a.page_size);
        const size_t at = (row * a.n_kv + kvh) * HD;
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
template <int DT, int NQ, int ND, class Span>
__device__ __forceinline__ void probabilities(const f4 (&s)[2][NQ], int kb, bool edge,
                                              const float (&sc)[NQ], const Span &span,
                                              float (&m)[NQ], float (&l)[NQ], f4 (&o)[NQ][ND],
                                              uint32_t (&pf)[NQ][Form<DT>::QP][4]) {
  constexpr bool F16 = Form<DT>::F16;
  const int g = (threadIdx.x & 63) >> 4;
  float t[NQ][8], top = -INFINITY;
#pragma unroll
  for (int n = 0; n < NQ; ++n)
#pragma unroll
    for (int j = 0; j < 8; ++j) t[n][j] = __builtin_fmaf(s[j >> 2][n][j & 3], sc[n], -m[n]);
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
        mx = fmaxf(mx, t[n][j] == -INFINITY ? -INFINITY : s[j >> 2][n][j & 3] * sc[n]);
      const float mn = fmaxf(m[n], max_groups(mx)), al = __builtin_amdgcn_exp2f(m[n] - mn);
      m[n] = mn;
      l[n] *= al;
#pragma unroll
      for (int d = 0; d < ND; ++d) o[n][d] *= al;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (t[n][j] != -INFINITY) t[n][j] = __builtin_fmaf(s[j >> 2][n][j & 3], sc[n], -mn);
    }
  }
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    float *p = t[n];
#pragma unroll
    for (int j = 0; j < 8; ++j) p[j] = __builtin_amdgcn_exp2f(F16 ? p[j] + kLift : p[j]);
    l[n] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
#pragma unroll
    for (int j = 0; j < 4; ++j)
      split2<F16, Form<DT>::QP>(p[2 * j], p[2 * j + 1], &pf[n][0][j], 4);
  }
}

// 2^k that brings the largest of fp16 queries' values below 2^15, and its inverse.
__device__ inline void lift_of(float big, float *up, float *down) {
  int e = big > 0.f && big < INFINITY ? 14 + 127 - (int)((__float_as_uint(big) >> 23) & 255) : 0;
  e = max(-126, min(126, e));
  *up = __uint_as_float((uint32_t)(127 + e) << 23);
  *down = __uint_as_float((uint32_t)(127 - e) << 23);
}

// KS 32-dim steps of a query's dims from qp on (that lane's eight of each), times `scale` (0.5 to 1 in
// size; one rounding), in parts, as the first product's operand; 0 where the query is not real.  What
// their product has to be multiplied by, a power of two: *down.
template <int DT, int KS>
__device__ __forceinline__ void load_q(const float *qp, bool real, float scale,
                                       u4 (&q)[KS][Form<DT>::QP], float *down) {
  constexpr bool F16 = Form<DT>::F16;
  constexpr int QP = Form<DT>::QP;
  f4 x[KS][2];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    x[ks][0] = ldg<f4>(qp + 32 * ks);
    x[ks][1] = ldg<f4>(qp + 32 * ks + 4);
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
// Dims of a value row that a lane of item_by_tile loads at once: 16 bytes, 8 at head dim 64.
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
//   S^T = K Q^T     A: lane l loads 8 dims of key l % 16 of a half tile (16 bytes of bf16).
//                   D: lane l has the scores of query l % 16 with keys 4 (l / 16) + e.
//   O^T = V^T P^T   B is those probabilities as they are: k index 8 (l / 16) + j stands for
//                   key 4 (l / 16) + j of the first half tile (j < 4) or key
//                   4 (l / 16) + j - 4 of the second.  A: lane l loads VD dims of its eight keys
//                   and turns them in its registers: MFMA t of a chunk of 16 VD dims takes
//                   dim VD (l % 16) + t.  D: dims VD (4 (l / 16) + e) + t of query l % 16.
// A value that is not finite makes the sums it is multiplied into not finite, with the
// zeros of masked keys too; where the end finds such a sum the item is done again key by
// key.
template <int HD, int DT, int NQ, int W>
__device__ __forceinline__ void item_by_tile(const PagedAttnArgs &a, const PagedItem &it, int kvh,
                                             char *lds) {
  using F = Form<DT>;
  constexpr bool F16 = F::F16;
  constexpr int SP = tile_split<HD>(), NG = W / SP, HW = HD / SP;
  constexpr int QP = F::QP, KP = F::KP, KS = HW / 32, ES = DT == MS_KV_F32 ? 4 : 2;
  constexpr int VD = v_dims<HD, DT>(), CD = 16 * VD, NC = HW / CD;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c16 = lane & 15, g = lane >> 4;
  const int grp = wave / SP, part = wave % SP;
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
  const char *kb0 = static_cast<const char *>(a.k) + ((size_t)kvh * HD + HW * part + 8 * g) * ES;
  const char *vb0 = static_cast<const char *>(a.v) + ((size_t)kvh * HD + HW * part + VD * c16) * ES;
  // The next tile's keys are loaded once this one's are multiplied, its values once these are, where
  // there are registers for it (not for fp32 pools and one query tile: 160 us with spills, 118 us with
  // the tile's own loads in it; 32 tokens over 4096 keys, 8 kv heads of 128 dims).  Of those the compiler
  // issues four of a tile's keys at a time, between the products, and most of the values behind them:
  // where a block has one tile that chain is most of its time.
  constexpr bool AHEAD = F16 ? NQ == 1 : ES == 2 || NQ == 2;
  u4 kr[2][KS][ES / 2], vr[8][NC];
  auto load_k = [&](int row) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const char *p = kb0 + (uint64_t)(uint32_t)__shfl(row, 16 * i + c16, 64) * row_bytes;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int j = 0; j < ES / 2; ++j) kr[i][ks][j] = ldg<u4>(p + ks * 32 * ES + 16 * j);
    }
  };
  auto load_v = [&](int row) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const char *p = vb0 + (uint64_t)(uint32_t)__shfl(row, 16 * (j >> 2) + 4 * g + (j & 3), 64) * row_bytes;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if constexpr (VD * ES == 16) {
          vr[j][c] = ldg<u4>(p + c * CD * ES);
        } else {
          const u2 y = ldg<u2>(p);
          vr[j][0] = u4{y[0], y[1], 0, 0};
        }
      }
    }
  };
  int ahead = grp;
  auto next = [&]() {  // pool row of the lane's key of the next tile
    const int row = page * a.page_rows + slot;
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
    const float *qp = a.q + (size_t)(it.row + t) * a.q_ld + (size_t)(kvh * a.G + h) * HD + 8 * g;
    load_q<DT, KS>(qp + HW * part, real, a.q_scale, q[n], &down[n]);
    sc[n] = SP == 1 ? a.s_scale * down[n] : a.s_scale;
  }

  f4 o[NQ][NC * VD] = {};
  float m[NQ], l[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    m[n] = kLow;
    l[n] = 0.f;
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
    f4 s[2][NQ] = {};
    if (work) {
      if (!AHEAD) {
        row = next();
        load_k(row);
        load_v(row);
      }
      // ---- scores (the products of the leading parts have a sum of their own: a running sum
      // that takes the small ones too rounds as often as there are products)
      f4 s_low[2][NQ] = {};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t kf[KP][4];
          if constexpr (ES == 2) {
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
              if (pa + pb >= F::TERMS) continue;
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
    probabilities<DT, NQ>(s, kb, kb < all_lo || kb + kTile - 1 > all_hi, sc, span, m, l, o, pf);

    // ---- values
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      uint32_t vf[VD][KP][4];
#pragma unroll
      for (int t = 0; t < VD; ++t)
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
          if (pa + pb >= F::TERMS) continue;
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
    l[n] = sum_groups(l[n]);
    bad |= !(fabsf(l[n]) < INFINITY);
#pragma unroll
    for (int d = 0; d < NC * VD; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) bad |= !(fabsf(o[n][d][e]) < INFINITY);
  }
  // (also: every wave is done with xs)
  if (__syncthreads_or(bad)) {
    item_by_key<HD, DT, 64 * W>(a, it, kvh, 16 * NQ, reinterpret_cast<float *>(lds));
    return;
  }
  float *ml = reinterpret_cast<float *>(lds);  // [2][group][16 NQ]
  constexpr int LD = CD + 4, ROWS = 16 * NQ;
  float *os = ml + 2 * NG * ROWS;              // [wave][16][LD]
  if (g == 0 && part == 0)
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      ml[grp * ROWS + 16 * n + c16] = m[n];
      ml[(NG + grp) * ROWS + 16 * n + c16] = l[n];
    }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    if (16 * n >= nrows) break;
    float top = kLow;
#pragma unroll
    for (int w = 0; w < NG; ++w) top = fmaxf(top, ml[w * ROWS + 16 * n + c16]);
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
      for (int i = tid; i < 16 * SP * (CD / 4); i += 64 * W) {
        const int d = i % (CD / 4) * 4, pt = i / (CD / 4) % SP, r16 = i / (CD / 4 * SP), r = 16 * n + r16;
        if (r >= nrows) break;
        float mt = kLow, ls = 0.f;
#pragma unroll
        for (int w = 0; w < NG; ++w) mt = fmaxf(mt, ml[w * ROWS + r]);
        f4 x = {};
#pragma unroll
        for (int w = 0; w < NG; ++w) {
          ls += ml[(NG + w) * ROWS + r] * __builtin_amdgcn_exp2f(ml[w * ROWS + r] - mt);
          x += *reinterpret_cast<const f4 *>(os + ((w * SP + pt) * 16 + r16) * LD + d);
        }
        const int dim = pt * HW + c * CD + d;
        if (it.part < 0) {
          const int t = (int)div_by(it.r0 + r, a.by_g), h = it.r0 + r - t * a.G;
          *reinterpret_cast<f4 *>(a.out + (size_t)(it.row + t) * a.out_ld + (size_t)(kvh * a.G + h) * HD + dim) =
              x / ls;
        } else {
          const size_t pr = ((size_t)it.part * a.n_kv + kvh) * a.part_rows + r;
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
  static constexpr int VD = HD / (16 * W) < 2 ? 2 : HD / (16 * W);  // dims of a value row a lane loads
  static constexpr int FRAG = kTile * HD * 2 * Form<DT>::KP;        // bytes of K's or V's fragments
  static constexpr int XS_AT = FRAG * (ONE ? 1 : 2), XS = SP > 1 ? W * NQ * 2 * 64 * 16 : 0;
  static constexpr int ROWS_AT = XS_AT + XS, USED = ROWS_AT + 2 * kTile * 4;
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
template <int HD, int DT>
__device__ __forceinline__ void item_by_block(const PagedAttnArgs &a, const PagedItem &it, int kvh,
                                              char *lds) {
  using F = Form<DT>;
  using B = Shape<HD, DT>;
  constexpr bool F16 = F::F16;
  constexpr int NQ = B::NQ, W = B::W, SP = B::SP;
  constexpr int QP = F::QP, KP = F::KP, KS = HD / 32, ES = DT == MS_KV_F32 ? 4 : 2;
  constexpr int VD = B::VD, CD = 16 * VD, NC = HD / CD;
  constexpr int KW = KS / SP, CW = NC / SP;  // a wave's 32-dim steps and chunks of CD dims
  constexpr int D8 = HD / 8, UK = kTile * D8 / (64 * W);  // K units of 8 dims a thread
  constexpr bool STRICT = KW * KP >= 8;
  constexpr int RING = 3;
  static_assert(CW >= 1 && UK >= 1 && 64 * W / D8 * UK == kTile, "shape");
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c16 = lane & 15, g = lane >> 4;
  const int grp = wave / SP, part = wave % SP;
  const int nrows = min(B::PAIRS, it.n_new * a.G - it.r0), base = it.len - it.n_new;
  u4 *kf = reinterpret_cast<u4 *>(lds);                        // [half][ks][part][64], slots turned by (ks, g)
  u4 *vf = B::ONE ? kf : kf + B::FRAG / 16;                    // [c][t][part][64]
  f4 *xs = reinterpret_cast<f4 *>(lds + B::XS_AT);             // [wave][nq][half][64]
  uint32_t *rows = reinterpret_cast<uint32_t *>(lds + B::ROWS_AT);  // [2][32]

  float sc[NQ], down[NQ], m[NQ], l[NQ];
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
  const char *vb0 = static_cast<const char *>(a.v) + ((size_t)kvh * HD + wave * CD + VD * c16) * ES;
  // Pool row of a tile's key `tid`, never one outside the attended keys; two tiles' rows in LDS.
  // Those of the next are written between the two barriers of a tile, in place of the last's,
  // whose readers are past the first of them.
  auto find = [&](int tile) {
    const int key = min(max(it.k0 + tile * kTile + tid, low_key), it.k1 - 1);
    const int pg = (int)div_by((uint32_t)key, a.by_page);
    return ldg<int32_t>(a.pages + (size_t)it.seq * a.stride + pg) * a.page_rows + key - pg * a.page_size;
  };
  uint32_t kr[UK][ES * 2];      // 8 dims of a key
  uint32_t vr[8][VD * ES / 4];  // VD dims of eight keys
  auto load_k = [&](int tile) {
    const uint32_t *row = rows + (tile & 1) * kTile + tid / D8;
#pragma unroll
    for (int u = 0; u < UK; ++u) {
      const char *p = kb0 + (uint64_t)row[64 * W / D8 * u] * row_bytes;
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
    const u4 r0 = row[0], r1 = row[4];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
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
  const bool v_busy = wave < NC;
  if (tid < kTile) rows[tid] = find(0);
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
    l[n] = 0.f;
    const float *qp = a.q + (size_t)(it.row + t) * a.q_ld + (size_t)(kvh * a.G + h) * HD + 8 * g;
    load_q<DT, KW>(qp + 32 * KW * part, real, a.q_scale, q[n], &down[n]);
    sc[n] = SP == 1 ? a.s_scale * down[n] : a.s_scale;
  }
  f4 o[NQ][CW * VD] = {};
  for (int tile = 0; tile < n_tiles; ++tile) {
    const int kb = it.k0 + tile * kTile;
    if (B::ONE && tile) __syncthreads();
#pragma unroll
    for (int u = 0; u < UK; ++u) {
      const int key = (tid + 64 * W * u) / D8, d8 = tid % D8;
      u4 *dst = kf + (((key >> 4) * KS + (d8 >> 2)) * KP) * 64 + (d8 & 3) * 16 + ((key ^ d8) & 15);
      if constexpr (ES == 2) {
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
    __syncthreads();
    int next = 0;
    if (tid < kTile) next = find(min(tile + 1, n_tiles - 1));
    uint32_t pf[NQ][QP][4];
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
          if (pa + pb >= F::TERMS) continue;
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
      if constexpr (SP == 1) probabilities<DT, NQ>(s, kb, edge, sc, span, m, l, o, pf);
    }
    if (B::ONE) __syncthreads();
    if (tid < kTile) rows[((tile + 1) & 1) * kTile + tid] = next;
    if (v_busy) {
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
      load_k(tile + 1);
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
        probabilities<DT, NQ>(s, kb, edge, sc, span, m, l, o, pf);
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
          if (pa + pb >= F::TERMS) continue;
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
    l[n] = sum_groups(l[n]);
    bad |= !(fabsf(l[n]) < INFINITY);
#pragma unroll
    for (int d = 0; d < CW * VD; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) bad |= !(fabsf(o[n][d][e]) < INFINITY);
  }
  if (__syncthreads_or(bad)) {
    item_by_key<HD, DT, 64 * W>(a, it, kvh, B::PAIRS, reinterpret_cast<float *>(lds));
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

// Items of at most 16 NQ pairs: single tokens, or a few of them.  (Two query tiles of three parts do
// not fit the registers of two waves a SIMD: with spills 110 us where one wave takes 72 us.)
template <int HD, int DT, int NQ>
__global__ __launch_bounds__(256, NQ == 2 && DT != MS_KV_F16 ? 1 : 2) void k_paged_tile(PagedAttnArgs a) {
  __shared__ __align__(16) char lds[tile_lds<HD, DT, NQ, 4>()];
  item_by_tile<HD, DT, NQ, 4>(a, a.items[blockIdx.x / a.n_kv], blockIdx.x % a.n_kv, lds);
}

// Items of longer chunks, and single tokens beside them.
template <int HD, int DT, int NT = 64 * Shape<HD, DT>::W>
__global__ __launch_bounds__(NT, 2) void k_paged_block(PagedAttnArgs a) {
  constexpr int A = tile_lds<HD, DT, 1, Shape<HD, DT>::W>(), B = Shape<HD, DT>::LDS;
  __shared__ __align__(16) char lds[A > B ? A : B];
  const PagedItem it = a.items[blockIdx.x / a.n_kv];
  if (it.n_new * a.G - it.r0 <= 16)
    item_by_tile<HD, DT, 1, Shape<HD, DT>::W>(a, it, blockIdx.x % a.n_kv, lds);
  else
    item_by_block<HD, DT>(a, it, blockIdx.x % a.n_kv, lds);
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

// Items of p->rows (row, head) pairs, their keys cut into spans so that the work fits
// `blocks` blocks at a time; the longest come first.
int make_plan(ms_paged_batch *b, PagedPlan *p, int blocks) {
  struct Span {
    int seq, r0, k0, k1, tiles, cost;  // cost: of a tile, in quarters of a block's step
  };
  std::vector<Span> spans;
  int64_t work = 0;
  int most = 0, longest = 0, most_tiles = 0;
  for (int s = 0; s < b->n_seqs; ++s) {
    const int pairs = b->n_new[s] * p->G, base = b->len[s] - b->n_new[s];
    most = std::max(most, std::min(pairs, p->rows));
    for (int r0 = 0; r0 < pairs; r0 += p->rows) {
      const int t0 = r0 / p->G, t1 = std::min((r0 + p->rows - 1) / p->G, b->n_new[s] - 1);
      const int lo = p->window ? std::max(0, base + t0 - p->window + 1) : 0;
      const int k0 = lo / kTile * kTile, k1 = base + t1 + 1, n = (k1 - k0 + kTile - 1) / kTile;
      spans.push_back({s, r0, k0, k1, n, p->block && pairs - r0 > 16 ? 4 : p->tile_cost});
      work += (int64_t)n * spans.back().cost;
      longest = std::max(longest, n * spans.back().cost);
      most_tiles = std::max(most_tiles, n);
    }
  }
  // The longest part a block gets, `per`: at least a step, and no more than kMaxParts of them; from an
  // even share up, where its end is soonest: all blocks at once are done with the longest, more of
  // them after about half of one more; then the merge, if there is anything to merge.
  auto cuts_of = [](const Span &x, int per) { return (x.tiles * x.cost + per - 1) / per; };
  // (by the tiles that the longest span has: a sliding window's are the same at every position)
  // (an even share of more than the longest span: nothing is cut; unbounded it passes 32 bits)
  const int64_t fill = std::min<int64_t>(longest, std::max((work * p->n_kv + blocks - 1) / blocks,
                                                           ((int64_t)most_tiles * 4 + kMaxParts - 1) / kMaxParts));
  int per = (int)((fill + 3) / 4 * 4);
  int64_t best = INT64_MAX;
  for (int64_t c = per;; c += std::max<int64_t>(4, c / 8 / 4 * 4)) {
    int64_t n = 0, top = 0;
    for (const Span &x : spans) {
      const int cuts = cuts_of(x, (int)c);
      n += cuts;
      top = std::max<int64_t>(top, (x.tiles + cuts - 1) / cuts * x.cost);
    }
    n *= p->n_kv;
    const bool cut = n > (int64_t)spans.size() * p->n_kv;
    const int64_t end = (n <= blocks ? top : std::max(top, work * p->n_kv / blocks) + top / 2) +
                        (cut ? p->merge_cost : 0);
    if (end < best) {
      best = end;
      per = (int)c;
    }
    if (c >= longest || c > 4 * fill + 64) break;
  }
  std::vector<PagedItem> items;
  std::vector<PagedMerge> merge;
  std::vector<std::pair<int, int>> order;
  int parts = 0, most_parts = 0;
  for (const Span &x : spans) {
    const int cuts = cuts_of(x, per), s = x.seq;
    most_parts = std::max(most_parts, cuts);
    if (cuts > 1) merge.push_back({b->first[s], b->n_new[s], x.r0, parts, cuts});
    for (int c = 0; c < cuts; ++c) {
      const int i0 = (int)((int64_t)x.tiles * c / cuts), i1 = (int)((int64_t)x.tiles * (c + 1) / cuts);
      order.push_back({-(i1 - i0) * x.cost, (int)items.size()});
      items.push_back({b->first[s], b->n_new[s], b->len[s], s, x.r0, x.k0 + i0 * kTile,
                       std::min(x.k1, x.k0 + i1 * kTile), cuts > 1 ? parts++ : -1});
    }
  }
  std::sort(order.begin(), order.end());
  p->n_items = (int)items.size();
  p->n_merge = (int)merge.size();
  p->n_parts = parts;
  p->most = most;
  p->most_parts = most_parts;
  p->merge_at = items.size() * sizeof(PagedItem);
  const size_t bytes = p->merge_at + merge.size() * sizeof(PagedMerge);
  if (int rc = p->up.reserve(bytes)) return rc;
  for (size_t i = 0; i < items.size(); ++i)
    reinterpret_cast<PagedItem *>(p->up.h)[i] = items[order[i].second];
  std::copy(merge.begin(), merge.end(), reinterpret_cast<PagedMerge *>(p->up.h + p->merge_at));
  if (int rc = p->up.send(bytes)) return rc;
  p->valid = true;
  return MS_OK;
}

int plan_for(ms_paged_batch *b, int G, int rows, bool block, int n_kv, int window, int blocks,
             int tile_cost, int merge_cost, PagedPlan **out) {
  PagedPlan *p = nullptr;
  for (PagedPlan *x : b->plans)
    if (x->G == G && x->rows == rows && x->block == block && x->n_kv == n_kv && x->window == window && x->blocks == blocks &&
        x->tile_cost == tile_cost && x->merge_cost == merge_cost)
      p = x;
  if (!p) {
    // (a model has a few shapes of layers; more than that reuse the oldest place)
    if (b->plans.size() < 8) {
      b->plans.reserve(8);
      b->plans.push_back(new PagedPlan());
    } else {
      std::rotate(b->plans.begin(), b->plans.begin() + 1, b->plans.end());
    }
    p = b->plans.back();
    p->valid = false;
    p->G = G;
    p->rows = rows;
    p->block = block;
    p->blocks = blocks;
    p->tile_cost = tile_cost;
    p->merge_cost = merge_cost;
    p->n_kv = n_kv;
    p->window = window;
  }
  *out = p;
  return p->valid ? MS_OK : make_plan(b, p, blocks);
}

template <int HD, int DT>
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
  const int w = block ? B::W : 4, cost = std::max(1, 4 * tile_split<HD>() / w);
  // A merge's launch takes 3.4 us; a step of a single token (4 in the plan's measure) 0.7 us at head dim 64,
  // 1.15 at 128 and 1.4 to 1.6 at 256 and 512 over 16-bit pools, 1.7 to 5 us over fp32 ones: one token over 250
  // keys of 64 dims (bf16) 5.4 us in one block a head, 9.0 us cut and merged; over 1500 keys 12.4 and 9.1 us.
  const int merge = block ? 8 : DT == MS_KV_F32 ? 4 : HD == 64 ? 20 : HD == 128 ? 12 : 8;
  if (int rc = plan_for(b, a.G, rows, block, a.n_kv, a.window, 8 / w * ctx().n_cu, cost, merge, &p)) return rc;
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
  const dim3 grid(p->n_items * a.n_kv);
  if (block) {
    hipLaunchKernelGGL((k_paged_block<HD, DT>), grid, dim3(64 * B::W), 0, st, a);
  } else if (rows == 16) {
    hipLaunchKernelGGL((k_paged_tile<HD, DT, 1>), grid, dim3(256), 0, st, a);
  } else {
    if constexpr (TWO) hipLaunchKernelGGL((k_paged_tile<HD, DT, 2>), grid, dim3(256), 0, st, a);
  }
  if (p->n_merge) {
    // about four parts a thread, more of them in a larger block
    const PagedMerge *merge = reinterpret_cast<const PagedMerge *>(p->up.d + p->merge_at);
    int rpb = 1024 / HD;
    while (rpb > 1 && 1024 / HD / rpb * 4 < p->most_parts) rpb /= 2;
    const dim3 mg(p->n_merge * a.n_kv, cdiv(p->most, rpb));
    if (1024 / HD * 4 < p->most_parts)
      hipLaunchKernelGGL((k_paged_merge<HD, 1024>), mg, dim3(1024), 0, st, a, merge, rpb);
    else
      hipLaunchKernelGGL((k_paged_merge<HD, 256>), mg, dim3(256), 0, st, a, merge, rpb);
  }
  MS_HIP_TRY(hipGetLastError());
  return MS_OK;
}
template <int HD>
int launch_type(PagedAttnArgs &a, ms_paged_batch *b, int dtype, int most, hipStream_t st) {
  if (dtype == MS_KV_F32) return launch<HD, MS_KV_F32>(a, b, most, st);
  if (dtype == MS_KV_BF16) return launch<HD, MS_KV_BF16>(a, b, most, st);
  return launch<HD, MS_KV_F16>(a, b, most, st);
}

}  // namespace
}  // namespace ms

using namespace ms;

extern "C" int ms_paged_attention(const ms_paged_layer *L, ms_paged_batch *b, const float *d_q,
                                  size_t q_stride, float *d_out, size_t out_stride) {
  MS_CHECK_ARG(L, "paged_attention: null layer or batch");
  // (log2(e) times it, what the kernels take, is finite too)
  MS_CHECK_ARG(std::fabs(L->scale * 1.4426950408889634) <= 0x1.fffffep+127,
               "paged_attention: the scale is not finite or too large");
  if (int rc = paged_check("paged_attention", L, b)) return rc;
  MS_CHECK_ARG((int64_t)b->rows * L->n_heads < ((int64_t)1 << 30),
               "paged_attention: too many rows for one call");
  const int q_dim = L->n_heads * L->head_dim, hd = L->head_dim, G = L->n_heads / L->n_kv_heads;
  int most = 0;
  for (int s = 0; s < b->n_seqs; ++s) {
    if (!b->n_new[s]) continue;
    const int lo = L->window ? std::max(0, b->len[s] - b->n_new[s] - L->window + 1) : 0;
    MS_CHECK_ARG(lo >= b->held[s], "paged_attention: sequence " + std::to_string(s) +
                                       " attends to a position whose page is -1");
    most = std::max(most, b->n_new[s] * G);
  }
  if (b->rows == 0) return require_init();
  MS_CHECK_ARG(d_q && d_out && aligned16(d_q) && aligned16(d_out) && q_stride % 4 == 0 &&
                   out_stride % 4 == 0 && q_stride >= (size_t)q_dim &&
                   out_stride >= (size_t)q_dim && q_stride < ((size_t)1 << 31) &&
                   out_stride < ((size_t)1 << 31),
               "paged_attention: bad q or output rows");
  MS_CHECK_ARG(!rows_overlap(d_q, q_stride, q_dim, d_out, out_stride, q_dim, b->rows),
               "paged_attention: d_q and d_out overlap");
  if (int rc = require_init()) return rc;
  OnDevice on;
  hipStream_t st = ctx().stream;
  PagedAttnArgs a{};
  a.q = d_q;
  a.out = d_out;
  a.q_ld = q_stride;
  a.out_ld = out_stride;
  a.k = L->k;
  a.v = L->v;
  a.pages = b->d_pages();
  a.stride = b->stride;
  a.n_kv = L->n_kv_heads;
  a.G = G;
  a.window = L->window;
  a.page_size = b->page_size;
  a.page_rows = page_rows(L, b);
  a.by_page = fast_div(b->page_size);
  a.by_g = fast_div(G);
  int e = 0;
  const double scale = (L->scale == 0.f ? 1.0 / std::sqrt((double)hd) : L->scale) * 1.4426950408889634;
  const double part = std::frexp(scale, &e);  // (e <= 128; 2^127 is the largest power that fp32 holds)
  a.q_scale = (float)(e > 127 ? 2 * part : part);
  a.s_scale = (float)std::ldexp(1.0, e > 127 ? e - 1 : e);
  try {
    switch (hd) {
      case 64: return launch_type<64>(a, b, L->dtype, most, st);
      case 128: return launch_type<128>(a, b, L->dtype, most, st);
      case 256: return launch_type<256>(a, b, L->dtype, most, st);
      default: return launch_type<512>(a, b, L->dtype, most, st);
    }
  } catch (const std::exception &e) {
    return fail(MS_E_NOMEM, std::string("paged_attention: ") + e.what());
  }
}
