// Attention of a ragged batch's new rows over a paged KV cache.
#include <algorithm>
#include <cmath>
#include <exception>

#include "devutil.h"
#include "paged.h"

namespace ms {
namespace {

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
  float scale;            // of the scores, log2(e) in it
  float *part_o, *part_ml;  // [part][kv head][16 nq][head dim], [part][kv head][16 nq][2]
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

constexpr float kLow = -3.0e38f;  // running maximum before the first key
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

// The item's rows one after the other, key by key, with 256 threads: a key that a row does
// not attend to is not multiplied by anything.  Parts lie 16 NQS rows apart.
template <int HD, int DT, int NQ, int NQS>
__device__ __forceinline__ void item_by_key(const PagedAttnArgs &a, const PagedItem &it, int kvh,
                                         float *lds) {
  constexpr int ND = (HD + 255) / 256;
  float *p_of = lds, *red = lds + 256;  // probabilities of 256 keys (-1: not attended); 8
  const int tid = threadIdx.x;
  const int nrows = min(16 * NQ, it.n_new * a.G - it.r0);
  for (int r = 0; r < nrows; ++r) {
    const int t = (it.r0 + r) / a.G, h = (it.r0 + r) % a.G;
    const int pos = it.len - it.n_new + t;
    const int lo = a.window && pos - a.window + 1 > 0 ? pos - a.window + 1 : 0;
    const float *q = a.q + (size_t)(it.row + t) * a.q_ld + (size_t)(kvh * a.G + h) * HD;
    float m = -INFINITY, l = 0.f, o[ND] = {};
    for (int k0 = it.k0; k0 < it.k1; k0 += 256) {
      const int key = k0 + tid;
      const bool on = key < it.k1 && key >= lo && key <= pos;
      float s = 0.f;
      if (on) {
        const uint32_t pg = div_by(key, a.by_page);
        const size_t row = (size_t)a.pages[(size_t)it.seq * a.stride + pg] * a.page_rows +
                           (key - pg * a.page_size);
        const size_t at = (row * a.n_kv + kvh) * HD;
        for (int d = 0; d < HD; ++d) s += q[d] * a.scale * load_kv<DT>(a.k, at + d);
      }
      float mx = on ? s : -INFINITY;
      for (int off = 1; off < 64; off <<= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
      if ((tid & 63) == 0) red[tid >> 6] = mx;
      __syncthreads();
      mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
      const float mn = fmaxf(m, mx), base = mn == -INFINITY ? 0.f : mn;
      // (lifted like the tiles' probabilities: parts of both kinds are merged)
      const float p = on ? __builtin_amdgcn_exp2f(Form<DT>::F16 ? s - base + kLift : s - base) : 0.f;
      p_of[tid] = on ? p : -1.f;
      float sum = p;
      for (int off = 1; off < 64; off <<= 1) sum += __shfl_xor(sum, off, 64);
      if ((tid & 63) == 0) red[4 + (tid >> 6)] = sum;
      __syncthreads();
      const float al = __builtin_amdgcn_exp2f(m - base);
      l = l * al + (red[4] + red[5]) + (red[6] + red[7]);
#pragma unroll
      for (int i = 0; i < ND; ++i) o[i] *= al;
      m = mn;
      for (int j = 0; j < 256 && k0 + j < it.k1; ++j) {
        const float pj = p_of[j];
        if (pj == -1.f) continue;
        const uint32_t pg = div_by(k0 + j, a.by_page);
        const size_t row = (size_t)a.pages[(size_t)it.seq * a.stride + pg] * a.page_rows +
                           (k0 + j - pg * a.page_size);
        const size_t at = (row * a.n_kv + kvh) * HD;
#pragma unroll
        for (int i = 0; i < ND; ++i)
          if (tid + 256 * i < HD) o[i] += pj * load_kv<DT>(a.v, at + tid + 256 * i);
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      const int d = tid + 256 * i;
      if (d >= HD) continue;
      if (it.part < 0) {
        a.out[(size_t)(it.row + t) * a.out_ld + (size_t)(kvh * a.G + h) * HD + d] = o[i] / l;
      } else {
        const size_t pr = ((size_t)it.part * a.n_kv + kvh) * (16 * NQS) + r;
        a.part_o[pr * HD + d] = o[i];
        if (d == 0) {
          a.part_ml[pr * 2] = m;
          a.part_ml[pr * 2 + 1] = l;
        }
      }
    }
  }
}

// The attention of one item: 16 NQ (row, head) pairs, the block's four waves taking its
// 32-key tiles in turn, each with sums of its own that are joined at the end.  No LDS and
// no barrier in the loop over the keys: K and V come from the pages straight into the
// registers that the MFMAs take them from.
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
// A maximum per query serves all its keys and may lag behind by kLag, so that a tile needs
// neither a cross-lane maximum nor a rescaling of the sums, unless a score exceeds it.
//
// A value that is not finite makes the sums it is multiplied into not finite, with the
// zeros of masked keys too; where the end finds such a sum the item is done again key by
// key.
template <int HD, int DT, int NQ, int NQS>
__device__ __forceinline__ void item_by_tile(const PagedAttnArgs &a, const PagedItem &it, int kvh,
                                             char *lds) {
  using F = Form<DT>;
  constexpr bool F16 = F::F16;
  constexpr int QP = F::QP, KP = F::KP, KS = HD / 32, ES = DT == MS_KV_F32 ? 4 : 2;
  constexpr int VD = HD >= 128 ? 8 : HD / 16, CD = 16 * VD, NC = HD / CD;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c16 = lane & 15, g = lane >> 4;
  const int nrows = min(16 * NQ, it.n_new * a.G - it.r0), base = it.len - it.n_new;

  // ---- q: parts in LDS in fragment order; per query its position and scale
  u4 *qf = reinterpret_cast<u4 *>(lds);  // [nq][s][part][64]
  float sc[NQ];
  int lim[NQ], low[NQ];
  const int t_first = it.r0 / a.G, t_last = (it.r0 + nrows - 1) / a.G;
  const int low_key = a.window ? max(it.k0, base + t_first - a.window + 1) : it.k0;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int r = 16 * n + c16, t = (it.r0 + r) / a.G, h = (it.r0 + r) - t * a.G;
    const bool real = r < nrows;
    lim[n] = real ? min(it.k1 - 1, base + t) : it.k1 - 1;
    low[n] = real && a.window ? max(low_key, base + t - a.window + 1) : low_key;
    const float *q = a.q + (size_t)(it.row + (real ? t : t_first)) * a.q_ld +
                     (size_t)(kvh * a.G + (real ? h : 0)) * HD + 8 * g;
    float x[(KS + 3) / 4][8];
    float big = 0.f;
    if constexpr (F16) {
      // (every wave needs the whole row's largest value)
      for (int s = 0; s < KS; ++s) {
        const f4 u = ldg<f4>(q + 32 * s), v = ldg<f4>(q + 32 * s + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) big = fmaxf(big, fmaxf(fabsf(u[j]), fabsf(v[j])));
      }
      big = max_groups(big);
    }
    // 2^(14 - exponent of the largest); 1 where there is none
    const int ex = big > 0.f && big < INFINITY ? 14 - (int)((__float_as_uint(big) >> 23) & 255) + 127 : 0;
    const int exc = max(-100, min(100, ex));
    const float up = F16 ? __uint_as_float((uint32_t)(exc + 127) << 23) : 1.f;
    sc[n] = F16 ? a.scale * __uint_as_float((uint32_t)(127 - exc) << 23) : a.scale;
#pragma unroll
    for (int si = 0; si < (KS + 3) / 4; ++si) {
      const int s = wave + 4 * si;
      if (s < KS) {
        const f4 u = ldg<f4>(q + 32 * s), v = ldg<f4>(q + 32 * s + 4);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[si][j] = real ? (j < 4 ? u[j] : v[j - 4]) * up : 0.f;
        uint32_t p[QP][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) split2<F16, QP>(x[si][2 * j], x[si][2 * j + 1], &p[0][j], 4);
#pragma unroll
        for (int i = 0; i < QP; ++i)
          qf[((n * KS + s) * QP + i) * 64 + lane] = u4{p[i][0], p[i][1], p[i][2], p[i][3]};
      }
    }
  }
  __syncthreads();

  f4 o[NQ][NC * VD] = {};
  float m[NQ], l[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    m[n] = kLow;
    l[n] = 0.f;
  }
  const int n_tiles = (it.k1 - it.k0 + kTile - 1) / kTile;
  // keys that every row attends to
  const int all_lo = a.window ? max(low_key, base + t_last - a.window + 1) : low_key;
  const int all_hi = min(it.k1 - 1, base + t_first);
  const int32_t *pages = a.pages + (size_t)it.seq * a.stride;
  const uint32_t row_bytes = (uint32_t)a.n_kv * HD * ES;
  const char *kb0 = static_cast<const char *>(a.k) + ((size_t)kvh * HD + 8 * g) * ES;
  const char *vb0 = static_cast<const char *>(a.v) + ((size_t)kvh * HD + VD * c16) * ES;
  // row of key kb + (lane & 31), never one outside the attended keys
  auto find = [&](int tile, int *page, int *slot) {
    const int key = min(max(it.k0 + tile * kTile + (lane & 31), low_key), it.k1 - 1);
    const int pg = (int)div_by((uint32_t)key, a.by_page);
    *slot = key - pg * a.page_size;
    *page = ldg<int32_t>(pages + pg);
  };
  int page = 0, slot = 0;
  if (wave < n_tiles) find(wave, &page, &slot);
  for (int tile = wave; tile < n_tiles; tile += 4) {
    const int kb = it.k0 + tile * kTile;
    const int row = page * a.page_rows + slot;
    const char *kp[2], *vp[8];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      kp[i] = kb0 + (uint64_t)(uint32_t)__shfl(row, 16 * i + c16, 64) * row_bytes;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      vp[j] = vb0 + (uint64_t)(uint32_t)__shfl(row, 16 * (j >> 2) + 4 * g + (j & 3), 64) * row_bytes;
    if (tile + 4 < n_tiles) find(tile + 4, &page, &slot);

    // ---- scores
    // (the products of the leading parts have a sum of their own: a running sum that takes
    // the small ones too rounds six times as often)
    f4 s[2][NQ] = {}, s_low[2][NQ] = {};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      uint32_t kf[2][KP][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if constexpr (ES == 2) {
          const u4 x = ldg<u4>(kp[i] + ks * 64);
#pragma unroll
          for (int j = 0; j < 4; ++j) kf[i][0][j] = x[j];
        } else {
          const f4 x = ldg<f4>(kp[i] + ks * 128), y = ldg<f4>(kp[i] + ks * 128 + 16);
          split2<false, KP>(x[0], x[1], &kf[i][0][0], 4);
          split2<false, KP>(x[2], x[3], &kf[i][0][1], 4);
          split2<false, KP>(y[0], y[1], &kf[i][0][2], 4);
          split2<false, KP>(y[2], y[3], &kf[i][0][3], 4);
        }
      }
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int pa = QP - 1; pa >= 0; --pa) {
          const u4 q = qf[((n * KS + ks) * QP + pa) * 64 + lane];
#pragma unroll
          for (int pb = KP - 1; pb >= 0; --pb) {
            if (pa + pb >= F::TERMS) continue;
#pragma unroll
            for (int i = 0; i < 2; ++i)
              (pa + pb ? s_low : s)[i][n] =
                  mfma<F16>(u4{kf[i][pb][0], kf[i][pb][1], kf[i][pb][2], kf[i][pb][3]}, q,
                            (pa + pb ? s_low : s)[i][n]);
          }
        }
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) s[i][n] += s_low[i][n];

    // ---- probabilities
    const bool whole = kb >= all_lo && kb + kTile - 1 <= all_hi;
    uint32_t pf[NQ][QP][4];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float t[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = __builtin_fmaf(s[j >> 2][n][j & 3], sc[n], -m[n]);
      if (!whole) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int key = kb + 16 * (j >> 2) + 4 * g + (j & 3);
          if (key > lim[n] || key < low[n]) t[j] = -INFINITY;
        }
      }
      float mx = t[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) mx = fmaxf(mx, t[j]);
      if (__any(mx > kLag)) {
        // (t is a score less the old maximum; taken anew from the scores, which near kLow
        // are lost in it)
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, t[j] == -INFINITY ? -INFINITY : s[j >> 2][n][j & 3] * sc[n]);
        const float mn = fmaxf(m[n], max_groups(top)), al = __builtin_amdgcn_exp2f(m[n] - mn);
        m[n] = mn;
        l[n] *= al;
#pragma unroll
        for (int d = 0; d < NC * VD; ++d) o[n][d] *= al;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (t[j] != -INFINITY) t[j] = __builtin_fmaf(s[j >> 2][n][j & 3], sc[n], -mn);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = __builtin_amdgcn_exp2f(F16 ? t[j] + kLift : t[j]);
      l[n] += ((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7]));
#pragma unroll
      for (int j = 0; j < 4; ++j) split2<F16, QP>(t[2 * j], t[2 * j + 1], &pf[n][0][j], 4);
    }

    // ---- values
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      uint32_t vf[VD][KP][4];
      if constexpr (ES == 2) {
        uint32_t x[8][VD / 2];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if constexpr (VD == 8) {
            const u4 y = ldg<u4>(vp[j] + c * CD * ES);
#pragma unroll
            for (int d = 0; d < 4; ++d) x[j][d] = y[d];
          } else {
            const u2 y = ldg<u2>(vp[j] + c * CD * ES);
            x[j][0] = y[0];
            x[j][1] = y[1];
          }
        }
#pragma unroll
        for (int t = 0; t < VD; ++t)
#pragma unroll
          for (int d = 0; d < 4; ++d)
            vf[t][0][d] = __builtin_amdgcn_perm(x[2 * d + 1][t / 2], x[2 * d][t / 2],
                                                t & 1 ? 0x07060302u : 0x05040100u);
      } else {
        float x[8][VD];
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int d = 0; d < VD / 4; ++d) {
            const f4 y = ldg<f4>(vp[j] + c * CD * ES + 16 * d);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[j][4 * d + e] = y[e];
          }
#pragma unroll
        for (int t = 0; t < VD; ++t)
#pragma unroll
          for (int d = 0; d < 4; ++d) split2<false, KP>(x[2 * d][t], x[2 * d + 1][t], &vf[t][0][d], 4);
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
  }

  // ---- the waves' sums joined
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
  // (also: every wave is done with q)
  if (__syncthreads_or(bad)) {
    item_by_key<HD, DT, NQ, NQS>(a, it, kvh, reinterpret_cast<float *>(lds));
    return;
  }
  float *ml = reinterpret_cast<float *>(lds);  // [2][wave][16 NQ]
  constexpr int LD = CD + 4;
  float *os = ml + 2 * 4 * 16 * NQ;            // [wave][16][LD]
  if (g == 0)
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      ml[wave * 16 * NQ + 16 * n + c16] = m[n];
      ml[(4 + wave) * 16 * NQ + 16 * n + c16] = l[n];
    }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const float *mw = ml + 16 * n + c16;
    const float top = fmaxf(fmaxf(mw[0], mw[16 * NQ]), fmaxf(mw[32 * NQ], mw[48 * NQ]));
    const float w = __builtin_amdgcn_exp2f(m[n] - top);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int t = 0; t < VD; t += 4) {
          f4 x;
#pragma unroll
          for (int u = 0; u < 4; ++u) x[u] = o[n][c * VD + t + u][e] * w;
          *reinterpret_cast<f4 *>(os + (wave * 16 + c16) * LD + VD * (4 * g + e) + t) = x;
        }
      __syncthreads();
      for (int i = tid; i < 4 * CD; i += 256) {
        const int r16 = i / (CD / 4), d = i % (CD / 4) * 4, r = 16 * n + r16;
        if (r >= nrows) continue;
        const float *mr = ml + r;
        const float m0 = mr[0], m1 = mr[16 * NQ], m2 = mr[32 * NQ], m3 = mr[48 * NQ];
        const float mt = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
        const float *lr = mr + 64 * NQ;
        const float ls = (lr[0] * __builtin_amdgcn_exp2f(m0 - mt) + lr[16 * NQ] * __builtin_amdgcn_exp2f(m1 - mt)) +
                         (lr[32 * NQ] * __builtin_amdgcn_exp2f(m2 - mt) + lr[48 * NQ] * __builtin_amdgcn_exp2f(m3 - mt));
        const float *p = os + r16 * LD + d;
        const f4 x = (*reinterpret_cast<const f4 *>(p) + *reinterpret_cast<const f4 *>(p + 16 * LD)) +
                     (*reinterpret_cast<const f4 *>(p + 32 * LD) + *reinterpret_cast<const f4 *>(p + 48 * LD));
        if (it.part < 0) {
          const int t = (it.r0 + r) / a.G, h = (it.r0 + r) - t * a.G;
          *reinterpret_cast<f4 *>(a.out + (size_t)(it.row + t) * a.out_ld + (size_t)(kvh * a.G + h) * HD +
                                  c * CD + d) = x / ls;
        } else {
          const size_t pr = ((size_t)it.part * a.n_kv + kvh) * (16 * NQS) + r;
          *reinterpret_cast<f4 *>(a.part_o + pr * HD + c * CD + d) = x;
          if (c == 0 && d == 0) {
            a.part_ml[pr * 2] = mt;
            a.part_ml[pr * 2 + 1] = ls;
          }
        }
      }
    }
  }
}

template <int HD, int DT, int NQ>
constexpr int attn_lds() {
  constexpr int q = Form<DT>::QP * NQ * HD * 32, vd = HD >= 128 ? 8 : HD / 16;
  constexpr int e = (128 * NQ + 64 * (16 * vd + 4)) * 4;
  return q > e ? q : e;
}

// At most 16 NQ pairs an item; items of at most 16 (single tokens in a call that has longer
// chunks too) take one query tile instead of NQ.
template <int HD, int DT, int NQ>
__global__ __launch_bounds__(256, HD * NQ >= 512 ? 1 : 2) void k_paged_attn(PagedAttnArgs a) {
  __shared__ __align__(16) char lds[attn_lds<HD, DT, NQ>()];
  const int kvh = blockIdx.x % a.n_kv;
  const PagedItem it = a.items[blockIdx.x / a.n_kv];
  if constexpr (NQ > 1) {
    if (it.n_new * a.G - it.r0 <= 16) return item_by_tile<HD, DT, 1, NQ>(a, it, kvh, lds);
  }
  item_by_tile<HD, DT, NQ, NQ>(a, it, kvh, lds);
}

// The parts of one result, weighted by e^(their maximum - the largest): a block per (row,
// head), its threads HD / 4 columns by 1024 / HD groups of parts.
constexpr int kMaxParts = 1024;
template <int HD, int NQ>
__global__ __launch_bounds__(256) void k_paged_merge(PagedAttnArgs a, const PagedMerge *merge) {
  constexpr int COLS = HD / 4, GRP = 256 / COLS;
  __shared__ float w[kMaxParts], red[8];
  __shared__ f4 os[GRP][COLS];
  const int tid = threadIdx.x, kvh = blockIdx.x % a.n_kv, r = blockIdx.y;
  const PagedMerge g = merge[blockIdx.x / a.n_kv];
  if (r >= g.n_new * a.G - g.r0) return;
  const size_t pr = ((size_t)g.part * a.n_kv + kvh) * (16 * NQ) + r, step = (size_t)a.n_kv * 16 * NQ;
  const int col = tid % COLS, grp = tid / COLS;
  float top = -INFINITY;
  for (int p = tid; p < g.n; p += 256) {
    w[p] = ldg<float>(a.part_ml + (pr + p * step) * 2);
    top = fmaxf(top, w[p]);
  }
  for (int off = 1; off < 64; off <<= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
  if ((tid & 63) == 0) red[tid >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  if (top == -INFINITY) top = 0.f;
  float l = 0.f;
  for (int p = tid; p < g.n; p += 256) {
    w[p] = __builtin_amdgcn_exp2f(w[p] - top);
    l += w[p] * ldg<float>(a.part_ml + (pr + p * step) * 2 + 1);
  }
  for (int off = 1; off < 64; off <<= 1) l += __shfl_xor(l, off, 64);
  if ((tid & 63) == 0) red[4 + (tid >> 6)] = l;
  __syncthreads();
  f4 o = {};
  const float *po = a.part_o + pr * HD + 4 * col;
#pragma unroll 4
  for (int p = grp; p < g.n; p += GRP) o += w[p] * ldg<f4>(po + p * step * HD);
  os[grp][col] = o;
  __syncthreads();
  if (tid >= COLS) return;
#pragma unroll
  for (int i = 1; i < GRP; ++i) o += os[i][col];
  const int t = (g.r0 + r) / a.G, h = (g.r0 + r) - t * a.G;
  *reinterpret_cast<f4 *>(a.out + (size_t)(g.row + t) * a.out_ld + (size_t)(kvh * a.G + h) * HD + 4 * col) =
      o / ((red[4] + red[5]) + (red[6] + red[7]));
}

// Blocks of 16 nq (row, head) pairs and spans of keys.  The spans are cut so that about
// `blocks` blocks have the same number of tiles each; the longest come first.
int make_plan(ms_paged_batch *b, PagedPlan *p, int blocks) {
  const int rows_of = 16 * p->nq;
  std::vector<PagedItem> items;
  std::vector<PagedMerge> merge;
  auto spans = [&](int s, int r0, int *k0, int *k1) {
    const int t0 = r0 / p->G, t1 = std::min((r0 + rows_of - 1) / p->G, b->n_new[s] - 1);
    const int base = b->len[s] - b->n_new[s];
    const int lo = p->window ? std::max(0, base + t0 - p->window + 1) : 0;
    *k0 = lo / kTile * kTile;
    *k1 = base + t1 + 1;
  };
  int64_t tiles = 0;
  for (int s = 0; s < b->n_seqs; ++s)
    for (int r0 = 0; r0 < b->n_new[s] * p->G; r0 += rows_of) {
      int k0, k1;
      spans(s, r0, &k0, &k1);
      tiles += (k1 - k0 + kTile - 1) / kTile;
    }
  // (a multiple of four, a tile for every wave; no more parts than a merge takes)
  const int64_t fill = std::max((tiles * p->n_kv + blocks - 1) / blocks,
                                ((int64_t)b->max_pos / kTile + kMaxParts) / kMaxParts);
  const int per = (int)((fill + 3) / 4 * 4);
  int parts = 0, most = 0;
  for (int s = 0; s < b->n_seqs; ++s)
    for (int r0 = 0; r0 < b->n_new[s] * p->G; r0 += rows_of) {
      int k0, k1;
      spans(s, r0, &k0, &k1);
      const int n = (k1 - k0 + kTile - 1) / kTile, cuts = (n + per - 1) / per;
      most = std::max(most, b->n_new[s] * p->G);
      if (cuts > 1) merge.push_back({b->first[s], b->n_new[s], r0, parts, cuts});
      for (int c = 0; c < cuts; ++c)
        items.push_back({b->first[s], b->n_new[s], b->len[s], s, r0,
                         k0 + (int)((int64_t)n * c / cuts) * kTile,
                         std::min(k1, k0 + (int)((int64_t)n * (c + 1) / cuts) * kTile),
                         cuts > 1 ? parts++ : -1});
    }
  std::stable_sort(items.begin(), items.end(), [](const PagedItem &x, const PagedItem &y) {
    return x.k1 - x.k0 > y.k1 - y.k0;
  });
  p->n_items = (int)items.size();
  p->n_merge = (int)merge.size();
  p->n_parts = parts;
  p->most = most;
  p->merge_at = items.size() * sizeof(PagedItem);
  const size_t bytes = p->merge_at + merge.size() * sizeof(PagedMerge);
  if (int rc = p->up.reserve(bytes)) return rc;
  std::copy(items.begin(), items.end(), reinterpret_cast<PagedItem *>(p->up.h));
  std::copy(merge.begin(), merge.end(), reinterpret_cast<PagedMerge *>(p->up.h + p->merge_at));
  if (int rc = p->up.send(bytes)) return rc;
  p->valid = true;
  return MS_OK;
}

int plan_for(ms_paged_batch *b, int G, int nq, int n_kv, int window, PagedPlan **out) {
  PagedPlan *p = nullptr;
  for (PagedPlan *x : b->plans)
    if (x->G == G && x->nq == nq && x->n_kv == n_kv && x->window == window) p = x;
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
    p->nq = nq;
    p->n_kv = n_kv;
    p->window = window;
  }
  *out = p;
  return p->valid ? MS_OK : make_plan(b, p, 2 * ctx().n_cu);
}

template <int HD, int DT, int NQ>
void launch(const PagedAttnArgs &a, const PagedPlan &p, hipStream_t st) {
  hipLaunchKernelGGL((k_paged_attn<HD, DT, NQ>), dim3(p.n_items * a.n_kv), dim3(256), 0, st, a);
  if (p.n_merge)
    hipLaunchKernelGGL((k_paged_merge<HD, NQ>), dim3(p.n_merge * a.n_kv, std::min(16 * NQ, p.most)), dim3(256), 0, st,
                       a,
                       reinterpret_cast<const PagedMerge *>(p.up.d + p.merge_at));
}
template <int HD, int DT>
void launch_nq(const PagedAttnArgs &a, const PagedPlan &p, hipStream_t st) {
  constexpr int MAXQ = HD >= 512 ? 1 : HD == 256 ? 2 : 4;
  if constexpr (MAXQ > 1) {
    if (p.nq > 1) return launch<HD, DT, MAXQ>(a, p, st);
  }
  launch<HD, DT, 1>(a, p, st);
}
template <int HD>
void launch_dt(const PagedAttnArgs &a, const PagedPlan &p, int dtype, hipStream_t st) {
  if (dtype == MS_KV_F32)
    launch_nq<HD, MS_KV_F32>(a, p, st);
  else if (dtype == MS_KV_BF16)
    launch_nq<HD, MS_KV_BF16>(a, p, st);
  else
    launch_nq<HD, MS_KV_F16>(a, p, st);
}

}  // namespace
}  // namespace ms

using namespace ms;

extern "C" int ms_paged_attention(const ms_paged_layer *L, ms_paged_batch *b, const float *d_q,
                                  size_t q_stride, float *d_out, size_t out_stride) {
  MS_CHECK_ARG(L, "paged_attention: null layer or batch");
  MS_CHECK_ARG(std::fabs(L->scale) < INFINITY, "paged_attention: the scale is not a finite number");
  if (int rc = paged_check("paged_attention", L, b)) return rc;
  const int q_dim = L->n_heads * L->head_dim, hd = L->head_dim, G = L->n_heads / L->n_kv_heads;
  int most = 0;
  for (int s = 0; s < b->n_seqs; ++s) {
    if (!b->n_new[s]) continue;
    const int lo = L->window ? std::max(0, b->len[s] - b->n_new[s] - L->window + 1) : 0;
    MS_CHECK_ARG(lo >= b->held[s], "paged_attention: sequence " + std::to_string(s) +
                                       " attends to a position whose page is -1");
    MS_CHECK_ARG((int64_t)b->n_new[s] * G < ((int64_t)1 << 30),
                 "paged_attention: too many rows for one call");
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
  const int nq = most <= 16 ? 1 : hd >= 512 ? 1 : hd == 256 ? 2 : 4;
  PagedPlan *p = nullptr;
  try {
    if (int rc = plan_for(b, G, nq, L->n_kv_heads, L->window, &p)) return rc;
  } catch (const std::exception &e) {
    return fail(MS_E_NOMEM, std::string("paged_attention: ") + e.what());
  }
  PagedAttnArgs a{};
  const size_t rows = (size_t)p->n_parts * L->n_kv_heads * 16 * nq;
  if (rows) {
    void *buf = nullptr;
    if (int rc = scratch(rows * (hd + 2) * 4, &buf)) return rc;
    a.part_o = static_cast<float *>(buf);
    a.part_ml = a.part_o + rows * hd;
  }
  a.q = d_q;
  a.out = d_out;
  a.q_ld = q_stride;
  a.out_ld = out_stride;
  a.k = L->k;
  a.v = L->v;
  a.pages = b->d_pages();
  a.stride = b->stride;
  a.items = reinterpret_cast<const PagedItem *>(p->up.d);
  a.n_kv = L->n_kv_heads;
  a.G = G;
  a.window = L->window;
  a.page_size = b->page_size;
  a.page_rows = page_rows(L, b);
  a.by_page = fast_div(b->page_size);
  a.by_g = fast_div(G);
  a.scale = (float)((L->scale == 0.f ? 1.0 / std::sqrt((double)hd) : L->scale) * 1.4426950408889634);
  switch (hd) {
    case 64: launch_dt<64>(a, *p, L->dtype, st); break;
    case 128: launch_dt<128>(a, *p, L->dtype, st); break;
    case 256: launch_dt<256>(a, *p, L->dtype, st); break;
    default: launch_dt<512>(a, *p, L->dtype, st); break;
  }
  MS_HIP_TRY(hipGetLastError());
  return MS_OK;
}
