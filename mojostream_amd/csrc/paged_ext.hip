// Paged KV cache: the append with normed heads, both rotations and 8-bit pools, and the pools read back.
#include <cmath>
#include <type_traits>

#include "devutil.h"
#include "paged.h"

namespace ms {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));

struct AppendExtArgs {
  const PagedRow *rows;
  const float *q, *k, *v, *cos_t, *sin_t, *q_gamma, *k_gamma;
  float *q_out;
  void *kp, *vp;
  float *k_scale, *v_scale;
  size_t q_ld, kv_ld, q_out_ld;
  int n_heads, n_kv, rot, page_rows, norm;
  float eps;
  int per_row;      // heads of a row
  long total;       // threads
  FastDiv by_row;   // heads / per_row
};

// The e4m3 code of t: rounded once.  (To fp32 first with what is lost kept in the last bit, so that the
// conversion's own rounding sees on which side of a middle t is.)
__device__ inline uint32_t e4m3_of(double t) {
  const float f = (float)fabs(t);
  const double r = fabs(t) - (double)f;
  uint32_t u = __float_as_uint(f);
  if (r != 0.0 && !(u & 1)) u = r > 0.0 ? u + 1 : u - 1;
  const float x = __uint_as_float(u | (t < 0.0 ? 0x80000000u : 0u));
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x, x, 0, false) & 0xFF;
}

template <class T>
__device__ inline T sum_over(T x, int lanes) {
  for (int o = 1; o < lanes; o <<= 1) x += __shfl_xor(x, o, 64);
  return x;
}
template <class T>
__device__ inline T max_over(T x, int lanes) {
  for (int o = 1; o < lanes; o <<= 1) {
    const T y = __shfl_xor(x, o, 64);
    x = x > y ? x : y;
  }
  return x;
}

// A group of lanes has one head of a row: q heads, k heads, v heads; a lane takes 2 N of its values at a time, N
// and the N that turn with them, or 2 N side by side.  x / sqrt(mean x^2 + eps) * gamma, then the rotation; 8-bit heads
// in 64 bits (their codes are then the nearest ones), the others in 32.  A head stays in its lanes' registers: sums and
// the largest value over them by lane moves, one pass over the rows.
// Bound by memory: 3001 rows of 40 + 8 + 8 heads of 128 dims, q and k normed, e4m3: 155 MB in 35 us (4.4 TB/s; a
// large copy 4.6 to 5.1).  One row of 8 + 2 + 2 heads of 512 dims: 4.2 us, the launch and a chain of loads.
template <int DT, int HD, int N, bool PAIRS>
__global__ __launch_bounds__(kBlock) void k_append_ext(AppendExtArgs a) {
  constexpr bool E8 = DT == MS_KV_E4M3 || DT == MS_KV_I8;
  constexpr int LANES = HD / (2 * N) < 64 ? HD / (2 * N) : 64, U = HD / (2 * N) / LANES;
  const long i = (long)blockIdx.x * kBlock + threadIdx.x;
  if (i >= a.total) return;
  const uint32_t head = (uint32_t)(i / LANES);
  const int lane = (int)(i % LANES), r = (int)div_by(head, a.by_row), hh = (int)(head - (uint32_t)r * a.per_row);
  const PagedRow w = a.rows[r];
  const int nq = a.q ? a.n_heads : 0, half = a.rot >> 1;
  const int what = hh < nq ? 0 : hh < nq + a.n_kv ? 1 : 2;
  const int h = what == 0 ? hh : what == 1 ? hh - nq : hh - nq - a.n_kv;
  const float *src = (what == 0 ? a.q + r * a.q_ld : (what == 1 ? a.k : a.v) + r * a.kv_ld) + h * HD;
  const float *gamma = what == 0 ? a.q_gamma : what == 1 ? a.k_gamma : nullptr;
  const bool normed = a.norm >> what & 1;
  typedef float V __attribute__((ext_vector_type(N)));
  using L = std::conditional_t<N == 1, float, V>;

  // ---- the lane's values: v[u][j] is dim at(u, j)
  int d0[U], d1[U];
  bool turn[U];
  float v[U][2 * N];
  auto get = [](const float *p, float *to) {
    const L x = ldg<L>(p);
    if constexpr (N == 1)
      to[0] = x;
    else
#pragma unroll
      for (int j = 0; j < N; ++j) to[j] = x[j];
  };
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int p = (u * LANES + lane) * N;
    turn[u] = what < 2 && p < half;
    const bool apart = !PAIRS && what < 2;
    d0[u] = !apart ? 2 * p : turn[u] ? p : a.rot + 2 * (p - half);
    d1[u] = apart && turn[u] ? p + half : d0[u] + N;
    get(src + d0[u], v[u]);
    get(src + d1[u], v[u] + N);
  }
  double inv = 1.0;
  if (normed) {
    double ss = 0.0;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < 2 * N; ++j) ss += (double)v[u][j] * (double)v[u][j];
    inv = 1.0 / sqrt(sum_over(ss, LANES) / HD + (double)a.eps);
  }

  auto finish = [&](auto zero) {
    using T = decltype(zero);
    T y[U][2 * N];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int j = 0; j < 2 * N; ++j) y[u][j] = normed ? (T)((double)v[u][j] * inv) : (T)v[u][j];
      if (normed && gamma) {
        float g[2 * N];
        get(gamma + d0[u], g);
        get(gamma + d1[u], g + N);
#pragma unroll
        for (int j = 0; j < 2 * N; ++j) y[u][j] *= (T)g[j];
      }
      if (turn[u]) {
        const size_t t = (size_t)w.pos * half + (u * LANES + lane) * N;
        float c[N], s[N];
        get(a.cos_t + t, c);
        get(a.sin_t + t, s);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          T &p = y[u][PAIRS ? 2 * j : j], &q = y[u][PAIRS ? 2 * j + 1 : N + j];
          const T p0 = p;
          p = p0 * (T)c[j] - q * (T)s[j];
          q = p0 * (T)s[j] + q * (T)c[j];
        }
      }
    }
    if constexpr (std::is_same_v<T, double>) {
      // ---- 8 bits
      constexpr double TOP = DT == MS_KV_E4M3 ? 448.0 : 127.0;
      constexpr float MOST = DT == MS_KV_E4M3 ? 0x1.249248p+119f : 0x1.020406p+121f;  // TOP times it is finite
      double big = 0.0;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < 2 * N; ++j) {
          const double m = fabs(y[u][j]);
          big = m > big ? m : m <= big ? big : (double)INFINITY;  // (NaN counts as infinite)
        }
      big = max_over(big, LANES);  // (a value past fp32's range is infinite: rotations and gammas may lead there)
      const float scale = big <= 0x1.fffffep+127 ? fminf(fmaxf((float)(big / TOP), 0x1p-126f), MOST) : NAN;
      uint8_t *pool = static_cast<uint8_t *>(what == 1 ? a.kp : a.vp) +
                      (((size_t)w.page * a.page_rows + w.slot) * a.n_kv + h) * HD;
      if (lane == 0)
        (what == 1 ? a.k_scale : a.v_scale)[((size_t)w.page * a.n_kv + h) * a.page_rows + w.slot] = scale;
      const double by = scale < INFINITY ? (double)scale : 1.0;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          uint32_t word = 0;
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const double t = scale < INFINITY ? y[u][N * part + j] / by : 0.0;
            const uint32_t c = DT == MS_KV_E4M3 ? e4m3_of(t) : (uint32_t)(int)rint(t) & 0xFF;
            word |= c << (8 * j);
          }
          uint8_t *to = pool + (part ? d1[u] : d0[u]);
          if constexpr (N == 4)
            *reinterpret_cast<uint32_t *>(to) = word;
          else
            *to = (uint8_t)word;
        }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          const int d = part ? d1[u] : d0[u];
          L x;
          if constexpr (N == 1)
            x = y[u][part];
          else
#pragma unroll
            for (int j = 0; j < N; ++j) x[j] = y[u][N * part + j];
          if (what == 0) {
            *reinterpret_cast<L *>(a.q_out + r * a.q_out_ld + h * HD + d) = x;
          } else if constexpr (!E8) {
            const size_t at = (((size_t)w.page * a.page_rows + w.slot) * a.n_kv + h) * HD + d;
            store_kv<DT>(what == 1 ? a.kp : a.vp, at, x);
          }
        }
    }
  };
  if (E8 && what > 0)
    finish(0.0);
  else
    finish(0.f);
}

template <int DT, int HD>
void launch_append(const AppendExtArgs &args, int rows, bool four, bool pairs, hipStream_t st) {
  AppendExtArgs a = args;
  a.total = (long)rows * a.per_row * (four ? HD / 8 : HD / 2 < 64 ? HD / 2 : 64);
  const dim3 grid(cdiv(a.total, kBlock)), blk(kBlock);
  if (four && pairs)
    hipLaunchKernelGGL((k_append_ext<DT, HD, 4, true>), grid, blk, 0, st, a);
  else if (four)
    hipLaunchKernelGGL((k_append_ext<DT, HD, 4, false>), grid, blk, 0, st, a);
  else if (pairs)
    hipLaunchKernelGGL((k_append_ext<DT, HD, 1, true>), grid, blk, 0, st, a);
  else
    hipLaunchKernelGGL((k_append_ext<DT, HD, 1, false>), grid, blk, 0, st, a);
}
template <int DT>
void launch_append(const AppendExtArgs &a, int hd, int rows, bool four, bool pairs, hipStream_t st) {
  switch (hd) {
    case 64: return launch_append<DT, 64>(a, rows, four, pairs, st);
    case 128: return launch_append<DT, 128>(a, rows, four, pairs, st);
    case 256: return launch_append<DT, 256>(a, rows, four, pairs, st);
    default: return launch_append<DT, 512>(a, rows, four, pairs, st);
  }
}

struct ReadArgs {
  const int32_t *pages;  // of the sequence
  const void *kp, *vp;
  const float *k_scale, *v_scale;
  float *k, *v;
  size_t ld;
  int pos0, n_kv, log_units, page_size, page_rows;
  uint32_t total;
  FastDiv by_page, by_row;
};

// Four values of a pool in fp32.
template <int DT>
__device__ inline f4 load4(const void *pool, size_t at) {
  if constexpr (DT == MS_KV_F32) {
    return ldg<f4>(static_cast<const float *>(pool) + at);
  } else if constexpr (DT == MS_KV_BF16) {
    return __builtin_convertvector(ldg<bf4>(static_cast<const __bf16 *>(pool) + at), f4);
  } else if constexpr (DT == MS_KV_F16) {
    return __builtin_convertvector(ldg<half4_t>(static_cast<const _Float16 *>(pool) + at), f4);
  } else {
    const uint32_t w = ldg<uint32_t>(static_cast<const uint8_t *>(pool) + at);
    if constexpr (DT == MS_KV_E4M3)
      return f4{__builtin_amdgcn_cvt_f32_fp8(w, 0), __builtin_amdgcn_cvt_f32_fp8(w, 1),
                __builtin_amdgcn_cvt_f32_fp8(w, 2), __builtin_amdgcn_cvt_f32_fp8(w, 3)};
    else
      return f4{(float)(int8_t)w, (float)(int8_t)(w >> 8), (float)(int8_t)(w >> 16), (float)(int8_t)(w >> 24)};
  }
}

// A thread has four values of k and of v of one position: 16 bytes of each written.  Bound by memory: 20011 positions of 8
// heads of 128 dims, int8, 206 MB, four fifths of them written, in 31 us (6.6 TB/s); 700 of 2 heads of 256 dims 2.9 us.
// Rows that are more than half of the last cache (256 MB) are written past the caches.  Of three layers in turn, int8, in the caches
// and past them: 64 MB 17.8 and 17.0 us, 128 MB 44 and 29, 160 MB 52 and 35, 256 MB 80 and 52, 400 MB 120 and 112; what
// reads them next pays for it where they would have been there: with a sum over both behind each 69 and 74, 105 and 112, 123
// and 127, 170 and 175, 255 and 248 (a sum over the same rows again and again, 164 MB, 90 and 83).  Rows of 160 MB
// out of bf16 pools 46 us, out of fp32 pools 60.
template <int DT, bool PAST>
__global__ __launch_bounds__(kBlock) void k_paged_read(ReadArgs a) {
  constexpr bool E8 = DT == MS_KV_E4M3 || DT == MS_KV_I8;
  const uint32_t i = blockIdx.x * kBlock + threadIdx.x;
  if (i >= a.total) return;
  const uint32_t r = div_by(i, a.by_row), u = i - r * (a.n_kv << a.log_units), h = u >> a.log_units;
  const uint32_t pos = a.pos0 + r, pg = div_by(pos, a.by_page), slot = pos - pg * a.page_size;
  const size_t page = (uint32_t)ldg<int32_t>(a.pages + pg);
  const size_t at = ((page * a.page_rows + slot) * a.n_kv << a.log_units) * 4 + 4 * u;
  const size_t sc = (page * a.n_kv + h) * a.page_rows + slot, to = (size_t)r * a.ld + 4 * u;
  auto put = [&](float *p, f4 x) {
    if constexpr (PAST)
      __builtin_nontemporal_store(x, reinterpret_cast<f4 *>(p));
    else
      *reinterpret_cast<f4 *>(p) = x;
  };
  if (a.k) {
    f4 x = load4<DT>(a.kp, at);
    if constexpr (E8) x *= ldg<float>(a.k_scale + sc);
    put(a.k + to, x);
  }
  if (a.v) {
    f4 x = load4<DT>(a.vp, at);
    if constexpr (E8) x *= ldg<float>(a.v_scale + sc);
    put(a.v + to, x);
  }
}

template <int DT>
void launch_read(const ReadArgs &a, bool past, hipStream_t st) {
  const dim3 grid(cdiv(a.total, kBlock)), blk(kBlock);
  if (past)
    hipLaunchKernelGGL((k_paged_read<DT, true>), grid, blk, 0, st, a);
  else
    hipLaunchKernelGGL((k_paged_read<DT, false>), grid, blk, 0, st, a);
}

}  // namespace
}  // namespace ms

using namespace ms;

extern "C" int ms_paged_append_ext(const ms_paged_layer_ext *X, const ms_paged_batch *b,
                                   const float *d_k, const float *d_v, size_t kv_stride,
                                   const float *d_q, size_t q_stride, float *d_q_out,
                                   size_t q_out_stride, const float *d_cos, const float *d_sin,
                                   int n_pos) {
  const char *what = "paged_append_ext";
  MS_CHECK_ARG(X, "paged_append_ext: null layer or batch");
  MS_CHECK_ARG(X->norm >= 0 && X->norm <= (MS_NORM_Q | MS_NORM_K | MS_NORM_V),
               "paged_append_ext: unknown norm");
  MS_CHECK_ARG(!X->norm || (X->norm_eps >= 0.f && X->norm_eps < INFINITY),
               "paged_append_ext: norm_eps must be finite and not negative");
  MS_CHECK_ARG(X->rope == MS_ROPE_HALVES || X->rope == MS_ROPE_PAIRS, "paged_append_ext: unknown rotation");
  MS_CHECK_ARG(((reinterpret_cast<uintptr_t>(X->q_gamma) | reinterpret_cast<uintptr_t>(X->k_gamma)) & 3) == 0,
               "paged_append_ext: the gammas must be 4-byte aligned");
  if (int rc = append_check(what, &X->base, X, b, d_k, d_v, kv_stride, d_q, q_stride,
                            d_q_out, q_out_stride, d_cos, d_sin, n_pos))
    return rc;
  const ms_paged_layer *L = &X->base;
  if (b->rows == 0) return require_init();
  if (!X->norm && !is_8bit(L->dtype) && (X->rope == MS_ROPE_HALVES || L->rot_dim == 0))
    return ms_paged_append(L, b, d_k, d_v, kv_stride, d_q, q_stride, d_q_out, q_out_stride, d_cos,
                           d_sin, n_pos);
  AppendExtArgs a{};
  a.rows = b->d_rows();
  a.q = d_q;
  a.k = d_k;
  a.v = d_v;
  a.cos_t = d_cos;
  a.sin_t = d_sin;
  a.q_gamma = X->q_gamma;
  a.k_gamma = X->k_gamma;
  a.q_out = d_q_out;
  a.kp = L->k;
  a.vp = L->v;
  a.k_scale = X->k_scale;
  a.v_scale = X->v_scale;
  a.q_ld = q_stride;
  a.kv_ld = kv_stride;
  a.q_out_ld = q_out_stride;
  a.n_heads = L->n_heads;
  a.n_kv = L->n_kv_heads;
  a.rot = L->rot_dim;
  a.page_rows = page_rows(L, b);
  a.norm = X->norm;
  a.eps = X->norm_eps;
  a.per_row = (d_q ? L->n_heads : 0) + 2 * L->n_kv_heads;
  a.by_row = fast_div(a.per_row);
  MS_CHECK_ARG((int64_t)b->rows * a.per_row * L->head_dim / 2 < ((int64_t)1 << 31),
               "paged_append_ext: too many rows for one call");
  // four values a load where they, their table entries and gammas are whole 16-byte words
  const bool four = L->rot_dim % 8 == 0 && (L->rot_dim == 0 || (aligned16(d_cos) && aligned16(d_sin))) &&
                    aligned16(X->q_gamma) && aligned16(X->k_gamma);
  const bool pairs = X->rope == MS_ROPE_PAIRS;
  if (int rc = require_init()) return rc;
  OnDevice on;
  hipStream_t st = ctx().stream;
  switch (L->dtype) {
    case MS_KV_F32: launch_append<MS_KV_F32>(a, L->head_dim, b->rows, four, pairs, st); break;
    case MS_KV_BF16: launch_append<MS_KV_BF16>(a, L->head_dim, b->rows, four, pairs, st); break;
    case MS_KV_F16: launch_append<MS_KV_F16>(a, L->head_dim, b->rows, four, pairs, st); break;
    case MS_KV_E4M3: launch_append<MS_KV_E4M3>(a, L->head_dim, b->rows, four, pairs, st); break;
    default: launch_append<MS_KV_I8>(a, L->head_dim, b->rows, four, pairs, st);
  }
  MS_HIP_TRY(hipGetLastError());
  return MS_OK;
}

extern "C" int ms_paged_read(const ms_paged_layer_ext *X, const ms_paged_batch *b, int seq,
                             int pos0, int n, float *d_k, float *d_v, size_t stride) {
  if (int rc = paged_check_ext("paged_read", X, b)) return rc;
  const ms_paged_layer *L = &X->base;
  MS_CHECK_ARG(seq >= 0 && seq < b->n_seqs, "paged_read: no such sequence");
  MS_CHECK_ARG(pos0 >= 0 && n >= 0 && (int64_t)pos0 + n <= b->len[seq],
               "paged_read: positions past the sequence");
  MS_CHECK_ARG(n == 0 || pos0 >= b->held[seq], "paged_read: a position whose page is -1");
  if (n == 0 || (!d_k && !d_v)) return require_init();
  const int kv_dim = L->n_kv_heads * L->head_dim;
  MS_CHECK_ARG(aligned16(d_k) && aligned16(d_v) && stride % 4 == 0 && stride >= (size_t)kv_dim &&
                   stride < ((size_t)1 << 31),
               "paged_read: bad output rows");
  MS_CHECK_ARG(!d_k || !d_v || !rows_overlap(d_k, stride, kv_dim, d_v, stride, kv_dim, n),
               "paged_read: d_k and d_v overlap");
  MS_CHECK_ARG((int64_t)n * kv_dim / 4 < ((int64_t)1 << 31), "paged_read: too many positions for one call");
  if (int rc = require_init()) return rc;
  OnDevice on;
  ReadArgs a{};
  a.pages = b->d_pages() + (size_t)seq * b->stride;
  a.kp = L->k;
  a.vp = L->v;
  a.k_scale = X->k_scale;
  a.v_scale = X->v_scale;
  a.k = d_k;
  a.v = d_v;
  a.ld = stride;
  a.pos0 = pos0;
  a.n_kv = L->n_kv_heads;
  while ((4 << a.log_units) < L->head_dim) ++a.log_units;
  a.page_size = b->page_size;
  a.page_rows = page_rows(L, b);
  a.by_page = fast_div(b->page_size);
  a.by_row = fast_div(kv_dim / 4);
  a.total = (uint32_t)n * (kv_dim / 4);
  const bool past = (int64_t)n * kv_dim * 4 * ((d_k != nullptr) + (d_v != nullptr)) > ((int64_t)1 << 27);
  hipStream_t st = ctx().stream;
  switch (L->dtype) {
    case MS_KV_F32: launch_read<MS_KV_F32>(a, past, st); break;
    case MS_KV_BF16: launch_read<MS_KV_BF16>(a, past, st); break;
    case MS_KV_F16: launch_read<MS_KV_F16>(a, past, st); break;
    case MS_KV_E4M3: launch_read<MS_KV_E4M3>(a, past, st); break;
    default: launch_read<MS_KV_I8>(a, past, st);
  }
  MS_HIP_TRY(hipGetLastError());
  return MS_OK;
}
