// Paged KV cache: the batch handle, the rotary tables and the append.
#include <cmath>
#include <cstring>
#include <exception>
#include <new>
#include <type_traits>

#include "devutil.h"
#include "paged.h"
#include "rope.h"

namespace ms {

int Upload::reserve(size_t bytes) {
  if (sent) MS_HIP_TRY(hipEventSynchronize(sent));
  if (bytes <= cap) return MS_OK;
  hipEvent_t keep = sent;
  if (!keep) MS_HIP_TRY(hipEventCreateWithFlags(&keep, hipEventDisableTiming));
  sent = nullptr;
  // (kernels in flight may still read the old copy)
  MS_HIP_TRY(hipStreamSynchronize(ctx().stream));
  release();
  sent = keep;
  bytes = (bytes + 4095) & ~(size_t)4095;
  if (hipHostMalloc(reinterpret_cast<void **>(&h), bytes, hipHostMallocDefault) != hipSuccess ||
      hipMalloc(reinterpret_cast<void **>(&d), bytes) != hipSuccess) {
    release();
    return fail(MS_E_NOMEM, "paged: no memory for the batch's tables");
  }
  cap = bytes;
  return MS_OK;
}

int Upload::send(size_t bytes) {
  MS_HIP_TRY(hipMemcpyAsync(d, h, bytes, hipMemcpyHostToDevice, ctx().stream));
  MS_HIP_TRY(hipEventRecord(sent, ctx().stream));
  return MS_OK;
}

void Upload::release() {
  if (sent) (void)hipEventDestroy(sent);
  if (h) (void)hipHostFree(h);
  if (d) (void)hipFree(d);
  h = d = nullptr;
  sent = nullptr;
  cap = 0;
}

int paged_check(const char *what, const ms_paged_layer *L, const ms_paged_batch *b) {
  auto w = [what](const char *msg) { return std::string(what) + msg; };
  MS_CHECK_ARG(L && b, w(": null layer or batch"));
  MS_CHECK_ARG(L->n_kv_heads >= 1 && L->n_heads >= 1 && L->n_heads % L->n_kv_heads == 0,
               w(": n_heads must be a multiple of n_kv_heads"));
  MS_CHECK_ARG(L->n_heads <= 1024, w(": at most 1024 query heads"));
  MS_CHECK_ARG(L->head_dim == 64 || L->head_dim == 128 || L->head_dim == 256 ||
                   L->head_dim == 512,
               w(": head_dim must be 64, 128, 256 or 512"));
  MS_CHECK_ARG(L->dtype == MS_KV_F32 || L->dtype == MS_KV_BF16 || L->dtype == MS_KV_F16,
               w(": unknown pool type"));
  MS_CHECK_ARG(L->window >= 0, w(": negative window"));
  MS_CHECK_ARG(L->page_rows == 0 || L->page_rows >= b->page_size,
               w(": page_rows is less than the page size"));
  MS_CHECK_ARG((int64_t)page_rows(L, b) * b->n_pages < ((int64_t)1 << 31),
               w(": a pool has fewer than 2^31 rows"));
  MS_CHECK_ARG(L->k && L->v, w(": null pool"));
  MS_CHECK_ARG(((reinterpret_cast<uintptr_t>(L->k) | reinterpret_cast<uintptr_t>(L->v)) & 15) == 0,
               w(": the pools must be 16-byte aligned"));
  MS_CHECK_ARG(b->set, w(": the batch was not set"));
  return MS_OK;
}

bool rows_overlap(const void *a, size_t stride_a, int na, const void *b, size_t stride_b, int nb,
                  int rows) {
  if (rows <= 0) return false;
  const uintptr_t a0 = reinterpret_cast<uintptr_t>(a), b0 = reinterpret_cast<uintptr_t>(b);
  const uintptr_t wa = (uintptr_t)na * 4, wb = (uintptr_t)nb * 4;
  if (a0 >= b0 + (rows - 1) * stride_b * 4 + wb || b0 >= a0 + (rows - 1) * stride_a * 4 + wa)
    return false;
  // rows of one stride side by side (q | k | v) are apart where, modulo the stride, b's row
  // starts behind a's and ends before a's next
  if (stride_a == stride_b) {
    const uintptr_t S = stride_a * 4, d = b0 >= a0 ? (b0 - a0) % S : (S - (a0 - b0) % S) % S;
    if (d >= wa && d + wb <= S) return false;
  }
  return true;
}

namespace {

// cos and sin of pos * theta^(-2i/rot) in 64 bits, rounded once.
__global__ void k_rope_table(float *cs, float *sn, int half, double step, int pos0, long total) {
  const long i = (long)blockIdx.x * kBlock + threadIdx.x;
  if (i >= total) return;
  const double ang = (double)(pos0 + i / half) * exp(step * (double)(i % half));
  cs[i] = (float)cos(ang);
  sn[i] = (float)sin(ang);
}

struct AppendArgs {
  const PagedRow *rows;
  const float *q, *k, *v, *cos_t, *sin_t;
  float *q_out;
  void *kp, *vp;
  size_t q_ld, kv_ld, q_out_ld;
  int n_heads, n_kv, hd, rot, page_rows;
  int log_units;  // log2 of a head's threads
  int per_row;    // threads of a row
  long total;
  FastDiv by_row;  // total < 2^31
};

typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));

// One or four values of a pool, rounded to nearest even.
template <int DT, class V>
__device__ inline void store_kv(void *pool, size_t at, V x) {
  constexpr bool ONE = sizeof(V) == 4;
  if constexpr (DT == MS_KV_F32)
    *reinterpret_cast<V *>(static_cast<float *>(pool) + at) = x;
  else if constexpr (DT == MS_KV_BF16 && ONE)
    static_cast<__bf16 *>(pool)[at] = (__bf16)x;
  else if constexpr (DT == MS_KV_BF16)
    *reinterpret_cast<bf4 *>(static_cast<__bf16 *>(pool) + at) = __builtin_convertvector(x, bf4);
  else if constexpr (ONE)
    static_cast<_Float16 *>(pool)[at] = (_Float16)x;
  else
    *reinterpret_cast<half4_t *>(static_cast<_Float16 *>(pool) + at) = __builtin_convertvector(x, half4_t);
}

// A thread takes N values and the N that turn with them (or 2 N side by side that do not turn) of
// one head of a row: q heads, k heads, v heads.  Bound by memory: 3001 rows of 40 + 8 + 8 heads
// of 128 dims into bf16 pools, 161 MB, in 30 us (with one pair a thread 43 us); a step of single
// tokens by its launch (2.2 to 2.6 us).
template <int DT, int N>
__global__ void k_paged_append(AppendArgs a) {
  typedef float V __attribute__((ext_vector_type(N)));
  using T = std::conditional_t<N == 1, float, V>;
  const long i = (long)blockIdx.x * kBlock + threadIdx.x;
  if (i >= a.total) return;
  const int r = (int)div_by((uint32_t)i, a.by_row), u = (int)(i - (long)r * a.per_row);
  const int hh = u >> a.log_units, p = (u & ((1 << a.log_units) - 1)) * N, half = a.rot >> 1;
  const PagedRow w = a.rows[r];
  const int nq = a.q ? a.n_heads : 0;
  const int what = hh < nq ? 0 : hh < nq + a.n_kv ? 1 : 2;
  const int h = what == 0 ? hh : what == 1 ? hh - nq : hh - nq - a.n_kv;
  const bool turn = what < 2 && p < half;
  const int d0 = what == 2 ? 2 * p : turn ? p : a.rot + 2 * (p - half), d1 = turn ? p + half : d0 + N;
  const float *src = (what == 0 ? a.q + r * a.q_ld : (what == 1 ? a.k : a.v) + r * a.kv_ld) + h * a.hd;
  T x = ldg<T>(src + d0), y = ldg<T>(src + d1);
  if (turn) {
    const size_t t = (size_t)w.pos * half + p;
    const T c = ldg<T>(a.cos_t + t), s = ldg<T>(a.sin_t + t), x0 = x;
    x = x0 * c - y * s;
    y = x0 * s + y * c;
  }
  if (what == 0) {
    float *o = a.q_out + r * a.q_out_ld + h * a.hd;
    *reinterpret_cast<T *>(o + d0) = x;
    *reinterpret_cast<T *>(o + d1) = y;
  } else {
    const size_t at = (((size_t)w.page * a.page_rows + w.slot) * a.n_kv + h) * a.hd;
    store_kv<DT>(what == 1 ? a.kp : a.vp, at + d0, x);
    store_kv<DT>(what == 1 ? a.kp : a.vp, at + d1, y);
  }
}

template <int N>
void launch_append(const AppendArgs &a, int dtype, hipStream_t st) {
  const dim3 grid(cdiv(a.total, kBlock)), blk(kBlock);
  if (dtype == MS_KV_F32)
    hipLaunchKernelGGL((k_paged_append<MS_KV_F32, N>), grid, blk, 0, st, a);
  else if (dtype == MS_KV_BF16)
    hipLaunchKernelGGL((k_paged_append<MS_KV_BF16, N>), grid, blk, 0, st, a);
  else
    hipLaunchKernelGGL((k_paged_append<MS_KV_F16, N>), grid, blk, 0, st, a);
}

}  // namespace
}  // namespace ms

using namespace ms;

extern "C" int ms_paged_batch_create(int page_size, int n_pages, int max_seqs, int max_rows,
                                     int max_pages, ms_paged_batch **out) {
  MS_CHECK_ARG(out, "paged_batch_create: null out pointer");
  *out = nullptr;
  MS_CHECK_ARG(page_size >= 1 && n_pages >= 1 && max_seqs >= 1 && max_rows >= 1 && max_pages >= 1,
               "paged_batch_create: sizes must be positive");
  MS_CHECK_ARG((int64_t)page_size * n_pages < ((int64_t)1 << 31) &&
                   (int64_t)page_size * max_pages <= ((int64_t)1 << 30),
               "paged_batch_create: fewer than 2^31 slots, at most 2^30 positions a sequence");
  MS_CHECK_ARG((int64_t)max_seqs * max_pages < ((int64_t)1 << 28) && max_seqs <= (1 << 20) &&
                   max_rows <= (1 << 24),
               "paged_batch_create: too many sequences, rows or pages");
  try {
    ms_paged_batch *b = new ms_paged_batch();
    b->page_size = page_size;
    b->n_pages = n_pages;
    b->max_seqs = max_seqs;
    b->max_rows = max_rows;
    b->max_pages = max_pages;
    *out = b;
    b->writer.assign(n_pages, 0);
  } catch (const std::exception &e) {
    delete *out;
    *out = nullptr;
    return fail(MS_E_NOMEM, std::string("paged_batch_create: ") + e.what());
  }
  return MS_OK;
}

extern "C" int ms_paged_batch_destroy(ms_paged_batch *b) {
  if (!b) return MS_OK;
  {
    OnDevice on;
    if (ctx().device >= 0) (void)hipStreamSynchronize(ctx().stream);
    b->up.release();
    for (PagedPlan *p : b->plans) {
      p->up.release();
      delete p;
    }
  }
  delete b;
  return MS_OK;
}

extern "C" int ms_paged_batch_set(ms_paged_batch *b, int n_seqs, const int32_t *h_new,
                                  const int32_t *h_len, const int32_t *h_pages) {
  MS_CHECK_ARG(b, "paged_batch_set: null batch");
  MS_CHECK_ARG(n_seqs >= 0 && n_seqs <= b->max_seqs, "paged_batch_set: too many sequences");
  MS_CHECK_ARG(n_seqs == 0 || (h_new && h_len && h_pages), "paged_batch_set: null argument");
  const int P = b->page_size;
  try {
    std::vector<int32_t> first(n_seqs), n_new(n_seqs), len(n_seqs), held(n_seqs);
    int64_t rows = 0;
    int stride = 0, max_pos = 0;
    const int64_t stamp = ++b->n_set;
    for (int s = 0; s < n_seqs; ++s) {
      auto w = [&](const std::string &msg) { return "paged_batch_set: sequence " + std::to_string(s) + ": " + msg; };
      const int n = h_new[s], l = h_len[s];
      MS_CHECK_ARG(n >= 0 && l >= n, w("the length is less than its new rows"));
      MS_CHECK_ARG((int64_t)l <= (int64_t)P * b->max_pages, w("more positions than its pages hold"));
      const int used = l == 0 ? 0 : (l - 1) / P + 1;
      const int32_t *pg = h_pages + (size_t)s * b->max_pages;
      int gone = 0;
      while (gone < used && pg[gone] == -1) ++gone;
      for (int i = gone; i < used; ++i)
        MS_CHECK_ARG(pg[i] >= 0 && pg[i] < b->n_pages,
                     w("page " + std::to_string(i) + " is " + std::to_string(pg[i])));
      MS_CHECK_ARG(n == 0 || (l - n) / P >= gone, w("a new row's page is missing"));
      for (int i = n ? (l - n) / P : used; i < used; ++i) {
        MS_CHECK_ARG(b->writer[pg[i]] != stamp,
                     w("page " + std::to_string(pg[i]) + " would be written twice"));
        b->writer[pg[i]] = stamp;
      }
      first[s] = (int)rows;
      n_new[s] = n;
      len[s] = l;
      held[s] = gone * P;
      rows += n;
      MS_CHECK_ARG(rows <= b->max_rows, w("more rows than the batch holds"));
      stride = used > stride ? used : stride;
      if (n && l > max_pos) max_pos = l;
    }
    if (int rc = require_init()) return rc;
    OnDevice on;
    const size_t rb = ((size_t)rows * sizeof(PagedRow) + 255) & ~(size_t)255;
    const size_t pb = (size_t)n_seqs * stride * 4;
    if (rb + pb) {
      b->set = false;  // (a batch that fails from here on has no tables)
      if (int rc = b->up.reserve(rb + pb)) return rc;
      PagedRow *rw = reinterpret_cast<PagedRow *>(b->up.h);
      int32_t *tab = reinterpret_cast<int32_t *>(b->up.h + rb);
      for (int s = 0; s < n_seqs; ++s) {
        const int32_t *pg = h_pages + (size_t)s * b->max_pages;
        for (int p = len[s] - n_new[s]; p < len[s]; ++p) *rw++ = PagedRow{p, pg[p / P], p % P, s};
        const int used = len[s] == 0 ? 0 : (len[s] - 1) / P + 1;
        if (used) std::memcpy(tab + (size_t)s * stride, pg, (size_t)used * 4);
        for (int i = used; i < stride; ++i) tab[(size_t)s * stride + i] = -1;
      }
      if (int rc = b->up.send(rb + pb)) return rc;
    }
    b->first.swap(first);
    b->n_new.swap(n_new);
    b->len.swap(len);
    b->held.swap(held);
    b->n_seqs = n_seqs;
    b->rows = (int)rows;
    b->stride = stride;
    b->max_pos = max_pos;
    b->pages_at = rb;
    b->set = true;
    for (PagedPlan *p : b->plans) p->valid = false;
  } catch (const std::exception &e) {
    return fail(MS_E_NOMEM, std::string("paged_batch_set: ") + e.what());
  }
  return MS_OK;
}

extern "C" int ms_rope_table(float *d_cos, float *d_sin, int rot_dim, float theta, int pos0,
                             int n_pos, int wide) {
  MS_CHECK_ARG(d_cos && d_sin, "rope_table: null table");
  MS_CHECK_ARG(rot_dim >= 2 && rot_dim % 2 == 0 && theta > 0.f && theta < INFINITY && pos0 >= 0 &&
                   n_pos >= 0 && (int64_t)pos0 + n_pos < ((int64_t)1 << 31),
               "rope_table: bad arguments");
  // (a launch has fewer than 2^32 threads)
  MS_CHECK_ARG((int64_t)n_pos * (rot_dim / 2) <= ((int64_t)1 << 31), "rope_table: table too large");
  if (int rc = require_init()) return rc;
  if (!n_pos) return MS_OK;
  OnDevice on;
  const long total = (long)n_pos * (rot_dim / 2);
  if (wide) {
    hipLaunchKernelGGL(k_rope_table, dim3(cdiv(total, kBlock)), dim3(kBlock), 0, ctx().stream,
                       d_cos, d_sin, rot_dim / 2, -2.0 * std::log((double)theta) / rot_dim, pos0,
                       total);
    MS_HIP_TRY(hipGetLastError());
    return MS_OK;
  }
  try {
    std::vector<float> cs, sn;
    rope_table_host(rot_dim, theta, pos0, n_pos, cs, sn);
    MS_HIP_TRY(hipMemcpyAsync(d_cos, cs.data(), cs.size() * 4, hipMemcpyHostToDevice, ctx().stream));
    MS_HIP_TRY(hipMemcpyAsync(d_sin, sn.data(), sn.size() * 4, hipMemcpyHostToDevice, ctx().stream));
    MS_HIP_TRY(hipStreamSynchronize(ctx().stream));  // the vectors end here
  } catch (const std::exception &e) {
    return fail(MS_E_NOMEM, std::string("rope_table: ") + e.what());
  }
  return MS_OK;
}

extern "C" int ms_paged_append(const ms_paged_layer *L, const ms_paged_batch *b, const float *d_k,
                               const float *d_v, size_t kv_stride, const float *d_q,
                               size_t q_stride, float *d_q_out, size_t q_out_stride,
                               const float *d_cos, const float *d_sin, int n_pos) {
  MS_CHECK_ARG(L, "paged_append: null layer or batch");
  MS_CHECK_ARG(L->rot_dim >= 0 && L->rot_dim % 2 == 0 && L->rot_dim <= L->head_dim,
               "paged_append: rot_dim must be even and at most head_dim");
  MS_CHECK_ARG(L->rot_dim == 0 || (d_cos && d_sin), "paged_append: rotary tables missing");
  if (int rc = paged_check("paged_append", L, b)) return rc;
  const int kv_dim = L->n_kv_heads * L->head_dim, q_dim = L->n_heads * L->head_dim;
  MS_CHECK_ARG(L->rot_dim == 0 || b->max_pos <= n_pos,
               "paged_append: a position past the rotary tables");
  if (b->rows == 0) return require_init();
  MS_CHECK_ARG(d_k && d_v && aligned16(d_k) && aligned16(d_v) && kv_stride % 4 == 0 &&
                   kv_stride >= (size_t)kv_dim && kv_stride < ((size_t)1 << 31),
               "paged_append: bad k or v rows");
  if (d_q) {
    MS_CHECK_ARG(d_q_out && aligned16(d_q) && aligned16(d_q_out) && q_stride % 4 == 0 &&
                     q_out_stride % 4 == 0 && q_stride >= (size_t)q_dim &&
                     q_out_stride >= (size_t)q_dim && q_stride < ((size_t)1 << 31) &&
                     q_out_stride < ((size_t)1 << 31),
                 "paged_append: bad q rows");
    MS_CHECK_ARG((d_q_out == d_q && q_out_stride == q_stride) ||
                     !rows_overlap(d_q, q_stride, q_dim, d_q_out, q_out_stride, q_dim, b->rows),
                 "paged_append: d_q and d_q_out overlap");
    MS_CHECK_ARG(!rows_overlap(d_k, kv_stride, kv_dim, d_q_out, q_out_stride, q_dim, b->rows) &&
                     !rows_overlap(d_v, kv_stride, kv_dim, d_q_out, q_out_stride, q_dim, b->rows),
                 "paged_append: d_q_out overlaps the k or v rows");
  }
  AppendArgs a{};
  a.rows = b->d_rows();
  a.q = d_q;
  a.k = d_k;
  a.v = d_v;
  a.q_out = d_q_out;
  a.cos_t = d_cos;
  a.sin_t = d_sin;
  a.kp = L->k;
  a.vp = L->v;
  a.q_ld = q_stride;
  a.kv_ld = kv_stride;
  a.q_out_ld = q_out_stride;
  a.n_heads = L->n_heads;
  a.n_kv = L->n_kv_heads;
  a.hd = L->head_dim;
  a.rot = L->rot_dim;
  a.page_rows = page_rows(L, b);
  // four pairs a thread where they and their table entries are whole 16-byte words
  const bool four = L->rot_dim % 8 == 0 && (L->rot_dim == 0 || (aligned16(d_cos) && aligned16(d_sin)));
  const int units = L->head_dim / (four ? 8 : 2);
  while ((1 << a.log_units) < units) ++a.log_units;
  a.per_row = ((d_q ? L->n_heads : 0) + 2 * L->n_kv_heads) * units;
  a.total = (long)a.per_row * b->rows;
  a.by_row = fast_div(a.per_row);
  MS_CHECK_ARG(a.total < ((long)1 << 31), "paged_append: too many rows for one call");
  if (int rc = require_init()) return rc;
  OnDevice on;
  if (four)
    launch_append<4>(a, L->dtype, ctx().stream);
  else
    launch_append<1>(a, L->dtype, ctx().stream);
  MS_HIP_TRY(hipGetLastError());
  return MS_OK;
}
