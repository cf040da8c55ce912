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

// The item's rows one after the other, key by key, with 256 threads: a key no row
// attends to is never multiplied by anything.
template <int HD, int DT, int NQ>
__device__ __noinline__ void item_by_key(const PagedAttnArgs &a, const PagedItem &it, int kvh,
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
      const float p = on ? __builtin_amdgcn_exp2f(s - base) : 0.f;
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
        const size_t pr = ((size_t)it.part * a.n_kv + kvh) * (16 * NQ) + r;
        a.part_o[pr * HD + d] = o[i];
        if (d == 0) {
          a.part_ml[pr * 2] = m;
          a.part_ml[pr * 2 + 1] = l;
        }
      }
    }
  }
}

template <int HD, int DT, int NQ>
__global__ __launch_bounds__(256) void k_paged_attn(PagedAttnArgs a) {
  __shared__ float lds[264];
  const int kvh = blockIdx.x % a.n_kv;
  const PagedItem it = a.items[blockIdx.x / a.n_kv];
  item_by_key<HD, DT, NQ>(a, it, kvh, lds);
}

// The parts of one result, weighted by e^(their maximum - the largest).
template <int HD, int NQ>
__global__ __launch_bounds__(256) void k_paged_merge(PagedAttnArgs a, const PagedMerge *merge) {
  const int kvh = blockIdx.x % a.n_kv;
  const PagedMerge g = merge[blockIdx.x / a.n_kv];
  const int nrows = min(16 * NQ, g.n_new * a.G - g.r0);
  for (int i = threadIdx.x; i < nrows * (HD / 4); i += 256) {
    const int r = i / (HD / 4), d = (i % (HD / 4)) * 4;
    const size_t pr = ((size_t)g.part * a.n_kv + kvh) * (16 * NQ) + r, step = (size_t)a.n_kv * 16 * NQ;
    float m = -INFINITY;
    for (int p = 0; p < g.n; ++p) m = fmaxf(m, ldg<float>(a.part_ml + (pr + p * step) * 2));
    const float base = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    float4_t o = {};
    for (int p = 0; p < g.n; ++p) {
      const float w = __builtin_amdgcn_exp2f(ldg<float>(a.part_ml + (pr + p * step) * 2) - base);
      l += w * ldg<float>(a.part_ml + (pr + p * step) * 2 + 1);
      o += w * ldg<float4_t>(a.part_o + (pr + p * step) * HD + d);
    }
    const int t = (g.r0 + r) / a.G, h = (g.r0 + r) % a.G;
    *reinterpret_cast<float4_t *>(a.out + (size_t)(g.row + t) * a.out_ld +
                                  (size_t)(kvh * a.G + h) * HD + d) = o / l;
  }
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
  const int per = (int)std::max<int64_t>(8, (tiles * p->n_kv + blocks - 1) / blocks);
  int parts = 0;
  for (int s = 0; s < b->n_seqs; ++s)
    for (int r0 = 0; r0 < b->n_new[s] * p->G; r0 += rows_of) {
      int k0, k1;
      spans(s, r0, &k0, &k1);
      const int n = (k1 - k0 + kTile - 1) / kTile, cuts = (n + per - 1) / per;
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
    hipLaunchKernelGGL((k_paged_merge<HD, NQ>), dim3(p.n_merge * a.n_kv), dim3(256), 0, st, a,
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
  a.scale = (L->scale == 0.f ? 1.0f / std::sqrt((float)hd) : L->scale) * 1.44269504088896340736f;
  switch (hd) {
    case 64: launch_dt<64>(a, *p, L->dtype, st); break;
    case 128: launch_dt<128>(a, *p, L->dtype, st); break;
    case 256: launch_dt<256>(a, *p, L->dtype, st); break;
    default: launch_dt<512>(a, *p, L->dtype, st); break;
  }
  MS_HIP_TRY(hipGetLastError());
  return MS_OK;
}
