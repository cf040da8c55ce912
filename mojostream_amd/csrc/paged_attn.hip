// Attention of a ragged batch's new rows over a paged KV cache: the split of the work and the entry
// point (the kernels: paged_attn.h).
#include <algorithm>
#include <cmath>
#include <exception>
#include <numeric>

#include "paged_attn.h"

namespace ms {
namespace {

constexpr int kMaxParts = 1024;  // about the most parts of one result

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
  // Whole spans that are taken in two to four turns, the last of which leaves half the blocks or more without
  // any: its spans, the shortest, are cut for them.  4096 rows over 16384 keys, 14B class, 1280 spans by 512
  // blocks, the last 256 cut in two: e4m3 2.59 -> 2.46 ms, bf16 capped 3.38 -> 3.01 ms.  (A fuller last turn cut as
  // well: 4 x 1500 rows over 9000 keys, 1888 spans, 0.99 -> 1.03 to 1.08 ms: the fewer blocks there are the
  // faster is each.)  One chunk behind 8000 keys, 64 spans a turn, e4m3, last turns of 8, 16, 24 and 32 in the second: 0.73,
  // 0.80, 0.90 and 0.93 of the time uncut; in the third 0.83, 0.88, -, 0.95; of 40 and 48 too 0.93 to 0.96, of 56 and 58
  // 1.01; bf16 capped the same or better; behind 1000 keys 0.94 to 1.03 whatever the last turn.
  std::vector<int> cut_in(spans.size(), 1);
  const int places = blocks / p->n_kv, n_spans = (int)spans.size(), last = places > 0 ? n_spans % places : 0;
  if (p->tail && per >= longest && last && 2 * last <= places && n_spans > places && n_spans < 4 * places) {
    std::vector<int> by_cost(n_spans);
    std::iota(by_cost.begin(), by_cost.end(), 0);
    std::stable_sort(by_cost.begin(), by_cost.end(),
                     [&](int x, int y) { return spans[x].tiles * spans[x].cost < spans[y].tiles * spans[y].cost; });
    for (int i = 0; i < last; ++i)  // (16 tiles a part at least: the merge costs about two)
      cut_in[by_cost[i]] = std::max(1, std::min(std::min(4, places / last), spans[by_cost[i]].tiles / 16));
  }
  // (every fourth page: a prefix that sequences share lies at the same places of theirs; 48 sequences of 256 pages 1.5 us)
  p->shared = false;
  if (p->count) {
    b->reader.resize(b->n_pages, 0);
    const int64_t stamp = ++b->n_counted;
    int64_t all = 0, again = 0;
    for (int s = 0; s < b->n_seqs; ++s) {
      if (!b->n_new[s]) continue;
      const int lo = p->window ? std::max(0, b->len[s] - b->n_new[s] - p->window + 1) : 0;
      const int32_t *pg = b->h_pages() + (size_t)s * b->stride;
      for (int i = (lo / b->page_size + 3) / 4 * 4; i <= (b->len[s] - 1) / b->page_size; i += 4) {
        ++all;
        again += b->reader[pg[i]] == stamp;
        b->reader[pg[i]] = stamp;
      }
    }
    p->shared = 3 * again > all;
  }
  std::vector<PagedItem> items;
  std::vector<PagedMerge> merge;
  std::vector<std::pair<int, int>> order;
  int parts = 0, most_parts = 0;
  for (const Span &x : spans) {
    const int cuts = std::max(cuts_of(x, per), cut_in[&x - spans.data()]), s = x.seq;
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

}  // namespace

int plan_for(ms_paged_batch *b, int G, int rows, bool block, int n_kv, int window, int blocks,
             int tile_cost, int merge_cost, bool tail, bool count, PagedPlan **out) {
  PagedPlan *p = nullptr;
  for (PagedPlan *x : b->plans)
    if (x->G == G && x->rows == rows && x->block == block && x->n_kv == n_kv && x->window == window && x->blocks == blocks &&
        x->tile_cost == tile_cost && x->merge_cost == merge_cost && x->tail == tail && x->count == count)
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
    p->tail = tail;
    p->count = count;
    p->n_kv = n_kv;
    p->window = window;
  }
  *out = p;
  return p->valid ? MS_OK : make_plan(b, p, blocks);
}

}  // namespace ms

using namespace ms;

namespace {

int attend(const char *what, const ms_paged_layer *L, const ms_paged_layer_ext *X, ms_paged_batch *b,
           const float *d_q, size_t q_stride, float *d_out, size_t out_stride) {
  auto w = [what](const std::string &msg) { return what + (": " + msg); };
  MS_CHECK_ARG(L, w("null layer or batch"));
  // (log2(e) times it, what the kernels take, is finite too)
  MS_CHECK_ARG(std::fabs(L->scale * 1.4426950408889634) <= 0x1.fffffep+127,
               w("the scale is not finite or too large"));
  const float cap = X ? X->score_cap : 0.f;
  MS_CHECK_ARG(cap == 0.f || (cap >= 0x1p-60f && cap <= 0x1p60f), w("score_cap must be 0 or 2^-60 to 2^60"));
  const double ratio = cap == 0.f || L->scale == 0.f ? 1.0 : std::fabs(L->scale / (double)cap);
  MS_CHECK_ARG(ratio >= 0x1p-126 && ratio <= 0x1.fffffep+127, w("the scale over score_cap must be 2^-126 to 2^127 in size"));
  if (int rc = X ? paged_check_ext(what, X, b) : paged_check(what, L, b)) return rc;
  MS_CHECK_ARG((int64_t)b->rows * L->n_heads < ((int64_t)1 << 30), w("too many rows for one call"));
  const int q_dim = L->n_heads * L->head_dim, hd = L->head_dim, G = L->n_heads / L->n_kv_heads;
  int most = 0;
  for (int s = 0; s < b->n_seqs; ++s) {
    if (!b->n_new[s]) continue;
    const int lo = L->window ? std::max(0, b->len[s] - b->n_new[s] - L->window + 1) : 0;
    MS_CHECK_ARG(lo >= b->held[s],
                 w("sequence " + std::to_string(s) + " attends to a position whose page is -1"));
    most = std::max(most, b->n_new[s] * G);
  }
  if (b->rows == 0) return require_init();
  MS_CHECK_ARG(d_q && d_out && aligned16(d_q) && aligned16(d_out) && q_stride % 4 == 0 &&
                   out_stride % 4 == 0 && q_stride >= (size_t)q_dim &&
                   out_stride >= (size_t)q_dim && q_stride < ((size_t)1 << 31) &&
                   out_stride < ((size_t)1 << 31),
               w("bad q or output rows"));
  MS_CHECK_ARG(!rows_overlap(d_q, q_stride, q_dim, d_out, out_stride, q_dim, b->rows),
               w("d_q and d_out overlap"));
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
  const double by = L->scale == 0.f ? 1.0 / std::sqrt((double)hd) : L->scale;
  const double scale = cap == 0.f ? by * 1.4426950408889634 : by / cap;
  const double part = std::frexp(scale, &e);  // (e <= 128; 2^127 is the largest power that fp32 holds)
  a.q_scale = (float)(e > 127 ? 2 * part : part);
  a.s_scale = (float)std::ldexp(1.0, e > 127 ? e - 1 : e);
  if (cap != 0.f) cap_args(&a, cap);
  if (X) {
    a.k_scale = X->k_scale;
    a.v_scale = X->v_scale;
  }
  try {
    if (L->dtype == MS_KV_E4M3) return launch_attn_e4m3(a, b, hd, most, st);
    if (L->dtype == MS_KV_I8) return launch_attn_i8(a, b, hd, most, st);
    if (cap != 0.f) return launch_attn_capped(a, b, L->dtype, hd, most, st);
    if (L->dtype == MS_KV_F32) return launch_dims<MS_KV_F32, false>(a, b, hd, most, st);
    if (L->dtype == MS_KV_BF16) return launch_dims<MS_KV_BF16, false>(a, b, hd, most, st);
    return launch_dims<MS_KV_F16, false>(a, b, hd, most, st);
  } catch (const std::exception &e) {
    return fail(MS_E_NOMEM, w(e.what()));
  }
}

}  // namespace

extern "C" int ms_paged_attention(const ms_paged_layer *L, ms_paged_batch *b, const float *d_q,
                                  size_t q_stride, float *d_out, size_t out_stride) {
  return attend("paged_attention", L, nullptr, b, d_q, q_stride, d_out, out_stride);
}

extern "C" int ms_paged_attention_ext(const ms_paged_layer_ext *L, ms_paged_batch *b,
                                      const float *d_q, size_t q_stride, float *d_out,
                                      size_t out_stride) {
  return attend("paged_attention_ext", L ? &L->base : nullptr, L, b, d_q, q_stride, d_out, out_stride);
}
