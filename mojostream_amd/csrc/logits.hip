// Penalties for tokens that occurred, biases and grammar masks on the logits.
#include <cmath>

#include "devutil.h"
#include "paged.h"

namespace ms {
namespace {

constexpr int kLogRows = 64;    // rows of a launch: their settings are kernel arguments
constexpr int kOwners = 1024;   // a power of two

struct LogitsArgs {
  const float *x;
  float *y;
  size_t x_ld, y_ld;
  int vocab, words, in_place;
  const int32_t *hist, *bias_ids;
  const float *bias;
  const uint32_t *masks;
  ms_logits_row rows[kLogRows];
};

// What a block knows of an id: seen, has a bias, times generated.
constexpr uint32_t kSeen = 0x80000000u, kBiased = 0x40000000u, kMade = 0x3FFFFFFFu;

// A block has 4 PER NT ids of one row.  It loads its logits (only those that the mask
// allows), counts the history's ids among them and adds up their biases in LDS meanwhile, and
// goes over them once.  48 rows of 262144 logits, 4000 ids of history and 300 biases each, half
// of them under a mask of 30%: 26 us for 95 MB (3.6 TB/s), bound by memory and by each block's
// chain of loads, of which 1024 threads a block hide the most (512: 27 us, 256: 36 to 57 us); one
// row 4.2 us, mostly its launch.  VEC: four ids side by side a thread, where rows are 16-byte aligned.  In
// place, four logits that nothing changes are neither loaded nor stored.
template <int NT, int PER, bool VEC>
__global__ __launch_bounds__(NT) void k_logits(LogitsArgs a) {
  constexpr int TILE = 4 * PER * NT;
  __shared__ uint32_t cnt[TILE];
  __shared__ float add[TILE];
  __shared__ int owner[kOwners];
  const int tid = threadIdx.x, t0 = blockIdx.x * TILE;
  const ms_logits_row &w = a.rows[blockIdx.y];
  const int nt = min(TILE, a.vocab - t0), nh = w.n_prompt + w.n_generated, nb = w.n_bias;
  const float *x = a.x + blockIdx.y * a.x_ld + t0;
  float *y = a.y + blockIdx.y * a.y_ld + t0;
  auto id = [&](int j, int e) { return VEC ? (j * NT + tid) * 4 + e : (j * 4 + e) * NT + tid; };
  auto load = [&](int j, uint32_t ok) {
    float4_t v = {};
    if (VEC && id(j, 3) < nt) {
      if (ok) v = ldg<float4_t>(x + id(j, 0));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (ok >> e & 1) v[e] = ldg<float>(x + id(j, e));
    }
    return v;
  };

  // ---- the first of the history and of the biases, on their way beside the mask's words
  const int32_t *h = a.hist + w.history;
  int32_t h_id[4] = {}, b_id = 0;
  float b_val = 0.f;
  auto load_h = [&](int i0) {
#pragma unroll
    for (int u = 0; u < 4; ++u) h_id[u] = ldg<int32_t>(h + min(i0 + u * NT, nh - 1));
  };
  auto load_b = [&](int i) {
    b_id = ldg<int32_t>(a.bias_ids + w.bias + min(i, nb - 1));
    b_val = ldg<float>(a.bias + w.bias + min(i, nb - 1));
  };
  if (nh > 0) load_h(tid);
  if (nb > 0) load_b(tid);

  // ---- what the mask allows of this thread's ids (those past the row: nothing), their logits
  uint32_t ok[PER];
  float4_t v[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    ok[j] = 0;
    if (VEC) {
      const int i = id(j, 0);
      if (i < nt) {
        ok[j] = w.mask < 0 ? 15u : ldg<uint32_t>(a.masks + (size_t)w.mask * a.words + ((t0 + i) >> 5)) >> ((t0 + i) & 31) & 15u;
        if (i + 3 >= nt) ok[j] &= (1u << (nt - i)) - 1;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = id(j, e);
        if (i < nt)
          ok[j] |= (w.mask < 0 ? 1u : ldg<uint32_t>(a.masks + (size_t)w.mask * a.words + ((t0 + i) >> 5)) >> ((t0 + i) & 31) & 1u) << e;
      }
    }
  }
  if (!a.in_place)
#pragma unroll
    for (int j = 0; j < PER; ++j) v[j] = load(j, ok[j]);

  // ---- history and biases
  if (nh + nb > 0) {
    for (int i = tid; i < TILE; i += NT) cnt[i] = 0;
    if (nb > 0) {
      for (int i = tid; i < TILE; i += NT) add[i] = 0.f;
      for (int i = tid; i < kOwners; i += NT) owner[i] = NT;
    }
    __syncthreads();
    for (int i0 = tid; i0 < nh; i0 += 4 * NT) {
      if (i0 > tid) load_h(i0);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + u * NT;
        const uint32_t at = (uint32_t)h_id[u] - (uint32_t)t0;
        if (i >= nh || at >= (uint32_t)nt) continue;
        if (i < w.n_prompt)
          atomicOr(&cnt[at], kSeen);
        else
          atomicAdd(&cnt[at], 1u);
      }
    }
    // Entries of one id add up in their order: of the threads that hold one, the lowest goes first.
    // (Threads whose ids share a place among the owners take turns too.)
    for (int i0 = 0; i0 < nb; i0 += NT) {
      if (i0) load_b(i0 + tid);
      const uint32_t at = (uint32_t)b_id - (uint32_t)t0;
      bool wait = i0 + tid < nb && at < (uint32_t)nt;
      while (__syncthreads_or(wait)) {
        if (wait) atomicMin(&owner[at & (kOwners - 1)], tid);
        __syncthreads();
        const bool mine = wait && owner[at & (kOwners - 1)] == tid;
        __syncthreads();
        if (mine) {
          add[at] += b_val;
          atomicOr(&cnt[at], kBiased);
          owner[at & (kOwners - 1)] = NT;
          wait = false;
        }
      }
    }
    __syncthreads();
  }

  // ---- once over the logits
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    uint32_t c[4] = {};
    if (nh + nb > 0)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (ok[j] >> e & 1) c[e] = cnt[id(j, e)];
    if (a.in_place) {
      if (ok[j] == 15 && !(c[0] | c[1] | c[2] | c[3])) continue;
      v[j] = load(j, ok[j]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float z = v[j][e];
      if (c[e]) {
        const uint32_t made = c[e] & kMade;
        if (c[e] & (kSeen | kMade)) z = z > 0.f ? z / w.repetition : z * w.repetition;
        if (made) z = z - w.frequency * (float)made - w.presence;
        if (c[e] & kBiased) z += add[id(j, e)];
      }
      v[j][e] = ok[j] >> e & 1 ? z : -INFINITY;
    }
    if (VEC && id(j, 3) < nt) {
      *reinterpret_cast<float4_t *>(y + id(j, 0)) = v[j];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (id(j, e) < nt) y[id(j, e)] = v[j][e];
    }
  }
}

template <int NT, int PER>
void launch_tiles(const LogitsArgs &a, int rows, bool vec, hipStream_t st) {
  const dim3 grid(cdiv(a.vocab, 4 * PER * NT), rows);
  if (vec)
    hipLaunchKernelGGL((k_logits<NT, PER, true>), grid, dim3(NT), 0, st, a);
  else
    hipLaunchKernelGGL((k_logits<NT, PER, false>), grid, dim3(NT), 0, st, a);
}

}  // namespace
}  // namespace ms

using namespace ms;

extern "C" int ms_logits_process(const float *d_logits, size_t in_stride, float *d_out,
                                 size_t out_stride, int rows, int vocab,
                                 const ms_logits_row *h_rows, const int32_t *d_history,
                                 size_t n_history, const int32_t *d_bias_ids, const float *d_bias,
                                 size_t n_bias, const uint32_t *d_masks, int n_masks) {
  MS_CHECK_ARG(rows >= 0 && vocab >= 1 && vocab <= (1 << 30) && n_masks >= 0,
               "logits_process: bad sizes");
  if (rows == 0) return require_init();
  MS_CHECK_ARG(d_logits && d_out && h_rows, "logits_process: null argument");
  MS_CHECK_ARG(in_stride >= (size_t)vocab && out_stride >= (size_t)vocab &&
                   in_stride < ((size_t)1 << 40) && out_stride < ((size_t)1 << 40),
               "logits_process: row stride less than the vocabulary");
  MS_CHECK_ARG((d_logits == d_out && in_stride == out_stride) ||
                   !rows_overlap(d_logits, in_stride, vocab, d_out, out_stride, vocab, rows),
               "logits_process: d_logits and d_out overlap");
  for (int r = 0; r < rows; ++r) {
    const ms_logits_row &w = h_rows[r];
    auto at = [r](const char *msg) { return "logits_process: row " + std::to_string(r) + ": " + msg; };
    MS_CHECK_ARG(w.repetition > 0.f && w.repetition < INFINITY,
                 at("the repetition penalty must be positive and finite"));
    MS_CHECK_ARG(std::fabs(w.frequency) < INFINITY && std::fabs(w.presence) < INFINITY,
                 at("a penalty is not a finite number"));
    MS_CHECK_ARG(w.n_prompt >= 0 && w.n_generated >= 0 && w.n_bias >= 0, at("negative count"));
    const int64_t h = (int64_t)w.n_prompt + w.n_generated;
    MS_CHECK_ARG(h < (1 << 30) && w.history >= 0 && (uint64_t)w.history <= n_history &&
                     (uint64_t)h <= n_history - (uint64_t)w.history && (h == 0 || d_history),
                 at("the history reaches past d_history"));
    MS_CHECK_ARG(w.n_bias < (1 << 30) && w.bias >= 0 && (uint64_t)w.bias <= n_bias &&
                     (uint64_t)w.n_bias <= n_bias - (uint64_t)w.bias &&
                     (w.n_bias == 0 || (d_bias_ids && d_bias)),
                 at("the biases reach past d_bias"));
    MS_CHECK_ARG(w.mask >= -1 && w.mask < n_masks && (w.mask < 0 || d_masks),
                 at("no such mask"));
  }
  if (int rc = require_init()) return rc;
  OnDevice on;
  LogitsArgs a;
  a.x_ld = in_stride;
  a.y_ld = out_stride;
  a.vocab = vocab;
  a.words = (vocab + 31) / 32;
  a.hist = d_history;
  a.bias_ids = d_bias_ids;
  a.bias = d_bias;
  a.masks = d_masks;
  a.in_place = d_logits == d_out;
  const bool vec = aligned16(d_logits) && aligned16(d_out) && in_stride % 4 == 0 && out_stride % 4 == 0;
  for (int r0 = 0; r0 < rows; r0 += kLogRows) {
    const int n = rows - r0 < kLogRows ? rows - r0 : kLogRows;
    a.x = d_logits + (size_t)r0 * in_stride;
    a.y = d_out + (size_t)r0 * out_stride;
    for (int r = 0; r < kLogRows; ++r) a.rows[r] = h_rows[r0 + (r < n ? r : 0)];
    // Every block reads its row's whole history: blocks of 8192 ids, smaller ones only where those
    // would leave compute units idle.
    if ((long)n * cdiv(vocab, 8192) >= ctx().n_cu)
      launch_tiles<1024, 2>(a, n, vec, ctx().stream);
    else
      launch_tiles<256, 1>(a, n, vec, ctx().stream);
    MS_HIP_TRY(hipGetLastError());
  }
  return MS_OK;
}
