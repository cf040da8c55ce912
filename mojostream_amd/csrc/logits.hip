// Penalties for tokens that occurred, biases and grammar masks on the logits.
#include <cmath>

#include "devutil.h"
#include "paged.h"

namespace ms {
namespace {

constexpr int kLogTile = 4096;  // logits of a block
constexpr int kLogRows = 64;    // rows of a launch: their settings are kernel arguments
constexpr int kLogNT = 256;

struct LogitsArgs {
  const float *x;
  float *y;
  size_t x_ld, y_ld;
  int vocab, words;
  const int32_t *hist, *bias_ids;
  const float *bias;
  const uint32_t *masks;
  ms_logits_row rows[kLogRows];
};

// A block has kLogTile ids of one row: it counts the history's ids among them and adds
// up their biases in LDS, then goes over its logits once.
__global__ __launch_bounds__(kLogNT) void k_logits(LogitsArgs a) {
  __shared__ uint32_t cnt[kLogTile];  // bit 31: seen; below: times generated
  __shared__ float add[kLogTile];
  __shared__ int owner[kLogTile];
  const int tid = threadIdx.x, t0 = blockIdx.x * kLogTile;
  const ms_logits_row &w = a.rows[blockIdx.y];
  const int nt = min(kLogTile, a.vocab - t0);
  for (int i = tid; i < nt; i += kLogNT) {
    cnt[i] = 0;
    add[i] = 0.f;
    owner[i] = kLogNT;
  }
  __syncthreads();
  for (int i = tid; i < w.n_prompt + w.n_generated; i += kLogNT) {
    const uint32_t at = (uint32_t)a.hist[w.history + i] - (uint32_t)t0;
    if (at >= (uint32_t)nt) continue;
    if (i < w.n_prompt)
      atomicOr(&cnt[at], 0x80000000u);
    else
      atomicAdd(&cnt[at], 1u);
  }
  // Entries of one id add up in their order: of the threads that hold one, the lowest
  // goes first.
  for (int i0 = 0; i0 < w.n_bias; i0 += kLogNT) {
    uint32_t at = 0;
    float v = 0.f;
    bool wait = false;
    if (i0 + tid < w.n_bias) {
      at = (uint32_t)a.bias_ids[w.bias + i0 + tid] - (uint32_t)t0;
      wait = at < (uint32_t)nt;
      if (wait) v = a.bias[w.bias + i0 + tid];
    }
    while (__syncthreads_or(wait)) {
      if (wait) atomicMin(&owner[at], tid);
      __syncthreads();
      const bool mine = wait && owner[at] == tid;
      __syncthreads();
      if (mine) {
        add[at] += v;
        owner[at] = kLogNT;
        wait = false;
      }
    }
  }
  __syncthreads();
  const float *x = a.x + blockIdx.y * a.x_ld + t0;
  float *y = a.y + blockIdx.y * a.y_ld + t0;
  for (int i = tid; i < nt; i += kLogNT) {
    const bool ok = w.mask < 0 ||
                    (a.masks[(size_t)w.mask * a.words + ((t0 + i) >> 5)] >> ((t0 + i) & 31) & 1);
    float v = -INFINITY;
    if (ok) {
      v = x[i];
      const uint32_t c = cnt[i], made = c & 0x7FFFFFFFu;
      if (c) v = v > 0.f ? v / w.repetition : v * w.repetition;
      if (made) v = v - w.frequency * (float)made - w.presence;
      v += add[i];
    }
    y[i] = v;
  }
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
    const std::string at = "logits_process: row " + std::to_string(r) + ": ";
    MS_CHECK_ARG(w.repetition > 0.f && w.repetition < INFINITY,
                 at + "the repetition penalty must be positive and finite");
    MS_CHECK_ARG(std::fabs(w.frequency) < INFINITY && std::fabs(w.presence) < INFINITY,
                 at + "a penalty is not a finite number");
    MS_CHECK_ARG(w.n_prompt >= 0 && w.n_generated >= 0 && w.n_bias >= 0, at + "negative count");
    const int64_t h = (int64_t)w.n_prompt + w.n_generated;
    MS_CHECK_ARG(h <= (1 << 30) && w.history >= 0 && (uint64_t)w.history <= n_history &&
                     (uint64_t)h <= n_history - (uint64_t)w.history && (h == 0 || d_history),
                 at + "the history reaches past d_history");
    MS_CHECK_ARG(w.bias >= 0 && (uint64_t)w.bias <= n_bias &&
                     (uint64_t)w.n_bias <= n_bias - (uint64_t)w.bias &&
                     (w.n_bias == 0 || (d_bias_ids && d_bias)),
                 at + "the biases reach past d_bias");
    MS_CHECK_ARG(w.mask >= -1 && w.mask < n_masks && (w.mask < 0 || d_masks),
                 at + "no such mask");
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
  for (int r0 = 0; r0 < rows; r0 += kLogRows) {
    const int n = rows - r0 < kLogRows ? rows - r0 : kLogRows;
    a.x = d_logits + (size_t)r0 * in_stride;
    a.y = d_out + (size_t)r0 * out_stride;
    for (int r = 0; r < kLogRows; ++r) a.rows[r] = h_rows[r0 + (r < n ? r : 0)];
    hipLaunchKernelGGL(k_logits, dim3(cdiv(vocab, kLogTile), n), dim3(kLogNT), 0, ctx().stream, a);
    MS_HIP_TRY(hipGetLastError());
  }
  return MS_OK;
}
