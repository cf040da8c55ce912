// A token id for each row of logits: temperature, top-k, top-p, min-p, a given random number.
//
// Id i weighs w_i = e^((x_i - max) / T), as a whole number of 2^-S, S = 63 - ceil(log2 n): sums over
// a row are exact in 64 bits and the same in any order.  What top-k, top-p and min-p leave is, in order of
// falling logits (the lower id first among equals), a first part of the row: all logits above a cut and the
// first few that are equal to it.
#include <cmath>

#include "devutil.h"
#include "paged.h"

namespace ms {
namespace {

constexpr int kRows = 128;  // rows of a launch: their settings are kernel arguments
constexpr int kNT = 1024;

struct SampleRowsArgs {
  const float *x;
  size_t ld;
  int n, bits;  // logits of a row; S
  const float *u;
  int32_t *ids, *kept;
  float *prob;
  ms_sample_row rows[kRows];
};

// Logits as unsigned numbers of the same order; -infinity and NaN, which are never drawn, as 0.
__device__ inline uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);  // (-0 and 0 are equal)
  return !(x > -INFINITY) ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ inline float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

__device__ inline uint64_t add_over_wave(uint64_t v) {
  for (int o = 1; o < 64; o <<= 1) v += __shfl_xor((unsigned long long)v, o, 64);
  return v;
}

// The whole of a row, by one block.  The cut is found digit by digit of the logits' keys: a histogram
// of the counts (top-k) or weights (top-p) of the logits that agree with the digits found so far.
__global__ __launch_bounds__(kNT) void k_sample_row(SampleRowsArgs a) {
  __shared__ uint32_t cnt[256];
  __shared__ unsigned long long wt[256];
  __shared__ unsigned long long part[16];
  __shared__ uint32_t red[16];
  __shared__ uint32_t s_key, s_count;
  __shared__ unsigned long long s_above;
  __shared__ int s_id;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = a.n;
  const ms_sample_row set = a.rows[blockIdx.x];
  const float *x = a.x + blockIdx.x * a.ld;

  // ---- maximum, and how many can be drawn
  uint32_t top = 0, real = 0;
  for (int i = tid; i < n; i += kNT) {
    const uint32_t k = key_of(ldg<float>(x + i));
    top = max(top, k);
    real += k != 0;
  }
  for (int o = 1; o < 64; o <<= 1) {
    top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
    real += __shfl_xor((int)real, o, 64);
  }
  if (lane == 0) {
    red[wave] = top;
    cnt[wave] = real;
  }
  __syncthreads();
  real = 0;
  for (int w = 0; w < kNT / 64; ++w) {
    top = max(top, red[w]);
    real += cnt[w];
  }
  if (real == 0) {
    if (tid == 0) {
      a.ids[blockIdx.x] = -1;
      if (a.prob) a.prob[blockIdx.x] = 0.f;
      if (a.kept) a.kept[blockIdx.x] = 0;
    }
    return;
  }
  const double vmax = of_key(top), temp = set.temperature;
  auto share = [&](float v) { return v == (float)vmax ? 1.0 : exp(((double)v - vmax) / temp); };
  auto weight = [&](float v) { return (unsigned long long)rint(ldexp(share(v), a.bits)); };

  // The cut where the count (or weight) from the top reaches `want`, of what lies at or above `floor` (of
  // those equal to it, floor_count): key, how many of the logits equal to it, what lies above it.
  uint32_t cut_key, cut_count;
  unsigned long long above;
  auto find = [&](bool by_weight, unsigned long long want, uint32_t floor, uint32_t floor_count) {
    uint32_t prefix = 0;
    above = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      if (tid < 256) {
        cnt[tid] = 0;
        wt[tid] = 0;
      }
      __syncthreads();
      for (int i = tid; i < n; i += kNT) {
        const float v = ldg<float>(x + i);
        const uint32_t k = key_of(v);
        if (k < floor || k == 0 || (shift < 24 && (k >> (shift + 8)) != prefix)) continue;
        atomicAdd(&cnt[k >> shift & 255], 1u);
        if (by_weight && k > floor) atomicAdd(&wt[k >> shift & 255], weight(v));
      }
      __syncthreads();
      if (tid == 0) {
        unsigned long long sum = above;
        const unsigned long long at_floor = by_weight ? floor_count * weight(of_key(floor)) : 0;
        int d = 255;
        for (; d > 0; --d) {
          unsigned long long w = cnt[d];
          if (by_weight) {
            w = wt[d];
            if ((prefix << 8 | d) == floor >> shift) w += at_floor;
          }
          if (sum + w >= want) break;
          sum += w;
        }
        s_key = prefix << 8 | d;
        s_above = sum;
        s_count = cnt[d];
      }
      __syncthreads();
      prefix = s_key;
      above = s_above;
    }
    cut_key = prefix;
    cut_count = s_count;
  };

  uint32_t key = 1;  // (below every number's)
  uint32_t eq = 0, eq_all = 0;  // of the logits equal to the cut, the first eq are left
  const unsigned long long all_k = set.temperature == 0.f ? 1 : set.top_k > 0 ? set.top_k : real;
  if (all_k < real) {
    find(false, all_k, 1, 0);
    key = cut_key;
    eq = (uint32_t)(all_k - above);
    eq_all = cut_count;
  }
  uint32_t last_eq = 0xFFFFFFFFu;  // the last id of those equal to the cut
  auto block_sum = [&](unsigned long long v) {
    v = add_over_wave(v);
    __syncthreads();
    if (lane == 0) part[wave] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < kNT / 64; ++w) v += part[w];
    return v;
  };
  if (set.temperature != 0.f && set.top_p < 1.f) {
    unsigned long long sum = 0;
    for (int i = tid; i < n; i += kNT) {
      const float v = ldg<float>(x + i);
      if (key_of(v) > key) sum += weight(v);
    }
    sum = block_sum(sum);
    const unsigned long long w_eq = key > 1 ? weight(of_key(key)) : 0;
    sum += eq * w_eq;
    unsigned long long want = (unsigned long long)ceil((double)set.top_p * (double)sum);
    if (want == 0) want = 1;
    find(true, want, key, key > 1 ? eq : 0);
    const uint32_t have = cut_key == key && key > 1 ? eq : cut_count;
    const unsigned long long w = weight(of_key(cut_key));
    const unsigned long long take = w ? (want - above + w - 1) / w : 1;
    key = cut_key;
    eq = (uint32_t)(take < have ? take : have);
    eq_all = cut_count;
  }
  if (eq < eq_all) {
    // ---- the eq-th id that is equal to the cut
    uint32_t seen = 0;
    for (int i0 = 0; i0 < n; i0 += kNT) {
      const int i = i0 + tid;
      const bool is = i < n && key_of(ldg<float>(x + i)) == key;
      const unsigned long long m = __ballot(is);
      __syncthreads();
      if (lane == 0) red[wave] = __popcll(m);
      __syncthreads();
      uint32_t before = seen;
      for (int w = 0; w < kNT / 64; ++w) {
        if (w < wave) before += red[w];
        seen += red[w];
      }
      if (is && before + __popcll(m & ((1ull << lane) - 1)) == eq - 1) s_id = i;
      if (seen >= eq) break;
    }
    __syncthreads();
    last_eq = (uint32_t)s_id;
  }
  auto left = [&](float v, int i) {
    const uint32_t k = key_of(v);
    if (k < key || k == 0 || (k == key && (uint32_t)i > last_eq)) return false;
    return k == top || share(v) >= (double)set.min_p;
  };
  // ---- the draw: the wave, then the sixteenth of its part, and so on, in which the running weight passes the target
  unsigned long long total = 0, target = 0, before = 0, count = 0;
  int lo = 0, len = n;
  for (bool first = true; len > 64 || first; first = false) {
    const int per = ((len + 15) / 16 + 63) / 64 * 64, b0 = lo + min(len, wave * per), b1 = lo + min(len, wave * per + per);
    unsigned long long sum = 0, num = 0;
    for (int i = b0 + lane; i < b1; i += 64) {
      const float v = ldg<float>(x + i);
      if (left(v, i)) {
        sum += weight(v);
        ++num;
      }
    }
    sum = add_over_wave(sum);
    if (first) num = block_sum(num);
    __syncthreads();
    if (lane == 0) part[wave] = sum;
    __syncthreads();
    if (first) {
      count = num;
      for (int w = 0; w < 16; ++w) total += part[w];
      const float u = ldg<float>(a.u + blockIdx.x);
      target = !(u > 0.f) ? 0 : u >= 1.f ? total - 1 : (unsigned long long)((double)u * (double)total);
      if (target >= total) target = total - 1;
    }
    int w = 0;
    while (w < 15 && before + part[w] <= target) before += part[w++];
    lo += min(len, w * per);
    len = min(len - min(len, w * per), per);
  }
  if (wave == 0) {
    const int i = lo + lane;
    unsigned long long w = 0;
    if (lane < len) {
      const float v = ldg<float>(x + i);
      if (left(v, i)) w = weight(v);
    }
    unsigned long long upto = w;
    for (int o = 1; o < 64; o <<= 1) {
      const unsigned long long y = __shfl_up(upto, o, 64);
      if (lane >= o) upto += y;
    }
    const unsigned long long hit = __ballot(before + upto > target);
    const int l = __ffsll((unsigned long long)hit) - 1;
    if (lane == l) {
      a.ids[blockIdx.x] = i;
      if (a.prob) a.prob[blockIdx.x] = (float)((double)w / (double)total);
      if (a.kept) a.kept[blockIdx.x] = (int)count;
    }
  }
}

}  // namespace
}  // namespace ms

using namespace ms;

extern "C" int ms_sample_rows(const float *d_logits, size_t in_stride, int rows, int vocab,
                              const ms_sample_row *h_rows, const float *d_u, int32_t *d_ids,
                              float *d_prob, int32_t *d_kept) {
  MS_CHECK_ARG(rows >= 0 && vocab >= 1 && vocab <= (1 << 30), "sample_rows: bad sizes");
  if (rows == 0) return require_init();
  MS_CHECK_ARG(d_logits && h_rows && d_u && d_ids, "sample_rows: null argument");
  MS_CHECK_ARG(in_stride >= (size_t)vocab && in_stride < ((size_t)1 << 40),
               "sample_rows: row stride less than the vocabulary");
  for (int r = 0; r < rows; ++r) {
    const ms_sample_row &w = h_rows[r];
    auto at = [r](const char *msg) { return "sample_rows: row " + std::to_string(r) + ": " + msg; };
    MS_CHECK_ARG(w.temperature >= 0.f && w.temperature < INFINITY,
                 at("the temperature must be finite and not negative"));
    MS_CHECK_ARG(w.top_k >= 0, at("negative top_k"));
    MS_CHECK_ARG(w.top_p >= 0.f && w.top_p <= 1.f, at("top_p must be 0 to 1"));
    MS_CHECK_ARG(w.min_p >= 0.f && w.min_p <= 1.f, at("min_p must be 0 to 1"));
  }
  if (int rc = require_init()) return rc;
  OnDevice on;
  SampleRowsArgs a;
  a.ld = in_stride;
  a.n = vocab;
  a.bits = 63;
  while ((1 << (63 - a.bits)) < vocab) --a.bits;
  for (int r0 = 0; r0 < rows; r0 += kRows) {
    const int m = rows - r0 < kRows ? rows - r0 : kRows;
    a.x = d_logits + (size_t)r0 * in_stride;
    a.u = d_u + r0;
    a.ids = d_ids + r0;
    a.prob = d_prob ? d_prob + r0 : nullptr;
    a.kept = d_kept ? d_kept + r0 : nullptr;
    for (int r = 0; r < kRows; ++r) a.rows[r] = h_rows[r0 + (r < m ? r : 0)];
    hipLaunchKernelGGL(k_sample_row, dim3(m), dim3(kNT), 0, ctx().stream, a);
    MS_HIP_TRY(hipGetLastError());
  }
  return MS_OK;
}
