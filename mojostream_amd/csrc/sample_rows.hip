// A token id for each row of logits: temperature, top-k, top-p, min-p, a given random number.
//
// Id i weighs w_i = e^((x_i - max) / T), as a whole number of 2^-S: sums over a row are exact in
// 64 bits and the same in any order.  What top-k, top-p and min-p leave is, in order of falling logits
// (the lower id first among equals), a first part of the row: all logits above a cut and the
// first few that are equal to it.
//
//  k_rows_scan  a block has a slice of a row: its maximum, and a histogram of counts (top-k) or weights
//               (top-p) over buckets of its logits
//  k_rows_pick  finds, from the slices' histograms, the bucket in which the cut lies; the slice once more: the
//               candidates (top-k: all down to the cut's bucket; top-p: those in it) into a list, the weights
//               of what lies above it added up by chunks of 1024 ids
//  k_rows_draw  a block a row: sorts the candidates, finds the cut and draws.  Rows that this does not
//               fit (more candidates than the list holds, a large top-k, infinite logits) it goes over digit by digit.
#include <climits>
#include <cmath>

#include "devutil.h"
#include "paged.h"

namespace ms {
namespace {

constexpr int kRows = 128;      // rows of a launch: their settings are kernel arguments
constexpr int kNT = 1024;
constexpr int kBins = 2048;     // buckets of a slice's histogram; the last takes what lies below
constexpr int kList = 8192;     // candidates of a row
constexpr int kMostK = 2048;    // the largest top-k by the list
constexpr int kPer = 16;        // logits of a thread; a wave's 1024 are a chunk
constexpr int kMostSlices = 64;
constexpr int kSliceBits = 49;  // S of a slice of up to 2^14 logits; S of a row is at most that

struct RowInfo {
  int state, bucket;         // kNone ..; the cut's bucket
  int ref;                   // weights are 2^(x log2(e) / T - ref)
  float top;                 // the largest logit
  unsigned long long want;   // top-p: weight still to be reached within the bucket
};
enum { kNone, kBest, kSum, kSlow };  // nothing to draw; by the list; by sums (and the list); digit by digit

struct SampleRowsArgs {
  const float *x;
  size_t ld;
  int n, bits;  // logits of a row; S
  int slices, slice;
  const float *u;
  int32_t *ids, *kept;
  float *prob;
  // workspace
  unsigned long long *hist;  // [row][slice][kBins], top-k: uint32
  unsigned long long *sum;   // [row][slice]: its whole weight
  float *top;                // [row][slice]
  uint32_t *real;            // [row][slice]: logits that can be drawn
  RowInfo *info;
  uint32_t *n_list;          // [row]
  unsigned long long *list;  // [row][kList]
  unsigned long long *chunk; // [row][slices * slice / 1024]
  uint32_t *chunk_n;
  ms_sample_row rows[kRows];
};

// Logits as unsigned numbers of the same order; -infinity and NaN, which are never drawn, as 0.
__device__ inline uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);  // (-0 and 0 are equal)
  return !(x > -INFINITY) ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ inline float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

// 2^t as a whole number of 2^-bits, bits <= 51: 2^(j/64) from a table, a polynomial of degree 5 over a 64th of an octave
// (its remainder is below 2^-54).
struct Exp2 {
  const double *table;  // LDS, [64]
  __device__ unsigned long long operator()(double t, int bits) const {
    if (!(t > -60.0)) return 0;
    const double n = rint(t * 64.0), r = __builtin_fma(t, 64.0, -n) * 0.010830424696249145;
    double p = __builtin_fma(r, 1.0 / 120, 1.0 / 24);
    p = __builtin_fma(r, p, 1.0 / 6);
    p = __builtin_fma(r, p, 0.5);
    p = __builtin_fma(r, p, 1.0);
    p = __builtin_fma(r, p, 1.0);
    const int e = (int)n;
    const double v = ldexp(p * table[e & 63], (e >> 6) + bits) + 0x1p52;
    return (unsigned long long)__double_as_longlong(v) & 0xFFFFFFFFFFFFFull;
  }
};
// A logit's weight by sums: the same instructions in every kernel, which count on the same number.
__device__ inline unsigned long long weight_of(const Exp2 &exp2, float x, double c, int ref, int bits) {
  return exp2(__builtin_fma((double)x, c, (double)-ref), bits);
}
// log2 of the least share, T and the largest logit in it, that min_p leaves
__device__ inline double least_of(float top, double c, float min_p) {
  return min_p > 0.f ? __builtin_fma((double)top, c, log2((double)min_p)) : -INFINITY;
}
__device__ inline void exp2_table(double *t) {
  if (threadIdx.x < 64) t[threadIdx.x] = exp2(threadIdx.x / 64.0);
}

// How a row is done.
__device__ inline int best_of(const ms_sample_row &s, int n) {  // ids that top-k leaves; 0: all
  return s.temperature == 0.f ? 1 : s.top_k > 0 && s.top_k < n ? s.top_k : 0;
}
__device__ inline bool by_sums(const ms_sample_row &s, int n) { return best_of(s, n) == 0; }
__device__ inline float grain(const ms_sample_row &s) { return 32.f * 1.44269504f / s.temperature; }
constexpr float kMostGrain = 0x1p60f;
// A logit's bucket, in the order of logits.  Top-k: the exponent and eight bits of the mantissa, whatever
// the logits' size; sums: 1/32 of an octave of the weights.
__device__ inline int bucket_of(float x, bool sums, float grain) {
  return sums ? (int)fminf(fmaxf(floorf(x * grain), -0x1p29f), 0x1p29f) : (int)(key_of(x) >> 15);
}

template <bool VEC>
__device__ inline void load_chunk(const float *x, int n, int at, float (&v)[kPer]) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int j = 0; j < kPer / 4; ++j) {
    const int i = at + 256 * j + 4 * lane;
    if (VEC && i + 3 < n) {
      const float4 y = ldg<float4>(x + i);
      v[4 * j] = y.x;
      v[4 * j + 1] = y.y;
      v[4 * j + 2] = y.z;
      v[4 * j + 3] = y.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * j + e] = i + e < n ? ldg<float>(x + i + e) : -INFINITY;
    }
  }
#pragma unroll
  for (int j = 0; j < kPer; ++j) v[j] = v[j] > -INFINITY ? v[j] : -INFINITY;  // (NaN too)
}

template <int NT, bool VEC>
__global__ __launch_bounds__(NT) void k_rows_scan(SampleRowsArgs a) {
  __shared__ __align__(16) unsigned long long hist[kBins];
  __shared__ double table[64];
  __shared__ float tops[NT / 64];
  __shared__ uint32_t reals[NT / 64];
  __shared__ unsigned long long sums[NT / 64];
  uint32_t *count = reinterpret_cast<uint32_t *>(hist);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.y;
  const ms_sample_row &set = a.rows[row];
  const int k = best_of(set, a.n);
  const bool sums_of = k == 0, bins = sums_of ? set.top_p < 1.f && grain(set) < kMostGrain : k <= kMostK;
  float v[kPer];
  load_chunk<VEC>(a.x + row * a.ld, a.n, blockIdx.x * a.slice + wave * 1024, v);
  if (bins) {
    for (int i = tid; i < (sums_of ? kBins : kBins / 2); i += NT) hist[i] = 0;
    exp2_table(table);
  }
  float top = -INFINITY;
  uint32_t real = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    top = fmaxf(top, v[j]);
    real += v[j] > -INFINITY;
  }
  for (int o = 1; o < 64; o <<= 1) {
    top = fmaxf(top, __shfl_xor(top, o, 64));
    real += (uint32_t)__shfl_xor((int)real, o, 64);
  }
  if (lane == 0) {
    tops[wave] = top;
    reals[wave] = real;
  }
  __syncthreads();
  real = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    top = fmaxf(top, tops[w]);
    real += reals[w];
  }
  const size_t at = (size_t)row * a.slices + blockIdx.x;
  if (tid == 0) {
    a.top[at] = top;
    a.real[at] = real;
    if (blockIdx.x == 0) a.n_list[row] = 0;
  }
  if (!bins || real == 0 || top == INFINITY) return;
  const float gr = grain(set);
  const int g_top = bucket_of(top, sums_of, gr);
  if (sums_of) {
    const Exp2 exp2{table};
    const double c = 1.4426950408889634 / (double)set.temperature;
    const int ref = (g_top >> 5) + 1;
    unsigned long long sum = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const unsigned long long w = weight_of(exp2, v[j], c, ref, kSliceBits);
      if (w) atomicAdd(&hist[min(max(g_top - bucket_of(v[j], true, gr), 0), kBins - 1)], w);
      sum += w;
    }
    for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
    if (lane == 0) sums[wave] = sum;
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int d = g_top - bucket_of(v[j], false, gr);
      if (d < kBins - 1) atomicAdd(&count[d], 1u);
    }
  }
  __syncthreads();
  if (sums_of) {
    for (int i = tid; i < kBins; i += NT) a.hist[at * kBins + i] = hist[i];
    if (tid == 0) {
      unsigned long long sum = 0;
      for (int w = 0; w < NT / 64; ++w) sum += sums[w];
      a.sum[at] = sum;
    }
  } else {
    for (int i = tid; i < kBins / 2; i += NT) a.hist[at * kBins + i] = hist[i];
  }
}

template <int NT, bool VEC>
__global__ __launch_bounds__(NT) void k_rows_pick(SampleRowsArgs a) {
  constexpr int GR = NT / 256;
  __shared__ double table[64];
  __shared__ int g_of[kMostSlices];
  __shared__ unsigned long long part[GR][256];
  __shared__ unsigned long long wsum[4], found_before;
  __shared__ int found;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.y;
  const ms_sample_row &set = a.rows[row];
  const int k = best_of(set, a.n);
  const bool sums = k == 0, cut = sums && set.top_p < 1.f;
  const int id0 = blockIdx.x * a.slice + wave * 1024;
  float v[kPer];
  load_chunk<VEC>(a.x + row * a.ld, a.n, id0, v);

  // ---- the row's maximum
  const size_t at = (size_t)row * a.slices;
  const float gr = grain(set);
  float top = lane < a.slices ? ldg<float>(a.top + at + lane) : -INFINITY;
  const float mine = top;
  uint32_t real = lane < a.slices ? ldg<uint32_t>(a.real + at + lane) : 0;
  for (int o = 1; o < 64; o <<= 1) {
    top = fmaxf(top, __shfl_xor(top, o, 64));
    real += (uint32_t)__shfl_xor((int)real, o, 64);
  }
  exp2_table(table);
  // (a weight's bucket is a whole number that fp32 holds to a quarter)
  int state = real == 0 ? kNone : top == INFINITY || k > kMostK ? kSlow : !sums ? kBest : kSum;
  if (state == kSum && !(fabsf(top) * gr < 0x1p22f && gr < kMostGrain)) state = kSlow;
  int bucket = INT_MIN, ref = 0;
  unsigned long long want = 0;
  const int g_top = state == kBest || state == kSum ? bucket_of(top, sums, gr) : 0;
  if (state == kSum) ref = (g_top >> 5) + 1;
  const double c = set.temperature == 0.f ? 0.0 : 1.4426950408889634 / (double)set.temperature;

  // ---- the bucket of the cut
  if (state == kBest || (state == kSum && cut)) {
    if (wave == 0) g_of[lane] = mine > -INFINITY ? bucket_of(mine, sums, gr) : INT_MIN;
    if (tid == 0) found = -1;
    __syncthreads();
    // a slice's weights in the row's unit, rounded
    auto in_unit = [&](unsigned long long w, int g) {
      const int sh = kSliceBits - a.bits + ref - ((g >> 5) + 1);
      return sh == 0 ? w : sh > 63 ? 0ull : ((w >> (sh - 1)) + 1) >> 1;
    };
    unsigned long long goal = (unsigned long long)k;
    if (sums) {
      unsigned long long all = 0;
      if (lane < a.slices && g_of[lane] != INT_MIN) all = in_unit(ldg<unsigned long long>(a.sum + at + lane), g_of[lane]);
      for (int o = 1; o < 64; o <<= 1) all += __shfl_xor(all, o, 64);
      goal = (unsigned long long)ceil((double)set.top_p * (double)all);
      if (goal == 0) goal = 1;
    }
    unsigned long long before = 0;
    for (int b0 = 0; b0 < kBins - 1; b0 += 256) {
      const int j = b0 + (tid & 255);
      unsigned long long s = 0;
      if (j < kBins - 1)
        for (int q = tid >> 8; q < a.slices; q += GR) {
          const int g = g_of[q], i = j - (g_top - g);
          if (g == INT_MIN || i < 0) continue;
          const unsigned long long *h = a.hist + (at + q) * kBins;
          s += sums ? in_unit(ldg<unsigned long long>(h + i), g) : ldg<uint32_t>(reinterpret_cast<const uint32_t *>(h) + i);
        }
      if (GR > 1) {
        part[tid >> 8][tid & 255] = s;
        __syncthreads();
        if (tid < 256) {
          s = 0;
#pragma unroll
          for (int q = 0; q < GR; ++q) s += part[q][tid];
        }
      }
      unsigned long long upto = s;
      for (int o = 1; o < 64; o <<= 1) {
        const unsigned long long y = __shfl_up(upto, o, 64);
        if (lane >= o) upto += y;
      }
      if (wave < 4 && lane == 63) wsum[wave] = upto;
      __syncthreads();
      if (tid < 256) {
        upto += before;
        for (int w = 0; w < wave; ++w) upto += wsum[w];
        if (upto >= goal && upto - s < goal) {
          found = j;
          found_before = upto - s;
        }
      }
      before += wsum[0] + wsum[1] + wsum[2] + wsum[3];
      __syncthreads();
      if (found >= 0) break;
    }
    if (found >= 0) {
      bucket = g_top - found;
      want = goal - found_before;
    } else if (sums || real > kList) {
      state = kSlow;
    }  // (else all that can be drawn is in the list)
  }
  if (blockIdx.x == 0 && tid == 0) a.info[row] = RowInfo{state, bucket, ref, top, want};
  if (state == kNone || state == kSlow) return;
  __syncthreads();  // (the table)

  // ---- the slice once more
  const Exp2 exp2{table};
  const double least = least_of(top, c, set.min_p);
  unsigned long long sum = 0;
  uint32_t num = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int g = bucket_of(v[j], sums, gr);
    const bool on = v[j] > -INFINITY && g >= bucket && (!sums || v[j] == top || (double)v[j] * c >= least);
    const bool listed = on && (!sums || (cut && g == bucket));
    const unsigned long long m = __ballot(listed);
    if (m) {
      uint32_t base = 0;
      if (lane == 0) base = atomicAdd(a.n_list + row, (uint32_t)__popcll(m));
      base = (uint32_t)__shfl((int)base, 0, 64) + __popcll(m & ((1ull << lane) - 1));
      if (listed && base < kList)
        a.list[(size_t)row * kList + base] = (unsigned long long)key_of(v[j]) << 32 |
                                             (0xFFFFFFFFu - (uint32_t)(id0 + 256 * (j / 4) + 4 * lane + j % 4));
    }
    if (sums && on && !listed) {
      sum += weight_of(exp2, v[j], c, ref, a.bits);
      ++num;
    }
  }
  if (sums) {
    for (int o = 1; o < 64; o <<= 1) {
      sum += __shfl_xor(sum, o, 64);
      num += (uint32_t)__shfl_xor((int)num, o, 64);
    }
    if (lane == 0) {
      const size_t ch = (size_t)row * a.slices * (a.slice / 1024) + id0 / 1024;
      a.chunk[ch] = sum;
      a.chunk_n[ch] = num;
    }
  }
}

__device__ inline uint64_t add_over_wave(uint64_t v) {
  for (int o = 1; o < 64; o <<= 1) v += __shfl_xor((unsigned long long)v, o, 64);
  return v;
}

struct DigitLds {
  uint32_t cnt[256];
  unsigned long long wt[256];
  unsigned long long part[16];
  uint32_t red[16];
  uint32_t s_key, s_count;
  unsigned long long s_above;
  int s_id;
};

// The whole of a row, by one block.  The cut is found digit by digit of the logits' keys: a histogram
// of the counts (top-k) or weights (top-p) of the logits that agree with the digits found so far.
__device__ void row_by_digits(const SampleRowsArgs &a, DigitLds &lds) {
  uint32_t *cnt = lds.cnt, *red = lds.red, &s_key = lds.s_key, &s_count = lds.s_count;
  unsigned long long *wt = lds.wt, *part = lds.part, &s_above = lds.s_above;
  int &s_id = lds.s_id;
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

// Falling order of n numbers, n a power of two.
__device__ inline void sort_falling(unsigned long long *x, int n) {
  for (int size = 2; size <= n; size <<= 1)
    for (int step = size / 2; step > 0; step >>= 1) {
      __syncthreads();
      for (int t = threadIdx.x; t < n / 2; t += kNT) {
        const int i = 2 * t - (t & (step - 1)), j = i + step;
        const unsigned long long p = x[i], q = x[j];
        if ((p < q) == ((i & size) == 0)) {
          x[i] = q;
          x[j] = p;
        }
      }
    }
  __syncthreads();
}
__device__ inline int power_of_two(int n) {
  int p = 64;
  while (p < n) p <<= 1;
  return p;
}

// Running sum over the block's threads, this one's value among it; *all: the whole.
__device__ inline unsigned long long run_sum(unsigned long long v, unsigned long long *part, unsigned long long *all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned long long y = __shfl_up(v, o, 64);
    if (lane >= o) v += y;
  }
  __syncthreads();
  if (lane == 63) part[wave] = v;
  __syncthreads();
  unsigned long long sum = 0;
#pragma unroll
  for (int w = 0; w < kNT / 64; ++w) {
    if (w == wave) v += sum;
    sum += part[w];
  }
  *all = sum;
  return v;
}

__device__ inline unsigned long long target_of(float u, unsigned long long total) {
  const unsigned long long t = !(u > 0.f) ? 0 : u >= 1.f ? total - 1 : (unsigned long long)((double)u * (double)total);
  return t < total ? t : total - 1;
}

__global__ __launch_bounds__(kNT) void k_rows_draw(SampleRowsArgs a) {
  __shared__ __align__(16) unsigned long long list[kList];
  __shared__ unsigned long long chunk[kMostSlices * 16];
  __shared__ double table[64];
  __shared__ unsigned long long part[16];
  __shared__ DigitLds digits;
  __shared__ int hit;
  __shared__ unsigned long long hit_before;
  const int tid = threadIdx.x, row = blockIdx.x;
  const ms_sample_row &set = a.rows[row];
  const RowInfo in = a.info[row];
  const uint32_t n_list = a.n_list[row];
  auto write = [&](int id, float prob, uint32_t kept) {
    a.ids[row] = id;
    if (a.prob) a.prob[row] = prob;
    if (a.kept) a.kept[row] = (int)kept;
  };
  if (in.state == kNone) {
    if (tid == 0) write(-1, 0.f, 0);
    return;
  }
  if (in.state == kSlow || n_list > kList) {
    row_by_digits(a, digits);
    return;
  }
  exp2_table(table);
  const Exp2 exp2{table};
  const float *x = a.x + row * a.ld;
  const double c = set.temperature == 0.f ? 0.0 : 1.4426950408889634 / (double)set.temperature;
  const int size = n_list ? power_of_two((int)n_list) : 0;
  for (int i = tid; i < size; i += kNT) list[i] = i < (int)n_list ? a.list[(size_t)row * kList + i] : 0;
  sort_falling(list, size);
  const float u = ldg<float>(a.u + row);
  auto id_of = [](unsigned long long e) { return 0xFFFFFFFFu - (uint32_t)e; };
  auto logit_of = [](unsigned long long e) { return of_key((uint32_t)(e >> 32)); };

  if (in.state == kBest) {
    // ---- everything that may be left is in the list: two of its first kMostK a thread
    const int best = best_of(set, a.n), nk = min(best, (int)n_list);
    unsigned long long w[2] = {};
    const double least = set.min_p > 0.f ? log2((double)set.min_p) : -INFINITY;
    uint32_t over = 0;  // of the two, how many min_p leaves
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = 2 * tid + e;
      if (i >= nk) continue;
      const float v = logit_of(list[i]);
      const double t = v == in.top ? 0.0 : ((double)v - (double)in.top) * c;
      w[e] = exp2(t, a.bits);
      over += v == in.top || t >= least;
    }
    unsigned long long total, left, most;
    unsigned long long upto = run_sum(w[0] + w[1], part, &total);
    unsigned long long goal = ~0ull;
    if (set.temperature != 0.f && set.top_p < 1.f) {
      goal = (unsigned long long)ceil((double)set.top_p * (double)total);
      if (goal == 0) goal = 1;
    }
    const uint32_t under = (2 * tid < nk && upto - w[0] - w[1] < goal) + (2 * tid + 1 < nk && upto - w[1] < goal);
    run_sum(under, part, &left);
    run_sum(over, part, &most);
    const int n = (int)(left < most ? left : most);
    // in order of ids: (id, place) sorted, the weights by their places
    __syncthreads();
    unsigned long long *by_place = list + 4096;
    uint32_t id[2] = {};
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (2 * tid + e < n) id[e] = id_of(list[2 * tid + e]);
    __syncthreads();
    const int size2 = power_of_two(n);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = 2 * tid + e;
      if (i < size2) list[i] = i < n ? (unsigned long long)(0xFFFFFFFFu - id[e]) << 32 | (uint32_t)i : 0;
      if (i < n) by_place[i] = w[e];
    }
    sort_falling(list, size2);
#pragma unroll
    for (int e = 0; e < 2; ++e) w[e] = 2 * tid + e < n ? by_place[(uint32_t)list[2 * tid + e]] : 0;
    upto = run_sum(w[0] + w[1], part, &total);
    const unsigned long long target = target_of(u, total);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const unsigned long long to = e ? upto : upto - w[1];
      if (to > target && to - w[e] <= target)
        write((int)(0xFFFFFFFFu - (uint32_t)(list[2 * tid + e] >> 32)), (float)((double)w[e] / (double)total), n);
    }
    return;
  }

  // ---- sums of the chunks; of the candidates as many as it takes
  const int n_chunks = a.slices * (a.slice / 1024);
  unsigned long long kept = 0, total;
  if (tid < n_chunks) {
    chunk[tid] = a.chunk[(size_t)row * n_chunks + tid];
    kept = a.chunk_n[(size_t)row * n_chunks + tid];
  }
  __syncthreads();
  unsigned long long before = 0;
  int taken = 0;
  for (int i0 = 0; i0 < (int)n_list; i0 += kNT) {
    const int i = i0 + tid;
    unsigned long long w = 0, all;
    if (i < (int)n_list) w = weight_of(exp2, logit_of(list[i]), c, in.ref, a.bits);
    const unsigned long long upto = run_sum(w, part, &all);
    const bool take = i < (int)n_list && before + upto - w < in.want;
    if (take) atomicAdd(&chunk[id_of(list[i]) >> 10], w);
    unsigned long long num;
    run_sum(take, part, &num);
    taken += (int)num;
    before += all;
    if (before >= in.want) break;
  }
  const unsigned long long cut = taken ? list[taken - 1] : ~0ull;
  __syncthreads();
  {
    unsigned long long num;
    run_sum(kept, part, &num);
    kept = num + taken;
  }
  const unsigned long long w = tid < n_chunks ? chunk[tid] : 0, upto = run_sum(w, part, &total);
  const unsigned long long target = target_of(u, total);
  if (upto > target && upto - w <= target) {
    hit = tid;
    hit_before = upto - w;
  }
  __syncthreads();
  {
    const int id = hit * 1024 + tid;
    const float v = id < a.n ? ldg<float>(x + id) : -INFINITY;
    unsigned long long w = 0, all;
    if (v > -INFINITY) {
      const int g = bucket_of(v, true, grain(set));
      const bool in_cut = g > in.bucket || ((unsigned long long)key_of(v) << 32 | (0xFFFFFFFFu - (uint32_t)id)) >= cut;
      if ((in.bucket == INT_MIN || in_cut) && (v == in.top || (double)v * c >= least_of(in.top, c, set.min_p)))
        w = weight_of(exp2, v, c, in.ref, a.bits);
    }
    const unsigned long long upto = hit_before + run_sum(w, part, &all);
    if (upto > target && upto - w <= target) write(id, (float)((double)w / (double)total), (uint32_t)kept);
  }
}

template <int NT>
void launch_slices(const SampleRowsArgs &a, int rows, bool vec, hipStream_t st) {
  const dim3 grid(a.slices, rows), blk(NT);
  if (vec) {
    hipLaunchKernelGGL((k_rows_scan<NT, true>), grid, blk, 0, st, a);
    hipLaunchKernelGGL((k_rows_pick<NT, true>), grid, blk, 0, st, a);
  } else {
    hipLaunchKernelGGL((k_rows_scan<NT, false>), grid, blk, 0, st, a);
    hipLaunchKernelGGL((k_rows_pick<NT, false>), grid, blk, 0, st, a);
  }
}

// Rows of more ids than the slices hold.
__global__ __launch_bounds__(kNT) void k_rows_digits(SampleRowsArgs a) {
  __shared__ DigitLds digits;
  row_by_digits(a, digits);
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
  hipStream_t st = ctx().stream;
  SampleRowsArgs a{};
  a.ld = in_stride;
  a.n = vocab;
  a.bits = kSliceBits;
  while (a.bits < 63 && (1 << (63 - a.bits)) < vocab) --a.bits;
  // Slices of 16384 logits where these are as many as compute units, else of 4096.
  const int m0 = rows < kRows ? rows : kRows;
  const bool large = vocab > kMostSlices * 4096 || (long)m0 * cdiv(vocab, 16384) >= ctx().n_cu;
  a.slice = large ? 16384 : 4096;
  a.slices = cdiv(vocab, a.slice);
  const bool sliced = a.slices <= kMostSlices, vec = aligned16(d_logits) && in_stride % 4 == 0;
  if (sliced) {
    const size_t cells = (size_t)m0 * a.slices, chunks = cells * (a.slice / 1024);
    void *buf = nullptr;
    if (int rc = scratch(cells * (kBins * 8 + 16) + chunks * 12 + m0 * (kList * 8 + sizeof(RowInfo) + 4) + 64, &buf)) return rc;
    a.hist = static_cast<unsigned long long *>(buf);
    a.sum = a.hist + cells * kBins;
    a.list = a.sum + cells;
    a.chunk = a.list + (size_t)m0 * kList;
    a.info = reinterpret_cast<RowInfo *>(a.chunk + chunks);
    a.top = reinterpret_cast<float *>(a.info + m0);
    a.real = reinterpret_cast<uint32_t *>(a.top + cells);
    a.n_list = a.real + cells;
    a.chunk_n = a.n_list + m0;
  }
  for (int r0 = 0; r0 < rows; r0 += kRows) {
    const int m = rows - r0 < kRows ? rows - r0 : kRows;
    a.x = d_logits + (size_t)r0 * in_stride;
    a.u = d_u + r0;
    a.ids = d_ids + r0;
    a.prob = d_prob ? d_prob + r0 : nullptr;
    a.kept = d_kept ? d_kept + r0 : nullptr;
    for (int r = 0; r < kRows; ++r) a.rows[r] = h_rows[r0 + (r < m ? r : 0)];
    if (!sliced) {
      hipLaunchKernelGGL(k_rows_digits, dim3(m), dim3(kNT), 0, st, a);
    } else {
      if (large)
        launch_slices<1024>(a, m, vec, st);
      else
        launch_slices<256>(a, m, vec, st);
      hipLaunchKernelGGL(k_rows_draw, dim3(m), dim3(kNT), 0, st, a);
    }
    MS_HIP_TRY(hipGetLastError());
  }
  return MS_OK;
}
