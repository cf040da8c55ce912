// A token id for each row of logits: temperature, top-k, top-p, min-p, a given random number.
//
// Id i weighs w_i = e^((x_i - max) / T), as a whole number of 2^-S: sums over a row are exact in
// 64 bits and the same in any order.  What top-k, top-p and min-p leave is, in order of falling logits
// (the lower id first among equals), a first part of the row: all logits above a cut and the
// first few that are equal to it.
//
// Where top-p cuts a whole row the same weights are whole numbers of 2^-S of their own octave: a slice's sums, which know
// nothing of the rest of the row, then are exact too, an octave's sum over all slices fits 64 bits and the row's, of
// 64 octaves, 128.  (As whole numbers of a slice's part, rounded to the row's, they were off by one or two: of two equal
// logits top-p 0.5 left both.)
//
//  k_rows_scan  a block has a slice of a row: its maximum, and a histogram of counts (top-k) or weights
//               (top-p) over buckets of its logits
//  k_rows_pick  finds, from the slices' histograms, the bucket in which the cut lies; the slice once more: the
//               candidates (top-k: all down to the cut's bucket; top-p: those in it) into a list, the weights
//               of what lies above it added up by chunks of a wave's 256 or 1024 ids
//  k_rows_draw  a block a row: sorts the candidates, finds the cut and draws.  Rows that this does not
//               fit (more candidates than the list holds, a large top-k, infinite logits) it goes over as a whole.
//
// Three launches, each with a chain of loads behind the last one's results: 4.8 + 7.6 + 7.2 us for a row of 262144 ids; 48 such
// rows, 50 MB, 17 + 17 + 12 us (the first without its weights and sums 17 as well; in slices of 28672 ids, whose
// blocks are all there at once, 20 + 16 + 14).
#include <climits>
#include <cmath>

#include "devutil.h"
#include "paged.h"

namespace ms {
namespace {

typedef unsigned __int128 u128;

constexpr float MAX32 = 0x1.fffffep+127f;
constexpr int kRows = 64;       // rows of a launch: their settings are kernel arguments
constexpr int kNT = 1024;
constexpr int kBins = 2048;     // buckets of a slice's histogram, in 64 groups of 32
constexpr int kList = 8192;     // candidates of a row
constexpr int kSliceList = 2048;  // of one of its slices
constexpr int kMostK = 2048;    // the largest top-k by the list
constexpr int kMostSlices = 64;
constexpr int kWave = 256;      // candidates that one wave goes through alone
constexpr int kMostBits = 49;   // S of up to 2^14 logits

struct RowInfo {
  int state;                // kNone ..
  int ref;                  // weights are 2^(x log2(e) / T - ref)
  float top;                // the largest logit
  float lo, hi;             // the cut lies among the logits lo <= x < hi (the candidates); what lies above stays
  unsigned long long want;  // top-p: weight (of its octave) that the bucket has to reach; top-k: ids of the cut's bucket
  int bucket;               // top-p: the one in which the cut lies, whatever min_p leaves of it
};
// A row's settings.
struct RowSet {
  double c64, by;   // 64 log2(e) / T (T = 0: 0), and its inverse
  double min64;     // 64 log2(min_p)
  float temperature, top_p, min_p;
  int k;            // ids that top-k leaves; 0: all
};
enum { kNone, kBest, kSum, kSlow };  // nothing to draw; by the list; by sums (and the list); as a whole

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
  unsigned long long *coarse;  // [row][slice][64]: of each group of buckets
  float *top;                // [row][slice]
  float *chunk_top;          // [row][slices * 16]
  uint32_t *real;            // [row][slice]: logits that can be drawn
  RowInfo *info;
  uint32_t *n_list;          // [row][slice]
  unsigned long long *list;  // [row][slice][kSliceList]
  unsigned long long *chunk; // [row][slices * 16]: of a wave's part of a slice
  uint32_t *chunk_n;
  RowSet rows[kRows];
};

// Logits as unsigned numbers of the same order; -infinity and NaN, which are never drawn, as 0.
__device__ inline uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);  // (-0 and 0 are equal)
  return !(x > -INFINITY) ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}
// (0: -infinity)
__device__ inline float of_key(uint32_t k) {
  return k == 0 ? -INFINITY : __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// One step across a wave's lanes: the value of a lane below (row_shr 1, 2, 4, 8 within 16 lanes; the last
// lane of a row of 16 to the next row, of the first half to the second), `old` where there is none.
template <int CTRL, int ROWS>
__device__ inline uint32_t from_below(uint32_t old, uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)old, (int)v, CTRL, ROWS, 15, false);
}
template <int CTRL, int ROWS>
__device__ inline unsigned long long from_below(unsigned long long old, unsigned long long v) {
  return (unsigned long long)from_below<CTRL, ROWS>((uint32_t)(old >> 32), (uint32_t)(v >> 32)) << 32 |
         from_below<CTRL, ROWS>((uint32_t)old, (uint32_t)v);
}
template <int CTRL, int ROWS>
__device__ inline u128 from_below(u128 old, u128 v) {
  return (u128)from_below<CTRL, ROWS>((unsigned long long)(old >> 64), (unsigned long long)(v >> 64)) << 64 |
         from_below<CTRL, ROWS>((unsigned long long)old, (unsigned long long)v);
}
// Running sum over a wave's lanes, a lane's own value in it.
template <class T>
__device__ inline T scan_wave(T v) {
  v += from_below<0x111, 15>((T)0, v);
  v += from_below<0x112, 15>((T)0, v);
  v += from_below<0x114, 15>((T)0, v);
  v += from_below<0x118, 15>((T)0, v);
  v += from_below<0x142, 10>((T)0, v);
  return v + from_below<0x143, 12>((T)0, v);
}
__device__ inline uint32_t last_lane(uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, 63); }
__device__ inline unsigned long long last_lane(unsigned long long v) {
  return (unsigned long long)last_lane((uint32_t)(v >> 32)) << 32 | last_lane((uint32_t)v);
}
__device__ inline u128 last_lane(u128 v) {
  return (u128)last_lane((unsigned long long)(v >> 64)) << 64 | last_lane((unsigned long long)v);
}
template <class T>
__device__ inline T sum_wave(T v) {
  return last_lane(scan_wave(v));
}
__device__ inline uint32_t max_wave(uint32_t v) {
  v = max(v, from_below<0x111, 15>(v, v));
  v = max(v, from_below<0x112, 15>(v, v));
  v = max(v, from_below<0x114, 15>(v, v));
  v = max(v, from_below<0x118, 15>(v, v));
  v = max(v, from_below<0x142, 10>(v, v));
  return last_lane(max(v, from_below<0x143, 12>(v, v)));
}

// 2^(j/64)
__device__ const double kExp2[64] = {
    0x1.0000000000000p+0, 0x1.02c9a3e778061p+0, 0x1.059b0d3158574p+0, 0x1.0874518759bc8p+0,
    0x1.0b5586cf9890fp+0, 0x1.0e3ec32d3d1a2p+0, 0x1.11301d0125b51p+0, 0x1.1429aaea92de0p+0,
    0x1.172b83c7d517bp+0, 0x1.1a35beb6fcb75p+0, 0x1.1d4873168b9aap+0, 0x1.2063b88628cd6p+0,
    0x1.2387a6e756238p+0, 0x1.26b4565e27cddp+0, 0x1.29e9df51fdee1p+0, 0x1.2d285a6e4030bp+0,
    0x1.306fe0a31b715p+0, 0x1.33c08b26416ffp+0, 0x1.371a7373aa9cbp+0, 0x1.3a7db34e59ff7p+0,
    0x1.3dea64c123422p+0, 0x1.4160a21f72e2ap+0, 0x1.44e086061892dp+0, 0x1.486a2b5c13cd0p+0,
    0x1.4bfdad5362a27p+0, 0x1.4f9b2769d2ca7p+0, 0x1.5342b569d4f82p+0, 0x1.56f4736b527dap+0,
    0x1.5ab07dd485429p+0, 0x1.5e76f15ad2148p+0, 0x1.6247eb03a5585p+0, 0x1.6623882552225p+0,
    0x1.6a09e667f3bcdp+0, 0x1.6dfb23c651a2fp+0, 0x1.71f75e8ec5f74p+0, 0x1.75feb564267c9p+0,
    0x1.7a11473eb0187p+0, 0x1.7e2f336cf4e62p+0, 0x1.82589994cce13p+0, 0x1.868d99b4492edp+0,
    0x1.8ace5422aa0dbp+0, 0x1.8f1ae99157736p+0, 0x1.93737b0cdc5e5p+0, 0x1.97d829fde4e50p+0,
    0x1.9c49182a3f090p+0, 0x1.a0c667b5de565p+0, 0x1.a5503b23e255dp+0, 0x1.a9e6b5579fdbfp+0,
    0x1.ae89f995ad3adp+0, 0x1.b33a2b84f15fbp+0, 0x1.b7f76f2fb5e47p+0, 0x1.bcc1e904bc1d2p+0,
    0x1.c199bdd85529cp+0, 0x1.c67f12e57d14bp+0, 0x1.cb720dcef9069p+0, 0x1.d072d4a07897cp+0,
    0x1.d5818dcfba487p+0, 0x1.da9e603db3285p+0, 0x1.dfc97337b9b5fp+0, 0x1.e502ee78b3ff6p+0,
    0x1.ea4afa2a490dap+0, 0x1.efa1bee615a27p+0, 0x1.f50765b6e4540p+0, 0x1.fa7c1819e90d8p+0};

// 2^((k + r)/64) as a whole number, |r| <= 1/2 or little more: 2^(j/64) from a table, a polynomial of degree 4 over a 64th of
// an octave (off by 4e-14 of it at most); sums with large constants round to whole numbers.  (With rint, ldexp and
// conversions in place of the constants the 12.6 million weights of 48 rows took 20 us more.)
struct Exp2 {
  const double *table;  // LDS, [64]
  // times 2^e in place of 2^(k/64 rounded down), e <= 49
  __device__ unsigned long long whole(int k, double r, int e) const {
    constexpr double L = 0.010830424696249145;  // ln(2) / 64
    double p = __builtin_fma(r, L * L * L * L / 24, L * L * L / 6);
    p = __builtin_fma(r, p, L * L / 2);
    p = __builtin_fma(r, p, L);
    p = __builtin_fma(r, p, 1.0);
    const long long t = __double_as_longlong(table[k & 63]) + ((long long)e << 52);
    return (unsigned long long)__double_as_longlong(__builtin_fma(p, __longlong_as_double(t), 0x1p52)) & 0xFFFFFFFFFFFFFull;
  }
  // 2^(z/64) as a whole number of 2^-bits
  __device__ unsigned long long operator()(double z, int bits) const {
    z = __builtin_fmax(z, -3840.0);  // (2^-60: none)
    const double m = z + 0x1.8p52, r = z - (m - 0x1.8p52);
    const int k = (int)__double_as_longlong(m);
    return whole(k, r, (k >> 6) + bits);
  }
};
__device__ inline void exp2_table(double *t) {
  if (threadIdx.x < 64) t[threadIdx.x] = kExp2[threadIdx.x];
}
// By sums a logit's place is x c64, k + r of it in 64ths of an octave, k its nearest whole number: the same whatever the
// logit is compared with, and so is the bucket of 1/32 of an octave that it lies in, k / 2 rounded down.
struct Place {
  int k;
  double r;
};
// (least: logits below it, none of which weighs anything, are taken as that)
__device__ inline Place place_of(float x, double least, double c64) {
  const double y = __builtin_fmax((double)x, least), m = __builtin_fma(y, c64, 0x1.8p52);
  return {(int)__double_as_longlong(m), __builtin_fma(y, c64, -(m - 0x1.8p52))};
}
// The reference of a largest logit: the end of its octave; a row's largest is at most 2^17 octaves from 0.  (A slice's at most
// 2^18: of a row in the range the slices past that weigh nothing, those between do.)
__device__ inline bool in_range(float top, double c64) { return fabs((double)top * c64) < 0x1p23; }
__device__ inline bool slice_in_range(float top, double c64) { return fabs((double)top * c64) < 0x1p24; }
__device__ inline int ref_of(float top, double c64) { return (place_of(top, -INFINITY, c64).k >> 6) + 1; }
// 66 octaves below it.
__device__ inline double least_of(int ref, const RowSet &set) { return (64.0 * ref - 4224.0) * set.by; }
// The weight by its own octave, and in the row's unit.
__device__ inline unsigned long long weight_of_octave(const Exp2 &exp2, Place p, int bits) { return exp2.whole(p.k, p.r, bits); }
__device__ inline unsigned long long weight_of(const Exp2 &exp2, Place p, int ref, int bits) {
  return exp2.whole(p.k, p.r, (p.k >> 6) - ref + bits);
}
// By counts: a bucket is the exponent and eight bits of the mantissa, whatever the logits' size.
__device__ inline int bucket_of(float x) { return (int)(key_of(x) >> 15); }
// The least number that is `ok`, as all larger ones are; z: its place, to a few roundings.  (by: 1 / c64, by which the first
// guess is off by one number at most)
template <class F>
__device__ inline float least_float(double z, double by, const F &ok) {
  const float x = fmaxf((float)(z * by), -MAX32), below = of_key(key_of(x) - 1);
  return !ok(x) ? of_key(key_of(x) + 1) : ok(below) ? below : x;
}
// The first logit of bucket b.
__device__ inline float least_of_bucket(int b, const RowSet &set) {
  return least_float(2.0 * b - 0.5, set.by, [&](float y) { return place_of(y, -INFINITY, set.c64).k >= 2 * b; });
}
// By sums min_p leaves the logits from this one on.
__device__ inline float least_of_min_p(float top, const RowSet &set) {
  if (!(set.min_p > 0.f)) return -MAX32;
  const double z = __builtin_fma((double)top, set.c64, set.min64);
  return fminf(top, least_float(z, set.by, [&](float y) { return (double)y * set.c64 >= z; }));
}

template <int PER, bool VEC>
__device__ inline void load_chunk(const float *x, int n, int at, float (&v)[PER]) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int j = 0; j < PER / 4; ++j) {
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
  for (int j = 0; j < PER; ++j) v[j] = v[j] > -INFINITY ? v[j] : -INFINITY;  // (NaN too)
}

// A slice's buckets are counted from the top of its largest logit's group of 32 down: those of two slices
// lie whole groups apart.  That group's number:
template <bool SUMS>
__device__ inline int group_of(float top, double c64) {
  if constexpr (SUMS) return ref_of(top, c64);
  return (bucket_of(top) >> 5) + 1;
}

__device__ inline unsigned long long share_of(float p, unsigned long long total) {
  const unsigned long long t = (unsigned long long)ceil((double)p * (double)total);
  return t ? t : 1;
}
// The least whole number of p of the total, p < 1, rounded nowhere: a number of equal weights may be just that.  (Below 2^-32:
// 1, which the largest weight reaches as well.)
__device__ inline u128 share_of(float p, u128 total) {
  if (p < 0x1p-32f) return 1;
  const uint32_t b = __float_as_uint(p), s = 150 - (b >> 23), f = (b & 0x7FFFFFu) | 0x800000u;  // p = f 2^-s, 24 <= s <= 55
  const u128 low = (u128)(unsigned long long)total * f, high = (total >> 64) * f + (low >> 64);
  const unsigned long long lo = (unsigned long long)low;
  return (high << (64 - s)) + (lo >> s) + ((lo & ((1ull << s) - 1)) != 0);
}
// By one wave, lane g holding the weight of the row's octave g (from the top, by that octave): the octave in which the running
// weight reaches p of the whole, and of that octave's what it has to reach.
__device__ inline int octave_of_share(float p, unsigned long long weight, unsigned long long *want) {
  const int lane = threadIdx.x & 63;
  const u128 w = (u128)weight << (63 - lane), upto = scan_wave(w), goal = share_of(p, last_lane(upto));
  const unsigned long long hit = __ballot(upto >= goal);
  const int g = __ffsll(hit) - 1;  // (the last octave's reaches the whole)
  const u128 rest = goal - (upto - w);
  const unsigned long long mine = (unsigned long long)((rest + (((u128)1 << (63 - lane)) - 1)) >> (63 - lane));
  *want = __shfl(mine, g, 64);
  return g;
}

struct CutLds {
  unsigned long long part[kNT / 64][64];
  unsigned long long goal;
  int group;
  RowInfo info;
};

// What a row's slices say: the state, and the bucket in which the cut lies.  Each wave adds up the buckets of its
// share of the slices, the first wave looks for the cut in the sum: among the groups, then in the one it lies in.  (By
// the first wave alone 11 us for 64 slices.)
template <bool SUMS>
__device__ inline void find_cut(const SampleRowsArgs &a, const RowSet &set, size_t at, CutLds &lds) {
  constexpr int W = kNT / 64, Q = kMostSlices / W;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float mine = lane < a.slices ? ldg<float>(a.top + at + lane) : -INFINITY;
  uint32_t real = lane < a.slices ? ldg<uint32_t>(a.real + at + lane) : 0;
  const float top = of_key(max_wave(key_of(mine)));
  real = sum_wave(real);
  RowInfo in{real == 0 ? kNone : top == INFINITY || set.k > kMostK ? kSlow : SUMS ? kSum : kBest, 0, top, -MAX32, -MAX32, 0, 0};
  if (in.state == kSum && !in_range(top, set.c64)) in.state = kSlow;
  const bool all = SUMS && set.top_p >= 1.f;
  const int group0 = in.state == kSum || in.state == kBest ? group_of<SUMS>(top, set.c64) : 0;
  if (in.state == kSum) in.ref = group0;
  if (in.state == kNone || in.state == kSlow || all) {
    if (wave == 0) {
      if (in.state == kSum) in.lo = in.hi = least_of_min_p(top, set);
      if (lane == 0) lds.info = in;
    }
    __syncthreads();
    return;
  }
  // groups that a slice's buckets begin below the row's
  const bool has = mine > -INFINITY && (!SUMS || slice_in_range(mine, set.c64));
  const int down = has ? group0 - group_of<SUMS>(mine, set.c64) : kBins;
  unsigned long long h[Q], s = 0;
  int d[Q];
#pragma unroll
  for (int e = 0; e < Q; ++e) {
    if (W * e >= a.slices) break;
    const int q = min(wave + W * e, a.slices - 1);
    d[e] = __builtin_amdgcn_readlane(down, q);
    h[e] = ldg<unsigned long long>(a.coarse + (at + q) * 64 + max(lane - d[e], 0));
  }
#pragma unroll
  for (int e = 0; e < Q; ++e) {
    if (W * e >= a.slices) break;
    s += wave + W * e < a.slices && lane >= d[e] ? h[e] : 0;
  }
  lds.part[wave][lane] = s;
  __syncthreads();
  if (wave == 0) {
    s = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) s += lds.part[w][lane];
    unsigned long long goal;
    int group;
    if constexpr (SUMS) {
      group = octave_of_share(set.top_p, s, &goal);
    } else {
      const unsigned long long upto = scan_wave(s), hit = __ballot(upto >= (unsigned long long)set.k);
      group = hit ? __ffsll(hit) - 1 : -1;
      goal = set.k - __shfl(upto - s, max(group, 0), 64);
    }
    if (lane == 0) {
      // (top-k, whose buckets end eight octaves below the largest logit: all that can be drawn is in the list, if it holds
      // that, and nothing is `want`ed of a bucket)
      if (group < 0 && real > kList) in.state = kSlow;
      if (!SUMS) in.hi = INFINITY;
      lds.info = in;
      lds.group = group;
      lds.goal = goal;
    }
  }
  __syncthreads();
  const int group = lds.group;
  if (group < 0) return;
  // ---- the group's 32 buckets: two slices at a time
  s = 0;
#pragma unroll
  for (int e = 0; e < Q / 2; ++e) {
    if (2 * W * e >= a.slices) break;
    const int q = min(2 * (wave + W * e) + (lane >> 5), a.slices - 1);
    d[e] = __shfl(down, q, 64);
    const size_t i = 32 * max(group - d[e], 0) + (lane & 31);
    const unsigned long long *from = a.hist + (at + q) * kBins;
    if constexpr (SUMS)
      h[e] = ldg<unsigned long long>(from + i);
    else
      h[e] = ldg<uint32_t>(reinterpret_cast<const uint32_t *>(from) + i);
  }
#pragma unroll
  for (int e = 0; e < Q / 2; ++e) {
    if (2 * W * e >= a.slices) break;
    s += 2 * (wave + W * e) + (lane >> 5) < a.slices && group >= d[e] ? h[e] : 0;
  }
  lds.part[wave][lane] = s;
  __syncthreads();
  if (wave == 0) {
    s = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) s += lds.part[w][lane & 31] + lds.part[w][32 + (lane & 31)];
    if (lane >= 32) s = 0;
    const unsigned long long goal = lds.goal, upto = scan_wave(s), hit = __ballot(upto >= goal && lane < 32);
    const int bin = __ffsll(hit) - 1;
    in.want = goal - __shfl(upto - s, bin, 64);
    const int bucket = 32 * (group0 - group) - 1 - bin;
    in.bucket = bucket;
    if constexpr (SUMS) {
      // (the first lane's and the others' bound)
      const float x = least_of_bucket(bucket + (lane > 0), set), least = least_of_min_p(top, set);
      in.lo = fmaxf(__shfl(x, 0, 64), least);
      in.hi = fmaxf(__shfl(x, 1, 64), least);
    } else {
      in.lo = of_key((uint32_t)bucket << 15);
      in.hi = INFINITY;
    }
    if (lane == 0) lds.info = in;
  }
  __syncthreads();
}

// A thread has PER logits, a wave a chunk of 64 PER.
template <int PER, bool VEC>
__global__ __launch_bounds__(kNT) void k_rows_scan(SampleRowsArgs a) {
  __shared__ __align__(16) unsigned long long hist[kBins];
  __shared__ double table[64];
  __shared__ uint32_t tops[kNT / 64], reals[kNT / 64];
  uint32_t *count = reinterpret_cast<uint32_t *>(hist);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.y;
  const RowSet &set = a.rows[row];
  const bool sums = set.k == 0, bins = sums ? set.top_p < 1.f : set.k <= kMostK;
  float v[PER];
  load_chunk<PER, VEC>(a.x + row * a.ld, a.n, blockIdx.x * a.slice + wave * 64 * PER, v);
  if (bins) {
    for (int i = tid; i < (sums ? kBins : kBins / 2); i += kNT) hist[i] = 0;
    exp2_table(table);
  }
  float most = -INFINITY;
  uint32_t real = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    most = fmaxf(most, v[j]);
    real += v[j] > -INFINITY;
  }
  uint32_t key = max_wave(key_of(most));
  real = sum_wave(real);
  const size_t at = (size_t)row * a.slices + blockIdx.x;
  if (lane == 0) {
    tops[wave] = key;
    reals[wave] = real;
    a.chunk_top[at * (kNT / 64) + wave] = of_key(key);
  }
  __syncthreads();
  key = 0;
#pragma unroll
  for (int w = 0; w < kNT / 64; ++w) key = max(key, tops[w]);
  const float top = of_key(key);
  if (tid == 0) {
    real = 0;
    for (int w = 0; w < kNT / 64; ++w) real += reals[w];
    a.top[at] = top;
    a.real[at] = real;
  }
  if (bins && top > -INFINITY && top < INFINITY && (!sums || slice_in_range(top, set.c64))) {
    if (sums) {
      const Exp2 exp2{table};
      const int ref = ref_of(top, set.c64);
      const double least = least_of(ref, set);
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const Place p = place_of(v[j], least, set.c64);
        const uint32_t d = 32 * ref - 1 - (p.k >> 1);
        if (d < kBins) atomicAdd(&hist[d], weight_of_octave(exp2, p, a.bits));
      }
    } else {
      const int base = bucket_of(top) | 31;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int d = base - bucket_of(v[j]);
        if (d < kBins) atomicAdd(&count[d], 1u);
      }
    }
    __syncthreads();
    // two buckets a thread, a group 16 threads
    unsigned long long two;
    if (sums) {
      const unsigned long long h0 = hist[2 * tid], h1 = hist[2 * tid + 1];
      a.hist[at * kBins + 2 * tid] = h0;
      a.hist[at * kBins + 2 * tid + 1] = h1;
      two = h0 + h1;
    } else {
      const unsigned long long h = hist[tid];
      a.hist[at * kBins + tid] = h;
      two = (h & 0xFFFFFFFFu) + (h >> 32);
    }
    for (int o = 1; o < 16; o <<= 1) two += __shfl_xor(two, o, 64);
    if ((tid & 15) == 0) a.coarse[at * 64 + tid / 16] = two;
  }
}

// Each block looks for the cut (in a kernel of its own, a block a row: 5 us and a launch, 2 to 4 us here); then a wave goes
// over its chunk once more, but for one whose largest logit lies below the cut.
template <int PER, bool VEC>
__global__ __launch_bounds__(kNT) void k_rows_pick(SampleRowsArgs a) {
  __shared__ double table[64];
  __shared__ uint32_t places[kNT / 64];
  __shared__ CutLds lds;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.y;
  const RowSet &set = a.rows[row];
  const bool sums = set.k == 0, cut = sums && set.top_p < 1.f;
  const size_t slice = (size_t)row * a.slices + blockIdx.x, ch = slice * (kNT / 64) + wave;
  const int id0 = blockIdx.x * a.slice + wave * 64 * PER;
  const float chunk_top = ldg<float>(a.chunk_top + ch);
  exp2_table(table);
  if (sums)
    find_cut<true>(a, set, (size_t)row * a.slices, lds);
  else
    find_cut<false>(a, set, (size_t)row * a.slices, lds);
  const RowInfo in = lds.info;
  if (blockIdx.x == 0 && tid == 0) a.info[row] = in;
  if (in.state == kNone || in.state == kSlow) return;
  const Exp2 exp2{table};
  const double least = least_of(in.ref, set);
  unsigned long long sum = 0;
  uint32_t num = 0, listed = 0;  // bit j: logit j goes to the list
  float v[PER];
  if (chunk_top >= in.lo) {
    load_chunk<PER, VEC>(a.x + row * a.ld, a.n, id0, v);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      listed |= (uint32_t)(v[j] >= in.lo && v[j] < in.hi) << j;
      if (v[j] >= in.hi) {
        sum += weight_of(exp2, place_of(v[j], least, set.c64), in.ref, a.bits);
        ++num;
      }
    }
    if (sums) {
      sum = sum_wave(sum);
      num = sum_wave(num);
    }
  }
  if (sums && lane == 0) {
    a.chunk[ch] = sum;
    a.chunk_n[ch] = num;
  }
  // the slice's candidates, in a place of their own (a list for the row, whose end blocks ask for by an atomic: 4 us, one
  // block after the other)
  if (!sums || cut) {
    const uint32_t mine = __popc(listed), upto = scan_wave(mine);
    if (lane == 63) places[wave] = upto;
    __syncthreads();
    uint32_t at = upto - mine, all = 0;
#pragma unroll
    for (int w = 0; w < kNT / 64; ++w) {
      const uint32_t p = places[w];
      at += w < wave ? p : 0;
      all += p;
    }
    if (tid == 0) a.n_list[slice] = all;
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (listed >> j & 1) {
        if (at < kSliceList)
          a.list[slice * kSliceList + at] = (unsigned long long)key_of(v[j]) << 32 |
                                            (0xFFFFFFFFu - (uint32_t)(id0 + 256 * (j / 4) + 4 * lane + j % 4));
        ++at;
      }
  } else if (tid == 0) {
    a.n_list[slice] = 0;
  }
}

// Falling order of n numbers, n a power of two from 64 on.  A wave does the steps within 128 numbers of its own
// without waiting for the others.
__device__ inline void sort_falling(unsigned long long *x, int n) {
  const int lane = threadIdx.x & 63;
  auto swap = [&](int t, int size, int step) {
    const int i = 2 * t - (t & (step - 1)), j = i + step;
    const unsigned long long p = x[i], q = x[j];
    if ((p < q) == ((i & size) == 0)) {
      x[i] = q;
      x[j] = p;
    }
  };
  auto near = [&](int size, int step) {  // steps of up to 64: pairs t of a wave lie among its 128 numbers
    for (int t = threadIdx.x; t - lane < n / 2; t += kNT)
      for (int s = step; s > 0; s >>= 1) {
        if (t < n / 2) swap(t, size, s);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (no instruction: LDS accesses stay in their order)
      }
  };
  __syncthreads();
  for (int size = 2; size <= 128 && size <= n; size <<= 1) near(size, size / 2);
  for (int size = 256; size <= n; size <<= 1) {
    for (int step = size / 2; step > 64; step >>= 1) {
      __syncthreads();
      for (int t = threadIdx.x; t < n / 2; t += kNT) swap(t, size, step);
    }
    __syncthreads();
    near(size, 64);
  }
  __syncthreads();
}
// The same by one wave, of n <= 64 E numbers that differ: each goes to the place that says how many are larger.
// (64 numbers 0.6 us; sorted as above 3.6 us, a chain of 21 LDS round trips)
template <int E>
__device__ inline void rank_by_wave(unsigned long long *x, int n) {
  const int lane = threadIdx.x & 63;
  unsigned long long v[E];
  int place[E] = {};
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = 64 * e + lane < n ? x[64 * e + lane] : 0;
#pragma unroll
  for (int f = 0; f < E; ++f)
    for (int l = 0; l < min(64, n - 64 * f); ++l) {
      const unsigned long long y = (unsigned long long)(uint32_t)__builtin_amdgcn_readlane((int)(v[f] >> 32), l) << 32 |
                                   (uint32_t)__builtin_amdgcn_readlane((int)v[f], l);
#pragma unroll
      for (int e = 0; e < E; ++e) place[e] += y > v[e];
    }
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (64 * e + lane < n) x[place[e]] = v[e];
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}
__device__ inline void sort_by_wave(unsigned long long *x, int n) {
  if (n <= 64)
    rank_by_wave<1>(x, n);
  else if (n <= 128)
    rank_by_wave<2>(x, n);
  else
    rank_by_wave<kWave / 64>(x, n);
}
__device__ inline int power_of_two(int n) {
  int p = 64;
  while (p < n) p <<= 1;
  return p;
}

// Running sum over the block's threads, this one's value among it; *all: the whole.
__device__ inline unsigned long long run_sum(unsigned long long v, unsigned long long *part, unsigned long long *all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = scan_wave(v);
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
__device__ inline uint32_t id_of(unsigned long long entry) { return 0xFFFFFFFFu - (uint32_t)entry; }
__device__ inline float logit_of(unsigned long long entry) { return of_key((uint32_t)(entry >> 32)); }
__device__ inline void write_row(const SampleRowsArgs &a, int row, int id, float prob, uint32_t kept) {
  a.ids[row] = id;
  if (a.prob) a.prob[row] = prob;
  if (a.kept) a.kept[row] = (int)kept;
}

struct RowLds {
  unsigned long long bin[kBins];
  unsigned long long part[kNT / 64];
  unsigned long long before, cut;
  int found;
  uint32_t num, kept;
};

// The bin (of two of each thread's) at which the running sum reaches goal: to lds.found, what lies before it to lds.before.
__device__ inline void find_bin(RowLds &lds, unsigned long long before, unsigned long long goal) {
  const unsigned long long h0 = lds.bin[2 * threadIdx.x], h1 = lds.bin[2 * threadIdx.x + 1];
  unsigned long long total;
  const unsigned long long upto = before + run_sum(h0 + h1, lds.part, &total);
  if (upto >= goal && upto - h0 - h1 < goal) {
    const bool second = upto - h1 < goal;
    lds.found = 2 * threadIdx.x + second;
    lds.before = second ? upto - h1 : upto - h0 - h1;
  }
  __syncthreads();
}

// The whole of a row, by one block (in: what is known of it, or null).  The cut's logit is found by histograms over the keys of a range,
// by counts (top-k) or weights (top-p), the range then being the bin that the cut lies in.  (One row of 262144
// logits that are all alike, about nine times over the row: 0.43 ms.)
__device__ inline void row_by_ranges(const SampleRowsArgs &a, const Exp2 &exp2, RowLds &lds, const RowInfo *in) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = a.n, row = blockIdx.x;
  const RowSet &set = a.rows[row];
  const float *x = a.x + row * a.ld;
  auto each = [&](int from, int to, int step, const auto &f) {  // eight loads in flight
    for (int i0 = from; i0 < to; i0 += 8 * step) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = ldg<float>(x + min(i0 + e * step, to - 1));
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (i0 + e * step < to) f(v[e], i0 + e * step);
    }
  };
  auto over_block = [&](unsigned long long v) {
    unsigned long long all;
    run_sum(v, lds.part, &all);
    __syncthreads();
    return all;
  };

  // ---- largest and least logit, and how many can be drawn
  uint32_t top = 0, least = 0xFFFFFFFFu, mine = 0;
  each(tid, n, kNT, [&](float v, int) {
    const uint32_t k = key_of(v);
    top = max(top, k);
    least = min(least, k ? k : 0xFFFFFFFFu);
    mine += k != 0;
  });
  const uint32_t real = (uint32_t)over_block(mine);
  if (real == 0) {
    if (tid == 0) write_row(a, row, -1, 0.f, 0);
    return;
  }
  if (tid == 0) lds.before = lds.cut = 0;
  __syncthreads();
  top = max_wave(top);
  least = ~max_wave(~least);
  if (lane == 0) {
    atomicMax(&lds.before, (unsigned long long)top);
    atomicMax(&lds.cut, (unsigned long long)~least);
  }
  __syncthreads();
  top = (uint32_t)lds.before;
  least = ~(uint32_t)lds.cut;
  const double vmax = of_key(top);
  // (whether the lists hold a row depends on how it was cut into slices: what is done to it here does not)
  const bool sums = set.k == 0 && in_range((float)vmax, set.c64);
  const int ref = sums ? ref_of((float)vmax, set.c64) : 0;
  const double from = least_of(ref, set);
  auto place = [&](float v) { return v == (float)vmax ? 0.0 : ((double)v - vmax) * set.c64; };
  auto weight = [&](float v) { return sums ? weight_of(exp2, place_of(v, from, set.c64), ref, a.bits) : exp2(place(v), a.bits); };

  // Where the count (or weight) from the top, `hi`, reaches `want`, of what lies at or above `floor` (of those equal
  // to it, floor_n): the key; what lies above it.
  enum By { kCount, kWeight, kOctave };
  unsigned long long above;
  auto find = [&](By by, unsigned long long want, uint32_t hi, uint32_t floor, uint32_t floor_n) {
    uint32_t lo = floor;
    above = 0;
    for (;;) {
      const int shift = hi - lo < kBins ? 0 : 21 - __clz(hi - lo);
      __syncthreads();
      for (int i = tid; i < kBins; i += kNT) lds.bin[i] = 0;
      __syncthreads();
      each(tid, n, kNT, [&](float v, int) {
        const uint32_t k = key_of(v);
        if (k >= lo && k <= hi && (by != kWeight || k > floor))
          atomicAdd(&lds.bin[(hi - k) >> shift],
                    by == kCount ? 1ull : by == kWeight ? weight(v) : weight_of_octave(exp2, place_of(v, from, set.c64), a.bits));
      });
      if (by == kWeight && tid == 0 && lo == floor) atomicAdd(&lds.bin[(hi - floor) >> shift], floor_n * weight(of_key(floor)));
      __syncthreads();
      find_bin(lds, above, want);
      above = lds.before;
      hi -= (uint32_t)lds.found << shift;
      if (shift == 0) return hi;
      lo = max(lo, hi - ((1u << shift) - 1));
    }
  };
  auto equal_to = [&](uint32_t key) {
    uint32_t num = 0;
    each(tid, n, kNT, [&](float v, int) { num += key_of(v) == key; });
    return (uint32_t)over_block(num);
  };

  uint32_t key = least, eq = 0xFFFFFFFFu;  // of the logits equal to the cut, the first eq are left
  if (set.k > 0 && (uint32_t)set.k < real) {
    key = find(kCount, set.k, top, least, 0);
    eq = (uint32_t)(set.k - above);
  }
  if (sums && set.top_p < 1.f && least == top) {
    eq = (uint32_t)share_of(set.top_p, (u128)real);
  } else if (sums && set.top_p < 1.f) {
    // the octave, its bucket and the logit in which the cut lies
    int bucket;
    unsigned long long want;
    if (in) {
      bucket = in->bucket;
      want = in->want;
    } else {
      for (int i = tid; i < kBins; i += kNT) lds.bin[i] = 0;
      __syncthreads();
      each(tid, n, kNT, [&](float v, int) {
        const Place p = place_of(v > -INFINITY ? v : -INFINITY, from, set.c64);
        const uint32_t d = 32 * ref - 1 - (p.k >> 1);
        if (d < kBins) atomicAdd(&lds.bin[d], weight_of_octave(exp2, p, a.bits));
      });
      __syncthreads();
      if (wave == 0) {
        unsigned long long w = 0, rest;
        for (int i = 0; i < 32; ++i) w += lds.bin[32 * lane + i];
        const int g = octave_of_share(set.top_p, w, &rest);
        const unsigned long long mine = lane < 32 ? lds.bin[32 * g + lane] : 0, upto = scan_wave(mine);
        const int b = __ffsll((unsigned long long)__ballot(upto >= rest)) - 1;
        rest -= __shfl(upto - mine, b, 64);
        if (lane == 0) {
          lds.found = 32 * ref - 1 - (32 * g + b);
          lds.cut = rest;
        }
      }
      __syncthreads();
      bucket = lds.found;
      want = lds.cut;
    }
    key = find(kOctave, want, min(top, key_of(least_of_bucket(bucket + 1, set)) - 1),
               max(least, key_of(least_of_bucket(bucket, set))), 0);
    const unsigned long long w = weight_of_octave(exp2, place_of(of_key(key), from, set.c64), a.bits);
    eq = (uint32_t)min((want - above + w - 1) / w, 0xFFFFFFFFull);
  } else if (set.temperature != 0.f && set.top_p < 1.f) {
    unsigned long long sum = 0;
    each(tid, n, kNT, [&](float v, int) {
      if (key_of(v) > key) sum += weight(v);
    });
    const uint32_t floor_n = min(eq, equal_to(key));
    sum = over_block(sum) + floor_n * weight(of_key(key));
    const unsigned long long want = share_of(set.top_p, sum);
    const uint32_t floor = key;
    key = find(kWeight, want, top, floor, floor_n);
    const unsigned long long w = weight(of_key(key)), take = (want - above + w - 1) / w;
    eq = (uint32_t)min(take, (unsigned long long)(key == floor ? floor_n : 0xFFFFFFFFu));
  }
  uint32_t last_eq = 0xFFFFFFFFu;  // the last id of those equal to the cut that is left
  if (eq < equal_to(key)) {
    uint32_t seen = 0;
    for (int i0 = 0; i0 < n; i0 += kNT) {
      const int i = i0 + tid;
      const bool is = i < n && key_of(ldg<float>(x + i)) == key;
      unsigned long long all;
      const uint32_t upto = seen + (uint32_t)run_sum(is, lds.part, &all);
      if (is && upto == eq) lds.found = i;
      seen += (uint32_t)all;
      if (seen >= eq) break;
    }
    __syncthreads();
    last_eq = (uint32_t)lds.found;
  }
  const float min_x = sums ? least_of_min_p((float)vmax, set) : 0.f;
  auto left = [&](float v, int i) {
    const uint32_t k = key_of(v);
    if (k < key || (k == key && (uint32_t)i > last_eq)) return false;
    return sums ? v >= min_x : k == top || place(v) >= set.min64;
  };
  // ---- the draw: the wave, then the sixteenth of its part, and so on, in which the running weight passes the target
  unsigned long long total = 0, target = 0, before = 0;
  uint32_t count = 0;
  int lo = 0, len = n;
  for (bool first = true; len > 64 || first; first = false) {
    const int per = ((len + 15) / 16 + 63) / 64 * 64, b0 = lo + min(len, wave * per), b1 = lo + min(len, wave * per + per);
    unsigned long long sum = 0;
    uint32_t num = 0;
    each(b0 + lane, b1, 64, [&](float v, int i) {
      if (left(v, i)) {
        sum += weight(v);
        ++num;
      }
    });
    if (first) count = (uint32_t)over_block(num);
    sum = sum_wave(sum);
    __syncthreads();
    if (lane == 0) lds.part[wave] = sum;
    __syncthreads();
    if (first) {
      for (int w = 0; w < 16; ++w) total += lds.part[w];
      target = target_of(ldg<float>(a.u + row), total);
    }
    int w = 0;
    while (w < 15 && before + lds.part[w] <= target) before += lds.part[w++];
    lo += min(len, w * per);
    len = min(len - min(len, w * per), per);
  }
  if (wave != 0) return;
  const int i = lo + lane;
  unsigned long long w = 0;
  if (lane < len) {
    const float v = ldg<float>(x + i);
    if (left(v, i)) w = weight(v);
  }
  const unsigned long long upto = before + scan_wave(w);
  if (upto > target && upto - w <= target) write_row(a, row, i, (float)((double)w / (double)total), count);
}

// The draw of a row whose best ids are the sorted list's first, nk of them, E of these a lane, by one wave.
template <int E>
__device__ inline void draw_few(const SampleRowsArgs &a, const RowSet &set, int row, float top, int nk, float u,
                                const Exp2 &exp2, unsigned long long *list, unsigned long long *by_place) {
  const int at = (threadIdx.x & 63) * E;
  unsigned long long w[E], sum = 0;
  uint32_t id[E], over = 0, under = 0;  // how many min_p leaves, and top-p
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const bool in = at + e < nk;
    const unsigned long long x = in ? list[at + e] : 0;
    const float v = logit_of(x);
    id[e] = id_of(x);
    const double z = v == top ? 0.0 : ((double)v - (double)top) * set.c64;
    w[e] = in ? exp2(z, a.bits) : 0;
    over += __popcll(__ballot(in && (v == top || z >= set.min64)));
    sum += w[e];
  }
  unsigned long long upto = scan_wave(sum), total = last_lane(upto);
  upto -= sum;
  const unsigned long long goal = set.temperature != 0.f && set.top_p < 1.f ? share_of(set.top_p, total) : ~0ull;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    under += __popcll(__ballot(at + e < nk && upto < goal));
    upto += w[e];
  }
  const int n = (int)min(over, under);
  // ---- in the order of ids: (id, place) sorted, the weights by their places
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (at + e < n) {
      list[at + e] = (unsigned long long)(0xFFFFFFFFu - id[e]) << 32 | (uint32_t)(at + e);
      by_place[at + e] = w[e];
    }
  sort_by_wave(list, n);
  sum = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const unsigned long long x = at + e < n ? list[at + e] : 0;
    id[e] = 0xFFFFFFFFu - (uint32_t)(x >> 32);
    w[e] = at + e < n ? by_place[(uint32_t)x] : 0;
    sum += w[e];
  }
  upto = scan_wave(sum);
  total = last_lane(upto);
  upto -= sum;
  const unsigned long long target = target_of(u, total);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (upto <= target && upto + w[e] > target) write_row(a, row, (int)id[e], (float)((double)w[e] / (double)total), n);
    upto += w[e];
  }
}

// The chunk in which the running weight passes the target, by one wave: *before, what the chunks before it weigh.
__device__ inline int find_chunk(const unsigned long long *chunk, int n_chunks, float u, unsigned long long *total,
                                 unsigned long long *target, unsigned long long *before) {
  const int lane = threadIdx.x & 63, per = (n_chunks + 63) / 64;
  unsigned long long sum = 0;
  for (int i = 0; i < per; ++i) sum += per * lane + i < n_chunks ? chunk[per * lane + i] : 0;
  const unsigned long long upto = scan_wave(sum);
  *total = last_lane(upto);
  *target = target_of(u, *total);
  const int l = __ffsll((unsigned long long)__ballot(upto > *target)) - 1;
  unsigned long long b = __shfl(upto - sum, l, 64);
  int hit = per * l;
  while (b + chunk[hit] <= *target) b += chunk[hit++];
  *before = b;
  return hit;
}

// The same of a longer list, by all threads.  Nothing is sorted but what lies in the bucket of a cut (top-k's, then
// top-p's) and in the chunk of ids in which the draw falls.  (Sorted as a whole, 1000 ids of 48 rows: 20 us.)
__device__ inline void draw_many(const SampleRowsArgs &a, const RowSet &set, int row, const RowInfo &in, int n_list,
                                 float u, const Exp2 &exp2, unsigned long long *list, unsigned long long *chunk,
                                 int n_chunks, int chunk_len, RowLds &lds) {
  constexpr int E = kList / kNT;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  unsigned long long x[E], w[E];
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = kNT * e + tid < n_list ? list[kNT * e + tid] : 0;
  // those that `which` says, into the list from its start, the largest first
  auto gather = [&](const auto &which) {
    __syncthreads();
    if (tid == 0) lds.num = 0;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (kNT * e >= n_list) break;
      const bool is = x[e] && which(x[e]);
      const unsigned long long m = __ballot(is);
      uint32_t at = 0;
      if (m) {
        if (lane == 0) at = atomicAdd(&lds.num, (uint32_t)__popcll(m));
        at = (uint32_t)__builtin_amdgcn_readfirstlane((int)at) + __popcll(m & ((1ull << lane) - 1));
      }
      if (is) list[at] = x[e];
    }
    __syncthreads();
    const int num = (int)lds.num;
    if (num <= kWave) {
      if (wave == 0) sort_by_wave(list, num);
      __syncthreads();
    } else {
      const int size = power_of_two(num);
      for (int i = num + tid; i < size; i += kNT) list[i] = 0;
      sort_falling(list, size);
    }
    return num;
  };

  // ---- top-k: of the last bucket's, as many as it takes; of all, where the buckets end above the cut
  if (n_list > set.k) {
    const uint32_t last = key_of(in.lo) >> 15;
    const bool beyond = in.want == 0;
    gather([&](unsigned long long y) { return beyond || (uint32_t)(y >> 47) == last; });
    const unsigned long long cut = list[(beyond ? (unsigned long long)set.k : in.want) - 1];
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (x[e] < cut) x[e] = 0;
  }
  // ---- weights, min_p, and for top-p their histogram
  const uint32_t base = key_of(in.top) >> 15;
  const bool cut_p = set.top_p < 1.f;
  for (int i = tid; i < kBins; i += kNT) lds.bin[i] = 0;
  for (int i = tid; i < n_chunks; i += kNT) chunk[i] = 0;
  if (tid == 0) lds.kept = 0;
  __syncthreads();
  auto bin_of = [&](unsigned long long y) { return min((int)(base - (uint32_t)(y >> 47)), kBins - 1); };
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (kNT * e >= n_list) break;
    const double z = logit_of(x[e]) == in.top ? 0.0 : ((double)logit_of(x[e]) - (double)in.top) * set.c64;
    w[e] = x[e] ? exp2(z, a.bits) : 0;
    if (cut_p && w[e]) atomicAdd(&lds.bin[bin_of(x[e])], w[e]);
  }
  if (cut_p) {
    __syncthreads();
    unsigned long long sum = 0, total;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (kNT * e < n_list) sum += w[e];
    run_sum(sum, lds.part, &total);
    const unsigned long long goal = share_of(set.top_p, total);
    find_bin(lds, 0, goal);
    const int found = lds.found;
    const int num = gather([&](unsigned long long y) { return bin_of(y) == found; });
    if (wave == 0) {
      unsigned long long before = lds.before, cut = 0;
      for (int i0 = 0; i0 < num && before < goal; i0 += 64) {
        const unsigned long long y = i0 + lane < num ? list[i0 + lane] : 0;
        const double z = logit_of(y) == in.top ? 0.0 : ((double)logit_of(y) - (double)in.top) * set.c64;
        const unsigned long long v = y ? exp2(z, a.bits) : 0, upto = before + scan_wave(v);
        const unsigned long long m = __ballot(y && upto - v < goal);
        if (m) cut = __shfl(y, 63 - __clzll(m), 64);
        before = last_lane(upto);
      }
      if (lane == 0) lds.cut = cut;
    }
    __syncthreads();
    const unsigned long long cut = lds.cut;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (x[e] < cut) x[e] = 0;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (kNT * e >= n_list) break;
    const float v = logit_of(x[e]);
    if (x[e] && !(v == in.top || ((double)v - (double)in.top) * set.c64 >= set.min64)) x[e] = 0;
    const unsigned long long m = __ballot(x[e] != 0);
    if (lane == 0 && m) atomicAdd(&lds.kept, (uint32_t)__popcll(m));
    if (x[e]) atomicAdd(&chunk[id_of(x[e]) / chunk_len], w[e]);
  }
  __syncthreads();
  unsigned long long total, target, before;
  int hit = 0;
  if (wave == 0) {
    hit = find_chunk(chunk, n_chunks, u, &total, &target, &before);
    if (lane == 0) lds.found = hit;
  }
  __syncthreads();
  hit = lds.found;
  // (turned to the order of ids: the lowest id first is the largest number)
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = x[e] ? x[e] << 32 | x[e] >> 32 : 0;
  const int num = gather([&](unsigned long long y) { return (int)((0xFFFFFFFFu - (uint32_t)(y >> 32)) / chunk_len) == hit; });
  if (wave != 0) return;
  for (int i0 = 0; i0 < num; i0 += 64) {
    const unsigned long long y = i0 + lane < num ? list[i0 + lane] : 0;
    const float v = of_key((uint32_t)y);
    const double z = v == in.top ? 0.0 : ((double)v - (double)in.top) * set.c64;
    const unsigned long long w = y ? exp2(z, a.bits) : 0, upto = before + scan_wave(w);
    if (upto > target && upto - w <= target)
      write_row(a, row, (int)(0xFFFFFFFFu - (uint32_t)(y >> 32)), (float)((double)w / (double)total), lds.kept);
    before = last_lane(upto);
  }
}

template <int PER>
__global__ __launch_bounds__(kNT) void k_rows_draw(SampleRowsArgs a) {
  __shared__ __align__(16) unsigned long long list[kList];
  __shared__ __align__(16) unsigned long long chunk[kMostSlices * 16];
  __shared__ double table[64];
  __shared__ RowLds lds;
  __shared__ uint32_t counted;
  constexpr int chunk_len = 64 * PER;
  const int tid = threadIdx.x, lane = tid & 63, row = blockIdx.x;
  const RowSet &set = a.rows[row];
  const RowInfo in = a.info[row];
  exp2_table(table);
  const Exp2 exp2{table};
  // the slices' candidates, one after the other; what a wave copies: every 16th slice's
  const size_t at = (size_t)row * a.slices;
  const int wave = tid >> 6;
  const uint32_t mine = in.state != kNone && in.state != kSlow && lane < a.slices ? ldg<uint32_t>(a.n_list + at + lane) : 0;
  const bool fits = !__any(mine > kSliceList);
  const uint32_t listed = scan_wave(mine), n_list = last_lane(listed);
  if (in.state == kNone) {
    if (tid == 0) write_row(a, row, -1, 0.f, 0);
    return;
  }
  if (in.state == kSlow || !fits || n_list > kList) {
    __syncthreads();  // (the table)
    row_by_ranges(a, exp2, lds, in.state == kSum ? &in : nullptr);
    return;
  }
  const float u = ldg<float>(a.u + row);
  const int n_chunks = a.slices * (kNT / 64);
  uint32_t kept = 0;
  if (in.state == kSum && tid < n_chunks) {
    chunk[tid] = a.chunk[at * (kNT / 64) + tid];
    kept = a.chunk_n[at * (kNT / 64) + tid];
  }
  for (int q = wave; q < a.slices; q += kNT / 64) {
    const int num = __builtin_amdgcn_readlane((int)mine, q), from = __builtin_amdgcn_readlane((int)(listed - mine), q);
    for (int i = lane; i < num; i += 64) list[from + i] = ldg<unsigned long long>(a.list + (at + q) * kSliceList + i);
  }
  if (tid == 0) counted = 0;
  __syncthreads();
  if (in.state == kBest) {
    if (n_list > kWave) {
      draw_many(a, set, row, in, (int)n_list, u, exp2, list, chunk, n_chunks, chunk_len, lds);
    } else if (wave == 0) {
      const int nk = min(set.k, (int)n_list);
      sort_by_wave(list, (int)n_list);
      if (nk <= 64)
        draw_few<1>(a, set, row, in.top, nk, u, exp2, list, list + kWave);
      else
        draw_few<kWave / 64>(a, set, row, in.top, nk, u, exp2, list, list + kWave);
    }
    return;
  }

  // ---- the weights of the chunks, and of the candidates as many as it takes
  kept = sum_wave(kept);
  if (lane == 0 && kept) atomicAdd(&counted, kept);
  if (n_list > kWave) {
    const int size = power_of_two((int)n_list);
    for (int i = (int)n_list + tid; i < size; i += kNT) list[i] = 0;
    sort_falling(list, size);
  } else {
    __syncthreads();
  }
  if (wave != 0) return;
  if (n_list <= kWave) sort_by_wave(list, (int)n_list);
  const double least = least_of(in.ref, set);
  unsigned long long before = 0, cut = ~0ull;
  uint32_t taken = 0;
  for (int i0 = 0; i0 < (int)n_list && before < in.want; i0 += 64) {
    const int i = i0 + lane;
    const unsigned long long x = i < (int)n_list ? list[i] : 0;
    const Place p = place_of(logit_of(x), least, set.c64);
    const unsigned long long w = i < (int)n_list ? weight_of_octave(exp2, p, a.bits) : 0;
    const unsigned long long upto = before + scan_wave(w);
    const bool take = i < (int)n_list && upto - w < in.want;
    if (take) atomicAdd(&chunk[id_of(x) / chunk_len], weight_of(exp2, p, in.ref, a.bits));
    const unsigned long long m = __ballot(take);
    if (m) cut = __shfl(x, 63 - __clzll(m), 64);
    taken += __popcll(m);
    before = last_lane(upto);
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  // ---- the chunk, then the id, at which the running weight passes the target
  unsigned long long total, target;
  const int hit = find_chunk(chunk, n_chunks, u, &total, &target, &before);
  const float *x = a.x + row * a.ld;
  const int id0 = hit * chunk_len + PER * lane;
  float v[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) v[e] = id0 + e < a.n ? ldg<float>(x + id0 + e) : -INFINITY;
  unsigned long long w[PER], sum = 0;
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    w[e] = 0;
    if (v[e] >= in.hi ||
        (v[e] >= in.lo && ((unsigned long long)key_of(v[e]) << 32 | (0xFFFFFFFFu - (uint32_t)(id0 + e))) >= cut))
      w[e] = weight_of(exp2, place_of(v[e], least, set.c64), in.ref, a.bits);
    sum += w[e];
  }
  unsigned long long upto = before + scan_wave(sum) - sum;
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    if (upto <= target && upto + w[e] > target)
      write_row(a, row, id0 + e, (float)((double)w[e] / (double)total), counted + taken);
    upto += w[e];
  }
}

template <int PER>
void launch_slices(const SampleRowsArgs &a, int rows, bool vec, hipStream_t st) {
  const dim3 grid(a.slices, rows), blk(kNT);
  if (vec) {
    hipLaunchKernelGGL((k_rows_scan<PER, true>), grid, blk, 0, st, a);
    hipLaunchKernelGGL((k_rows_pick<PER, true>), grid, blk, 0, st, a);
  } else {
    hipLaunchKernelGGL((k_rows_scan<PER, false>), grid, blk, 0, st, a);
    hipLaunchKernelGGL((k_rows_pick<PER, false>), grid, blk, 0, st, a);
  }
  hipLaunchKernelGGL(k_rows_draw<PER>, dim3(rows), blk, 0, st, a);
}

// Rows of more ids than the slices hold.
__global__ __launch_bounds__(kNT) void k_rows_whole(SampleRowsArgs a) {
  __shared__ double table[64];
  __shared__ RowLds lds;
  exp2_table(table);
  __syncthreads();
  row_by_ranges(a, Exp2{table}, lds, nullptr);
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
  a.bits = kMostBits;
  while (a.bits < 63 && (1 << (63 - a.bits)) < vocab) --a.bits;
  // Slices of 16384 logits where these are as many as compute units, else of 4096.
  const int m0 = rows < kRows ? rows : kRows;
  const bool large = vocab > kMostSlices * 4096 || (long)m0 * cdiv(vocab, 16384) >= ctx().n_cu;
  a.slice = large ? 16384 : 4096;
  a.slices = cdiv(vocab, a.slice);
  const bool sliced = a.slices <= kMostSlices, vec = aligned16(d_logits) && in_stride % 4 == 0;
  if (sliced) {
    const size_t cells = (size_t)m0 * a.slices, chunks = cells * (kNT / 64);
    void *buf = nullptr;
    if (int rc = scratch(cells * ((kBins + 64 + kSliceList) * 8 + 12) + chunks * 16 + m0 * sizeof(RowInfo) + 64, &buf)) return rc;
    a.hist = static_cast<unsigned long long *>(buf);
    a.coarse = a.hist + cells * kBins;
    a.list = a.coarse + cells * 64;
    a.chunk = a.list + cells * kSliceList;
    a.info = reinterpret_cast<RowInfo *>(a.chunk + chunks);
    a.top = reinterpret_cast<float *>(a.info + m0);
    a.real = reinterpret_cast<uint32_t *>(a.top + cells);
    a.n_list = a.real + cells;
    a.chunk_n = a.n_list + cells;
    a.chunk_top = reinterpret_cast<float *>(a.chunk_n + chunks);
  }
  for (int r0 = 0; r0 < rows; r0 += kRows) {
    const int m = rows - r0 < kRows ? rows - r0 : kRows;
    a.x = d_logits + (size_t)r0 * in_stride;
    a.u = d_u + r0;
    a.ids = d_ids + r0;
    a.prob = d_prob ? d_prob + r0 : nullptr;
    a.kept = d_kept ? d_kept + r0 : nullptr;
    for (int r = 0; r < kRows; ++r) {
      const ms_sample_row &w = h_rows[r0 + (r < m ? r : 0)];
      const bool best = w.temperature == 0.f;
      a.rows[r].c64 = best ? 0.0 : 64 * 1.4426950408889634 / (double)w.temperature;
      a.rows[r].by = best ? 0.0 : 1.0 / a.rows[r].c64;
      a.rows[r].min64 = w.min_p > 0.f ? 64 * std::log2((double)w.min_p) : -INFINITY;
      a.rows[r].temperature = w.temperature;
      a.rows[r].top_p = w.top_p;
      a.rows[r].min_p = w.min_p;
      a.rows[r].k = best ? 1 : w.top_k > 0 && w.top_k < vocab ? w.top_k : 0;
    }
    if (!sliced) {
      hipLaunchKernelGGL(k_rows_whole, dim3(m), dim3(kNT), 0, st, a);
    } else {
      if (large)
        launch_slices<16>(a, m, vec, st);
      else
        launch_slices<4>(a, m, vec, st);
    }
    MS_HIP_TRY(hipGetLastError());
  }
  return MS_OK;
}
