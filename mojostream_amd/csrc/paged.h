// Paged KV cache: the batch handle and what its kernels share.
#pragma once
#include <vector>

#include "common.h"

namespace ms {

// The calling thread's current device is the library's while this lives (a
// caller may have made another current).
class OnDevice {
 public:
  OnDevice() {
    if (ctx().device < 0) return;
    if (hipGetDevice(&was_) != hipSuccess) was_ = -1;
    if (was_ != ctx().device) (void)hipSetDevice(ctx().device);
  }
  ~OnDevice() {
    if (was_ >= 0 && was_ != ctx().device) (void)hipSetDevice(was_);
  }

 private:
  int was_ = -1;
};

// A host table and its device copy: fill `h` (after reserve), then send().
struct Upload {
  char *h = nullptr;  // pinned
  char *d = nullptr;
  size_t cap = 0;
  hipEvent_t sent = nullptr;
  int reserve(size_t bytes);  // also waits until the last send() has read `h`
  int send(size_t bytes);
  void release();
};

// Where a new row goes.
struct PagedRow {
  int32_t pos, page, slot, seq;
};

// One block's part of the attention (per kv head): pairs from r0 on (the plan's rows of them) of
// the sequence's new * G (row, query head) pairs, numbered row * G + head, over the
// keys k0 .. k1 - 1.
struct PagedItem {
  int32_t row, n_new, len, seq;  // the sequence: first row, new rows, positions
  int32_t r0, k0, k1;
  int32_t part;  // its place among the parts that are merged, -1: the whole result
};
// Parts part .. part + n - 1 of rows r0.. make one result.
struct PagedMerge {
  int32_t row, n_new, r0, part, n;
};

// A split of the batch's work, for layers of the same shape.
struct PagedPlan {
  int G = 0, rows = 0, n_kv = 0, window = 0, blocks = 0, tile_cost = 0, merge_cost = 0;
  bool block = false;  // items of more than 16 pairs go to item_by_block
  bool valid = false;
  int n_items = 0, n_merge = 0, n_parts = 0;
  int most = 0, most_parts = 0;  // (row, head) pairs of the longest item; parts of one result
  size_t merge_at = 0;  // byte offset of the merge list
  Upload up;
};

}  // namespace ms

struct ms_paged_batch {
  int page_size, n_pages, max_seqs, max_rows, max_pages;
  bool set = false;
  int n_seqs = 0, rows = 0, stride = 0;      // stride: pages per sequence in the device table
  int max_pos = 0;                           // highest position of a new row + 1
  std::vector<int32_t> first, n_new, len;    // per sequence: first row, new rows, positions
  std::vector<int32_t> held;                 // per sequence: first position whose page is there
  std::vector<int64_t> writer;               // per page: the last set() that writes it
  int64_t n_set = 0;
  ms::Upload up;                             // PagedRow [rows], then pages [n_seqs][stride]
  size_t pages_at = 0;
  std::vector<ms::PagedPlan *> plans;
  const ms::PagedRow *d_rows() const { return reinterpret_cast<const ms::PagedRow *>(up.d); }
  const int32_t *d_pages() const { return reinterpret_cast<const int32_t *>(up.d + pages_at); }
};

namespace ms {

// n / d for 0 <= n < 2^31 by a multiplication: (n * mul) >> 31 >> shift.
struct FastDiv {
  uint32_t mul, shift;
};
inline FastDiv fast_div(uint32_t d) {
  uint32_t s = 0;
  while ((1ull << s) < d) ++s;  // 2^s >= d
  // ceil(2^(31 + s) / d) < 2^32 and n * error < 2^(31 + s) for n < 2^31
  return {(uint32_t)(((1ull << (31 + s)) + d - 1) / d), s};
}
__device__ inline uint32_t div_by(uint32_t n, FastDiv f) {
  return (uint32_t)(((uint64_t)n * f.mul) >> 31 >> f.shift);
}

// The layer's shape and pools, and that they fit the batch.
int paged_check(const char *what, const ms_paged_layer *L, const ms_paged_batch *b);
inline int page_rows(const ms_paged_layer *L, const ms_paged_batch *b) {
  return L->page_rows ? L->page_rows : b->page_size;
}
inline size_t kv_bytes(int dtype) { return dtype == MS_KV_F32 ? 4 : 2; }
// Whether `rows` rows of na floats at a and of nb floats at b overlap.
bool rows_overlap(const void *a, size_t stride_a, int na, const void *b, size_t stride_b, int nb,
                  int rows);
inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace ms
