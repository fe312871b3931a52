// The paged 4-bit K / V cache as the kernels see it (layout: include/b200_hstu.h).
#pragma once

#include "common.cuh"

namespace b200hstu {

constexpr int PAGED_GROUP = 64;   // values that share a scale

struct PagedCache {
  uint8_t *pages;
  const int32_t *table;
  int64_t num_pages, table_stride;
  int B, H, d, width;
  int page_shift;                 // log2 of the positions of a page

  __host__ __device__ __forceinline__ int page_size() const { return 1 << page_shift; }
  // positions that a sequence can have pages for
  __device__ __forceinline__ int positions() const {
    return (int)min((int64_t)width << page_shift, (int64_t)0x7ffffc00);
  }
  __host__ __device__ __forceinline__ int code_bytes() const { return d >> 1; }                    // of a row
  __host__ __device__ __forceinline__ int scale_bytes() const { return 2 * (d / PAGED_GROUP); }    // of a row
  __host__ __device__ __forceinline__ int64_t page_bytes() const {
    return (int64_t)2 * (code_bytes() + scale_bytes()) << page_shift;
  }
  // Number of the page that position `pos` of sequence b is in; -1 where the sequence has none there or names
  // one outside the pool.
  __device__ __forceinline__ int64_t page_of(int b, int64_t pos) const {
    const int64_t i = pos >> page_shift;
    if (pos < 0 || i >= width) return -1;
    const int32_t p = table[b * table_stride + i];
    return p >= 0 && p < num_pages ? p : -1;
  }
  __device__ __forceinline__ uint8_t *page(int64_t p, int h) const { return pages + (p * H + h) * page_bytes(); }
  // within a page of one head; kv: 0 K, 1 V
  __host__ __device__ __forceinline__ int codes_at(int kv) const { return (kv * code_bytes()) << page_shift; }
  __host__ __device__ __forceinline__ int scales_at(int kv) const {
    return (2 * code_bytes() + kv * scale_bytes()) << page_shift;
  }
};

// What a row sees.  On the mask's clamped ids (common.cuh) the columns of an id below the row's, and those within
// the window, are intervals, so a row at position p sees [lo, hi) and itself.
struct RowSees {
  int lo, hi, self;   // self = -1: a row before the sequence's start, which sees nothing
  __host__ __device__ __forceinline__ bool operator()(int j) const { return (j >= lo && j < hi) || j == self; }
  __host__ __device__ __forceinline__ bool past(int end) const { return (hi > lo && hi > end) || self >= end; }
};
__host__ __device__ __forceinline__ RowSees row_sees(int p, int len, int num_targets, int c, int W) {
  RowSees r{0, 0, p};
  if (p < 0) {
    r.self = -1;
    return r;
  }
  const SeqMask m = make_seq_mask(len, len, num_targets, c, W, 0);
  const int shift = c > 0 ? c - 1 : 0;              // ids above 0 are positions less this
  const int id = m.id(p);
  if (c > 0 && id == 0) {                           // a contextual row sees every id below the last
    r.hi = m.max_id > 0 ? m.max_id + shift : 0;
  } else if (id > 0) {
    r.hi = id + shift;
    if (W > 0 && id > W) r.lo = id - W + shift;
  }
  r.hi = r.hi < len ? r.hi : len;
  return r;
}

int check_paged_cache(const char *what, const b200_hstu_paged_cache &c, PagedCache &out);

}  // namespace b200hstu
