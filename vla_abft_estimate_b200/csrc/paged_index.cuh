// paged_index.cuh - index arithmetic of the paged key-value cache.
//
// Everything that turns lengths, table entries and split numbers (device
// data, which the host cannot check) into offsets goes through here, and is
// plain arithmetic that also runs on the host, where the tests call it.
#pragma once

#include <stdint.h>

namespace abft {

// The part of abft_paged_kv the kernels index with.
struct PagedView {
  void* k_pages;
  void* v_pages;
  int64_t k_page_stride, v_page_stride;  // elements
  const int32_t* page_table;
  int64_t table_stride;
  const int32_t* seq_lens;
  uint32_t* status;
  int32_t num_pages, page_shift, kv_heads, batch, max_pages;
};

// A length as the kernels use it: within [0, max_pages * page_size], which
// is kept below 2^31 by the host's checks.
__host__ __device__ __forceinline__ int paged_clamp_len(int len, int max_pages, int page_shift, bool* bad) {
  const int cap = max_pages << page_shift;
  *bad = len < 0 || len > cap;
  return len < 0 ? 0 : (len > cap ? cap : len);
}

// Element offset of head `head`, slot `slot` of page `page` (rows of
// 2^hd_shift elements); 64-bit throughout, since a pool passes 2^31 elements
// at 4 GB.
__host__ __device__ __forceinline__ int64_t paged_offset(int page, int64_t page_stride, int head, int slot,
                                                         int page_shift, int hd_shift) {
  return static_cast<int64_t>(page) * page_stride +
         ((((static_cast<int64_t>(head)) << page_shift) + slot) << hd_shift);
}

// A sequence's packed rows [begin, end), within [0, tokens] whatever cu holds:
// none when its boundaries fall or lie outside.
__host__ __device__ __forceinline__ void packed_range(const int32_t* cu, int b, int tokens, int* begin, int* end) {
  const int lo = cu[b], hi = cu[b + 1];
  const bool ok = lo >= 0 && lo <= hi && hi <= tokens;
  *begin = ok ? lo : 0;
  *end = ok ? hi : 0;
}

// Tiles [begin, end) of piece `split` when `tiles` tiles are cut into at
// most `splits` pieces of equal size (the last one shorter, later ones empty).
__host__ __device__ __forceinline__ void split_tiles(int tiles, int splits, int split, int* begin, int* end) {
  const int per = (tiles + splits - 1) / splits;
  const int64_t b = static_cast<int64_t>(per) * split;
  *begin = b < tiles ? static_cast<int>(b) : tiles;
  *end = b + per < tiles ? static_cast<int>(b + per) : tiles;
}

// Pieces that are not empty.
__host__ __device__ __forceinline__ int split_count(int tiles, int splits) {
  if (tiles <= 0) return 0;
  const int per = (tiles + splits - 1) / splits;
  return (tiles + per - 1) / per;
}

// `total` tiles dealt to `shares` equal shares (they differ by one tile at
// most): the first tile of share w ...
__host__ __device__ __forceinline__ int share_start(int total, int shares, int w) {
  const int base = total / shares, rest = total - base * shares;
  return w * base + (w < rest ? w : rest);
}
// ... and the share that holds tile u < total.
__host__ __device__ __forceinline__ int share_of(int total, int shares, int u) {
  const int base = total / shares, rest = total - base * shares;
  const int cut = rest * (base + 1);
  return u < cut ? u / (base + 1) : rest + (u - cut) / base;
}

}  // namespace abft
