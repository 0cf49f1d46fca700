// What the kernels of the paged KV cache share: page tables and pools.
#pragma once

#include "common.cuh"

namespace sn {
namespace {

// A page table: its entry for a block of page_size positions of stream b, or -1 where there is none.
struct PageMap {
  const int* table;  // [batch, table_stride]
  int64_t table_stride;
  int max_pages, num_pages, page_size;
};
__device__ __forceinline__ int page_of(const PageMap& m, int b, int block) {
  if (block < 0 || block >= m.max_pages) return -1;
  const int pg = m.table[static_cast<int64_t>(b) * m.table_stride + block];
  return static_cast<unsigned>(pg) < static_cast<unsigned>(m.num_pages) ? pg : -1;
}
// Length of a stream, within the page table's reach.
__device__ __forceinline__ int length_of(const PageMap& m, const int* seq_lens, int b) {
  const int n = seq_lens[b];
  const int64_t cap = static_cast<int64_t>(m.max_pages) * m.page_size;
  if (n < 0 || n > cap) {
    record_status(SN_ERR_INVALID_ARGUMENT);
    return n < 0 ? 0 : static_cast<int>(cap);
  }
  return n;
}
// Pages that hold n >= 0 positions (their sum with a page's size fits without a sign only).
__device__ __forceinline__ int pages_of(const PageMap& m, int n) {
  return static_cast<int>((static_cast<unsigned>(n) + static_cast<unsigned>(m.page_size) - 1u) / static_cast<unsigned>(m.page_size));
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
struct PoolStrides {  // elements
  int64_t page, head, tok;
};
inline bool pool_ok(int64_t page, int64_t head, int64_t tok, int nheads, int page_size, int hd) {
  // rows dense, axes in any order but not overlapping below the row
  return tok >= hd && head >= hd && page >= hd && nheads >= 1 && page_size >= 1;
}
inline bool rows16(const void* base, int64_t a, int64_t b, int64_t c) {
  return aligned16(base) && a % 8 == 0 && b % 8 == 0 && c % 8 == 0;
}

// The stream of token t: the last b with cu[b] <= t (binary search).
__device__ __forceinline__ int stream_of(const int* cu, int batch, int t) {
  int lo = 0, hi = batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= t) lo = mid; else hi = mid - 1;
  }
  return lo;
}

}  // namespace
}  // namespace sn
