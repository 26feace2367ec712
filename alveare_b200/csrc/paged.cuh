// Device view of a paged bf16 KV cache and of the ragged batch of new tokens
// that reads it: shared by the q/k norm + rotation + append kernel and the
// attention kernels.
//
// One layer's cache is pages of [kv head][position in page][head_dim], reached
// by strides; sequence b's position j lives in page table[b][j / page_size].
// The batch's new tokens are the last q_start[b+1] - q_start[b] of the
// kv_lens[b] positions of sequence b.  Lengths and tables live in device
// memory, so a launch can be captured in a CUDA graph and replayed while they
// change; every index that comes from them is checked before it is used (a
// bad one is skipped and sets kStatusBadIndex).
#pragma once

#include "common.cuh"

namespace alv {

constexpr int64_t kMaxMapStride = int64_t{1} << 39;  // elements: a tensor map's strides are below 2^40 bytes

struct PagedView {
  uint16_t* k;
  uint16_t* v;
  int64_t page_stride, head_stride, row_stride;  // elements
  int pages, page_size, nkv;
  const int* table;
  int64_t table_stride;
  int table_width;
  const int* q_start;  // [batch + 1]
  const int* kv_lens;  // [batch]
  int batch, tokens;
  uint32_t* status;
};

struct SeqSpan {
  int q0;    // first new token (row of q)
  int qlen;  // new tokens
  int kv;    // positions in the cache, the new tokens' included
};

// Sequence b's span; an inconsistent one is reported and comes back empty.
__device__ __forceinline__ SeqSpan seq_span(const PagedView& p, int b) {
  const int a = p.q_start[b], e = p.q_start[b + 1], n = p.kv_lens[b];
  if (a < 0 || e < a || e > p.tokens || n < 0 ||
      static_cast<int64_t>(n) > static_cast<int64_t>(p.table_width) * p.page_size) {
    atomicOr(p.status, kStatusBadIndex);
    return {0, 0, 0};
  }
  return {a, e - a, n};
}

// The page that holds position j of sequence b, or -1 (reported) if the table
// has no valid page there.
__device__ __forceinline__ int page_of(const PagedView& p, int b, int j) {
  const int page = p.table[static_cast<int64_t>(b) * p.table_stride + j / p.page_size];
  if (page >= 0 && page < p.pages) return page;
  atomicOr(p.status, kStatusBadIndex);
  return -1;
}

}  // namespace alv
