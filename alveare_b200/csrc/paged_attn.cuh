// Attention of new tokens over a paged cache, for row blocks of up to 16
// query rows (a row = one query head of one new token; the heads of a kv
// group share its keys, so they share a block).
//
//   o_r = sum_j p_rj v_j,   p_r = softmax_j(scale q_r . k_j)   over visible j:
//   j <= pos_r and (no window, or j > pos_r - window, or j < sinks)
//
// One pass with a running maximum m and sum l (base 2, fp32):
//   m' = max(m, max_j s_j),  l' = l 2^(m-m') + sum_j 2^(s_j-m'),
//   O' = O 2^(m-m') + sum_j 2^(s_j-m') v_j
// The positions are cut into slices of 32 (16 for 256-wide heads), four slices
// to a unit, one for each warp of a CTA.  Every warp streams its slices' k and
// v rows through a private ring of tensor copies (128-byte swizzle; no barrier
// between warps in the loop) and keeps its own m, l and O in registers; the
// warps' states are joined at the end.  The products run on mma.sync
// m16n8k16: the work is bound by the cache's bytes, and 16 rows are all there
// is to a block.  p is rounded to bf16 for the product with v (the tensor
// core's operand type; the result is rounded to bf16 anyway), l sums the
// unrounded fp32 p.
//
// The blocks (sequence, kv head, 16 rows), in order, are laid end to end, each
// as long as its units and a few more for what a block costs by itself, and
// cut into equal runs, one per CTA (two CTAs per SM: one joins while the other
// streams).  A block cut between CTAs leaves parts (m, l, O); the CTA that
// finishes last joins them in a fixed order.
//
// Bound: the cache's bytes.  64 sequences' next tokens, 200 to 9,000 positions
// each, 32 heads over 8 of 128 (538 MB of cache): 98.6 us, 5.46 TB/s, 85% of
// the rate of a plain copy; 32 over 8 heads of 256 in a window of 1,024 with 4
// first tokens (269 MB): 49 us, 5.48 TB/s.  One sequence at 331 positions: 10.1
// us called from the host, no bytes to speak of: launch, look-ups, one fetch
// from memory, join.
#pragma once

#include <cuda.h>

#include "internal.h"
#include "paged.cuh"

namespace alv {

struct AttnArgs {
  PagedView c;
  const uint16_t* q;
  int64_t q_tok, q_head;  // elements
  uint16_t* out;
  int64_t o_tok, o_head;
  int nq, group;
  int window, sinks;      // window 0: none
  float scale_log2;       // scale * log2(e)
  int row_max;            // row-block kernel: sequences with more rows are not its
};

// The tensor-core form's tile, and what an item counts beyond its tiles.
template <int HD>
struct ChunkTile {
  static constexpr int kBN = HD == 256 ? 64 : 128, kExtra = 256 / kBN;
};
// Whether it takes a mixed batch's short sequences too (`length`: of their
// items, one per kv head): up to six tiles per CTA, 6 to 8 us, where the
// row-block kernel beside it adds some 15 us for however little (start, one
// fetch from memory, join).  13 sequences of 1 to 517 new tokens, three of them
// single: 98 us with both kernels, 86 with one.
__device__ __forceinline__ bool chunk_takes_few(int64_t length, int ctas) { return length <= 6ll * ctas; }

// The tensor-core form for chunks (paged_chunk.cu): sequences with at least
// row_min rows (new tokens x heads of a kv group).  mixed: the row-block
// kernel for the others is launched between it and its join (without it
// row_min is 1: every sequence is somebody's).
bool chunk_takes(const AttnArgs& a);
int launch_chunk(alv_ctx* ctx, const AttnArgs& a, int hd, int max_q_len, int row_min, bool mixed, cudaStream_t st);
// The row-block kernel (paged_attn.cu); its scratch starts at byte `scratch`
// of the context's work area.  early: it does not wait for the kernel before
// it, only ends after it.
size_t rows_scratch(alv_ctx* ctx, int hd);
int launch_rows(alv_ctx* ctx, const AttnArgs& a, int hd, size_t scratch, bool early, cudaStream_t st);

constexpr int kRowsPerBlock = 16;
constexpr int kRowWarps = 4;

template <int HD>
struct RowRing {
  static constexpr int kSlice = HD == 256 ? 16 : 32;  // positions
  // half-slices (k or v rows of a slice) in a warp's ring: 96 KB over 4 warps
  static constexpr uint32_t kSlotBytes = kSlice * HD * 2;
  static constexpr int kSlots = 96 * 1024 / kRowWarps / kSlotBytes;
  static constexpr uint32_t kRingBytes = kRowWarps * kSlots * kSlotBytes;
  static constexpr uint32_t kQBytes = kRowsPerBlock * HD * 2;
  // joining the warps: m and l of every warp and row, then O
  static constexpr uint32_t kJoinBytes = kRowWarps * kRowsPerBlock * (HD + 2) * 4;
  static constexpr uint32_t kBytes = kQBytes + (kRingBytes > kJoinBytes ? kRingBytes : kJoinBytes) + 1024;
  static constexpr int kPart = kRowsPerBlock * (HD + 2);  // floats of a part: m[16], l[16], O[16][HD]
  // A unit is 32 KB (64-wide heads) or 64 KB of cache, 1.5 or 3 us of a CTA's
  // share of the memory; starting and joining a block takes about 3 us, so a
  // block counts kExtra units more.  A run is at least kMinUnits, and blocks
  // of up to kWhole units are not cut: joining parts costs another 4 us.
  static constexpr int kExtra = HD == 64 ? 2 : 1;
  static constexpr int kMinUnits = 2;
  static constexpr int kWhole = 6;
};

__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
// 2^x (x <= 0 here; -inf gives 0).
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf2_rn(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ bool bf2_nonfinite(uint32_t x) {
  return (x & 0x7F80u) == 0x7F80u || (x & 0x7F800000u) == 0x7F800000u;
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
          dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
      : "memory");
}
// Tensor maps of a layer's k and v pages with boxes of 64 dims x `box`
// positions; *head_first: the map's order is (dim, head, row, page) instead of
// (dim, row, head, page).
int encode_cache(alv_ctx* ctx, const PagedView& c, int hd, int box, CUtensorMap* kmap, CUtensorMap* vmap, int* head_first);
// The largest power of two that divides page sizes, at most `most`.
inline int box_rows(int page_size, int most) {
  int b = 16;
  while (b < most && page_size % (2 * b) == 0) b *= 2;
  return b;
}

// Which positions a row at position `pos` sees.
__device__ __forceinline__ bool sees(int j, int pos, int window, int sinks) {
  return j <= pos && (window == 0 || j > pos - window || j < sinks);
}

// x * y / z for x < 2^40 and y, z <= 2^16: in 32 bits where it fits.
__device__ __forceinline__ int64_t mul_div(int64_t x, int y, int z) {
  if (x < (1 << 21) && y < (1 << 10)) return static_cast<uint32_t>(x) * static_cast<uint32_t>(y) / static_cast<uint32_t>(z);
  return x * y / z;
}

// The slices that any row at positions [p0, p1] sees: [0, n_sink) and
// [first, first + n_main), with [0, n_sink) ending at or before `first`.
struct SliceRange {
  int n_sink, first, n_main;
  int lo, hi;  // visible to some row: j < hi and (j >= lo or j < sinks)
  __device__ __forceinline__ int count() const { return n_sink + n_main; }
  __device__ __forceinline__ int slice(int i) const { return i < n_sink ? i : first + (i - n_sink); }
};
template <int TILE>
__device__ __forceinline__ SliceRange slice_range(int p0, int p1, int window, int sinks) {
  SliceRange r{0, 0, 0, 0, 0};
  if (p1 < 0) return r;
  r.hi = p1 + 1;
  r.lo = window == 0 || p0 < window ? 0 : p0 - window + 1;
  r.first = r.lo / TILE;
  r.n_main = (p1 / TILE + 1) - r.first;
  const int seen = sinks < r.lo ? sinks : r.lo;
  const int ns = seen / TILE + (seen % TILE != 0);
  r.n_sink = ns < r.first ? ns : r.first;
  return r;
}

}  // namespace alv
