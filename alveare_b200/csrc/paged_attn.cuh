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
// The positions are cut into slices of 16 (a slice never crosses a page: page
// sizes are multiples of 16), four slices to a unit, one for each warp of a
// CTA.  Every warp streams its slices' k and v rows through a private cp.async
// ring (no barrier between warps in the loop) and keeps its own m, l and O in
// registers; the warps' states are joined at the end.  The products run on
// mma.sync m16n8k16: the work is bound by the cache's bytes, and 16 rows are
// all there is to a block.  p is rounded to bf16 for the product with v (the
// tensor core's operand type; the result is rounded to bf16 anyway), l sums
// the unrounded fp32 p.
//
// The units of all blocks (sequence, kv head, 16 rows), in order, are cut into
// equal runs, one per CTA (two CTAs per SM: one joins while the other
// streams).  A block cut between CTAs leaves parts (m, l, O); the CTA that
// finishes last joins them in a fixed order.
#pragma once

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

// The tensor-core form for chunks (paged_chunk.cu): sequences with at least
// row_min rows (new tokens x heads of a kv group).
bool chunk_takes(const AttnArgs& a);
int launch_chunk(alv_ctx* ctx, const AttnArgs& a, int hd, int row_min, cudaStream_t st);

constexpr int kRowsPerBlock = 16;
constexpr int kSlice = 16;
constexpr int kRowWarps = 4;
constexpr int kUnit = kSlice * kRowWarps;  // positions of a unit

// Half-slices (16 rows of k or of v) in a warp's ring: 96 KB over 4 warps.
template <int HD>
struct RowRing {
  static constexpr int kSlots = 96 * 1024 / kRowWarps / (kSlice * HD * 2);
  static constexpr uint32_t kSlotBytes = kSlice * HD * 2;
  static constexpr uint32_t kRingBytes = kRowWarps * kSlots * kSlotBytes;
  static constexpr uint32_t kQBytes = kRowsPerBlock * HD * 2;
  // joining the warps: m and l of every warp and row, then O
  static constexpr uint32_t kJoinBytes = kRowWarps * kRowsPerBlock * (HD + 2) * 4;
  static constexpr uint32_t kBytes = kQBytes + (kRingBytes > kJoinBytes ? kRingBytes : kJoinBytes);
  static constexpr int kPart = kRowsPerBlock * (HD + 2);  // floats of a part: m[16], l[16], O[16][HD]
  // A run is at least kMinUnits, and blocks of up to kWhole units are not cut:
  // joining parts costs about 4 us, a unit a CTA alone about 0.3 us (64-wide
  // heads) to 0.8 us (256-wide).
  static constexpr int kMinUnits = HD == 256 ? 2 : 4;
  static constexpr int kWhole = HD == 256 ? 6 : 12;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t src_bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
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
