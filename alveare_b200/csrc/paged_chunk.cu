// Attention of chunks of new tokens over a paged cache on the tensor cores
// (tcgen05, TMEM).  Same mathematics as paged_attn.cuh, tiles of 128 query
// rows (tokens x the heads of a kv group) against tiles of BN positions:
//
//   S = Q K^T          tcgen05.mma, Q and K tiles in shared memory, S in TMEM
//   P = 2^(S c - m)    softmax warps: two threads per row, half of its columns
//                      each, TMEM -> registers; P goes back to TMEM as bf16
//                      over S's own columns
//   O += P V           tcgen05.mma with P from TMEM, O stays in TMEM
//
// Head sizes 64 and 128: two query tiles per CTA (TMEM: 2 x (S 128 + O HD)
// columns), each with its own softmax warps, so the tensor cores work for one
// tile while the other's softmax runs.  Head size 256: O alone takes 256
// columns, so one query tile with two S buffers of 64 positions.
//
// The running maximum only moves when a row's new maximum exceeds the one in
// use by 2^8 (p stays below 2^8 then, exact in fp32 sums and in range of
// bf16), so O is rescaled in TMEM on the first few tiles and hardly ever
// after; rows take p = 2^(s - m) of whatever m they use, and l sums the same.
//
// Work: the items (sequence, query tiles, kv head), in order, are laid end to
// end, each as long as its tiles and a few more for what an item costs by
// itself, and cut into equal runs, one per CTA, so that a short chunk over a
// long past fills the GPU and ragged batches balance; an item cut between CTAs
// leaves unnormalised parts (O, m, l) that a second launch joins in a fixed
// order.  (Joined instead by the CTA that finishes last, as the row blocks are,
// the parts cost 5 us more at 64-wide heads and 25 at 256: one CTA at the end
// against all of them.)
//
// Bound: the special-function unit and the tensor cores about alike.  A tile
// pair of 256 rows x 128 positions of 128-wide heads is 1.1 us of products and
// 0.85 of exponentials (a quarter of them on the FMA pipe) and takes 2.2 with
// the power limit reached, 1.9 before: neither pipe is full (57 and 43 %), since
// P V of a tile waits for all of its P and only the other query tile's work
// fills the time.  2,048 tokens of 32 heads over 16,001 positions (503 GFLOP):
// 517 to 534 us back to back by GPU, 944 to 972 TFLOP/s, and 445 us, 1130
// TFLOP/s, when the GPU rests between calls.  64-wide heads do half the
// products for the same exponentials: 1.55 us a pair.  256-wide: one query tile
// of 128 rows, each 64 positions 1.35 us against 0.55 of products: nothing
// covers the softmax's latency but the product before, and the k and v of a
// tile (64 KB) come out of L2 for 128 rows only.  Short batches also pay 7 to 9
// us until the first scores (start, look-ups, first fetch) and 8 to 12 for the
// join.
#include <cuda.h>

#include "gemm_tc.cuh"
#include "internal.h"
#include "paged_attn.cuh"

namespace alv {
namespace {

int encode(alv_ctx* ctx, CUtensorMap* map, uint32_t rank, const void* p, const cuuint64_t* dims, const cuuint64_t* strides,
           const cuuint32_t* box) {
  EncodeTiledFn enc = nullptr;
  int rc = tensor_map_encoder(ctx, &enc);
  if (rc) return rc;
  const cuuint32_t one[4] = {1, 1, 1, 1};
  const CUresult cr = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(p), dims, strides, box, one,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (cr != CUDA_SUCCESS)
    return fail(ctx, ALV_ERR_CUDA, "paged_attention: cuTensorMapEncodeTiled failed (" + std::to_string(cr) + ")");
  return ALV_OK;
}

constexpr int kChunkRows = 128;

template <int HD>
struct Chunk {
  static constexpr int kNQ = HD == 256 ? 1 : 2;    // query tiles per item
  static constexpr int kBN = HD == 256 ? 64 : 128; // positions per tile
  static constexpr int kSB = HD == 256 ? 2 : 1;    // S buffers per query tile
  static constexpr int kStages = HD == 64 ? 3 : 2; // K and V stages each
  static constexpr uint32_t kQTile = kChunkRows * HD * 2;
  static constexpr uint32_t kKV = kBN * HD * 2;
  static constexpr uint32_t kBytes = kNQ * kQTile + 2 * kStages * kKV + 1024;
  static constexpr int kHalf = kBN / 2;            // columns of S a softmax thread takes
  // a CTA's run at least (a part costs about as much as 256 positions), and what
  // an item counts for its start and end (query tile, first scores, store)
  static constexpr int kMinRun = 512 / kBN, kExtra = 256 / kBN;
  static_assert(kBN == ChunkTile<HD>::kBN && kExtra == ChunkTile<HD>::kExtra, "the row-block kernel counts the same");
  static constexpr int kSoftWarps = 8 * kNQ;
  static constexpr int kThreads = (kSoftWarps + 4) * 32;  // + copy, issue and two scan warps
  static constexpr uint32_t kSCol = 0;      // S (and P) of tile q, buffer b: (q + b) * kBN
  static constexpr uint32_t kOCol = 256;    // O of tile q: 256 + q * HD
};

struct ChunkArgs {
  AttnArgs a;
  int tpt;        // tokens per query tile: 128 / group
  int box;        // positions per tensor copy
  int head_first; // cache tensor map order: (hd, head, row, page) instead of (hd, row, head, page)
  int row_min;    // sequences with at least this many rows are this kernel's in any case
  float* parts;   // [2 * grid][kNQ * 128][HD + 2]
  int4* cuts;     // [grid]: item (b, pair, kvh) that the run starts inside, and where (x = -1: none)
  int64_t* total; // [2] length of all items; rows of the shortest sequence taken
  int max_pairs;  // query-tile pairs of the longest sequence
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
// D[tmem] (+)= A[tmem] B[smem]
__device__ __forceinline__ void umma_bf16_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Shared-memory descriptor of an operand whose M/N index is contiguous
// (128-byte swizzle): 64 values per 128-byte row, rows along K; `chunk` bytes
// from one 64-value column to the next, 1024 bytes from 8 rows to the next 8.
__device__ __forceinline__ uint64_t umma_desc_mn_sw128(uint32_t saddr, uint32_t chunk) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(chunk >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
#define ALV_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define ALV_I8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
// 32 consecutive columns of this thread's TMEM lane (complete after tmem_wait_ld).
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : ALV_R8(r, 0), ALV_R8(r, 8), ALV_R8(r, 16), ALV_R8(r, 24)
      : "r"(addr));
}
__device__ __forceinline__ void tmem_ld16u(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : ALV_R8(r, 0), ALV_R8(r, 8)
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::ALV_I8(r, 0),
      ALV_I8(r, 8), "r"(addr)
      : "memory");
}
#undef ALV_R8
#undef ALV_I8
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// True in one lane of the (converged) warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
// NaN if one of them is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Two fp32 values in a register pair.
__device__ __forceinline__ uint64_t pack_f2(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ float lo_f2(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float hi_f2(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }
__device__ __forceinline__ uint64_t fma_f2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add_f2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// The lowest n bits.
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1; }
// Scores of 32 columns that the row does not see (it sees e <= hi with e > lo
// or e < sinks) -> -inf.
__device__ __forceinline__ void mask32(uint32_t (&s)[32], int hi, int lo, int sinks) {
  const uint32_t seen = low_bits(hi + 1) & (~low_bits(lo + 1) | low_bits(sinks));
#pragma unroll
  for (int e = 0; e < 32; ++e)
    if (!(seen & (1u << e))) s[e] = 0xFF800000u;
}
// 2^x of two values x >= -126 on the FMA pipe: x = n + f with n the nearest
// integer (the low bits of x + 1.5 2^23), 2^f by the cubic of least relative
// error on [-1/2, 1/2] (7.5e-5: a fiftieth of p's rounding to bf16; the fp32 sum
// l adds the same p, so the output is off by no more than that), n added to
// the exponent.  (Of NaN it gives any number: the row's maximum sees to that.)
__device__ __forceinline__ uint64_t exp2_poly2(uint64_t x) {
  const uint64_t magic = pack_f2(12582912.f, 12582912.f), minus_magic = pack_f2(-12582912.f, -12582912.f);
  const uint64_t r = add_f2(x, magic);
  const uint64_t f = fma_f2(add_f2(r, minus_magic), pack_f2(-1.f, -1.f), x);
  uint64_t p = fma_f2(pack_f2(0.05517167f, 0.05517167f), f, pack_f2(0.24261113f, 0.24261113f));
  p = fma_f2(p, f, pack_f2(0.69326097f, 0.69326097f));
  p = fma_f2(p, f, pack_f2(0.99992806f, 0.99992806f));
  const uint32_t lo = static_cast<uint32_t>(p) + (static_cast<uint32_t>(r) << 23);
  const uint32_t hi = static_cast<uint32_t>(p >> 32) + (static_cast<uint32_t>(r >> 32) << 23);
  return static_cast<uint64_t>(lo) | static_cast<uint64_t>(hi) << 32;
}
// p = 2^(s scale - m) of 32 scores, added to the sums, as 16 packed bf16 pairs
// in s[0 .. 16).  Where every score counts (POLY) a quarter of the
// exponentials goes to the FMA pipe: the special-function unit's 16 a cycle
// are as scarce as the tensor cores' cycles (2,048 tokens over 16,001 positions
// of 128: 455 us, none there 480; of 256-wide heads, which wait for one tile's
// softmax, none is better: 78.5 us against 80 for three windowed chunks).
template <bool POLY>
__device__ __forceinline__ void probs32(uint32_t (&s)[32], uint64_t scale2, uint64_t sub2, uint64_t (&sum)[2]) {
#pragma unroll
  for (int e = 0; e < 32; e += 2) {
    const uint64_t x = fma_f2(pack_f2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), scale2, sub2);
    uint64_t p;
    if (POLY && e % 8 == 6) p = exp2_poly2(pack_f2(fmaxf(lo_f2(x), -126.f), fmaxf(hi_f2(x), -126.f)));
    else p = pack_f2(exp2_fast(lo_f2(x)), exp2_fast(hi_f2(x)));
    sum[e / 2 & 1] = add_f2(sum[e / 2 & 1], p);
    s[e / 2] = pack_bf2_rn(lo_f2(p), hi_f2(p));
  }
}

// Items (b, pair, kvh) in order, kv heads fastest.
template <int HD>
struct Walk {
  using C = Chunk<HD>;
  int b, pair, kvh, pairs;
  SeqSpan s;
  SliceRange r;      // tiles of the current item
  int p0, p1;        // positions of the item's first and last new token
  int row_min;       // sequences of fewer rows are left out

  __device__ __forceinline__ void load(const ChunkArgs& c) {
    p0 = s.kv - s.qlen + pair * C::kNQ * c.tpt;
    p1 = min(p0 + C::kNQ * c.tpt, s.kv) - 1;
    r = slice_range<C::kBN>(p0, p1, c.a.window, c.a.sinks);
    // an item that sees nothing still has one (masked) tile: it writes zeros
    if (r.count() == 0) r.n_main = 1;
  }
  __device__ __forceinline__ int pairs_of(const ChunkArgs& c) const {
    if (s.qlen <= 0 || static_cast<int64_t>(s.qlen) * c.a.group < row_min) return 0;
    return min((s.qlen + C::kNQ * c.tpt - 1) / (C::kNQ * c.tpt), c.max_pairs);
  }
  // Sequence and pair number e of batch x max_pairs; false where there is none.
  __device__ __forceinline__ bool at(const ChunkArgs& c, int64_t e) {
    b = e <= INT_MAX ? static_cast<int>(static_cast<uint32_t>(e) / static_cast<uint32_t>(c.max_pairs))
                     : static_cast<int>(e / c.max_pairs);
    pair = static_cast<int>(e - static_cast<int64_t>(b) * c.max_pairs);
    kvh = 0;
    s = seq_span(c.a.c, b);
    pairs = pairs_of(c);
    if (pair >= pairs) return false;
    load(c);
    return true;
  }
  __device__ __forceinline__ int length() const { return r.count() + C::kExtra; }
  __device__ __forceinline__ void next(const ChunkArgs& c) {
    if (++kvh < c.a.c.nkv) return;
    kvh = 0;
    if (++pair == pairs) {
      pair = 0;
      do {
        if (++b >= c.a.c.batch) return;
        s = seq_span(c.a.c, b);
        pairs = pairs_of(c);
      } while (pairs == 0);
    }
    load(c);
  }
  // The next item of the run [u, u1), at place x of the current one, of which
  // tiles [t, t + n) are this run's; false at the run's end.  After each item
  // the caller moves on with next() if u < u1.
  __device__ __forceinline__ bool take(const ChunkArgs& c, int64_t& u, int64_t u1, int& x, int& t, int& n) {
    while (u < u1) {
      const int len = length();
      t = max(0, x - C::kExtra);
      n = max(0, static_cast<int>(min(static_cast<int64_t>(len), x + (u1 - u))) - C::kExtra) - t;
      u += len - x;
      x = 0;
      if (n > 0) return true;
      if (u < u1) next(c);
    }
    return false;
  }
};
// CTAs that get a run, and the run that holds a place: the last c with total * c / g <= place.
__device__ __forceinline__ int runs_of(int64_t total, int min_run, int grid) {
  return static_cast<int>(min((total + min_run - 1) / min_run, static_cast<int64_t>(grid)));
}
__device__ __forceinline__ int run_of(int64_t place, int64_t total, int g) {
  return static_cast<int>(((place + 1) * g - 1) / total);
}

template <int HD>
struct ChunkShared {
  using C = Chunk<HD>;
  uint64_t kfull[C::kStages], kempty[C::kStages], vfull[C::kStages], vempty[C::kStages], vscan[C::kStages];
  uint64_t qfull, qempty, sfull[C::kNQ][C::kSB], pfull[C::kNQ][C::kSB], odone[C::kNQ], pvdone;
  uint32_t tmem;
  volatile uint32_t failed;  // a wait gave up: report, wait no more, run to the end
  float mx[C::kNQ][2][2][kChunkRows];  // a row's maximum over each half, two tiles deep
  float lx[C::kNQ][2][kChunkRows];
  Walk<HD> walk[C::kSoftWarps];  // each softmax warp's place (its registers hold scores)
  // i + 1 of the run's last item i so far with v values that are not finite in
  // a tile that only some rows see whole; it never goes back.  An item's store
  // adds such values if it is this item or an earlier one: the scan may be any
  // number of items ahead of it, and an item without them has none to add.
  uint32_t odd;
  // the CTA's run
  int64_t sums[C::kThreads / 32], few[C::kThreads / 32];
  int64_t u0, u1;
  int64_t start_e;     // batch x pair number the run starts in
  int64_t start_rest;  // and how far into its kv heads' items
};

// A CTA's part of a cut item: m, l of the rows of a query tile, then O as
// [dims / 4][row][4].  Slot 0: the item its run starts inside, 1: the one it
// ends inside.
__device__ __forceinline__ float* part_of(const ChunkArgs& c, int cta, int slot, int floats) {
  return c.parts + (static_cast<int64_t>(cta) * 2 + slot) * floats;
}

// Whether every row of the item sees the whole tile of positions j0 ...
template <int HD>
__device__ __forceinline__ bool sees_all(const AttnArgs& a, const Walk<HD>& w, int j0) {
  constexpr int BN = Chunk<HD>::kBN;
  return j0 + BN - 1 <= w.p0 && (a.window == 0 || j0 > w.p1 - a.window || j0 + BN <= a.sinks);
}

// Add to 32 of a row's sums the values that are not finite and were left out
// of its products: those it sees in tiles that not every row sees whole.
template <int HD>
__device__ __forceinline__ void add_odd(const ChunkArgs& c, const Walk<HD>& w, int t0, int t1, int pos, int d0, uint32_t (&o)[32]) {
  for (int t = t0; t < t1; ++t) {
    const int j0 = w.r.slice(t) * Chunk<HD>::kBN;
    if (sees_all(c.a, w, j0)) continue;
    for (int j = j0; j < j0 + Chunk<HD>::kBN; ++j) {
      if (!sees(j, pos, c.a.window, c.a.sinks)) continue;
      const int page = page_of(c.a.c, w.b, j);
      if (page < 0) continue;
      const uint16_t* v = c.a.c.v + page * c.a.c.page_stride + w.kvh * c.a.c.head_stride +
                          (j % c.a.c.page_size) * c.a.c.row_stride + d0;
#pragma unroll
      for (int x = 0; x < 32; ++x)
        if ((v[x] & 0x7F80u) == 0x7F80u) o[x] = __float_as_uint(__uint_as_float(o[x]) + bf16_bits_to_f32(v[x]));
    }
  }
}

template <int HD>
__global__ void __launch_bounds__(Chunk<HD>::kThreads, 1)
    paged_chunk_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                       const __grid_constant__ CUtensorMap vmap, const ChunkArgs c) {
  using C = Chunk<HD>;
  constexpr int NQ = C::kNQ, BN = C::kBN, ST = C::kStages;
  extern __shared__ uint8_t smem_dyn[];
  __shared__ ChunkShared<HD> sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t base = (smem_u32(smem_dyn) + 1023u) & ~1023u;
  const uint32_t q_sm = base, k_sm = base + NQ * C::kQTile, v_sm = k_sm + ST * C::kKV;

  if (threadIdx.x == 0) {
    prefetch_map(&qmap);
    prefetch_map(&kmap);
    prefetch_map(&vmap);
    for (int i = 0; i < ST; ++i) {
      mbar_init(&sh.kfull[i], 1);
      mbar_init(&sh.kempty[i], 1);
      mbar_init(&sh.vfull[i], 1);
      mbar_init(&sh.vempty[i], 1);
      mbar_init(&sh.vscan[i], 2);
    }
    mbar_init(&sh.qfull, 1);
    mbar_init(&sh.qempty, 1);
    for (int q = 0; q < NQ; ++q) {
      for (int i = 0; i < C::kSB; ++i) {
        mbar_init(&sh.sfull[q][i], 1);
        // per S buffer: with two, a warp may be a tile ahead of its fellows
        mbar_init(&sh.pfull[q][i], 8);
      }
      mbar_init(&sh.odone[q], 1);
    }
    mbar_init(&sh.pvdone, 1);
    fence_mbar_init();
    sh.failed = 0;
    sh.odd = 0;
  }
  // query rows past tpt * group are never loaded: keep them zero
  for (uint32_t i = threadIdx.x; i < NQ * C::kQTile / 16; i += C::kThreads)
    *reinterpret_cast<uint4*>(smem_dyn + (base - smem_u32(smem_dyn)) + i * 16) = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();

  // The row-block kernel of a mixed batch may start where this one's CTAs end.
  pdl_wait();
  pdl_trigger();
  // ---- the CTA's run: thread t adds up the lengths of its sequences and
  // pairs, a scan over the threads finds where the run starts
  Walk<HD> w{};
  w.row_min = 1;
  const int64_t n_e = static_cast<int64_t>(c.a.c.batch) * c.max_pairs, per = (n_e + C::kThreads - 1) / C::kThreads;
  const int64_t e0 = threadIdx.x * per, e1 = min(e0 + per, n_e);
  int64_t mine = 0, few = 0;  // few: of the sequences short enough for row blocks
  for (int64_t e = e0; e < e1; ++e)
    if (w.at(c, e)) (w.s.qlen * static_cast<int64_t>(c.a.group) < c.row_min ? few : mine) += static_cast<int64_t>(w.length()) * c.a.c.nkv;
  int64_t incl = mine, incl_few = few;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, incl, o), z = __shfl_up_sync(0xffffffffu, incl_few, o);
    if (lane >= o) incl += y, incl_few += z;
  }
  if (lane == 31) sh.sums[warp] = incl, sh.few[warp] = incl_few;
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  __syncthreads();
  int64_t before = incl - mine, total = 0, before_few = incl_few - few, total_few = 0;
  for (int i = 0; i < C::kThreads / 32; ++i) {
    if (i < warp) before += sh.sums[i], before_few += sh.few[i];
    total += sh.sums[i];
    total_few += sh.few[i];
  }
  w.row_min = c.row_min;
  if (chunk_takes_few(total_few, gridDim.x)) {
    w.row_min = 1;
    mine += few;
    before += before_few;
    total += total_few;
  }
  const int g = runs_of(total, C::kMinRun, gridDim.x);
  const int64_t u0 = static_cast<int>(blockIdx.x) < g ? mul_div(total, blockIdx.x, g) : total;
  const int64_t u1 = static_cast<int>(blockIdx.x) < g ? mul_div(total, blockIdx.x + 1, g) : total;
  if (blockIdx.x == 0 && threadIdx.x == 0) c.total[0] = total, c.total[1] = w.row_min;
  if (u0 < u1 && before <= u0 && u0 < before + mine) {  // this thread's range holds the start
    int64_t at = before;
    for (int64_t e = e0; e < e1; ++e) {
      if (!w.at(c, e)) continue;
      const int64_t len = static_cast<int64_t>(w.length()) * c.a.c.nkv;
      if (u0 < at + len) {
        sh.start_e = e;
        sh.start_rest = u0 - at;
        break;
      }
      at += len;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;

  int x0 = 0;  // where the run starts inside its first item
  if (u0 < u1) {
    w.at(c, sh.start_e);
    w.kvh = static_cast<int>(sh.start_rest) / w.length();
    x0 = static_cast<int>(sh.start_rest) - w.kvh * w.length();
  }
  if (threadIdx.x == 0)
    c.cuts[blockIdx.x] = x0 > C::kExtra ? make_int4(w.b, w.pair, w.kvh, x0) : make_int4(-1, 0, 0, 0);
  int64_t u = u0;
  int x = x0, t = 0, n = 0;

  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (mbar_try_wait_s(smem_u32(bar), parity) || sh.failed || mbar_wait_bounded_slow(smem_u32(bar), parity)) return;
    atomicOr(c.a.c.status, kStatusMbarTimeout);
    sh.failed = 1;
  };

  if (warp == C::kSoftWarps) {
    // ---- copies: lane i fetches box i of a tile's k and v.  Tile by tile: k,
    // then v of the tile before (the order the products need them in); the
    // next tile's page is looked up meanwhile.
    const int boxes = BN / c.box;
    uint32_t it = 0, item = 0;
    int i = -1;
    // the tile to come: its first position here, whether some row sees this
    // box (others are not fetched, their pages may be gone), its page
    int j = 0, raw = -1;
    bool live = false;
    auto step = [&]() -> bool {
      if (++i >= n) {
        if (item > 0 && u < u1) w.next(c);
        if (!w.take(c, u, u1, x, t, n)) return false;
        i = 0;
        ++item;
      }
      j = w.r.slice(t + i) * BN + lane * c.box;
      live = lane < boxes && j < w.r.hi && (j + c.box > w.r.lo || j < c.a.sinks);
      raw = live ? c.a.c.table[static_cast<int64_t>(w.b) * c.a.c.table_stride + j / c.a.c.page_size] : -1;
      return true;
    };
    auto fetch = [&](uint32_t k, bool v, uint32_t n_live, bool mine, int page, int row, int kvh) {
      const uint32_t stage = k % ST;
      if (k >= ST) wait(v ? &sh.vempty[stage] : &sh.kempty[stage], ((k / ST) & 1) ^ 1);
      __syncwarp();
      const uint32_t full = smem_u32(v ? &sh.vfull[stage] : &sh.kfull[stage]);
      if (lane == 0) mbar_arrive_expect_tx_s(full, n_live * c.box * HD * 2);
      __syncwarp();
      if (mine) {
        const uint32_t dst = (v ? v_sm : k_sm) + stage * C::kKV + lane * c.box * 128;
        const CUtensorMap* map = v ? &vmap : &kmap;
        for (int d = 0; d < HD / 64; ++d) {
          if (c.head_first) tma_load_4d(dst + d * (BN * 128), map, d * 64, kvh, row, page, full);
          else tma_load_4d(dst + d * (BN * 128), map, d * 64, row, kvh, page, full);
        }
      }
      __syncwarp();
    };
    uint32_t v_live = 0;
    bool v_mine = false;
    int v_page = 0, v_row = 0, v_kvh = 0;
    while (step()) {
      const bool mine = live;
      const uint32_t n_live = __popc(__ballot_sync(0xffffffffu, mine));
      const int row = j % c.a.c.page_size, kvh = w.kvh;
      int page = raw;
      if (page < 0 || page >= c.a.c.pages) {
        if (mine) atomicOr(c.a.c.status, kStatusBadIndex);
        page = c.a.c.pages;  // past the end: the copy reads zeros
      }
      fetch(it, false, n_live, mine, page, row, kvh);
      if (it > 0) fetch(it - 1, true, v_live, v_mine, v_page, v_row, v_kvh);
      ++it;
      if (i == 0) {  // the item's query tiles
        const int tok = w.pair * NQ * c.tpt, nq = NQ == 2 && tok + c.tpt < w.s.qlen ? 2 : 1;
        if (item > 1) wait(&sh.qempty, item & 1);
        __syncwarp();
        if (lane == 0) {
          mbar_arrive_expect_tx(&sh.qfull, nq * c.tpt * c.a.group * HD * 2);
          for (int q = 0; q < nq; ++q)
            for (int d = 0; d < HD / 64; ++d)
              tma_load_3d(q_sm + q * C::kQTile + d * (kChunkRows * 128), &qmap, d * 64, w.kvh * c.a.group,
                          w.s.q0 + tok + q * c.tpt, smem_u32(&sh.qfull));
        }
      }
      v_live = n_live, v_mine = mine, v_page = page, v_row = row, v_kvh = kvh;
    }
    if (it > 0) fetch(it - 1, true, v_live, v_mine, v_page, v_row, v_kvh);
    // every armed stage lands before the CTA may exit
    for (uint32_t k = it > ST ? it - ST : 0; k < it; ++k) {
      mbar_wait_bounded_s(smem_u32(&sh.kfull[k % ST]), (k / ST) & 1);
      mbar_wait_bounded_s(smem_u32(&sh.vfull[k % ST]), (k / ST) & 1);
    }
    if (item > 0) mbar_wait_bounded_s(smem_u32(&sh.qfull), (item - 1) & 1);
  } else if (warp == C::kSoftWarps + 1) {
    // ---- tensor-core issue.  The whole warp walks the run and one lane
    // issues: addresses and counters stay warp-uniform (scalar registers); with
    // one lane in the loop every operand would be moved there one by one, 95
    // cycles an instruction against the 64 it takes.
    const bool leader = elect_one();
    const uint32_t s_idesc = umma_idesc_bf16_f32(kChunkRows, BN);
    const uint32_t o_idesc = umma_idesc_bf16_f32(kChunkRows, HD) | (1u << 16);  // B's N index contiguous
    // stage of K (and of V), phases
    uint32_t ks = 0, kph = 0, vs = 0, vph = 0, item = 0, pph = 0;
    auto qk = [&](int q, int buf) {
      const uint64_t kd = umma_desc_sw128(k_sm + ks * C::kKV), qd = umma_desc_sw128(q_sm + q * C::kQTile);
      const uint32_t d_addr = tmem + C::kSCol + (q + buf) * BN;
      if (leader) {
#pragma unroll
        for (int d = 0; d < HD / 16; ++d)
          umma_bf16(d_addr, qd + (d / 4) * (kChunkRows * 8) + 2 * (d % 4), kd + (d / 4) * (BN * 8) + 2 * (d % 4), s_idesc, d != 0);
        umma_commit(smem_u32(&sh.sfull[q][buf]));
      }
      __syncwarp();
    };
    auto pv = [&](int q, int buf, bool acc) {
      const uint64_t vd = umma_desc_mn_sw128(v_sm + vs * C::kKV, BN * 128);
      const uint32_t d_addr = tmem + C::kOCol + q * HD, p_addr = tmem + C::kSCol + (q + buf) * BN;
      if (leader) {
#pragma unroll
        for (int j = 0; j < BN / 16; ++j)
          umma_bf16_ts(d_addr, p_addr + j / (C::kHalf / 16) * C::kHalf + j % (C::kHalf / 16) * 8, vd + j * 128, o_idesc,
                       acc || j != 0);
      }
      __syncwarp();
    };
    auto commit = [&](uint64_t* bar) {
      if (leader) umma_commit(smem_u32(bar));
      __syncwarp();
    };
    auto next_k = [&] {
      commit(&sh.kempty[ks]);
      if (++ks == ST) ks = 0, kph ^= 1;
    };
    int items = 0;  // of the run: a first walk, so that the loop below is uniform
    for (Walk<HD> w2 = w; w2.take(c, u, u1, x, t, n);) {
      ++items;
      if (u < u1) w2.next(c);
    }
    u = u0;
    x = x0;
    items = __shfl_sync(0xffffffffu, items, 0);
    for (int it = 0; it < items; ++it) {
      w.take(c, u, u1, x, t, n);
      n = __shfl_sync(0xffffffffu, n, 0);
      const int nq = NQ == 1 ? 1 : __shfl_sync(0xffffffffu, w.pair * NQ * c.tpt + c.tpt < w.s.qlen ? 2 : 1, 0);
      wait(&sh.qfull, item & 1);
      wait(&sh.kfull[ks], kph);
      tc_fence_after();
      qk(0, 0);
      if (nq == 2) qk(NQ - 1, 0);
      next_k();
      if (n == 1) commit(&sh.qempty);
      for (int i = 0; i < n; ++i) {
        const bool more = i + 1 < n;
        if (NQ == 1 && more) {  // the next scores before this tile's P V
          wait(&sh.kfull[ks], kph);
          tc_fence_after();
          qk(0, (i + 1) & 1);
          next_k();
          if (i + 2 == n) commit(&sh.qempty);
        }
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          if (q >= nq) break;
          const int buf = C::kSB == 2 ? i & 1 : 0;
          wait(&sh.pfull[q][buf], pph >> (2 * q + buf) & 1);
          if (q == 0) wait(&sh.vscan[vs], vph);  // (it follows the copy's arrival)
          pph ^= 1u << (2 * q + buf);
          tc_fence_after();
          pv(q, buf, i > 0);
          if (NQ == 1) commit(&sh.pvdone);
          if (!more) commit(&sh.odone[q]);
          if (NQ == 2 && more) {
            if (q == 0) wait(&sh.kfull[ks], kph);
            tc_fence_after();
            qk(q, 0);
          }
        }
        commit(&sh.vempty[vs]);
        if (++vs == ST) vs = 0, vph ^= 1;
        if (NQ == 2 && more) {
          next_k();
          if (i + 2 == n) commit(&sh.qempty);
        }
      }
      ++item;
      if (u < u1) w.next(c);
    }
  } else if (warp > C::kSoftWarps + 1) {
    // ---- scan of v.  A row's p is 0 where it does not see, but 0 * inf is not:
    // in tiles that not every row sees whole, zero the v rows no one sees and
    // the values that are not finite (the rows that see those take them in the
    // end).
    uint32_t vs = 0, vph = 0, item = 0;
    while (w.take(c, u, u1, x, t, n)) {
      for (int i = 0; i < n; ++i) {
        const int j0 = w.r.slice(t + i) * BN;
        wait(&sh.vfull[vs], vph);
        __syncwarp();
        if (!sees_all(c.a, w, j0)) {
          const uint32_t v = v_sm + vs * C::kKV;
          bool odd = false;
          for (int r = threadIdx.x - (C::kSoftWarps + 2) * 32; r < BN; r += 64) {  // a thread per row
            const int j = j0 + r;
            auto at = [&](int ch) { return v + (ch / 8) * (BN * 128) + r * 128 + (((ch % 8) ^ (r & 7)) << 4); };
            if (j >= w.r.hi || (j < w.r.lo && j >= c.a.sinks)) {
#pragma unroll 8
              for (int ch = 0; ch < HD / 8; ++ch)
                asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(at(ch)), "r"(0) : "memory");
              continue;
            }
            uint32_t any = 0;  // an exponent of all ones carries into the sign's place
#pragma unroll 8
            for (int ch = 0; ch < HD / 8; ++ch) {
              const uint4 val = lds128_at<0>(at(ch));
              any |= ((val.x & 0x7F807F80u) + 0x00800080u) | ((val.y & 0x7F807F80u) + 0x00800080u) |
                     ((val.z & 0x7F807F80u) + 0x00800080u) | ((val.w & 0x7F807F80u) + 0x00800080u);
            }
            if (!(any & 0x80008000u)) continue;
            odd = true;
            for (int ch = 0; ch < HD / 8; ++ch) {
              const uint4 val = lds128_at<0>(at(ch));
              uint32_t x4[4] = {val.x, val.y, val.z, val.w};
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                if ((x4[y] & 0x7F80u) == 0x7F80u) x4[y] &= 0xFFFF0000u;
                if ((x4[y] & 0x7F800000u) == 0x7F800000u) x4[y] &= 0xFFFFu;
              }
              asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at(ch)), "r"(x4[0]), "r"(x4[1]), "r"(x4[2]), "r"(x4[3])
                           : "memory");
            }
          }
          if (odd) atomicMax(&sh.odd, item + 1);
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (lane == 0) mbar_arrive(&sh.vscan[vs]);
        if (++vs == ST) vs = 0, vph ^= 1;
      }
      ++item;
      if (u < u1) w.next(c);
    }
  } else {
    // ---- softmax: a thread has half of the columns of a row of query tile q
    constexpr int HB = C::kHalf;
    const int q = warp >> 3, half = (warp >> 2) & 1, row = (warp & 3) * 32 + lane;
    const uint32_t lane_addr = tmem + (((warp & 3) * 32) << 16);
    const uint32_t o_addr = lane_addr + C::kOCol + q * HD + half * (HD / 2);
    const float scale = c.a.scale_log2;
    auto both_halves = [&] { asm volatile("bar.sync %0, 256;" ::"r"(1 + q) : "memory"); };
    uint32_t sph = 0, oph = 0, it = 0, item = 0;  // S tiles seen, items stored, tiles and items of the run
    Walk<HD>& sw = sh.walk[warp];  // lane 0 walks
    if (lane == 0) sw = w;
    while (true) {
      int more = 0;
      if (lane == 0) more = sw.take(c, u, u1, x, t, n);
      more = __shfl_sync(0xffffffffu, more, 0);
      t = __shfl_sync(0xffffffffu, t, 0);
      n = __shfl_sync(0xffffffffu, n, 0);
      if (!more) break;
      __syncwarp();
      const int tok0 = (sw.pair * NQ + q) * c.tpt, tok = tok0 + row / c.a.group;
      const bool active = q == 0 || tok0 < sw.s.qlen;
      const bool real = row < c.tpt * c.a.group && tok < sw.s.qlen;
      const int pfirst = sw.s.kv - sw.s.qlen;
      const int pos = real ? pfirst + tok : -1;
      // every row of the item sees the whole tile at j0: j0 <= all_hi and (j0 > all_lo or j0 <= all_sink)
      const int all_hi = sw.p0 - BN + 1, all_lo = c.a.window ? sw.p1 - c.a.window : -1, all_sink = c.a.sinks - BN;
      float m = -INFINITY, l = 0.f;
      for (int i = 0; active && i < n; ++i) {
        const int j0 = sw.r.slice(t + i) * BN;
        const uint32_t buf = C::kSB == 2 ? (i & 1) : 0;
        wait(&sh.sfull[q][buf], C::kSB == 2 ? (sph >> buf) & 1 : sph & 1);
        __syncwarp();
        if (C::kSB == 2) sph ^= 1u << buf;
        else ++sph;
        tc_fence_after();
        const bool whole = j0 <= all_hi && (j0 > all_lo || j0 <= all_sink);
        const uint32_t s_addr = lane_addr + C::kSCol + (q + buf) * BN + half * HB;
        uint32_t sa[32], sb[32];
        tmem_ld32(s_addr, sa);
        if constexpr (HB == 64) tmem_ld32(s_addr + 32, sb);
        tmem_wait_ld();
        if (!whole) {
          const int jh = j0 + half * HB, hi = pos - jh;
          const int lo = c.a.window ? pos - c.a.window - jh : -BN - 1, sk = c.a.window ? c.a.sinks - jh : 0;
          mask32(sa, hi, lo, sk);
          if constexpr (HB == 64) mask32(sb, hi - 32, lo - 32, sk - 32);
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          mx[e / 2 & 1] = max3_nan(mx[e / 2 & 1], __uint_as_float(sa[e]), __uint_as_float(sa[e + 1]));
          if constexpr (HB == 64) mx[2 + (e / 2 & 1)] = max3_nan(mx[2 + (e / 2 & 1)], __uint_as_float(sb[e]), __uint_as_float(sb[e + 1]));
        }
        const float mine = max_nan(max_nan(mx[0], mx[1]), max_nan(mx[2], mx[3]));
        sh.mx[q][i & 1][half][row] = mine;
        both_halves();
        const float mt = max_nan(mine, sh.mx[q][i & 1][half ^ 1][row]) * scale;
        // Also from -inf.  A score that is NaN or +inf leaves the row nothing
        // defined: its maximum becomes NaN, and with it the sum and the output.
        const bool move = !(mt <= m + 8.f);
        if (__any_sync(0xffffffffu, move)) {
          const float f = move ? (m == -INFINITY ? 0.f : exp2_fast(m - mt)) : 1.f;
          if (move) m = mt == INFINITY ? NAN : mt;
          l *= f;
          if (i > 0) {
            if (NQ == 1) {  // O must hold the last product (with two tiles S's arrival says so)
              wait(&sh.pvdone, (it + i - 1) & 1);
              __syncwarp();
              tc_fence_after();
            }
#pragma unroll 1
            for (int e = 0; e < HD / 2; e += 16) {
              uint32_t o[16];
              tmem_ld16u(o_addr + e, o);
              tmem_wait_ld();
#pragma unroll
              for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
              tmem_st16(o_addr + e, o);
            }
          }
        }
        const float sub = m == -INFINITY ? 0.f : m;
        const uint64_t scale2 = pack_f2(scale, scale), sub2 = pack_f2(-sub, -sub);
        uint64_t sum[2] = {};
        if (whole) {
          probs32<HD != 256>(sa, scale2, sub2, sum);
          tmem_st16(s_addr, sa);
          if constexpr (HB == 64) {
            probs32<HD != 256>(sb, scale2, sub2, sum);
            tmem_st16(s_addr + 16, sb);
          }
        } else {
          probs32<false>(sa, scale2, sub2, sum);
          tmem_st16(s_addr, sa);
          if constexpr (HB == 64) {
            probs32<false>(sb, scale2, sub2, sum);
            tmem_st16(s_addr + 16, sb);
          }
        }
        const uint64_t sums = add_f2(sum[0], sum[1]);
        l += lo_f2(sums) + hi_f2(sums);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.pfull[q][buf]);
      }
      // ---- the item's rows (or this CTA's part of them): half of the dims each
      if (active) {
        wait(&sh.odone[q], oph & 1);
        ++oph;
        sh.lx[q][half][row] = l;
        both_halves();
        l = sh.lx[q][0][row] + sh.lx[q][1][row];
        tc_fence_after();
        const bool part = t > 0 || n < sw.r.count();
        const int head = sw.kvh * c.a.group + row % c.a.group;
        uint16_t* dst = !real ? nullptr : c.a.out + static_cast<int64_t>(sw.s.q0 + tok) * c.a.o_tok + head * c.a.o_head + half * (HD / 2);
        float* pd = part_of(c, blockIdx.x, t > 0 ? 0 : 1, NQ * kChunkRows * (HD + 2)) + q * kChunkRows * (HD + 2);
        const bool odd = *const_cast<volatile uint32_t*>(&sh.odd) > item;
        // A row before the first position sees nothing and gives zeros; any other
        // sees itself at least, and with no score above -inf it gives NaN.
        const float inv = pos < 0 ? 0.f : 1.f / l;
        if (part && half == 0) pd[row] = m, pd[kChunkRows + row] = l;
        pd += 2 * kChunkRows + half * (HD / 2) * kChunkRows;
#pragma unroll 1
        for (int e = 0; e < HD / 2; e += 32) {
          uint32_t o[32];
          __syncwarp();
          tmem_ld32(o_addr + e, o);
          tmem_wait_ld();
          if (odd) add_odd<HD>(c, sw, t, t + n, pos, half * (HD / 2) + e, o);
          if (part) {  // [dims / 4][row][4]: a warp writes 512 bytes in a row
#pragma unroll
            for (int y = 0; y < 32; y += 4)
              *reinterpret_cast<uint4*>(pd + (e + y) * kChunkRows + row * 4) = make_uint4(o[y], o[y + 1], o[y + 2], o[y + 3]);
          } else {
            // four lanes exchange the 16-byte quarters of their rows: a store
            // then writes 64 bytes in a row of eight rows, not 16 of 32
            uint32_t p[16];
#pragma unroll
            for (int y = 0; y < 16; ++y)
              p[y] = pack_bf2_rn(__uint_as_float(o[2 * y]) * inv, __uint_as_float(o[2 * y + 1]) * inv);
#pragma unroll
            for (int b = 1; b < 4; b *= 2)
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                if (k & b) continue;
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                  uint32_t &lo = p[4 * k + z], &hi = p[4 * (k | b) + z];
                  const uint32_t got = __shfl_xor_sync(0xffffffffu, lane & b ? lo : hi, b);
                  if (lane & b) lo = got;
                  else hi = got;
                }
              }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              uint16_t* d = reinterpret_cast<uint16_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(dst), (lane & 28) + k));
              if (d) *reinterpret_cast<uint4*>(d + e + 8 * (lane & 3)) = make_uint4(p[4 * k], p[4 * k + 1], p[4 * k + 2], p[4 * k + 3]);
            }
          }
        }
        __syncwarp();
        tc_fence_before();
      }
      it += n;
      ++item;
      __syncwarp();
      if (lane == 0 && u < u1) sw.next(c);
      __syncwarp();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// Join the parts of items cut between CTAs: block (c, y) joins rows 32 y ..
// 32 y + 31 (a lane each) of the item that cut c is the first inside; warps
// take the dims in fours.
template <int HD>
__global__ void __launch_bounds__(256) paged_join_kernel(const ChunkArgs c, int grid) {
  using C = Chunk<HD>;
  constexpr int kFloats = C::kNQ * kChunkRows * (HD + 2), G = HD / 32;  // G: groups of four dims per warp
  pdl_wait();
  const int cut = blockIdx.x + 1;
  const int4 it = c.cuts[cut];
  if (it.x < 0) return;
  const int64_t total = *c.total;
  const int g = runs_of(total, C::kMinRun, grid);
  if (cut >= g) return;
  Walk<HD> w{};
  w.row_min = static_cast<int>(c.total[1]);
  w.at(c, static_cast<int64_t>(it.x) * c.max_pairs + it.y);
  w.kvh = it.z;
  const int64_t first = mul_div(total, cut, g) - it.w + C::kExtra;  // the item's first tile
  const int c0 = run_of(first, total, g), c1 = run_of(first + w.r.count() - 1, total, g);
  if (c0 + 1 != cut) return;  // an earlier cut is inside the item
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int q = blockIdx.y / 4, row = blockIdx.y % 4 * 32 + lane;
  const int tok = (w.pair * C::kNQ + q) * c.tpt + row / c.a.group;
  const bool real = row < c.tpt * c.a.group && tok < w.s.qlen;
  if (!__any_sync(0xffffffffu, real)) return;
  float m = -INFINITY, l = 0.f;
  float4 o[G];
#pragma unroll
  for (int i = 0; i < G; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int cta = c0; cta <= c1; ++cta) {
    const float* p = part_of(c, cta, cta == c0 ? 1 : 0, kFloats) + q * kChunkRows * (HD + 2);
    const float pm = p[row], pl = p[kChunkRows + row];
    float4 v[G];
#pragma unroll
    for (int i = 0; i < G; ++i)
      v[i] = *reinterpret_cast<const float4*>(p + 2 * kChunkRows + ((warp + 8 * i) * kChunkRows + row) * 4);
    const float mn = fmaxf(m, pm), base = mn == -INFINITY ? 0.f : mn;
    const float f0 = exp2_fast(m - base), f1 = exp2_fast(pm - base);
    l = l * f0 + pl * f1;
    m = mn;
#pragma unroll
    for (int i = 0; i < G; ++i) {
      o[i].x = o[i].x * f0 + v[i].x * f1;
      o[i].y = o[i].y * f0 + v[i].y * f1;
      o[i].z = o[i].z * f0 + v[i].z * f1;
      o[i].w = o[i].w * f0 + v[i].w * f1;
    }
  }
  if (!real) return;
  const float inv = w.s.kv - w.s.qlen + tok < 0 ? 0.f : 1.f / l;
  const int head = w.kvh * c.a.group + row % c.a.group;
  uint16_t* dst = c.a.out + static_cast<int64_t>(w.s.q0 + tok) * c.a.o_tok + head * c.a.o_head;
#pragma unroll
  for (int i = 0; i < G; ++i)
    *reinterpret_cast<uint2*>(dst + (warp + 8 * i) * 4) =
        make_uint2(pack_bf2_rn(o[i].x * inv, o[i].y * inv), pack_bf2_rn(o[i].z * inv, o[i].w * inv));
}

template <int HD>
int launch_chunk_t(alv_ctx* ctx, const AttnArgs& a, int max_q_len, int row_min, bool mixed, cudaStream_t st) {
  using C = Chunk<HD>;
  ChunkArgs c{};
  c.a = a;
  c.tpt = kChunkRows / a.group;
  c.row_min = row_min;
  c.max_pairs = (max_q_len + C::kNQ * c.tpt - 1) / (C::kNQ * c.tpt);
  c.box = box_rows(a.c.page_size, C::kBN);
  CUtensorMap qmap, kmap, vmap;
  {
    const cuuint64_t dims[3] = {HD, static_cast<cuuint64_t>(a.nq), static_cast<cuuint64_t>(a.c.tokens)};
    const cuuint64_t str[2] = {static_cast<cuuint64_t>(a.q_head) * 2, static_cast<cuuint64_t>(a.q_tok) * 2};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(a.group), static_cast<cuuint32_t>(c.tpt)};
    const int rc = encode(ctx, &qmap, 3, a.q, dims, str, box);
    if (rc) return rc;
  }
  if (const int rc = encode_cache(ctx, a.c, HD, c.box, &kmap, &vmap, &c.head_first)) return rc;
  const int grid = ctx->num_sms;
  const size_t o_cuts = 256, o_parts = o_cuts + align_up(static_cast<size_t>(grid) * sizeof(int4), 256);
  const size_t o_rows = align_up(o_parts + static_cast<size_t>(grid) * 2 * C::kNQ * kChunkRows * (HD + 2) * 4, 256);
  int rc = ensure_scratch(ctx, o_rows + (mixed ? rows_scratch(ctx, HD) : 0));
  if (rc) return rc;
  c.total = reinterpret_cast<int64_t*>(work_ptr(ctx));
  c.cuts = reinterpret_cast<int4*>(work_ptr(ctx) + o_cuts);
  c.parts = reinterpret_cast<float*>(work_ptr(ctx) + o_parts);
  c.a.c.status = status_ptr(ctx);
  auto k = paged_chunk_kernel<HD>;
  if ((rc = prepare_kernel(ctx, k, C::kBytes))) return rc;
  if ((rc = launch_ex(ctx, k, dim3(grid), dim3(C::kThreads), C::kBytes, st, true, qmap, kmap, vmap, c))) return rc;
  if (mixed && (rc = launch_rows(ctx, a, HD, o_rows, true, st))) return rc;
  if (grid < 2) return ALV_OK;
  return launch_ex(ctx, paged_join_kernel<HD>, dim3(grid - 1, C::kNQ * 4), dim3(256), 0, st, true, c, grid);
}

}  // namespace

int encode_cache(alv_ctx* ctx, const PagedView& c, int hd, int box, CUtensorMap* kmap, CUtensorMap* vmap, int* head_first) {
  const bool hf = c.head_stride < c.row_stride;
  *head_first = hf;
  const cuuint64_t rows = c.page_size, heads = c.nkv, rs = c.row_stride * 2, hs = c.head_stride * 2;
  const cuuint32_t bx = static_cast<cuuint32_t>(box);
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(hd), hf ? heads : rows, hf ? rows : heads,
                              static_cast<cuuint64_t>(c.pages)};
  const cuuint64_t str[3] = {hf ? hs : rs, hf ? rs : hs, static_cast<cuuint64_t>(c.page_stride) * 2};
  const cuuint32_t bdim[4] = {64, hf ? 1 : bx, hf ? bx : 1, 1};
  const int rc = encode(ctx, kmap, 4, c.k, dims, str, bdim);
  return rc ? rc : encode(ctx, vmap, 4, c.v, dims, str, bdim);
}

// The tensor-core form takes whole kv groups as rows of one tile, a positive
// scale (masked scores are -inf before the scale), and q strides a tensor map
// can hold; anything else runs on the row-block kernel.
bool chunk_takes(const AttnArgs& a) {
  return a.group <= kChunkRows && a.scale_log2 > 0.f && a.q_head > 0 && a.q_tok > 0 && a.q_tok < kMaxMapStride &&
         a.q_head < kMaxMapStride;
}

int launch_chunk(alv_ctx* ctx, const AttnArgs& a, int hd, int max_q_len, int row_min, bool mixed, cudaStream_t st) {
  switch (hd) {
    case 64: return launch_chunk_t<64>(ctx, a, max_q_len, row_min, mixed, st);
    case 128: return launch_chunk_t<128>(ctx, a, max_q_len, row_min, mixed, st);
    default: return launch_chunk_t<256>(ctx, a, max_q_len, row_min, mixed, st);
  }
}

}  // namespace alv
