// Host side of the C ABI, part 10: token sampling from given uniform numbers.
//
//   s_i = l_i / T,  w_i = exp(s_i - max s),  mass_i = floor(w_i 2^40)
//   top-k: the k first in the order (s descending, index ascending);
//   top-p: the shortest prefix of those with mass >= ceil(p * their mass);
//   min-p: of those, w_i >= min_p;
//   token: the first, in index order, whose running mass passes floor(u * total).
//
// The masses are integers (a vocabulary of 2^19 sums to at most 2^59), so sums
// of any order and atomics give one result.
//
// A cluster of CTAs takes a row and keeps it in its shared memory, so the
// logits are read once; the CTAs exchange sums and histograms through
// distributed shared memory.  The end of a prefix is found by a histogram over
// max - s (2048 even bins; counts for top-k, masses for top-p, whose bins also
// add up to the mass that p is a share of), the bin where the k-th element (or
// the wanted mass) falls, and then among that bin's elements, which every CTA
// gathers and compares each with each; a bin with too many elements is cut
// again by the bits of s.  Elements equal to the last one kept enter in index
// order.  The bins before the last one also give every CTA's kept mass, so only
// the CTA that the draw falls into goes over its elements again.  Where top-k
// leaves few elements, one CTA finishes the row by itself.
//
// Bound: not the logits' bytes (15 us of HBM for 192 rows of 128,256 fp32
// values) but the passes over shared memory (nearly every value has mass, so
// nearly every one is binned by atomics) and waiting at meetings: 44 % of the
// issue slots are used.  192 such rows at top-p 0.9 take 145
// us: a row's cluster is busy 23 us, of them 5 loading, 7 in the exponentials
// and atomics of the histogram, and most of the rest in four meetings of the
// cluster; two CTAs per SM cover for each other.  One row of 128,256 bf16
// values with top-k 40 and top-p: 14.5 us, of it 4.4 until the row is loaded, 3
// in the one CTA that finishes it, the rest in passes of a few instructions and
// meetings.
#include <cooperative_groups.h>

#include "common.cuh"
#include "internal.h"

namespace alv {
namespace {

namespace cg = cooperative_groups;

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kBins = 2048;
constexpr int kCand = kSampleThreads;  // elements of the last bin compared each with each
constexpr int kMaxCluster = 8;
constexpr float kMaxDist = 27.75f;     // exp(-27.75) < 2^-40: no mass beyond
constexpr int kMaxSlice = 65536;       // elements per CTA: 65,536 16-bit digits add up below 2^32
constexpr int kSlice18 = 16384;        // up to here 18-bit digits do: most masses are then one digit long
typedef unsigned long long u64;

struct SampleArgs {
  const void* logits;
  int64_t stride;
  const float* u;
  int* tokens;
  float* logprobs;
  const float *t_rows, *p_rows, *m_rows;
  const int* k_rows;
  int vocab, k, slice;  // slice: elements of the row per CTA
  float t, p, m;
};

// Bits of s in an order that unsigned comparison follows.
__device__ __forceinline__ uint32_t key_of(float s) {
  const uint32_t b = __float_as_uint(s);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// floor(w 2^40) for w in [0, 1], by two additions that round down: at 2 a
// float's step is 2^-22, at 2^-17 it is 2^-40.  hi 2^18 + lo, lo < 2^18.
__device__ __forceinline__ void mass_digits(float w, uint32_t* hi, uint32_t* lo) {
  const float a = __fadd_rz(w, 2.0f);
  const float b = __fadd_rz(__fsub_rn(w, __fsub_rn(a, 2.0f)), 7.62939453125e-06f);
  *hi = __float_as_uint(a) - 0x40000000u;
  *lo = __float_as_uint(b) & 0x3FFFFu;
}
__device__ __forceinline__ u64 mass_of(float w) {
  uint32_t hi, lo;
  mass_digits(w, &hi, &lo);
  return (static_cast<u64>(hi) << 18) + lo;
}

struct Cut {  // kept: s > last, and the first `ties` (in index order) of s == last
  float last;
  uint32_t ties, of;  // of: how many equal `last`
};

constexpr int kCoarse = 64;  // runs of 32 bins

struct SampleShared {
  uint32_t bins[3][kBins];  // counts in the first, or masses as three digits' sums
  u64 coarse[4][kCoarse];   // their sums over runs of bins, one slot per use
  u64 tmp[kMaxCluster][kCoarse];
  // this CTA's elements of the bin in question, then the cluster's
  uint32_t lkey[kCand], lidx[kCand], n_list;
  uint32_t ckey[kCand], cidx[kCand];
  u64 cmass[kCand];
  u64 scan[32];
  u64 sum;  // kept mass
  u64 few_all, few_before, few_own;  // of a last bin's elements: kept mass, that before this CTA's slice, in it
  uint32_t best_key, best_idx, kmin, kmax;
  struct { int bin; u64 before, in, want; uint32_t last_key, ties, of; } found;
  uint32_t wties[kSampleWarps];
  u64 wmass[kSampleWarps];
};

// Inclusive prefix sum over the CTA; *total in every thread.
__device__ __forceinline__ u64 cta_scan(u64 v, u64* total, u64* sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) sh[warp] = x;
  __syncthreads();
  u64 before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSampleWarps; ++w) {
    const u64 y = sh[w];
    if (w < warp) before += y;
    all += y;
  }
  *total = all;
  return x + before;
}

// The row's values, in shared memory (RES) or read again where they do not fit.
template <bool BF16, bool RES>
struct Row {
  const void* base;  // this CTA's slice
  float* vals;
  int n, first;      // elements of the slice, index of its first
  int slice;         // elements of a full slice
  float temp;
  bool greedy;
  bool infinite;  // without a copy: +inf is the largest value and reads as 0, the rest as -inf
  __device__ __forceinline__ float value(float x) const {
    return !greedy && temp != 1.0f ? scaled<true>(x) : scaled<false>(x);
  }
  template <bool DIV>
  __device__ __forceinline__ float scaled(float x) const {
    if (DIV) x = __fdiv_rn(x, temp);
    return fmaxf(x + 0.0f, -INFINITY);  // -0 counts as +0, NaN as -inf
  }
  __device__ __forceinline__ float raw(int i) const {
    return BF16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(base)[i]) : static_cast<const float*>(base)[i];
  }
  __device__ __forceinline__ float at(int i) const {
    if (RES) return vals[i];
    const float x = value(raw(i));
    return !infinite ? x : x == INFINITY ? 0.f : -INFINITY;
  }
  // f(i, value) for i in [i0, i1) (i0 a multiple of 4), `step` threads from
  // `first`, four values at a time; in shared memory -inf may follow past i1.
  template <class F>
  __device__ __forceinline__ void each(int i0, int i1, int first, int step, F f) const {
    if (RES) {
#pragma unroll 2
      for (int i = i0 + 4 * first; i < i1; i += 4 * step) {
        const float4 v = *reinterpret_cast<const float4*>(vals + i);
        f(i, v.x);
        f(i + 1, v.y);
        f(i + 2, v.z);
        f(i + 3, v.w);
      }
    } else {
#pragma unroll 4
      for (int i = i0 + first; i < i1; i += step) f(i, at(i));
    }
  }
  // Reads the slice (RES: into vals), 16 bytes a load where aligned; this
  // thread's largest value.
  __device__ __forceinline__ float load() const { return !greedy && temp != 1.0f ? load_t<true>() : load_t<false>(); }
  template <bool DIV>
  __device__ __forceinline__ float load_t() const {
    constexpr int V = BF16 ? 8 : 4;
    float best = -INFINITY;
    int i0 = 0;
    if ((reinterpret_cast<uintptr_t>(base) & 15) == 0) {
      const uint4* p = static_cast<const uint4*>(base);
      const int nv = n / V;
#pragma unroll 4
      for (int c = threadIdx.x; c < nv; c += kSampleThreads) {
        const uint4 x = p[c];
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
        float v[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
          v[e] = scaled<DIV>(BF16 ? bf16_bits_to_f32(e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xFFFFu) : __uint_as_float(w[e & 3]));
          best = fmaxf(best, v[e]);
        }
#pragma unroll
        for (int e = 0; e < V; e += 4)
          if (RES) *reinterpret_cast<float4*>(vals + c * V + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
      }
      i0 = nv * V;
    }
    for (int i = i0 + threadIdx.x; i < n; i += kSampleThreads) {
      const float v = scaled<DIV>(raw(i));
      best = fmaxf(best, v);
      if (RES) vals[i] = v;
    }
    return best;
  }
};

// Sums over the CTAs before this one and over all, in every thread (a lane
// reads a CTA's).
__device__ __forceinline__ void cluster_sums(cg::cluster_group& cl, SampleShared& sh, u64* before, u64* all) {
  const unsigned lane = threadIdx.x & 31, nb = cl.num_blocks();
  const u64 v = lane < nb ? cl.map_shared_rank(&sh, lane)->sum : 0;
  u64 x = v, y = lane < cl.block_rank() ? v : 0;
#pragma unroll
  for (int o = kMaxCluster / 2; o > 0; o >>= 1) {
    x += __shfl_xor_sync(0xffffffffu, x, o);
    y += __shfl_xor_sync(0xffffffffu, y, o);
  }
  *all = __shfl_sync(0xffffffffu, x, 0);
  *before = __shfl_sync(0xffffffffu, y, 0);
}

__device__ __forceinline__ u64 lane_sum(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ u64 lane_scan(u64 v) {  // inclusive
  const unsigned lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  return v;
}

// The histogram's crossing: with `bin_of(s)` (-1: not in question) of every
// element, the bin in which the count (MASS: the mass) starting from `acc`
// reaches the wanted one, what lies before it and what it holds (found.*).
// `want_of(total)` gives the wanted one from the sum of all bins; 0: found.bin
// = -1.  Every CTA shows the sums of its runs of 32 bins; each then finds the
// run and adds up that run's bins itself, so the cluster meets once.  Leaves the
// list empty for a gather (by the meeting, every CTA has read the last one's).
template <bool MASS, bool BF16, bool RES, class B, class W>
__device__ __forceinline__ void crossing(cg::cluster_group& cl, SampleShared& sh, const Row<BF16, RES>& row, float top,
                                         u64 acc, int slot, B bin_of, W want_of) {
  const unsigned nb = cl.num_blocks();
  const int lane = threadIdx.x & 31;
  const int digit = row.slice <= kSlice18 ? 18 : 16;
  for (int b = threadIdx.x; b < kBins * (MASS ? 3 : 1); b += kSampleThreads) (&sh.bins[0][0])[b] = 0;
  __syncthreads();
  auto add = [&](int b, uint32_t m0, uint32_t m1, uint32_t m2) {
    if (m0) atomicAdd(&sh.bins[0][b], m0);
    if (m1) atomicAdd(&sh.bins[1][b], m1);
    if (m2) atomicAdd(&sh.bins[2][b], m2);
  };
  if (!MASS) {
    row.each(0, row.n, threadIdx.x, kSampleThreads, [&](int, float s) {
      const int b = bin_of(s);
      if (b >= 0) atomicAdd(&sh.bins[0][b], 1u);
    });
  } else if (digit == 18) {
    row.each(0, row.n, threadIdx.x, kSampleThreads, [&](int, float s) {
      const int b = bin_of(s);
      uint32_t hi, lo;  // an element not in question has no mass
      mass_digits(b < 0 ? 0.f : expf(s - top), &hi, &lo);
      add(b, lo, hi & 0x3FFFFu, hi >> 18);
    });
  } else {
    row.each(0, row.n, threadIdx.x, kSampleThreads, [&](int, float s) {
      const int b = bin_of(s);
      if (b < 0) return;
      const u64 m = mass_of(expf(s - top));
      add(b, static_cast<uint32_t>(m) & 0xFFFFu, static_cast<uint32_t>(m >> 16) & 0xFFFFu, static_cast<uint32_t>(m >> 32));
    });
  }
  __syncthreads();
  {
    constexpr int kPer = kBins / kSampleThreads, kLanes = 32 / kPer;  // bins per thread, threads per run
    u64 v = 0;
#pragma unroll
    for (int x = 0; x < (MASS ? 3 : 1); ++x) {
      const uint4 q = *reinterpret_cast<const uint4*>(&sh.bins[x][threadIdx.x * kPer]);
      v += (static_cast<u64>(q.x) + q.y + q.z + q.w) << (digit * x);
    }
    static_assert(kPer == 4, "four bins per thread");
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (threadIdx.x % kLanes == 0) sh.coarse[slot][threadIdx.x / kLanes] = v;
  }
  cl.sync();
  if (threadIdx.x == 0) sh.n_list = 0, sh.few_all = 0, sh.few_before = 0, sh.few_own = 0;
  for (unsigned i = threadIdx.x; i < nb * kCoarse; i += kSampleThreads)
    sh.tmp[i / kCoarse][i % kCoarse] = cl.map_shared_rank(&sh, i / kCoarse)->coarse[slot][i % kCoarse];
  __syncthreads();
  if (threadIdx.x < 32) {
    u64 v0 = 0, v1 = 0;  // runs 2 lane, 2 lane + 1
#pragma unroll
    for (unsigned r = 0; r < kMaxCluster; ++r)
      if (r < nb) {
        v0 += sh.tmp[r][2 * lane];
        v1 += sh.tmp[r][2 * lane + 1];
      }
    const u64 upto = lane_scan(v0 + v1);
    const u64 want = want_of(__shfl_sync(0xffffffffu, upto, 31));
    const u64 b0 = acc + upto - v0 - v1, b1 = b0 + v0, b2 = b1 + v1;
    const int here = want == 0 ? -1 : b0 < want && want <= b1 ? 2 * lane : b1 < want && want <= b2 ? 2 * lane + 1 : -1;
    const uint32_t who = __ballot_sync(0xffffffffu, here >= 0);
    if (lane == 0) sh.found.bin = -1;
    __syncwarp();
    if (who) {
      const int src = __ffs(who) - 1, run = __shfl_sync(0xffffffffu, here, src);
      u64 before = __shfl_sync(0xffffffffu, here & 1 ? b1 : b0, src);
      uint32_t w[MASS ? 3 : 1][kMaxCluster];  // all in flight at once
#pragma unroll
      for (unsigned r = 0; r < kMaxCluster; ++r) {
        const SampleShared* o = cl.map_shared_rank(&sh, r < nb ? r : 0);
#pragma unroll
        for (int x = 0; x < (MASS ? 3 : 1); ++x) w[x][r] = r < nb ? o->bins[x][run * 32 + lane] : 0;
      }
      u64 v = 0;
#pragma unroll
      for (unsigned r = 0; r < kMaxCluster; ++r)
#pragma unroll
        for (int x = 0; x < (MASS ? 3 : 1); ++x) v += static_cast<u64>(w[x][r]) << (digit * x);
      before += lane_scan(v) - v;
      if (before < want && want <= before + v) {
        sh.found.bin = run * 32 + lane;
        sh.found.before = before;
        sh.found.in = v;
        sh.found.want = want;
      }
      if (MASS) {  // this CTA's mass before the bin
        const int bin = run * 32 + __ffs(__ballot_sync(0xffffffffu, before < want && want <= before + v)) - 1;
        u64 own = 0;
        if (2 * lane < run) own += sh.coarse[slot][2 * lane];
        if (2 * lane + 1 < run) own += sh.coarse[slot][2 * lane + 1];
        if (run * 32 + lane < bin)
#pragma unroll
          for (int x = 0; x < (MASS ? 3 : 1); ++x) own += static_cast<u64>(sh.bins[x][run * 32 + lane]) << (digit * x);
        own = lane_sum(own);
        if (lane == 0) sh.sum = own;
      }
    }
  }
  __syncthreads();
}

// Bins of max - s, even up to kMaxDist.
__device__ __forceinline__ int even_bin(float top, float s) {
  const float d = top - s;
  if (!(d <= kMaxDist)) return -1;
  return static_cast<int>(__float_as_uint(__fmaf_rz(d, kBins / kMaxDist * 0.99999f, 8388608.0f)) & 0x7FFFFFu);
}
// A range of s around bins b0 .. b1 with a bin to spare on either side: two
// comparisons that spare most elements the bin.
struct Near {
  float lo, hi;
  __device__ __forceinline__ Near(float top, int b0, int b1)
      : lo(top - (b1 + 2) * (kMaxDist / kBins)), hi(top - (b0 - 1) * (kMaxDist / kBins)) {}
  __device__ __forceinline__ bool has(float s) const { return s >= lo && s <= hi; }
};

// Put the elements with in(s) into this CTA's list; once the cluster has met,
// how many there are (more than kCand: the lists are cut off), and in lane r's
// *n_mine how many of CTA r.
template <bool BF16, bool RES, class F>
__device__ __forceinline__ uint32_t gather(cg::cluster_group& cl, SampleShared& sh, const Row<BF16, RES>& row,
                                           uint32_t* n_mine, F in) {
  row.each(0, row.n, threadIdx.x, kSampleThreads, [&](int i, float s) {
    if (!in(s)) return;
    const uint32_t at = atomicAdd(&sh.n_list, 1u);
    if (at < kCand) {
      sh.lkey[at] = key_of(s);
      sh.lidx[at] = row.first + i;
    }
  });
  cl.sync();
  const unsigned lane = threadIdx.x & 31;
  *n_mine = lane < cl.num_blocks() ? cl.map_shared_rank(&sh, lane)->n_list : 0;
  return __reduce_add_sync(0xffffffffu, *n_mine);
}

// The kept mass, found along with the end of the prefix.
struct Sums {
  bool known;
  u64 total, before, own;  // of the row, before this CTA's slice, of the slice
  uint32_t listed;    // elements in ckey / cidx
};

// The cluster's lists (n <= kCand elements, n_mine of them in the CTA whose
// rank is this lane's) into ckey / cidx of this CTA.
__device__ __forceinline__ void pull(cg::cluster_group& cl, SampleShared& sh, uint32_t n, uint32_t n_mine) {
  const uint32_t i = threadIdx.x;
  uint32_t at = 0, from = 0, skip = 0;
#pragma unroll
  for (int r = 0; r < kMaxCluster; ++r) {  // the list that element i is in
    const uint32_t m = __shfl_sync(0xffffffffu, n_mine, r);
    if (i >= at && i < at + m) from = r, skip = at;
    at += m;
  }
  if (i < n) {
    const SampleShared* o = cl.map_shared_rank(&sh, from);
    sh.ckey[i] = o->lkey[i - skip];
    sh.cidx[i] = o->lidx[i - skip];
  }
  __syncthreads();
}

// The prefix of the row, in (s descending, index ascending) order, that ends
// with the element where the count (MASS: the mass) reaches the wanted one:
// called once the histogram over even bins has found the bin (found.*).  Every
// CTA compares the bin's elements by itself, so nothing is told around.  MASS:
// with what the histogram says of the bins before, that gives the kept mass of
// every CTA too, unless min-p takes some of it away.
template <bool MASS, bool BF16, bool RES>
__device__ Cut select(cg::cluster_group& cl, SampleShared& sh, const Row<BF16, RES>& row, float top, float floor_s,
                      float min_p, Sums* sums) {
  const unsigned nb = cl.num_blocks();
  const int lane = threadIdx.x & 31;
  const u64 want = sh.found.want;
  uint32_t kmin = 0, kmax = 0;  // after the first round: the keys of the bin that is cut again
  int shift = 0;
  for (int round = 0;; ++round) {
    auto bin_of = [&](float s) -> int {
      if (round == 0) return s >= floor_s ? even_bin(top, s) : -1;
      const uint32_t k = key_of(s);
      return k >= kmin && k <= kmax ? static_cast<int>((kmax - k) >> shift) : -1;
    };
    if (round > 0) crossing<MASS>(cl, sh, row, top, sh.found.before, round & 1, bin_of, [&](u64) { return want; });
    const int bin = sh.found.bin;
    const u64 pre0 = sh.found.before;
    uint32_t n_mine;
    const Near near(top, bin, bin);
    const uint32_t n = round == 0 ? gather(cl, sh, row, &n_mine, [&](float s) {
      return near.has(s) && even_bin(top, s) == bin && s >= floor_s;
    })
                                  : gather(cl, sh, row, &n_mine, [&](float s) { return bin_of(s) == bin; });
    if (n <= kCand) {
      if (MASS && round == 0) cluster_sums(cl, sh, &sums->before, &sums->total);
      pull(cl, sh, n, n_mine);
      const uint32_t i = threadIdx.x;
      uint32_t k = 0, idx = 0, ties = 1, of = 0;
      u64 m = 0;
      if (i < n) {
        k = sh.ckey[i];
        idx = sh.cidx[i];
        m = MASS ? mass_of(expf(key_value(k) - top)) : 1;
        sh.cmass[i] = m;
      }
      __syncthreads();
      if (i < n) {
        u64 pre = pre0;
        for (uint32_t j = 0; j < n; ++j) {
          const uint32_t kj = sh.ckey[j];
          const bool earlier = kj == k && sh.cidx[j] < idx;
          if (kj > k || earlier) pre += sh.cmass[j];
          ties += earlier;
          of += kj == k;
        }
        if (pre < want && want <= pre + m) {
          sh.found.last_key = k;
          sh.found.ties = ties;
          sh.found.of = of;
        }
      }
      __syncthreads();
      const uint32_t last = sh.found.last_key;
      if (MASS && round == 0 && expf(key_value(last) - top) >= min_p) {
        if ((i & ~31u) < n) {
          const bool keep = i < n && (k > last || (k == last && ties <= sh.found.ties));
          const u64 all = lane_sum(keep ? m : 0);
          const u64 pre = lane_sum(keep && idx < static_cast<uint32_t>(row.first) ? m : 0);
          const u64 own = lane_sum(keep && idx - row.first < static_cast<uint32_t>(row.n) ? m : 0);
          if (lane == 0) {
            atomicAdd(&sh.few_all, all);
            atomicAdd(&sh.few_before, pre);
            atomicAdd(&sh.few_own, own);
          }
        }
        __syncthreads();
        sums->before += sh.few_before;
        sums->total += sh.few_all;
        sums->own = sh.sum + sh.few_own;
        sums->known = true;
        sums->listed = n;
      }
      return {key_value(last), sh.found.ties, sh.found.of};
    }
    // too many: the range of their keys, to cut it again
    if (threadIdx.x == 0) {
      sh.kmin = 0xFFFFFFFFu;
      sh.kmax = 0;
    }
    __syncthreads();
    uint32_t lo = 0xFFFFFFFFu, hi = 0;
    row.each(0, row.n, threadIdx.x, kSampleThreads, [&](int, float s) {
      if (bin_of(s) != bin) return;
      lo = min(lo, key_of(s));
      hi = max(hi, key_of(s));
    });
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if (lane == 0 && hi >= lo) {
      atomicMin(&sh.kmin, lo);
      atomicMax(&sh.kmax, hi);
    }
    cl.sync();
    const SampleShared* o = cl.map_shared_rank(&sh, lane < static_cast<int>(nb) ? lane : 0);
    kmin = __reduce_min_sync(0xffffffffu, o->kmin);
    kmax = __reduce_max_sync(0xffffffffu, o->kmax);
    if (kmin == kmax) {  // all equal
      const u64 each = MASS ? mass_of(expf(key_value(kmin) - top)) : 1;
      return {key_value(kmin), static_cast<uint32_t>((want - pre0 + each - 1) / each), n};
    }
    shift = 0;
    while (((kmax - kmin) >> shift) >= kBins) ++shift;
  }
}

// The rest of a row whose top k are among CTA 0's list: ranks by comparing each
// with each (a warp an element: this CTA is alone by now, and 40 elements take 3
// us of it, 5.3 with a thread for each), then top-p over the ranks, min-p, and
// the draw in index order.
__device__ void finish_few(SampleShared& sh, const SampleArgs& a, int r, uint32_t n, uint32_t k, float p, float min_p,
                           float top) {
  const uint32_t i = threadIdx.x, lane = i & 31;
  for (uint32_t e = i / 32; e < n; e += kSampleWarps) {  // a warp compares element e with all
    const uint32_t ke = sh.ckey[e], ie = sh.cidx[e];
    uint32_t before = 0;
    for (uint32_t j = lane; j < n; j += 32) {
      const uint32_t kj = sh.ckey[j];
      before += kj > ke || (kj == ke && sh.cidx[j] < ie);
    }
    before = __reduce_add_sync(0xffffffffu, before);
    if (lane == 0) sh.lkey[e] = before;  // (the CTA's own list is read)
  }
  __syncthreads();
  uint32_t rank = 0xFFFFFFFFu;
  u64 m = 0;
  float w = 0.f;
  if (i < n) {
    rank = sh.lkey[i];
    if (rank < k) {
      w = expf(key_value(sh.ckey[i]) - top);
      m = mass_of(w);
    }
  }
  sh.cmass[i] = 0;
  __syncthreads();
  if (i < n) sh.cmass[rank] = m;  // by rank
  __syncthreads();
  u64 total;
  const u64 upto = cta_scan(sh.cmass[i], &total, sh.scan);
  uint32_t last = k;  // ranks below are kept
  if (p < 1.f) {
    const double x = ceil(static_cast<double>(total) * static_cast<double>(p));
    const u64 goal = x >= 1.0 ? static_cast<u64>(x) : 1;
    if (upto >= goal && upto - sh.cmass[i] < goal) sh.found.last_key = i + 1;
    __syncthreads();
    last = sh.found.last_key;
  }
  __syncthreads();
  const bool keep = i < n && rank < last && rank < k && w >= min_p;
  sh.cmass[i] = keep ? m : 0;  // by place in the list
  __syncthreads();
  u64 kept = 0;
  for (uint32_t j = lane; j < n; j += 32) kept += sh.cmass[j];
  kept = lane_sum(kept);
  const u64 x = static_cast<u64>(fmax(floor(static_cast<double>(a.u[r]) * static_cast<double>(kept)), 0.0));
  const u64 goal = x < kept ? x : kept - 1;
  for (uint32_t e = i / 32; e < n; e += kSampleWarps) {
    const u64 me = sh.cmass[e];
    if (me == 0) continue;
    const uint32_t ie = sh.cidx[e];
    u64 before = 0;
    for (uint32_t j = lane; j < n; j += 32)
      if (sh.cidx[j] < ie) before += sh.cmass[j];
    before = lane_sum(before);
    if (lane == 0 && before <= goal && goal < before + me) {
      a.tokens[r] = static_cast<int>(ie);
      if (a.logprobs) a.logprobs[r] = static_cast<float>(log(static_cast<double>(me) / static_cast<double>(kept)));
    }
  }
}

template <bool BF16, bool RES>
__global__ void __launch_bounds__(kSampleThreads, 2) sample_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) uint8_t dyn[];
  SampleShared& sh = *reinterpret_cast<SampleShared*>(dyn);
  cg::cluster_group cl = cg::this_cluster();
  const unsigned rank = cl.block_rank(), nb = cl.num_blocks();
  const int r = blockIdx.x / nb, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Row<BF16, RES> row;
  pdl_wait();
  pdl_trigger();
  row.first = min(static_cast<int>(rank) * a.slice, a.vocab);
  row.slice = a.slice;
  row.n = min(a.slice, a.vocab - row.first);
  row.base = static_cast<const char*>(a.logits) + (r * a.stride + row.first) * (BF16 ? 2 : 4);
  row.vals = reinterpret_cast<float*>(dyn + (sizeof(SampleShared) + 15) / 16 * 16);
  row.temp = a.t_rows ? a.t_rows[r] : a.t;
  row.greedy = !(row.temp > 0.f);
  row.infinite = false;
  const int k = a.k_rows ? a.k_rows[r] : a.k;
  const float p = a.p_rows ? a.p_rows[r] : a.p, min_p = fminf(a.m_rows ? a.m_rows[r] : a.m, 1.f);

  // ---- the row into shared memory; its largest value
  const float best = row.load();
  if (RES && threadIdx.x < 4 && (row.n & 3) && threadIdx.x >= (row.n & 3)) row.vals[(row.n & ~3) + threadIdx.x] = -INFINITY;
  {
    uint32_t bk = __reduce_max_sync(0xffffffffu, key_of(best));
    if (lane == 0) sh.wties[warp] = bk;
    __syncthreads();
    bk = __reduce_max_sync(0xffffffffu, sh.wties[lane % kSampleWarps]);
    if (threadIdx.x == 0) sh.best_key = bk, sh.best_idx = 0xFFFFFFFFu;
  }
  cl.sync();
  float top = key_value(__reduce_max_sync(0xffffffffu, cl.map_shared_rank(&sh, lane < static_cast<int>(nb) ? lane : 0)->best_key));
  if (row.greedy || top == -INFINITY) {  // the same in every CTA of the cluster
    uint32_t idx = 0xFFFFFFFFu;  // the first index of the largest
    row.each(0, row.n, threadIdx.x, kSampleThreads, [&](int i, float s) {
      if (s == top) idx = min(idx, static_cast<uint32_t>(row.first + i));
    });
    idx = __reduce_min_sync(0xffffffffu, idx);
    if (lane == 0 && idx != 0xFFFFFFFFu) atomicMin(&sh.best_idx, idx);
    cl.sync();
    if (rank == 0 && warp == 0) {
      idx = __reduce_min_sync(0xffffffffu, cl.map_shared_rank(&sh, lane < static_cast<int>(nb) ? lane : 0)->best_idx);
      if (lane == 0) {
        a.tokens[r] = top == -INFINITY ? -1 : static_cast<int>(idx);
        if (a.logprobs) a.logprobs[r] = top == -INFINITY ? -INFINITY : 0.f;
      }
    }
    cl.sync();  // no CTA leaves while another reads its words
    return;
  }
  if (top == INFINITY) {  // only the infinite ones count, all alike: as 0 among -inf
    row.infinite = true;
    top = 0.f;
    if (RES) {
      __syncthreads();
      for (int i = threadIdx.x; i < row.n; i += kSampleThreads) row.vals[i] = row.vals[i] == INFINITY ? 0.f : -INFINITY;
    }
  }
  __syncthreads();

  // ---- where the kept prefix ends
  Cut cut{-INFINITY, 0, 0};
  bool all = true;
  Sums sums{};
  if (k > 0 && k < a.vocab) {
    // elements without mass do not matter: if fewer than k have some, all do
    crossing<false>(cl, sh, row, top, 0, 2, [&](float s) { return even_bin(top, s); },
                    [&](u64 n) { return n > static_cast<u64>(k) ? static_cast<u64>(k) : 0; });
    const int bin = sh.found.bin;
    if (bin >= 0 && sh.found.before + sh.found.in <= kCand) {
      uint32_t n_mine;
      const Near near(top, 0, bin);
      const uint32_t n = gather(cl, sh, row, &n_mine, [&](float s) {
        if (!near.has(s)) return false;
        const int b = even_bin(top, s);
        return b >= 0 && b <= bin;
      });
      if (rank == 0) pull(cl, sh, n, n_mine);
      cl.barrier_arrive();  // the lists are read
      if (rank == 0) finish_few(sh, a, r, n, static_cast<uint32_t>(k), p, min_p, top);
      cl.barrier_wait();
      return;
    }
    if (bin >= 0) {
      cut = select<false>(cl, sh, row, top, -INFINITY, min_p, nullptr);
      all = false;
    }
  }
  if (p < 1.f) {
    // the mass that p is a share of: all of it, or the k largest (of the
    // elements equal to the last one only some)
    const u64 each = all ? 0 : mass_of(expf(cut.last - top));
    const u64 beyond = all ? 0 : (cut.of - cut.ties) * each;
    crossing<true>(cl, sh, row, top, 0, 3, [&](float s) { return s >= cut.last ? even_bin(top, s) : -1; }, [&](u64 m) {
      const double goal = ceil(static_cast<double>(m - beyond) * static_cast<double>(p));
      return goal >= 1.0 ? static_cast<u64>(goal) : static_cast<u64>(1);
    });
    cut = select<true>(cl, sh, row, top, cut.last, min_p, &sums);
    all = false;
  }

  // ---- the CTA whose slice holds the token
  const bool ranked = !all && cut.ties < cut.of;  // only some of the equals are kept
  const int seg = (row.n + kSampleWarps * 128 - 1) / (kSampleWarps * 128) * 128;  // a warp's run of the slice
  const int i0 = min(warp * seg, row.n), i1 = min(i0 + seg, row.n);
  uint32_t tie0 = 0, ties;  // equals of the last one before this warp's run, and so far
  auto kept_mass = [&](int i) -> u64 {  // lanes take consecutive elements
    const float s = i < i1 ? row.at(i) : -INFINITY;
    bool keep = i < i1 && (all || s >= cut.last);
    if (ranked) {
      const uint32_t eq = __ballot_sync(0xffffffffu, i < i1 && s == cut.last);
      if (i < i1 && s == cut.last) keep = ties + __popc(eq & ((1u << lane) - 1)) < cut.ties;
      ties += __popc(eq);
    }
    if (!keep) return 0;
    const float w = expf(s - top);
    return w >= min_p ? mass_of(w) : 0;
  };
  auto run_mass = [&] {  // of this warp's run
    u64 m = 0;
    ties = tie0;
    if (ranked) {
      for (int b = i0; b < i1; b += 32) m += kept_mass(b + lane);
    } else {
      const float least = all ? -INFINITY : cut.last;
      row.each(i0, i1, lane, 32, [&](int, float s) {
        if (!(s >= least)) return;
        const float w = expf(s - top);
        if (w >= min_p) m += mass_of(w);
      });
    }
    m = lane_sum(m);
    if (lane == 0) sh.wmass[warp] = m;
    __syncthreads();
    return m;
  };
  u64 m = 0;
  if (!sums.known) {
    if (ranked) {
      uint32_t n = 0;
      for (int i = i0 + lane; i < i1; i += 32) n += row.at(i) == cut.last;
      n = __reduce_add_sync(0xffffffffu, n);
      if (lane == 0) sh.wties[warp] = n;
      cl.sync();
      for (unsigned o = 0; o <= rank; ++o) {
        const SampleShared* q = cl.map_shared_rank(&sh, o);
        for (int w = 0; w < (o == rank ? warp : kSampleWarps); ++w) tie0 += q->wties[w];
      }
    }
    m = run_mass();
    for (int w = 0; w < kSampleWarps; ++w) sums.own += sh.wmass[w];
    if (threadIdx.x == 0) sh.sum = sums.own;
    cl.sync();
    cluster_sums(cl, sh, &sums.before, &sums.total);
  }
  cl.barrier_arrive();  // its words are read; no CTA leaves before all have read
  const u64 total = sums.total;
  const u64 x = static_cast<u64>(fmax(floor(static_cast<double>(a.u[r]) * static_cast<double>(total)), 0.0));
  const u64 goal = x < total ? x : total - 1;
  u64 before = sums.before;
  if (goal < before || goal >= before + sums.own) {
    cl.barrier_wait();
    return;
  }

  // ---- the warp whose run does, and there the token
  if (sums.known) {
    if (ranked) {  // the equals are all among the last bin's elements
      const uint32_t key = key_of(cut.last), first = static_cast<uint32_t>(row.first + i0);
      for (uint32_t j = lane; j < sums.listed; j += 32) tie0 += sh.ckey[j] == key && sh.cidx[j] < first;
      tie0 = __reduce_add_sync(0xffffffffu, tie0);
    }
    m = run_mass();
  }
  for (int w = 0; w < warp; ++w) before += sh.wmass[w];
  if (before <= goal && goal < before + m) {  // this warp's run holds the token
    int b = i0;
    ties = tie0;
    if (!ranked) {  // 32 blocks of the run at a time: a lane adds up a block, then the right block is taken apart
      for (; b < i1; b += 1024) {
        u64 e = 0;
        for (int j = 0; j < 32; ++j) {  // rotated, so that the lanes use different banks
          const int i = b + 32 * lane + ((j + lane) & 31);
          const float s = i < i1 ? row.at(i) : -INFINITY;
          if (i >= i1 || !(all || s >= cut.last)) continue;
          const float w = expf(s - top);
          if (w >= min_p) e += mass_of(w);
        }
        u64 upto = e;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const u64 y = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += y;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, before + upto > goal);
        if (past) {
          const int blk = __ffs(past) - 1;
          before += __shfl_sync(0xffffffffu, upto - e, blk);
          b += 32 * blk;
          break;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
      }
    }
    for (; b < i1; b += 32) {
      const u64 e = kept_mass(b + lane);
      u64 upto = e;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      if (before + upto > goal && before + upto - e <= goal) {
        a.tokens[r] = row.first + b + lane;
        if (a.logprobs) a.logprobs[r] = static_cast<float>(log(static_cast<double>(e) / static_cast<double>(total)));
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
      if (before > goal) break;
    }
  }
  cl.barrier_wait();
}

template <bool BF16, bool RES>
int launch_sample(alv_ctx* ctx, const SampleArgs& a, int rows, int cluster, cudaStream_t st) {
  auto k = sample_kernel<BF16, RES>;
  const size_t smem = (sizeof(SampleShared) + 15) / 16 * 16 + (RES ? static_cast<size_t>(a.slice) * 4 : 0);
  int rc = prepare_kernel(ctx, k, smem);
  if (rc) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * cluster);
  cfg.blockDim = dim3(kSampleThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  ALV_CUDA(ctx, cudaLaunchKernelEx(&cfg, k, a));
  return ALV_OK;
}

}  // namespace
}  // namespace alv

using namespace alv;

extern "C" int alv_sample(alv_ctx* ctx, const alv_sample_args* s, void* stream) {
  if (!ctx || !s) return fail(ctx, ALV_ERR_ARG, "sample: bad argument");
  if (s->rows < 0 || s->vocab < 1 || !valid_dtype(s->logits_dtype) || (s->rows && (!s->logits || !s->u || !s->tokens)) ||
      s->logits_stride < 0)
    return fail(ctx, ALV_ERR_ARG, "sample: bad argument");
  if (s->vocab > kMaxCluster * kMaxSlice) return fail(ctx, ALV_ERR_UNSUPPORTED, "sample: at most 524,288 tokens");
  if (reinterpret_cast<uintptr_t>(s->logits) & (s->logits_dtype == ALV_F32 ? 3 : 1))
    return fail(ctx, ALV_ERR_ARG, "sample: logits must be aligned to their type");
  if ((!s->temperature_rows && !(s->temperature >= 0.f)) || (!s->top_p_rows && !(s->top_p >= 0.f)) ||
      (!s->min_p_rows && !(s->min_p >= 0.f && s->min_p <= 1.f)))
    return fail(ctx, ALV_ERR_ARG, "sample: temperature and top_p must be >= 0, min_p in [0, 1]");
  int rc = set_device(ctx);
  if (rc) return rc;
  if (s->rows == 0) return ALV_OK;
  SampleArgs a{};
  a.logits = s->logits;
  a.stride = s->logits_stride;
  a.u = s->u;
  a.tokens = s->tokens;
  a.logprobs = s->logprobs;
  a.t_rows = s->temperature_rows;
  a.p_rows = s->top_p_rows;
  a.m_rows = s->min_p_rows;
  a.k_rows = s->top_k_rows;
  a.vocab = s->vocab;
  a.k = s->top_k;
  a.t = s->temperature;
  a.p = s->top_p;
  a.m = s->min_p;
  // CTAs per row: as few as keep a CTA's slice at 16 K elements (64 KB: two
  // CTAs of other rows share the SM); more, down to slices of 2 K, while the
  // rows alone leave SMs idle.
  int cluster = 1;
  auto slice_of = [&](int c) { return static_cast<int>(align_up((s->vocab + c - 1) / c, 8)); };
  while (cluster < kMaxCluster &&
         (slice_of(cluster) > 16384 || (static_cast<int64_t>(s->rows) * cluster * 2 <= ctx->num_sms && slice_of(cluster) > 2048)))
    cluster *= 2;
  if (static_cast<int64_t>(s->rows) * cluster > INT_MAX) return fail(ctx, ALV_ERR_UNSUPPORTED, "sample: too many rows");
  a.slice = slice_of(cluster);
  const bool fits = a.slice <= 45056;  // 176 KB; a longer slice is read again in every pass
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (s->logits_dtype == ALV_BF16)
    return fits ? launch_sample<true, true>(ctx, a, s->rows, cluster, st) : launch_sample<true, false>(ctx, a, s->rows, cluster, st);
  return fits ? launch_sample<false, true>(ctx, a, s->rows, cluster, st) : launch_sample<false, false>(ctx, a, s->rows, cluster, st);
}
