// Host side of the C ABI, part 8: attention over a paged cache, and its
// kernel for row blocks (paged_attn.cuh has the mathematics).
#include "internal.h"
#include "paged_attn.cuh"

namespace alv {
namespace {

struct RowArgs {
  AttnArgs a;
  int box, head_first;  // positions per tensor copy, order of the cache's maps
  int early;            // wait for the kernel before at the end, not at the start
  float* parts;    // [2 * grid][kPart]: slot 0 where a run starts inside a block, 1 where it ends inside one
  uint32_t* done;  // [grid]: finished parts of the block that cut c is the first inside; zero between launches
};

// Blocks (sequence, kv head, 16 rows) in order, rows fastest.
template <int HD>
struct RowWalk {
  using R = RowRing<HD>;
  int b, kvh, blk, blks;
  SeqSpan s;
  SliceRange r;  // slices of the current block
  int p0, p1, nrow;

  __device__ __forceinline__ int blocks_of(const AttnArgs& a, const SeqSpan& q) const {
    const int64_t rows = static_cast<int64_t>(q.qlen) * a.group;
    return rows > a.row_max ? 0 : static_cast<int>((rows + kRowsPerBlock - 1) / kRowsPerBlock);
  }
  __device__ __forceinline__ void load(const AttnArgs& a) {
    // (rows of one kv head fit 31 bits: q itself would be larger than memory)
    const int r0 = blk * kRowsPerBlock;
    nrow = min(kRowsPerBlock, s.qlen * a.group - r0);
    p0 = s.kv - s.qlen + r0 / a.group;
    p1 = s.kv - s.qlen + (r0 + nrow - 1) / a.group;
    r = slice_range<R::kSlice>(p0, p1, a.window, a.sinks);
  }
  // A block that sees nothing still has one (empty) unit: it writes zeros.
  __device__ __forceinline__ int units() const { return max(1, (r.count() + kRowWarps - 1) / kRowWarps); }
  __device__ __forceinline__ int length() const { return units() + R::kExtra; }
  __device__ __forceinline__ int64_t length_of(const AttnArgs& a, const SeqSpan& q) {  // of one kv head's blocks
    s = q;
    const int n = blocks_of(a, q);
    int64_t u = 0;
    for (blk = 0; blk < n; ++blk) {
      load(a);
      u += length();
    }
    return u;
  }
  __device__ __forceinline__ void next(const AttnArgs& a) {
    if (++blk == blks) {
      blk = 0;
      if (++kvh == a.c.nkv) {
        kvh = 0;
        do {
          if (++b >= a.c.batch) return;
          s = seq_span(a.c, b);
          blks = blocks_of(a, s);
        } while (blks == 0);
      }
    }
    load(a);
  }
};

template <int HD>
__global__ void __launch_bounds__(kRowWarps * 32, 2)
    paged_rows_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const RowArgs ra) {
  using R = RowRing<HD>;
  constexpr int NS = R::kSlots, SL = R::kSlice, CH = HD / 8;  // CH: 16-byte chunks per row
  const AttnArgs& a = ra.a;
  extern __shared__ uint8_t smem_dyn[];
  __shared__ __align__(8) uint64_t full[kRowWarps][NS];
  __shared__ int64_t sums[kRowWarps], few[kRowWarps];
  __shared__ int longest[kRowWarps], shortest[kRowWarps];  // blocks
  __shared__ RowWalk<HD> start;                              // where the run starts, at its sequence's first block
  __shared__ int64_t start_rest, start_head;                 // how far into the sequence; the length of a kv head's blocks
  __shared__ uint32_t arrived;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* smem = smem_dyn + (((smem_u32(smem_dyn) + 1023u) & ~1023u) - smem_u32(smem_dyn));
  if (lane < NS) mbar_init(&full[warp][lane], 1);
  if (threadIdx.x == 0) {
    prefetch_map(&kmap);
    prefetch_map(&vmap);
  }
  fence_mbar_init();
  // Programmatic launch: inputs are touched once the kernel before is done.
  // Beside a chunk kernel (which has waited itself, and triggered after that)
  // nothing is shared, so only the end waits, for the join that follows.
  if (!ra.early) pdl_wait();
  pdl_trigger();

  // ---- this CTA's run [u0, u1) of the blocks laid end to end
  RowWalk<HD> w{};
  int64_t total, u0, u1;
  int G;  // CTAs that get a run
  bool cut = true;
  {
    const int per = (a.c.batch + kRowWarps * 32 - 1) / (kRowWarps * 32);
    const int b0 = threadIdx.x * per, b1 = min(b0 + per, a.c.batch);
    int64_t mine = 0, theirs = 0;  // theirs: as items of the chunk kernel
    int most = 0, least = INT_MAX;
    for (int b = b0; b < b1; ++b) {
      const int64_t len = w.length_of(a, seq_span(a.c, b));
      if (ra.early && len) {
        const SliceRange r = slice_range<ChunkTile<HD>::kBN>(w.s.kv - w.s.qlen, w.s.kv - 1, a.window, a.sinks);
        theirs += static_cast<int64_t>(max(r.count(), 1) + ChunkTile<HD>::kExtra) * a.c.nkv;
      }
      mine += len * a.c.nkv;
      if (len) {
        most = max(most, w.length());
        least = min(least, w.length());
      }
    }
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    most = __reduce_max_sync(0xffffffffu, most);
    least = __reduce_min_sync(0xffffffffu, least);
    if (ra.early) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) theirs += __shfl_xor_sync(0xffffffffu, theirs, o);
      if (lane == 0) few[warp] = theirs;
    }
    if (lane == 31) {
      sums[warp] = incl;
      longest[warp] = most;
      shortest[warp] = least;
    }
    __syncthreads();
    int64_t before = incl - mine;
    total = 0;
#pragma unroll
    for (int i = 0; i < kRowWarps; ++i) {
      if (i < warp) before += sums[i];
      total += sums[i];
      most = max(most, longest[i]);
      least = min(least, shortest[i]);
    }
    if (ra.early) {
      int64_t all = 0;
#pragma unroll
      for (int i = 0; i < kRowWarps; ++i) all += few[i];
      if (chunk_takes_few(all, gridDim.x / 2)) total = 0;  // (two CTAs per SM here, one there)
    }
    G = static_cast<int>(min((total + R::kMinUnits - 1) / R::kMinUnits, static_cast<int64_t>(gridDim.x)));
    if (blockIdx.x >= G) {
      if (ra.early) pdl_wait();
      return;
    }
    u0 = mul_div(total, blockIdx.x, G);
    u1 = mul_div(total, blockIdx.x + 1, G);
    // Blocks all about as long as a run: one each is as even as cutting, and
    // nothing is joined.  (A sequence's last block stands for its others.)
    const int64_t run = total / G;
    if (8 * static_cast<int64_t>(least) >= 7 * run && 4 * static_cast<int64_t>(most) <= 5 * run) cut = false;
    if (before <= u0 && u0 < before + mine) {
      int64_t at = before;
      for (int b = b0; b < b1; ++b) {
        const int64_t head = w.length_of(a, seq_span(a.c, b)), u = head * a.c.nkv;
        if (u0 < at + u) {
          w.b = b;
          w.blks = w.blocks_of(a, w.s);
          w.blk = w.kvh = 0;
          w.load(a);
          start = w;
          start_rest = u0 - at;
          start_head = head;
          break;
        }
        at += u;
      }
    }
    __syncthreads();
  }
  w = start;
  int x;  // where the run is inside the current block
  {
    int64_t rem = start_rest;
    if (rem >= start_head) {
      w.kvh = static_cast<int>(mul_div(rem, 1, static_cast<int>(min(start_head, static_cast<int64_t>(INT_MAX)))));
      rem -= w.kvh * start_head;
    }
    while (rem >= w.length()) {
      rem -= w.length();
      ++w.blk;
      w.load(a);
    }
    x = static_cast<int>(rem);
  }

  // the run that holds place x: the last c with total * c / G <= x
  auto run_of = [&](int64_t at) { return static_cast<int>(((at + 1) * G - 1) / total); };
  const uint32_t q_sm = smem_u32(smem), ring = q_sm + R::kQBytes + warp * NS * R::kSlotBytes;
  // the ring: next slot (and its barrier's phase) to fill and to use
  int fill = 0, use = 0;
  uint32_t phase = 0;
  bool dead = false;  // a copy never came: report, copy and wait no more
  for (int64_t u = u0; u < u1;) {
    const SeqSpan& s = w.s;
    const int units = w.units(), r0 = w.blk * kRowsPerBlock, nrow = w.nrow;
    int t0 = 0, t1 = units;  // units of this block that are this run's
    if (!cut || units <= R::kWhole) {
      if (x > 0) t1 = 0;  // a block that is not cut belongs to the run it begins in
    } else {
      t0 = max(0, x - R::kExtra);
      t1 = max(0, static_cast<int>(min(static_cast<int64_t>(units + R::kExtra), x + (u1 - u))) - R::kExtra);
    }
    const int64_t g0 = u - x;  // where the block begins
    u = g0 + units + R::kExtra;
    x = 0;
    if (t0 >= t1) {
      if (u < u1) w.next(a);
      continue;
    }
    const int pfirst = s.kv - s.qlen, p0 = w.p0, p1 = w.p1;

    // slices warp, warp + 4, ... of the run's units
    const int first = t0 * kRowWarps + warp;
    const int n_mine = max(0, (min(w.r.count(), t1 * kRowWarps) - first + kRowWarps - 1) / kRowWarps);
    auto j_of = [&](int i) { return w.r.slice(first + i * kRowWarps) * SL; };
    // Pages of the boxes to come: lane l holds box base + l (box b is part
    // b % sub of slice b / sub).
    const int sub = SL / ra.box;
    int page = 0, row = 0;
    auto look_up = [&](int i) {
      const int bx = i * sub + lane, sl = bx / sub, j = sl < n_mine ? j_of(sl) + bx % sub * ra.box : w.r.hi;
      page = a.c.pages;  // past the end: the copy reads zeros
      row = 0;
      if (j < w.r.hi && (j + ra.box > w.r.lo || j < a.sinks)) {
        const int pg = page_of(a.c, w.b, j);
        if (pg >= 0) page = pg, row = j % a.c.page_size;
      }
    };
    // Copy k or v of slice i into the next slot: lane l fetches box l / (HD / 64), dims 64 (l % (HD / 64)) ...
    auto copy = [&](int i, bool v) {
      if (i < n_mine && !dead) {
        const int per = 32 / sub;
        if (!v && i % per == 0) look_up(i);
        const int bx = lane / (HD / 64), d = lane % (HD / 64);
        const int pg = __shfl_sync(0xffffffffu, page, (i % per) * sub + (bx < sub ? bx : 0));
        const int rw = __shfl_sync(0xffffffffu, row, (i % per) * sub + (bx < sub ? bx : 0));
        const uint32_t bar = smem_u32(&full[warp][fill]);
        if (lane == 0) mbar_arrive_expect_tx_s(bar, R::kSlotBytes);
        __syncwarp();
        if (bx < sub) {
          const uint32_t dst = ring + fill * R::kSlotBytes + d * (SL * 128) + bx * ra.box * 128;
          if (ra.head_first) tma_load_4d(dst, v ? &vmap : &kmap, d * 64, w.kvh, rw, pg, bar);
          else tma_load_4d(dst, v ? &vmap : &kmap, d * 64, rw, w.kvh, pg, bar);
        }
      }
      if (i < n_mine) fill = fill + 1 == NS ? 0 : fill + 1;
    };
    auto arrive = [&]() {  // wait for the slot in use
      if (!dead && !__all_sync(0xffffffffu, mbar_wait_bounded_s(smem_u32(&full[warp][use]), phase))) {
        dead = true;
        if (lane == 0) atomicOr(a.c.status, kStatusMbarTimeout);
      }
      __syncwarp();
    };
    auto release = [&]() {
      __syncwarp();
      if (++use == NS) use = 0, phase ^= 1;
    };
    for (int h = 0; h < NS - 1; ++h) copy(h >> 1, h & 1);
    // q rows (row r = token r / group, head kvh * group + r % group)
    for (int e = threadIdx.x; e < kRowsPerBlock * CH; e += kRowWarps * 32) {
      const int r = e / CH, c = e % CH;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (r < nrow) {
        const int tok = s.q0 + (r0 + r) / a.group, head = w.kvh * a.group + (r0 + r) % a.group;
        v = *reinterpret_cast<const uint4*>(a.q + tok * a.q_tok + head * a.q_head + c * 8);
      }
      *reinterpret_cast<uint4*>(smem + r * HD * 2 + ((c ^ (r & 7)) << 4)) = v;
    }
    float o[HD / 8][4];  // C fragments: rows g, g + 8, dims 8n + 2t, +1
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < HD / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    const int pr[2] = {pfirst + (r0 + g) / a.group, pfirst + (r0 + g + 8) / a.group};  // positions of this lane's rows
    const bool one_token = p0 == p1;
    __syncthreads();  // q
    // this lane's part of ldmatrix addresses: q and v rows lane % 16, k rows (lane & 7) + 8 (lane / 16)
    const uint32_t lrow = lane & 15, lhi = lane >> 4, krow = (lane & 7) + ((lane >> 4) << 3), khi = (lane >> 3) & 1;
    for (int i = 0; i < n_mine; ++i) {
      const int j0 = j_of(i);
      // scores of the slice: n-tiles of 8 positions
      arrive();
      copy(i + (NS - 1) / 2, (NS - 1) & 1);
      float sc[SL / 8][4] = {};
      const uint32_t ks = ring + use * R::kSlotBytes;
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        uint32_t qa[4];
        ldsm4(q_sm + lrow * (HD * 2) + (((2 * k + lhi) ^ (lrow & 7)) << 4), qa);
#pragma unroll
        for (int n = 0; n < SL / 16; ++n) {
          uint32_t kb[4];
          ldsm4(ks + (k / 4) * (SL * 128) + (16 * n + krow) * 128 + (((2 * (k % 4) + khi) ^ (krow & 7)) << 4), kb);
          mma_16816(sc[2 * n], qa[0], qa[1], qa[2], qa[3], kb[0], kb[1]);
          mma_16816(sc[2 * n + 1], qa[0], qa[1], qa[2], qa[3], kb[2], kb[3]);
        }
      }
      release();
      // every row sees the whole slice?
      const bool whole = j0 + SL - 1 <= p0 && (a.window == 0 || j0 > p1 - a.window || j0 + SL <= a.sinks);
#pragma unroll
      for (int n = 0; n < SL / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[n][e] *= a.scale_log2;
      if (!whole) {
#pragma unroll
        for (int n = 0; n < SL / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!sees(j0 + 8 * n + 2 * t + (e & 1), pr[e >> 1], a.window, a.sinks)) sc[n][e] = -INFINITY;
      }
      float f[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float mx = m[r];
#pragma unroll
        for (int n = 0; n < SL / 8; ++n) mx = fmaxf(mx, fmaxf(sc[n][2 * r], sc[n][2 * r + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float base = mx == -INFINITY ? 0.f : mx;
        f[r] = exp2_fast(m[r] - base);
        m[r] = mx;
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < SL / 8; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float p = exp2_fast(sc[n][2 * r + e] - base);
            sc[n][2 * r + e] = p;
            sum += p;
          }
        l[r] = l[r] * f[r] + sum;  // this lane's columns; lanes are added at the end
      }
      if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
        for (int n = 0; n < HD / 8; ++n) {
          o[n][0] *= f[0];
          o[n][1] *= f[0];
          o[n][2] *= f[1];
          o[n][3] *= f[1];
        }
      }
      arrive();
      copy(i + NS / 2, NS & 1);
      const uint32_t vs = ring + use * R::kSlotBytes;
      // positions no row sees hold anything: their v counts as zero
      const bool edge = j0 + SL > w.r.hi || (j0 < w.r.lo && j0 + SL > a.sinks);
      uint32_t pa[SL / 16][4], live[SL / 16][2];
#pragma unroll
      for (int k = 0; k < SL / 16; ++k) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          pa[k][e] = pack_bf2_rn(sc[2 * k + (e >> 1)][2 * (e & 1)], sc[2 * k + (e >> 1)][2 * (e & 1) + 1]);
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const int j = j0 + 16 * k + 8 * hh + 2 * t;
          live[k][hh] = !edge ? 0xFFFFFFFFu
                              : (j < w.r.hi && (j >= w.r.lo || j < a.sinks) ? 0xFFFFu : 0u) |
                                    (j + 1 < w.r.hi && (j + 1 >= w.r.lo || j + 1 < a.sinks) ? 0xFFFF0000u : 0u);
        }
      }
      auto v_at = [&](int k, int n) {
        return vs + (n / 4) * (SL * 128) + (16 * k + lrow) * 128 + (((2 * (n % 4) + lhi) ^ (lrow & 7)) << 4);
      };
      // A value that is not finite must not reach the rows that do not see its
      // position (0 * inf): then each token's rows take their own product.
      bool odd = false;
      if (!whole && !one_token) {
        uint32_t any = 0;
#pragma unroll 1
        for (int k = 0; k < SL / 16; ++k)
#pragma unroll 4
          for (int n = 0; n < HD / 16; ++n) {
            uint32_t vb[4];
            ldsm4_t(v_at(k, n), vb);
#pragma unroll
            for (int e = 0; e < 4; ++e) any |= bf2_nonfinite(vb[e] & live[k][e & 1]);
          }
        odd = __any_sync(0xffffffffu, any);
      }
      if (!odd) {
#pragma unroll
        for (int k = 0; k < SL / 16; ++k)
#pragma unroll
          for (int n = 0; n < HD / 16; ++n) {
            uint32_t vb[4];
            ldsm4_t(v_at(k, n), vb);
            if (edge) {
#pragma unroll
              for (int e = 0; e < 4; ++e) vb[e] &= live[k][e & 1];
            }
            mma_16816(o[2 * n], pa[k][0], pa[k][1], pa[k][2], pa[k][3], vb[0], vb[1]);
            mma_16816(o[2 * n + 1], pa[k][0], pa[k][1], pa[k][2], pa[k][3], vb[2], vb[3]);
          }
      } else {
#pragma unroll
        for (int n = 0; n < HD / 16; ++n)
          for (int pt = p0; pt <= p1; ++pt)
#pragma unroll
            for (int k = 0; k < SL / 16; ++k) {
              uint32_t vb[4];
              ldsm4_t(v_at(k, n), vb);
#pragma unroll
              for (int hh = 0; hh < 2; ++hh) {
                uint32_t mk[2];
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                  const int j = j0 + 16 * k + 8 * y + 2 * t;
                  mk[y] = (sees(j, pt, a.window, a.sinks) ? 0xFFFFu : 0u) |
                          (sees(j + 1, pt, a.window, a.sinks) ? 0xFFFF0000u : 0u);
                }
                float tmp[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) tmp[e] = o[2 * n + hh][e];
                mma_16816(tmp, pa[k][0], pa[k][1], pa[k][2], pa[k][3], vb[2 * hh] & mk[0], vb[2 * hh + 1] & mk[1]);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (pr[e >> 1] == pt) o[2 * n + hh][e] = tmp[e];
              }
            }
      }
      release();
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
    // ---- join the warps in warp order
    __syncthreads();
    float* jm = reinterpret_cast<float*>(smem + R::kQBytes);
    float* jl = jm + kRowWarps * kRowsPerBlock;
    float* jo = jl + kRowWarps * kRowsPerBlock;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = warp * kRowsPerBlock + g + 8 * r;
      if (t == 0) {
        jm[row] = m[r];
        jl[row] = l[r];
      }
      if (g + 8 * r < nrow) {
#pragma unroll
        for (int n = 0; n < HD / 8; ++n)
          *reinterpret_cast<float2*>(jo + row * HD + 8 * n + 2 * t) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
      }
    }
    __syncthreads();
    const bool part = t0 > 0 || t1 < units;
    float* mypart = ra.parts + (static_cast<int64_t>(blockIdx.x) * 2 + (t0 > 0 ? 0 : 1)) * R::kPart;
    // (a row before the first position sees nothing and gives zeros; any other
    // sees itself at least, and with no score above -inf it gives NaN)
    auto share = [&](int r, float sum) { return pfirst + (r0 + r) / a.group < 0 ? 0.f : 1.f / sum; };
    auto store = [&](int r, int d, float x, float y) {  // two dims of a finished row
      const int tok = s.q0 + (r0 + r) / a.group, head = w.kvh * a.group + (r0 + r) % a.group;
      *reinterpret_cast<uint32_t*>(a.out + tok * a.o_tok + head * a.o_head + d) = pack_bf2_rn(x, y);
    };
    for (int e = threadIdx.x; e < nrow * (HD / 2); e += kRowWarps * 32) {
      const int r = e / (HD / 2), d = (e % (HD / 2)) * 2;
      float mm = -INFINITY;
#pragma unroll
      for (int x = 0; x < kRowWarps; ++x) mm = fmaxf(mm, jm[x * kRowsPerBlock + r]);
      const float base = mm == -INFINITY ? 0.f : mm;
      float ll = 0.f, x = 0.f, y = 0.f;
#pragma unroll
      for (int k = 0; k < kRowWarps; ++k) {
        const int row = k * kRowsPerBlock + r;
        const float f = exp2_fast(jm[row] - base);
        const float2 v = *reinterpret_cast<const float2*>(jo + row * HD + d);
        ll += f * jl[row];
        x += f * v.x;
        y += f * v.y;
      }
      if (part) {
        if (d == 0) mypart[r] = mm, mypart[kRowsPerBlock + r] = ll;
        *reinterpret_cast<float2*>(mypart + 2 * kRowsPerBlock + r * HD + d) = make_float2(x, y);
      } else {
        const float inv = share(r, ll);
        store(r, d, x * inv, y * inv);
      }
    }
    if (part) {
      // CTAs c0 .. c1 hold the block's parts; the last to finish joins them
      const int c0 = run_of(g0 + R::kExtra), c1 = run_of(g0 + R::kExtra + units - 1);
      __syncthreads();
      if (threadIdx.x == 0) {
        __threadfence();
        arrived = atomicAdd(ra.done + c0 + 1, 1u);
      }
      __syncthreads();
      if (arrived == static_cast<uint32_t>(c1 - c0)) {
        __threadfence();
        if (threadIdx.x == 0) ra.done[c0 + 1] = 0;
        // warp w joins parts w, w + 4, ... (m, l in registers of its lanes as
        // row = lane; O summed in shared memory), then the warps are joined
        auto part_at = [&](int c) {
          return ra.parts + (static_cast<int64_t>(c) * 2 + (c == c0 ? 1 : 0)) * R::kPart;
        };
        float wm = -INFINITY, wl = 0.f;
        if (lane < nrow)
          for (int c = c0 + warp; c <= c1; c += kRowWarps) wm = fmaxf(wm, __ldcg(part_at(c) + lane));
        const float base = wm == -INFINITY ? 0.f : wm;
        if (lane < nrow)
          for (int c = c0 + warp; c <= c1; c += kRowWarps)
            wl += exp2_fast(__ldcg(part_at(c) + lane) - base) * __ldcg(part_at(c) + kRowsPerBlock + lane);
        if (lane < kRowsPerBlock) {
          jm[warp * kRowsPerBlock + lane] = wm;
          jl[warp * kRowsPerBlock + lane] = wl;
        }
        __syncwarp();
        for (int e = lane; e < nrow * (HD / 4); e += 32) {
          const int r = e / (HD / 4), d = (e % (HD / 4)) * 4;
          const float rm = jm[warp * kRowsPerBlock + r], rb = rm == -INFINITY ? 0.f : rm;
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
          for (int c = c0 + warp; c <= c1; c += kRowWarps) {
            const float f = exp2_fast(__ldcg(part_at(c) + r) - rb);
            const float4 v = __ldcg(reinterpret_cast<const float4*>(part_at(c) + 2 * kRowsPerBlock + r * HD + d));
            acc.x += f * v.x;
            acc.y += f * v.y;
            acc.z += f * v.z;
            acc.w += f * v.w;
          }
          *reinterpret_cast<float4*>(jo + (warp * kRowsPerBlock + r) * HD + d) = acc;
        }
        __syncthreads();
        for (int e = threadIdx.x; e < nrow * (HD / 2); e += kRowWarps * 32) {
          const int r = e / (HD / 2), d = (e % (HD / 2)) * 2;
          float mm = -INFINITY;
#pragma unroll
          for (int x = 0; x < kRowWarps; ++x) mm = fmaxf(mm, jm[x * kRowsPerBlock + r]);
          const float b2 = mm == -INFINITY ? 0.f : mm;
          float ll = 0.f, x = 0.f, y = 0.f;
#pragma unroll
          for (int k = 0; k < kRowWarps; ++k) {
            const int row = k * kRowsPerBlock + r;
            const float f = exp2_fast(jm[row] - b2);
            const float2 v = *reinterpret_cast<const float2*>(jo + row * HD + d);
            ll += f * jl[row];
            x += f * v.x;
            y += f * v.y;
          }
          const float inv = share(r, ll);
          store(r, d, x * inv, y * inv);
        }
      }
    }
    if (u < u1) {
      w.next(a);
      fence_proxy_async_smem();  // the join's words lie where copies will
      __syncthreads();
    }
  }
  if (ra.early) pdl_wait();
}

template <int HD>
int launch_rows_t(alv_ctx* ctx, const AttnArgs& a, size_t scratch, bool early, cudaStream_t st) {
  using R = RowRing<HD>;
  auto k = paged_rows_kernel<HD>;
  int rc = prepare_kernel(ctx, k, R::kBytes);
  if (rc) return rc;
  if ((rc = ensure_scratch(ctx, scratch + rows_scratch(ctx, HD)))) return rc;
  RowArgs ra{};
  ra.a = a;
  ra.a.c.status = status_ptr(ctx);
  ra.parts = reinterpret_cast<float*>(work_ptr(ctx) + scratch);
  ra.done = counters_ptr(ctx);
  ra.early = early;
  CUtensorMap kmap, vmap;
  ra.box = box_rows(a.c.page_size, R::kSlice);
  if ((rc = encode_cache(ctx, a.c, HD, ra.box, &kmap, &vmap, &ra.head_first))) return rc;
  return launch_ex(ctx, k, dim3(ctx->num_sms * 2), dim3(kRowWarps * 32), R::kBytes, st, true, kmap, vmap, ra);
}

}  // namespace

size_t rows_scratch(alv_ctx* ctx, int hd) {
  return static_cast<size_t>(ctx->num_sms) * 2 * 2 * kRowsPerBlock * (hd + 2) * 4;
}

int launch_rows(alv_ctx* ctx, const AttnArgs& a, int hd, size_t scratch, bool early, cudaStream_t st) {
  switch (hd) {
    case 64: return launch_rows_t<64>(ctx, a, scratch, early, st);
    case 128: return launch_rows_t<128>(ctx, a, scratch, early, st);
    default: return launch_rows_t<256>(ctx, a, scratch, early, st);
  }
}

}  // namespace alv

using namespace alv;

extern "C" int alv_paged_attention(alv_ctx* ctx, const alv_paged* cache, const alv_attention_args* args, void* stream) {
  if (!ctx || !cache || !args) return fail(ctx, ALV_ERR_ARG, "paged_attention: bad argument");
  int rc = set_device(ctx);
  if (rc) return rc;
  AttnArgs a{};
  if ((rc = make_paged_view(ctx, "paged_attention", cache, &a.c))) return rc;
  if ((cache->tokens && (!args->q || !args->out)) || args->heads < 1 || args->max_q_len < 0 || args->window < 0 || args->sinks < 0 ||
      !std::isfinite(args->scale))
    return fail(ctx, ALV_ERR_ARG, "paged_attention: bad argument");
  if (args->heads % cache->kv_heads) return fail(ctx, ALV_ERR_SHAPE, "paged_attention: heads must be a multiple of kv_heads");
  if (((reinterpret_cast<uintptr_t>(args->q) | reinterpret_cast<uintptr_t>(args->out)) & 15) || args->q_token_stride % 8 ||
      args->q_head_stride % 8 || args->out_token_stride % 8 || args->out_head_stride % 8 || args->q_token_stride < 0 ||
      args->q_head_stride < 0 || args->out_token_stride < 0 || args->out_head_stride < 0)
    return fail(ctx, ALV_ERR_ARG, "paged_attention: q and out must be 16-byte aligned with strides of whole 16 bytes");
  if (cache->batch == 0 || cache->tokens == 0 || args->max_q_len == 0) return ALV_OK;
  a.q = args->q;
  a.q_tok = args->q_token_stride;
  a.q_head = args->q_head_stride;
  a.out = args->out;
  a.o_tok = args->out_token_stride;
  a.o_head = args->out_head_stride;
  a.nq = args->heads;
  a.group = args->heads / cache->kv_heads;
  a.window = args->window;
  a.sinks = args->sinks;
  a.scale_log2 = static_cast<float>(static_cast<double>(args->scale) * 1.4426950408889634);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // Sequences of more than 16 rows go to the tensor-core form; a batch may hold
  // both kinds (the lengths are on the device).
  a.row_max = INT_MAX;
  if (static_cast<int64_t>(args->max_q_len) * a.group > kRowsPerBlock && chunk_takes(a)) {
    a.row_max = kRowsPerBlock;
    // Room for max_q_len tokens of every sequence: a uniform batch, which leaves
    // nothing for row blocks.  A captured one may be replayed with shorter
    // sequences, so the tensor-core form, alone, takes those too.
    const bool mixed = static_cast<int64_t>(cache->batch) * args->max_q_len != cache->tokens;
    return launch_chunk(ctx, a, cache->head_dim, args->max_q_len, mixed ? kRowsPerBlock + 1 : 1, mixed, st);
  }
  return launch_rows(ctx, a, cache->head_dim, 0, false, st);
}
