// Host side of the C ABI, part 9: page bookkeeping of a shared cache pool
// (drop, fork, extend with copy-on-write, compaction) and the page copies it
// asks for.
//
// One CTA does the bookkeeping: it is a few dependent passes over small
// integer arrays, bound by latency.  It leaves a list of (from, to) pages in
// the scratch arena; a second launch copies them, in every layer, with the
// whole GPU (bound by HBM: each moved byte is read once and written once).
// Dropping 56 branches of 8 sequences, forking 56 and extending all by a token,
// with some 50 shared last pages of 32 KB (k and v) copied in each of 4 layers:
// 16 to 17.5 us for both launches, launch latency and the passes.  Dropped and
// forked rows are read whole by the one CTA: 56 drops and 56 forks take 2 us more
// with rows of 256 entries (4,096 positions of 16) than where only the entries in
// use were read, 10 us more with 1,024 and 75 with 8,192.  Compaction that moves 234 pages of 64 KB in each of 16 layers:
// 84 to 90 us, 5.4 to 5.8 TB/s.
// Counts change by integer atomics, so their order does not matter.
#include "internal.h"

namespace alv {
namespace {

constexpr int kPageThreads = 1024;

struct PagesArgs {
  int *table, *lens, *refs;
  int64_t table_stride;
  int pages, page_size, slots, width;
  const int *free_ids, *fork, *extend;
  int n_free, n_fork, n_extend;
  int* info;
  uint32_t* status;
  // scratch: number of moves, moves (from, to), free page ids
  int* n_moves;
  int2* moves;
  int* avail;
  int* cow;    // [n_extend] the shared last page an extend copies, or -1
  int* drops;  // [pages] pages to drop at the end
};

// Exclusive prefix sum over the CTA; `total` in every thread.
__device__ __forceinline__ int64_t cta_scan(int64_t v, int64_t* total, int64_t* sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) sh[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int64_t w = sh[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    sh[lane] = w;
  }
  __syncthreads();
  *total = sh[31];
  return x - v + (warp ? sh[warp - 1] : 0);
}

__device__ __forceinline__ int pages_for(int64_t len, int ps) { return static_cast<int>((len + ps - 1) / ps); }

__device__ __forceinline__ bool slot_ok(const PagesArgs& a, int slot) {
  if (slot >= 0 && slot < a.slots) return true;
  atomicOr(a.status, kStatusBadIndex);
  return false;
}

__device__ __forceinline__ void count(const PagesArgs& a, int page, int by) {
  if (page >= 0 && page < a.pages) atomicAdd(a.refs + page, by);
  else if (page >= a.pages) atomicOr(a.status, kStatusBadIndex);
}

// Which lists name a slot twice (bit 0: free, bit 1: fork, as a child or as a
// child that is another pair's parent, bit 2: extend), by three bitmaps in
// shared memory.
__device__ int lists_clash(const PagesArgs& a, uint32_t* bits) {
  const int words = (a.slots + 31) / 32;
  int clash = 0;
  auto mark = [&](uint32_t* set, int slot, int bit) {
    if (slot >= 0 && slot < a.slots && (atomicOr(set + slot / 32, 1u << (slot % 32)) >> (slot % 32) & 1)) clash |= bit;
  };
  for (int i = threadIdx.x; i < 3 * words; i += blockDim.x) bits[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < a.n_free; i += blockDim.x) mark(bits, a.free_ids[i], 1);
  for (int i = threadIdx.x; i < a.n_fork; i += blockDim.x) mark(bits + words, a.fork[2 * i + 1], 2);
  for (int i = threadIdx.x; i < a.n_extend; i += blockDim.x) mark(bits + 2 * words, a.extend[2 * i], 4);
  __syncthreads();
  for (int i = threadIdx.x; i < a.n_fork; i += blockDim.x) {
    const int par = a.fork[2 * i];
    if (par >= 0 && par < a.slots && par != a.fork[2 * i + 1] && (bits[words + par / 32] >> (par % 32) & 1)) clash |= 2;
  }
  return __syncthreads_or(clash & 1) * 1 | (__syncthreads_or(clash & 2) ? 2 : 0) | (__syncthreads_or(clash & 4) ? 4 : 0);
}

// Whole rows are dropped and forked: a caller may have lowered lens (rejected
// tokens), and the entries past it still name pages.  A warp takes kRowPart
// entries of a list's row at a time, their loads in flight together.
constexpr int kRowLoads = 8, kRowPart = 32 * kRowLoads;

// f(list entry, first table entry of the part) for every part of rows i0 .. i1.
template <class F>
__device__ __forceinline__ void each_part(const PagesArgs& a, int i0, int i1, F f) {
  const int warp = threadIdx.x >> 5, nw = blockDim.x >> 5, parts = (a.width + kRowPart - 1) / kRowPart;
  int i = i0 + warp / parts, part = warp % parts;
  while (i < i1) {
    f(i, part * kRowPart);
    for (part += nw; part >= parts; part -= parts) ++i;
  }
}
__device__ __forceinline__ void load_part(const PagesArgs& a, const int* row, int e0, int (&page)[kRowLoads]) {
#pragma unroll
  for (int x = 0; x < kRowLoads; ++x) {
    const int e = e0 + 32 * x + (threadIdx.x & 31);
    page[x] = e < a.width ? row[e] : -1;
  }
}

// Slots free_ids[i0 .. i1).
__device__ void drop_slots(const PagesArgs& a, int i0, int i1) {
  const int lane = threadIdx.x & 31;
  each_part(a, i0, i1, [&](int i, int e0) {
    const int slot = a.free_ids[i];
    if (!slot_ok(a, slot)) return;
    int* row = a.table + slot * a.table_stride;
    int page[kRowLoads];
    load_part(a, row, e0, page);
#pragma unroll
    for (int x = 0; x < kRowLoads; ++x)
      if (page[x] != -1) {
        count(a, page[x], -1);
        row[e0 + 32 * x + lane] = -1;
      }
    if (e0 == 0 && lane == 0) a.lens[slot] = 0;
  });
}

__device__ void fork_slots(const PagesArgs& a, int i0, int i1) {
  const int lane = threadIdx.x & 31;
  each_part(a, i0, i1, [&](int i, int e0) {
    const int par = a.fork[2 * i], kid = a.fork[2 * i + 1];
    if (!slot_ok(a, par) || !slot_ok(a, kid) || par == kid) return;
    int* to = a.table + kid * a.table_stride;
    int page[kRowLoads], old[kRowLoads];
    load_part(a, a.table + par * a.table_stride, e0, page);
    load_part(a, to, e0, old);
#pragma unroll
    for (int x = 0; x < kRowLoads; ++x)
      if (page[x] != old[x]) {
        count(a, old[x], -1);
        count(a, page[x], 1);
        to[e0 + 32 * x + lane] = page[x];
      }
    if (e0 == 0 && lane == 0) a.lens[kid] = a.lens[par];
  });
}

struct Need {
  int slot, len, have, want, cow;  // cow: the shared, partly filled last page, or -1
  bool ok;
};
__device__ __forceinline__ Need need_of(const PagesArgs& a, int i) {
  Need n{a.extend[2 * i], 0, 0, 0, -1, false};
  const int more = a.extend[2 * i + 1];
  if (!slot_ok(a, n.slot) || more < 0) {
    if (more < 0) atomicOr(a.status, kStatusBadIndex);
    n.slot = -1;
    n.ok = true;  // skipped: needs nothing
    return n;
  }
  n.len = max(a.lens[n.slot], 0);
  n.have = pages_for(n.len, a.page_size);
  const int64_t want = (static_cast<int64_t>(n.len) + more + a.page_size - 1) / a.page_size;
  n.ok = want <= a.width && static_cast<int64_t>(n.len) + more <= INT_MAX && n.have <= a.width;
  if (!n.ok) return n;
  n.want = static_cast<int>(want);
  if (more > 0 && n.len % a.page_size) {
    const int last = a.table[n.slot * a.table_stride + n.have - 1];
    if (last >= 0 && last < a.pages && a.refs[last] > 1) n.cow = last;
  }
  return n;
}

// A page that an extend puts another in the place of: its count goes down when
// all extends are done, so that no later one of the call is given the page
// while a copy from it is still to be made.  (Never more than pages handed out.)
__device__ __forceinline__ void drop_later(const PagesArgs& a, int page, int* n_drops) {
  const int at = atomicAdd(n_drops, 1);
  if (at < a.pages) a.drops[at] = page;
}

// Extends i0 .. i1 (no slot twice).  Returns the index of the first that does
// not fit, or i1.  `used`, `moves` and `n_drops` (shared) accumulate the call's
// totals.
__device__ int extend_slots(const PagesArgs& a, int i0, int i1, int64_t* used, int* moves, int* n_drops, int64_t* sh) {
  __shared__ int first_bad;
  __shared__ int64_t given;
  // pages wanted by the whole list, up to an entry past the table's width;
  // which last pages are shared is decided before any count changes
  if (threadIdx.x == 0) first_bad = INT_MAX;
  __syncthreads();
  Need n{-1, 0, 0, 0, -1, true};  // the entry of the last round: the only one of a list of up to 1024
  int64_t total = 0, t, mine = 0;
  for (int base = i0; base < i1; base += blockDim.x) {
    const int i = base + threadIdx.x;
    if (i < i1) {
      n = need_of(a, i);
      if (!n.ok) atomicMin(&first_bad, i);
      else mine += n.slot < 0 ? 0 : n.want - n.have + (n.cow >= 0);
      a.cow[i] = n.cow;
    }
  }
  cta_scan(mine, &total, sh);  // (of entries past first_bad too: more pages are listed than handed out)
  const int stop = min(i1, first_bad);
  // free pages in ascending order, as many as wanted
  int64_t have = 0;
  for (int base = 0; base < a.pages; base += 4 * blockDim.x) {
    int is_free[4], c = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int p = base + 4 * threadIdx.x + e;
      is_free[e] = p < a.pages && a.refs[p] == 0;
      c += is_free[e];
    }
    int64_t r = have + cta_scan(c, &t, sh);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (is_free[e]) {
        if (r < total) a.avail[r] = base + 4 * threadIdx.x + e;
        ++r;
      }
    have += t;
  }
  __syncthreads();
  // hand them out in list order
  const bool kept = i1 - i0 <= static_cast<int>(blockDim.x);
  int64_t at = 0;
  int n_moves = *moves;
  int fail = stop;
  for (int base = i0; base < stop; base += blockDim.x) {
    const int i = base + threadIdx.x;
    if (!kept) {
      n = Need{-1, 0, 0, 0, -1, true};
      if (i < stop) {
        n = need_of(a, i);
        n.cow = a.cow[i];
      }
    }
    const int64_t want = i < stop && n.slot >= 0 ? n.want - n.have + (n.cow >= 0) : 0;
    // pages and copies in one sum: copies in the high part
    const int64_t both = cta_scan(want + (i < stop && n.slot >= 0 && n.cow >= 0 ? int64_t{1} << 44 : 0), &t, sh);
    const int64_t first = at + (both & ((int64_t{1} << 44) - 1));
    const bool fits = i < stop && first + want <= have;
    if (threadIdx.x == 0) {
      first_bad = INT_MAX;
      given = at;
    }
    __syncthreads();
    if (i < stop && !fits) atomicMin(&first_bad, i);
    __syncthreads();
    const int unmet = first_bad;
    const bool apply = fits && i < unmet && n.slot >= 0;
    if (apply) {
      if (unmet != INT_MAX) atomicMax(reinterpret_cast<unsigned long long*>(&given), static_cast<unsigned long long>(first + want));
      int* row = a.table + n.slot * a.table_stride;
      int64_t next = first;
      if (n.cow >= 0) {
        const int dst = a.avail[next++];
        a.moves[n_moves + static_cast<int>(both >> 44)] = make_int2(n.cow, dst);
        atomicSub(a.refs + n.cow, 1);
        a.refs[dst] = 1;
        row[n.have - 1] = dst;
      }
      for (int e = n.have; e < n.want; ++e) {
        const int page = a.avail[next++], old = row[e];
        if (old != -1) drop_later(a, old, n_drops);  // (left by a caller that lowered lens)
        a.refs[page] = 1;
        row[e] = page;
      }
      a.lens[n.slot] = n.len + a.extend[2 * i + 1];
    }
    if (unmet != INT_MAX) {
      n_moves += __syncthreads_count(apply && n.cow >= 0);
      at = given;
      fail = unmet;
      break;
    }
    n_moves += static_cast<int>(t >> 44);
    at += t & ((int64_t{1} << 44) - 1);
  }
  *moves = n_moves;
  *used += at;
  return fail;
}

__global__ void __launch_bounds__(kPageThreads, 1) pages_update_kernel(const PagesArgs a) {
  extern __shared__ uint32_t bits[];
  __shared__ int64_t sh[32];
  __shared__ int n_drops;
  if (threadIdx.x == 0) n_drops = 0;
  pdl_wait();
  pdl_trigger();
  // A list that names a slot twice is taken one entry at a time.
  const int clash = lists_clash(a, bits);
  bool one = clash & 1;
  for (int i = 0; i < a.n_free; i = one ? i + 1 : a.n_free) {
    drop_slots(a, i, one ? i + 1 : a.n_free);
    __syncthreads();
  }
  one = clash & 2;
  for (int i = 0; i < a.n_fork; i = one ? i + 1 : a.n_fork) {
    fork_slots(a, i, one ? i + 1 : a.n_fork);
    __syncthreads();
  }
  one = clash & 4;
  int moves = 0, done = 0;
  int64_t used = 0;
  while (done < a.n_extend) {
    const int end = one ? done + 1 : a.n_extend;
    done = extend_slots(a, done, end, &used, &moves, &n_drops, sh);
    __syncthreads();
    if (done < end) break;
  }
  for (int i = threadIdx.x; i < min(n_drops, a.pages); i += blockDim.x) count(a, a.drops[i], -1);
  __syncthreads();
  if (threadIdx.x == 0) {
    *a.n_moves = moves;
    if (a.info) {
      a.info[1] = static_cast<int>(used);
      a.info[2] = moves;
      a.info[3] = done < a.n_extend ? done : -1;
    }
  }
  if (a.info) {  // a page whose last holder copied it counts as free
    int64_t n = 0, t;
    for (int p = threadIdx.x; p < a.pages; p += blockDim.x) n += a.refs[p] == 0;
    cta_scan(n, &t, sh);
    if (threadIdx.x == 0) a.info[0] = static_cast<int>(t);
  }
}

struct CompactArgs {
  const int *refs;
  int* refs_out;
  int pages;
  int* info;
  int* n_moves;
  int2* moves;
  int* to;      // [pages] new id of every page
  int* holes;   // [pages]
};

__global__ void __launch_bounds__(kPageThreads, 1) pages_compact_kernel(const CompactArgs a) {
  __shared__ int64_t sh[32];
  pdl_wait();
  pdl_trigger();
  int64_t t, n = 0;
  for (int p = threadIdx.x; p < a.pages; p += blockDim.x) n += a.refs[p] > 0;
  cta_scan(n, &t, sh);
  const int live = static_cast<int>(t);
  int64_t nh = 0, nm = 0;
  for (int base = 0; base < a.pages; base += blockDim.x) {
    const int p = base + threadIdx.x;
    const bool used = p < a.pages && a.refs[p] > 0;
    const bool hole = p < live && !used, mover = p >= live && used;
    // holes in the low, movers in the high half of the sum
    const int64_t r = cta_scan((hole ? 1 : 0) + (static_cast<int64_t>(mover) << 32), &t, sh);
    if (hole) a.holes[nh + (r & 0xFFFFFFFF)] = p;
    if (mover) a.moves[nm + (r >> 32)].x = p;
    if (p < a.pages) a.to[p] = p;
    nh += t & 0xFFFFFFFF;
    nm += t >> 32;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nm; i += blockDim.x) {
    const int src = a.moves[i].x, dst = a.holes[i];
    a.moves[i].y = dst;
    a.to[src] = dst;
  }
  __syncthreads();
  for (int p = threadIdx.x; p < live; p += blockDim.x)
    if (a.refs[p] > 0) a.refs_out[p] = a.refs[p];
  __syncthreads();
  for (int i = threadIdx.x; i < nm; i += blockDim.x) a.refs_out[a.moves[i].y] = a.refs[a.moves[i].x];
  __syncthreads();
  for (int p = live + threadIdx.x; p < a.pages; p += blockDim.x) a.refs_out[p] = 0;
  if (threadIdx.x == 0) {
    *a.n_moves = static_cast<int>(nm);
    if (a.info) {
      a.info[0] = live;
      a.info[1] = static_cast<int>(nm);
    }
  }
}

struct CopyArgs {
  uint8_t *k, *v;
  int64_t layer_stride, page_stride, page_bytes;
  int layers;
  const int* n_moves;
  const int2* moves;
  // compaction also renumbers the table
  const int* table;
  int* table_out;
  int64_t table_stride;
  int slots, width, pages;
  const int* to;
  uint32_t* status;
};

constexpr int kCopyThreads = 256;
constexpr int kCopyVec = 8;  // 16-byte loads in flight per thread

__global__ void __launch_bounds__(kCopyThreads) pages_copy_kernel(const CopyArgs a) {
  pdl_wait();
  const int n = *a.n_moves;
  if (a.table_out) {
    const int64_t entries = static_cast<int64_t>(a.slots) * a.width;
    for (int64_t e = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; e < entries;
         e += static_cast<int64_t>(gridDim.x) * blockDim.x) {
      int page = a.table[e / a.width * a.table_stride + e % a.width];
      if (page >= a.pages) atomicOr(a.status, kStatusBadIndex);
      else if (page >= 0) page = a.to[page];
      a.table_out[e] = page;
    }
  }
  // work unit: kCopyThreads * kCopyVec * 16 bytes of one page of one layer's k or v
  constexpr int64_t kUnit = kCopyThreads * kCopyVec * 16;
  const int64_t per_page = (a.page_bytes + kUnit - 1) / kUnit;
  const int64_t units = n * per_page * a.layers * 2;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int64_t part = u % per_page, blk = u / per_page;
    const int kv = static_cast<int>(blk & 1);
    const int64_t ml = blk >> 1;
    const int layer = static_cast<int>(ml % a.layers);
    const int2 mv = a.moves[ml / a.layers];
    uint8_t* base = (kv ? a.v : a.k) + layer * a.layer_stride;
    const uint4* src = reinterpret_cast<const uint4*>(base + mv.x * a.page_stride);
    uint4* dst = reinterpret_cast<uint4*>(base + mv.y * a.page_stride);
    const int64_t n16 = a.page_bytes / 16, i0 = part * (kUnit / 16) + threadIdx.x;
    uint4 r[kCopyVec];
#pragma unroll
    for (int i = 0; i < kCopyVec; ++i)
      if (i0 + i * kCopyThreads < n16) r[i] = __ldcs(src + i0 + i * kCopyThreads);
#pragma unroll
    for (int i = 0; i < kCopyVec; ++i)
      if (i0 + i * kCopyThreads < n16) __stcs(dst + i0 + i * kCopyThreads, r[i]);
  }
}

int check_pages(alv_ctx* ctx, const char* who, const alv_pages* p) {
  const std::string w(who);
  if (!p->k || !p->v || !p->table || !p->refs)
    return fail(ctx, ALV_ERR_ARG, w + ": null pointer in the page pool");
  if (p->layers < 1 || p->pages < 1 || p->page_size < 1 || p->slots < 1 || p->table_width < 1 ||
      p->table_stride < p->table_width || p->page_bytes < 16)
    return fail(ctx, ALV_ERR_ARG, w + ": every size of the page pool must be positive");
  if (p->page_bytes % 16 || p->page_stride % 16 || p->layer_stride % 16 || p->page_stride < p->page_bytes ||
      p->layer_stride < 0 || ((reinterpret_cast<uintptr_t>(p->k) | reinterpret_cast<uintptr_t>(p->v)) & 15))
    return fail(ctx, ALV_ERR_ARG, w + ": pages must be 16-byte aligned blocks of whole 16 bytes");
  if (p->slots > 1 << 19) return fail(ctx, ALV_ERR_UNSUPPORTED, w + ": at most 524,288 slots");
  return ALV_OK;
}

CopyArgs copy_args(alv_ctx* ctx, const alv_pages* p) {
  CopyArgs c{};
  c.k = static_cast<uint8_t*>(p->k);
  c.v = static_cast<uint8_t*>(p->v);
  c.layer_stride = p->layer_stride;
  c.page_stride = p->page_stride;
  c.page_bytes = p->page_bytes;
  c.layers = p->layers;
  c.pages = p->pages;
  c.status = status_ptr(ctx);
  return c;
}

int launch_copy(alv_ctx* ctx, const CopyArgs& c, cudaStream_t st) {
  return launch_ex(ctx, pages_copy_kernel, dim3(ctx->num_sms * 4), dim3(kCopyThreads), 0, st, true, c);
}

}  // namespace
}  // namespace alv

using namespace alv;

extern "C" int alv_pages_update(alv_ctx* ctx, const alv_pages* p, const int32_t* free, int n_free, const int32_t* fork,
                                int n_fork, const int32_t* extend, int n_extend, int32_t* info, void* stream) {
  if (!ctx || !p) return fail(ctx, ALV_ERR_ARG, "pages_update: bad argument");
  int rc = check_pages(ctx, "pages_update", p);
  if (rc) return rc;
  if (n_free < 0 || n_fork < 0 || n_extend < 0 || !p->lens || (n_free && !free) || (n_fork && !fork) || (n_extend && !extend))
    return fail(ctx, ALV_ERR_ARG, "pages_update: a list is missing");
  if ((rc = set_device(ctx))) return rc;
  const size_t o_moves = 256, o_cow = o_moves + align_up(static_cast<size_t>(n_extend) * 8, 256),
               o_avail = o_cow + align_up(static_cast<size_t>(n_extend) * 4, 256),
               o_drops = o_avail + align_up(static_cast<size_t>(p->pages) * 4, 256);
  if ((rc = ensure_scratch(ctx, o_drops + static_cast<size_t>(p->pages) * 4))) return rc;
  uint8_t* ws = work_ptr(ctx);
  PagesArgs a{};
  a.table = p->table;
  a.lens = p->lens;
  a.refs = p->refs;
  a.table_stride = p->table_stride;
  a.pages = p->pages;
  a.page_size = p->page_size;
  a.slots = p->slots;
  a.width = p->table_width;
  a.free_ids = free;
  a.n_free = n_free;
  a.fork = fork;
  a.n_fork = n_fork;
  a.extend = extend;
  a.n_extend = n_extend;
  a.info = info;
  a.status = status_ptr(ctx);
  a.n_moves = reinterpret_cast<int*>(ws);
  a.moves = reinterpret_cast<int2*>(ws + o_moves);
  a.cow = reinterpret_cast<int*>(ws + o_cow);
  a.avail = reinterpret_cast<int*>(ws + o_avail);
  a.drops = reinterpret_cast<int*>(ws + o_drops);
  const size_t smem = static_cast<size_t>((p->slots + 31) / 32) * 12;  // three bitmaps
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if ((rc = prepare_kernel(ctx, pages_update_kernel, smem))) return rc;
  if ((rc = launch_ex(ctx, pages_update_kernel, dim3(1), dim3(kPageThreads), smem, st, true, a))) return rc;
  if (n_extend == 0) return ALV_OK;
  CopyArgs c = copy_args(ctx, p);
  c.n_moves = a.n_moves;
  c.moves = a.moves;
  return launch_copy(ctx, c, st);
}

extern "C" int alv_pages_compact(alv_ctx* ctx, const alv_pages* p, int32_t* table_out, int32_t* refs_out, int32_t* info,
                                 void* stream) {
  if (!ctx || !p || !table_out || !refs_out) return fail(ctx, ALV_ERR_ARG, "pages_compact: bad argument");
  int rc = check_pages(ctx, "pages_compact", p);
  if (rc) return rc;
  if (table_out == p->table && p->table_stride != p->table_width)
    return fail(ctx, ALV_ERR_ARG, "pages_compact: a table renumbered in place must be contiguous");
  if ((rc = set_device(ctx))) return rc;
  const size_t np = static_cast<size_t>(p->pages), o_moves = 256, o_to = o_moves + align_up(np * 8, 256),
               o_holes = o_to + align_up(np * 4, 256);
  if ((rc = ensure_scratch(ctx, o_holes + np * 4))) return rc;
  uint8_t* ws = work_ptr(ctx);
  CompactArgs a{};
  a.refs = p->refs;
  a.refs_out = refs_out;
  a.pages = p->pages;
  a.info = info;
  a.n_moves = reinterpret_cast<int*>(ws);
  a.moves = reinterpret_cast<int2*>(ws + o_moves);
  a.to = reinterpret_cast<int*>(ws + o_to);
  a.holes = reinterpret_cast<int*>(ws + o_holes);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if ((rc = launch_ex(ctx, pages_compact_kernel, dim3(1), dim3(kPageThreads), 0, st, true, a))) return rc;
  CopyArgs c = copy_args(ctx, p);
  c.n_moves = a.n_moves;
  c.moves = a.moves;
  c.table = p->table;
  c.table_out = table_out;
  c.table_stride = p->table_stride;
  c.slots = p->slots;
  c.width = p->table_width;
  c.to = a.to;
  return launch_copy(ctx, c, st);
}
