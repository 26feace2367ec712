// Host side of the C ABI, part 7: per-head q/k norm, rotation and cache
// append of a ragged batch of new tokens, in one pass over [q | k | v].
//
//   h  = x w / sqrt(mean(x^2) + eps)          (only where a norm weight is given)
//   y_i        = h_i cos_i - h_{i+r/2} sin_i
//   y_{i+r/2}  = h_{i+r/2} cos_i + h_i sin_i  (i < r/2; dims >= r pass through)
//
// q goes to q_out, k and v to the token's slot of the paged cache.  fp32
// throughout, one rounding to bf16 at the stores.
//
// Bound: HBM (each value of qkv is read once and written once).  A CTA takes up
// to 8 tokens and looks up their sequence, page and table rows once for all
// heads; one token per CTA for small batches, which wait for memory and not for
// bytes.  7,000 tokens of 32 + 8 + 8 heads of 128 with norms (176 MB): 39 us,
// 4.5 TB/s, 70 % of a copy's rate (what is in flight is one head ahead per
// thread, in registers); a step of four tokens 8.9 us called from the host, 2.7 us in a CUDA
// graph.
#include "internal.h"
#include "paged.cuh"

namespace alv {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeTokens = 8;  // tokens of a CTA at most

struct RopeArgs {
  PagedView c;
  const void* qkv;
  int64_t qkv_stride;      // elements per token
  uint16_t* q_out;
  int64_t q_tok, q_head;   // elements
  const void* table;       // [max_pos][2 rot]: cos (rot) | sin (rot)
  int max_pos, rot, nq, tokens_per_cta;
  const float *qw, *kw;
  float eps;
};

// Eight consecutive values as fp32.
template <bool F32>
__device__ __forceinline__ void load8(const void* base, int64_t at, float (&v)[8]) {
  if (F32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
    const float4 a = p[0], b = p[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = bf16_bits_to_f32(w[i] & 0xFFFFu);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
}

__device__ __forceinline__ void store8(uint16_t* dst, const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack_bf2(bf16_bits_rn(v[2 * i]), bf16_bits_rn(v[2 * i + 1]));
  *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
}

// The sequence that token t belongs to: the last b with q_start[b] <= t.
__device__ __forceinline__ int seq_of(const PagedView& c, int t) {
  int lo = 0, hi = c.batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (c.q_start[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Eight values as they lie in memory.
template <bool F32>
struct Raw8 {
  uint4 v[F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void* base, int64_t at) {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const char*>(base) + at * (F32 ? 4 : 2));
#pragma unroll
    for (int i = 0; i < (F32 ? 2 : 1); ++i) v[i] = p[i];
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < (F32 ? 2 : 1); ++i) {
      const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (F32) {
          x[4 * i + e] = __uint_as_float(w[e]);
        } else {
          x[2 * e] = bf16_bits_to_f32(w[e] & 0xFFFFu);
          x[2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u);
        }
      }
    }
  }
};

// A CTA takes `tokens_per_cta` tokens (1, 2, 4 or 8), 8 / tokens_per_cta warps
// each: first their sequences, positions and cache slots (a thread each), then
// all heads of a token, one per group of HD / 16 lanes and step.  Each lane
// holds two groups of eight values: a rotation pair's two halves, or 16 that
// pass through; its place in the head never changes, so it keeps the cos, sin
// and weights of it, and reads only values, the next head's ahead.  (7,000
// tokens of 48 heads of 128 with norms: 39.4 us; cos, sin and weights read again
// for every head, at 40 registers and six CTAs per SM, 45.7; four CTAs per SM
// that spill 42.7; two heads ahead 41.)
template <int HD, bool F32, bool TF32>
__global__ void __launch_bounds__(kRopeThreads, 3) qk_norm_rope_kernel(const RopeArgs a) {
  constexpr int LPH = HD / 16;
  __shared__ int pos_of[kRopeTokens];          // -1: skipped
  __shared__ int64_t slot_of[kRopeTokens];     // element of the cache, -1: no page
  const PagedView& c = a.c;
  const int t0 = blockIdx.x * a.tokens_per_cta, nt = min(a.tokens_per_cta, c.tokens - t0);
  pdl_wait();
  pdl_trigger();
  if (threadIdx.x < nt) {
    const int t = t0 + threadIdx.x, b = seq_of(c, t);
    const SeqSpan s = seq_span(c, b);
    int pos = s.kv - s.qlen + (t - s.q0);
    int64_t slot = -1;
    if (t < s.q0 || t >= s.q0 + s.qlen || pos < 0 || pos >= a.max_pos) {
      // (a row before the first sequence or past the last is nobody's, and no error)
      if (t >= c.q_start[0] && t < c.q_start[c.batch]) atomicOr(c.status, kStatusBadIndex);
      pos = -1;
    } else {
      const int page = page_of(c, b, pos);
      if (page >= 0) slot = page * c.page_stride + (pos % c.page_size) * c.row_stride;
    }
    pos_of[threadIdx.x] = pos;
    slot_of[threadIdx.x] = slot;
  }
  const int per = kRopeThreads / a.tokens_per_cta;  // threads of a token
  const int ti = threadIdx.x / per, step = per / LPH, heads = a.nq + 2 * c.nkv;
  const int l = threadIdx.x % LPH, pairs = a.rot / 16;
  const int d0 = l < pairs ? 8 * l : a.rot + 16 * (l - pairs);
  const int d1 = l < pairs ? a.rot / 2 + 8 * l : d0 + 8;
  if (ti >= nt) {
    __syncthreads();
    return;
  }
  int head = (threadIdx.x % per) / LPH;
  const int64_t row = static_cast<int64_t>(t0 + ti) * a.qkv_stride;
  Raw8<F32> n0, n1;
  if (head < heads) {
    n0.load(a.qkv, row + head * HD + d0);
    n1.load(a.qkv, row + head * HD + d1);
  }
  __syncthreads();
  const int pos = pos_of[ti];
  if (pos < 0) return;
  Raw8<TF32> cs, sn;
  if (l < pairs) {
    const int64_t at = static_cast<int64_t>(pos) * 2 * a.rot + d0;
    cs.load(a.table, at);
    sn.load(a.table, at + a.rot);
  }
  float w0[8], w1[8];
  const float* held = nullptr;
  // (a warp's lanes stay together: the first lane's head is the lowest)
  for (; head - static_cast<int>(threadIdx.x & 31) / LPH < heads; head += step) {
    const bool real = head < heads, is_q = head < a.nq, is_k = !is_q && head < a.nq + c.nkv;
    float x0[8] = {}, x1[8] = {};
    if (real) {
      n0.get(x0);
      n1.get(x1);
    }
    if (head + step < heads) {
      n0.load(a.qkv, row + (head + step) * HD + d0);
      n1.load(a.qkv, row + (head + step) * HD + d1);
    }
    const float* w = is_q ? a.qw : (is_k ? a.kw : nullptr);
    if (a.qw || a.kw) {
      if (w && w != held) {
        load8<true>(w, d0, w0);
        load8<true>(w, d1, w1);
        held = w;
      }
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += x0[e] * x0[e] + x1[e] * x1[e];
#pragma unroll
      for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (w) {
        const float inv = 1.0f / sqrtf(ss / static_cast<float>(HD) + a.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x0[e] = x0[e] * inv * w0[e];
          x1[e] = x1[e] * inv * w1[e];
        }
      }
    }
    if (!real) continue;
    if (l < pairs && (is_q || is_k)) {
      float co[8], si[8];
      cs.get(co);
      sn.get(si);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y0 = x0[e] * co[e] - x1[e] * si[e], y1 = x1[e] * co[e] + x0[e] * si[e];
        x0[e] = y0;
        x1[e] = y1;
      }
    }
    uint16_t* dst;
    if (is_q) {
      dst = a.q_out + static_cast<int64_t>(t0 + ti) * a.q_tok + head * a.q_head;
    } else {
      if (slot_of[ti] < 0) continue;
      dst = (is_k ? c.k : c.v) + slot_of[ti] + (head - a.nq - (is_k ? 0 : c.nkv)) * c.head_stride;
    }
    store8(dst + d0, x0);
    store8(dst + d1, x1);
  }
}

template <int HD>
int launch_rope(alv_ctx* ctx, const RopeArgs& a, bool xf, bool tf, cudaStream_t st) {
  auto k = xf ? (tf ? qk_norm_rope_kernel<HD, true, true> : qk_norm_rope_kernel<HD, true, false>)
              : (tf ? qk_norm_rope_kernel<HD, false, true> : qk_norm_rope_kernel<HD, false, false>);
  const unsigned grid = static_cast<unsigned>((a.c.tokens + a.tokens_per_cta - 1) / a.tokens_per_cta);
  return launch_ex(ctx, k, dim3(grid), dim3(kRopeThreads), 0, st, true, a);
}

}  // namespace

int make_paged_view(alv_ctx* ctx, const char* who, const alv_paged* p, PagedView* out) {
  const std::string w(who);
  if (!p || p->batch < 0 || p->tokens < 0 || !p->k || !p->v || (p->batch && (!p->table || !p->q_start || !p->kv_lens)))
    return fail(ctx, ALV_ERR_ARG, w + ": null pointer or negative size in the paged cache");
  if (p->pages < 1 || p->kv_heads < 1 || p->page_size < 1 || p->table_width < 1 || p->table_stride < 0)
    return fail(ctx, ALV_ERR_ARG, w + ": pages, kv_heads, page_size and table_width must be positive, table_stride not negative");
  if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256)
    return fail(ctx, ALV_ERR_SHAPE, w + ": head_dim must be 64, 128 or 256");
  if (p->page_size % 16) return fail(ctx, ALV_ERR_SHAPE, w + ": page_size must be a multiple of 16");
  if (static_cast<int64_t>(p->table_width) * p->page_size > INT_MAX)
    return fail(ctx, ALV_ERR_UNSUPPORTED, w + ": a sequence may hold at most 2^31 - 1 positions");
  if (p->row_stride < p->head_dim || p->head_stride < 1 || p->page_stride < 1 || p->row_stride >= kMaxMapStride ||
      p->head_stride >= kMaxMapStride || p->page_stride >= kMaxMapStride)
    return fail(ctx, ALV_ERR_ARG, w + ": the pages' strides must be positive (no broadcast), rows of head_dim values apart");
  if (p->row_stride % 8 || p->head_stride % 8 || p->page_stride % 8 || ((reinterpret_cast<uintptr_t>(p->k) | reinterpret_cast<uintptr_t>(p->v)) & 15))
    return fail(ctx, ALV_ERR_ARG, w + ": k, v must be 16-byte aligned with strides of whole 16 bytes");
  int rc = ensure_scratch(ctx, 0);
  if (rc) return rc;
  *out = PagedView{p->k,         p->v,           p->page_stride, p->head_stride, p->row_stride, p->pages, p->page_size,
                   p->kv_heads,  p->table,       p->table_stride, p->table_width, p->q_start,   p->kv_lens, p->batch,
                   p->tokens,    status_ptr(ctx)};
  return ALV_OK;
}

}  // namespace alv

using namespace alv;

extern "C" int alv_qk_norm_rope(alv_ctx* ctx, const alv_paged* cache, const alv_qk_norm_rope_args* args, void* stream) {
  if (!ctx || !cache || !args) return fail(ctx, ALV_ERR_ARG, "qk_norm_rope: bad argument");
  int rc = set_device(ctx);
  if (rc) return rc;
  RopeArgs a{};
  if ((rc = make_paged_view(ctx, "qk_norm_rope", cache, &a.c))) return rc;
  const int hd = cache->head_dim;
  if ((cache->tokens && (!args->qkv || !args->q_out)) || !args->rope || !valid_dtype(args->qkv_dtype) || !valid_dtype(args->rope_dtype) ||
      args->heads < 1 || args->max_pos < 1 || !(args->eps >= 0.f))
    return fail(ctx, ALV_ERR_ARG, "qk_norm_rope: bad argument");
  if (args->rot < 16 || args->rot > hd || args->rot % 16)
    return fail(ctx, ALV_ERR_SHAPE, "qk_norm_rope: the rotated dims must be a multiple of 16, at most head_dim");
  if (args->qkv_stride < 0 || args->qkv_stride % 8 || args->q_token_stride % 8 ||
      args->q_head_stride % 8 || args->q_token_stride < 0 || args->q_head_stride < 0 ||
      ((reinterpret_cast<uintptr_t>(args->qkv) | reinterpret_cast<uintptr_t>(args->q_out) |
        reinterpret_cast<uintptr_t>(args->rope) | reinterpret_cast<uintptr_t>(args->q_weight) |
        reinterpret_cast<uintptr_t>(args->k_weight)) & 15))
    return fail(ctx, ALV_ERR_ARG, "qk_norm_rope: buffers must be 16-byte aligned with strides of whole 16 bytes");
  a.qkv = args->qkv;
  a.qkv_stride = args->qkv_stride;
  a.q_out = args->q_out;
  a.q_tok = args->q_token_stride;
  a.q_head = args->q_head_stride;
  a.table = args->rope;
  a.max_pos = args->max_pos;
  a.rot = args->rot;
  a.nq = args->heads;
  a.qw = args->q_weight;
  a.kw = args->k_weight;
  a.eps = args->eps;
  if (cache->tokens == 0 || cache->batch == 0) return ALV_OK;
  // a token per CTA while that leaves SMs idle, then up to 8: the look-up of a
  // CTA's tokens is shared, and a warp's cos, sin and weights by more heads
  a.tokens_per_cta = 1;
  while (a.tokens_per_cta < kRopeTokens && cache->tokens >= ctx->num_sms * 8 * a.tokens_per_cta) a.tokens_per_cta *= 2;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool xf = args->qkv_dtype == ALV_F32, tf = args->rope_dtype == ALV_F32;
  switch (hd) {
    case 64: return launch_rope<64>(ctx, a, xf, tf, st);
    case 128: return launch_rope<128>(ctx, a, xf, tf, st);
    default: return launch_rope<256>(ctx, a, xf, tf, st);
  }
}
