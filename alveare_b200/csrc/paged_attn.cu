// Host side of the C ABI, part 8: attention over a paged cache, and its
// kernel for row blocks (paged_attn.cuh has the mathematics).
#include "internal.h"
#include "paged_attn.cuh"

namespace alv {
namespace {

// One warp's online-softmax state over the slices it takes.
template <int HD>
struct RowState {
  float o[HD / 8][4];  // C fragments: rows g, g + 8 (g = lane / 4), dims 8n + 2t, +1 (t = lane % 4)
  float m[2], l[2];
};

template <int HD>
__global__ void __launch_bounds__(kRowWarps * 32, 1) paged_rows_kernel(const AttnArgs a) {
  using R = RowRing<HD>;
  constexpr int NS = R::kSlots, CH = HD / 8;  // 16-byte chunks per row
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int kvh = blockIdx.y, b = blockIdx.z;
  const SeqSpan s = seq_span(a.c, b);
  const int r0 = blockIdx.x * kRowsPerBlock;
  const int64_t rows = static_cast<int64_t>(s.qlen) * a.group;
  const int nrow = static_cast<int>(min(static_cast<int64_t>(kRowsPerBlock), rows - r0));
  if (nrow <= 0 || rows > a.row_max) return;
  const int pfirst = s.kv - s.qlen;  // position of the sequence's first new token
  const int p0 = pfirst + r0 / a.group, p1 = pfirst + (r0 + nrow - 1) / a.group;
  const SliceRange sr = slice_range<kSlice>(p0, p1, a.window, a.sinks);

  // q rows (row r = token r / group, head kvh * group + r % group)
  uint8_t* qs = smem;
  const uint32_t q_sm = smem_u32(smem), ring = q_sm + R::kQBytes + warp * NS * R::kSlotBytes;
  for (int e = threadIdx.x; e < kRowsPerBlock * CH; e += blockDim.x) {
    const int r = e / CH, c = e % CH;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r < nrow) {
      const int tok = s.q0 + (r0 + r) / a.group, head = kvh * a.group + (r0 + r) % a.group;
      v = *reinterpret_cast<const uint4*>(a.q + tok * a.q_tok + head * a.q_head + c * 8);
    }
    *reinterpret_cast<uint4*>(qs + r * HD * 2 + ((c ^ (r & 7)) << 4)) = v;
  }
  __syncthreads();

  const int n_mine = (sr.count() - warp + kRowWarps - 1) / kRowWarps;  // slices warp, warp + 8, ...
  // Start the copy of half h (k of slice h / 2, or v) into its slot.
  auto copy = [&](int h) {
    if (h < 2 * n_mine) {
      const int j0 = sr.slice(warp + (h >> 1) * kRowWarps) * kSlice;
      const int page = page_of(a.c, b, j0);
      const uint16_t* base = ((h & 1) ? a.c.v : a.c.k) + max(page, 0) * a.c.page_stride + kvh * a.c.head_stride +
                             (j0 % a.c.page_size) * a.c.row_stride;
      const uint32_t dst = ring + (h % NS) * R::kSlotBytes;
#pragma unroll
      for (int e = lane; e < kSlice * CH; e += 32) {
        const int r = e / CH, c = e % CH, j = j0 + r;
        const bool ok = page >= 0 && j < sr.hi && (j >= sr.lo || j < a.sinks);  // else zeros: never read
        cp_async16(dst + r * HD * 2 + ((c ^ (r & 7)) << 4), base + (ok ? r * a.c.row_stride + c * 8 : 0), ok ? 16u : 0u);
      }
    }
    cp_async_commit();
  };
  RowState<HD> st;
#pragma unroll
  for (int n = 0; n < HD / 8; ++n) st.o[n][0] = st.o[n][1] = st.o[n][2] = st.o[n][3] = 0.f;
  st.m[0] = st.m[1] = -INFINITY;
  st.l[0] = st.l[1] = 0.f;
  // positions of this lane's two rows
  const int pr[2] = {pfirst + (r0 + g) / a.group, pfirst + (r0 + g + 8) / a.group};
  const bool one_token = p0 == p1;
  for (int h = 0; h < NS - 1; ++h) copy(h);
  for (int i = 0; i < n_mine; ++i) {
    const int j0 = sr.slice(warp + i * kRowWarps) * kSlice;
    // scores of the slice: two n-tiles of 8 positions
    cp_async_wait<NS - 2>();
    __syncwarp();
    copy(2 * i + NS - 1);
    float sc[2][4] = {};
    const uint32_t ks = ring + ((2 * i) % NS) * R::kSlotBytes;
#pragma unroll
    for (int k = 0; k < HD / 16; ++k) {
      uint32_t qa[4], kb[4];
      const int qr = lane & 15, qc = 2 * k + (lane >> 4);
      ldsm4(q_sm + qr * HD * 2 + ((qc ^ (qr & 7)) << 4), qa);
      const int kr = (lane & 7) + ((lane >> 4) << 3), kc = 2 * k + ((lane >> 3) & 1);
      ldsm4(ks + kr * HD * 2 + ((kc ^ (kr & 7)) << 4), kb);
      mma_16816(sc[0], qa[0], qa[1], qa[2], qa[3], kb[0], kb[1]);
      mma_16816(sc[1], qa[0], qa[1], qa[2], qa[3], kb[2], kb[3]);
    }
    // every row sees the whole slice?
    const bool whole = j0 + kSlice - 1 <= p0 && (a.window == 0 || j0 > p1 - a.window || j0 + kSlice <= a.sinks);
    const bool paged = page_of(a.c, b, j0) >= 0;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = j0 + 8 * n + 2 * t + (e & 1);
        sc[n][e] = paged && (whole || sees(j, pr[e >> 1], a.window, a.sinks)) ? sc[n][e] * a.scale_log2 : -INFINITY;
      }
    float f[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float mx = fmaxf(fmaxf(sc[0][2 * r], sc[0][2 * r + 1]), fmaxf(sc[1][2 * r], sc[1][2 * r + 1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      mx = fmaxf(mx, st.m[r]);
      const float base = mx == -INFINITY ? 0.f : mx;
      f[r] = exp2_fast(st.m[r] - base);
      st.m[r] = mx;
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float p = exp2_fast(sc[n][2 * r + e] - base);
          sc[n][2 * r + e] = p;
          sum += p;
        }
      st.l[r] = st.l[r] * f[r] + sum;  // this lane's four columns; lanes are added at the end
    }
    if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
      for (int n = 0; n < HD / 8; ++n) {
        st.o[n][0] *= f[0];
        st.o[n][1] *= f[0];
        st.o[n][2] *= f[1];
        st.o[n][3] *= f[1];
      }
    }
    const uint32_t pa[4] = {pack_bf2_rn(sc[0][0], sc[0][1]), pack_bf2_rn(sc[0][2], sc[0][3]),
                            pack_bf2_rn(sc[1][0], sc[1][1]), pack_bf2_rn(sc[1][2], sc[1][3])};
    cp_async_wait<NS - 2>();
    __syncwarp();
    copy(2 * i + NS);
    const uint32_t vs = ring + ((2 * i + 1) % NS) * R::kSlotBytes;
    const bool mixed = !whole && !one_token;
#pragma unroll
    for (int n = 0; n < HD / 16; ++n) {
      uint32_t vb[4];
      const int vr = lane & 15, vc = 2 * n + (lane >> 4);
      ldsm4_t(vs + vr * HD * 2 + ((vc ^ (vr & 7)) << 4), vb);
      // A value that is not finite must not reach the rows that do not see
      // its position (0 * inf): then each token's rows take their own product.
      if (mixed && __any_sync(0xffffffffu, bf2_nonfinite(vb[0]) | bf2_nonfinite(vb[1]) | bf2_nonfinite(vb[2]) |
                                               bf2_nonfinite(vb[3]))) {
        for (int pt = p0; pt <= p1; ++pt) {
          uint32_t mk[2];
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            const int j = j0 + 8 * hh + 2 * t;
            mk[hh] = (sees(j, pt, a.window, a.sinks) ? 0xFFFFu : 0u) |
                     (sees(j + 1, pt, a.window, a.sinks) ? 0xFFFF0000u : 0u);
          }
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            float tmp[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) tmp[e] = st.o[2 * n + hh][e];
            mma_16816(tmp, pa[0], pa[1], pa[2], pa[3], vb[2 * hh] & mk[0], vb[2 * hh + 1] & mk[1]);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (pr[e >> 1] == pt) st.o[2 * n + hh][e] = tmp[e];
          }
        }
      } else {
        mma_16816(st.o[2 * n], pa[0], pa[1], pa[2], pa[3], vb[0], vb[1]);
        mma_16816(st.o[2 * n + 1], pa[0], pa[1], pa[2], pa[3], vb[2], vb[3]);
      }
    }
  }
  cp_async_wait<0>();
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    st.l[r] += __shfl_xor_sync(0xffffffffu, st.l[r], 1);
    st.l[r] += __shfl_xor_sync(0xffffffffu, st.l[r], 2);
  }
  // join the warps in warp order
  __syncthreads();
  float* jm = reinterpret_cast<float*>(smem + R::kQBytes);
  float* jl = jm + kRowWarps * kRowsPerBlock;
  float* jo = jl + kRowWarps * kRowsPerBlock;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = warp * kRowsPerBlock + g + 8 * r;
    if (t == 0) {
      jm[row] = st.m[r];
      jl[row] = st.l[r];
    }
    if (g + 8 * r < nrow) {
#pragma unroll
      for (int n = 0; n < HD / 8; ++n)
        *reinterpret_cast<float2*>(jo + row * HD + 8 * n + 2 * t) = make_float2(st.o[n][2 * r], st.o[n][2 * r + 1]);
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < nrow * (HD / 2); e += blockDim.x) {
    const int r = e / (HD / 2), d = (e % (HD / 2)) * 2;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) m = fmaxf(m, jm[w * kRowsPerBlock + r]);
    const float base = m == -INFINITY ? 0.f : m;
    float l = 0.f, x = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) {
      const int row = w * kRowsPerBlock + r;
      const float f = exp2_fast(jm[row] - base);
      const float2 o = *reinterpret_cast<const float2*>(jo + row * HD + d);
      l += f * jl[row];
      x += f * o.x;
      y += f * o.y;
    }
    const float inv = m == -INFINITY ? 0.f : 1.f / l;  // a row that sees nothing gives zeros
    const int tok = s.q0 + (r0 + r) / a.group, head = kvh * a.group + (r0 + r) % a.group;
    *reinterpret_cast<uint32_t*>(a.out + tok * a.o_tok + head * a.o_head + d) = pack_bf2_rn(x * inv, y * inv);
  }
}

template <int HD>
int launch_rows(alv_ctx* ctx, const AttnArgs& a, int max_q_len, cudaStream_t st) {
  auto k = paged_rows_kernel<HD>;
  const size_t smem = RowRing<HD>::kBytes;
  int rc = prepare_kernel(ctx, k, smem);
  if (rc) return rc;
  const int64_t rows = std::min<int64_t>(static_cast<int64_t>(max_q_len) * a.group, a.row_max);
  const dim3 grid(static_cast<unsigned>((rows + kRowsPerBlock - 1) / kRowsPerBlock), a.c.nkv, a.c.batch);
  k<<<grid, kRowWarps * 32, smem, st>>>(a);
  ALV_CUDA(ctx, cudaGetLastError());
  return ALV_OK;
}

}  // namespace
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
  if (cache->batch > 65535 || cache->kv_heads > 65535)
    return fail(ctx, ALV_ERR_UNSUPPORTED, "paged_attention: at most 65,535 sequences and kv heads in one call");
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
    if ((rc = launch_chunk(ctx, a, cache->head_dim, kRowsPerBlock + 1, st))) return rc;
    // all sequences as long as the longest: none is left for the row blocks
    if (static_cast<int64_t>(cache->batch) * args->max_q_len == cache->tokens) return ALV_OK;
  }
  switch (cache->head_dim) {
    case 64: return launch_rows<64>(ctx, a, args->max_q_len, st);
    case 128: return launch_rows<128>(ctx, a, args->max_q_len, st);
    default: return launch_rows<256>(ctx, a, args->max_q_len, st);
  }
}
