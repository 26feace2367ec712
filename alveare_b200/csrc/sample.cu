// Host side of the C ABI, part 10: token sampling from given uniform numbers.
//
//   s_i = l_i / T,  w_i = exp(s_i - max s),  mass_i = floor(w_i 2^40)
//   top-k: the k first in the order (s descending, index ascending);
//   top-p: the shortest prefix of those with mass >= ceil(p * their mass);
//   min-p: of those, w_i >= min_p;
//   token: the first, in index order, whose running mass passes floor(u * total).
//
// The masses are integers (w is exact to 2^-40 below 1, a vocabulary of 2^20
// sums to at most 2^60), so sums of any order and atomics give one result.
// The prefix's end is found by radix selection on s's bits (mapped so that
// unsigned order is s's order): a histogram of counts and masses per digit,
// the digit where the k-th element (or the wanted mass) falls, then the next
// digit among its elements.  Elements equal to the last one kept enter in
// index order.
#include "internal.h"

namespace alv {
namespace {

constexpr int kSampleThreads = 1024;
typedef unsigned long long u64;

struct SampleArgs {
  const void* logits;
  int64_t stride;
  const float* u;
  int* tokens;
  float* logprobs;
  const float *t_rows, *p_rows, *m_rows;
  const int* k_rows;
  int vocab, k;
  float t, p, m;
};

// s's bits, ordered: key(a) < key(b) exactly when a < b (-0 counts as +0, NaN as -inf).
__device__ __forceinline__ uint32_t key_of(float s) {
  if (s != s) s = -INFINITY;
  const uint32_t b = __float_as_uint(s + 0.0f == 0.0f ? 0.0f : s);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// w of the element with key k when the row's largest value is `top`.
__device__ __forceinline__ float weight(uint32_t k, float top) {
  const float s = key_value(k);
  if (top == INFINITY) return s == INFINITY ? 1.f : 0.f;
  return expf(s - top);
}
__device__ __forceinline__ u64 mass_of(float w) { return static_cast<u64>(w * 1099511627776.0f); }

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
  if (warp == 0) {
    u64 w = sh[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    sh[lane] = w;
  }
  __syncthreads();
  *total = sh[31];
  return x + (warp ? sh[warp - 1] : 0);
}

struct Cut {  // kept: key > key_last, and the first `ties` (in index order) of key == key_last
  uint32_t key;
  u64 ties;
  u64 mass;  // of everything kept
};

template <bool BF16>
struct Row {
  const void* base;
  int vocab;
  float temp;
  bool greedy;
  __device__ __forceinline__ uint32_t key(int i) const {
    float x = BF16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(base)[i]) : static_cast<const float*>(base)[i];
    if (!greedy) x = __fdiv_rn(x, temp);
    return key_of(x);
  }
};

// The prefix of the row (in (s descending, index ascending) order) that ends
// where the count reaches `want_n`, or (by_mass) the mass reaches `want_m`.
template <bool BF16>
__device__ Cut select(const Row<BF16>& row, float top, bool by_mass, u64 want_n, u64 want_m, unsigned* hn, u64* hm) {
  __shared__ uint32_t pick;
  __shared__ u64 before_n, before_m, in_n, in_m;
  uint32_t prefix = 0;
  u64 acc_n = 0, acc_m = 0, cnt = 0, ms = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int d = threadIdx.x; d < 256; d += blockDim.x) hn[d] = 0, hm[d] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < row.vocab; i += blockDim.x) {
      const uint32_t k = row.key(i);
      if (shift < 24 && (k >> (shift + 8)) != prefix) continue;
      atomicAdd(hn + ((k >> shift) & 255), 1u);
      atomicAdd(hm + ((k >> shift) & 255), mass_of(weight(k, top)));
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      u64 n = acc_n, m = acc_m;
      int d = 255;
      for (; d > 0; --d) {
        if (by_mass ? m + hm[d] >= want_m : n + hn[d] >= want_n) break;
        n += hn[d];
        m += hm[d];
      }
      pick = d;
      before_n = n;
      before_m = m;
      in_n = hn[d];
      in_m = hm[d];
    }
    __syncthreads();
    prefix = (prefix << 8) | pick;
    acc_n = before_n;
    acc_m = before_m;
    cnt = in_n;
    ms = in_m;
    __syncthreads();
  }
  // every element left equals the key; each holds the same mass
  const u64 each = cnt ? ms / cnt : 0;
  u64 ties = by_mass ? (each && want_m > acc_m ? (want_m - acc_m + each - 1) / each : 1) : want_n - acc_n;
  if (ties > cnt) ties = cnt;
  return {prefix, ties, acc_m + ties * each};
}

template <bool BF16>
__global__ void __launch_bounds__(kSampleThreads, 1) sample_kernel(const SampleArgs a) {
  __shared__ unsigned hn[256];
  __shared__ u64 hm[256], sh[32];
  __shared__ uint32_t wk[32];
  __shared__ int wi[32], chosen;
  __shared__ u64 chosen_mass;
  const int r = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Row<BF16> row;
  row.base = static_cast<const char*>(a.logits) + r * a.stride * (BF16 ? 2 : 4);
  row.vocab = a.vocab;
  row.temp = a.t_rows ? a.t_rows[r] : a.t;
  row.greedy = !(row.temp > 0.f);
  const int k = a.k_rows ? a.k_rows[r] : a.k;
  const float p = a.p_rows ? a.p_rows[r] : a.p, min_p = fminf(a.m_rows ? a.m_rows[r] : a.m, 1.f);

  // the largest value and its first index
  uint32_t best = 0;
  int bi = INT_MAX;
  for (int i = threadIdx.x; i < a.vocab; i += blockDim.x) {
    const uint32_t key = row.key(i);
    if (key > best) best = key, bi = i;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint32_t ok = __shfl_xor_sync(0xffffffffu, best, o);
    const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
    if (ok > best || (ok == best && oi < bi)) best = ok, bi = oi;
  }
  if (lane == 0) wk[warp] = best, wi[warp] = bi;
  __syncthreads();
  for (int w = 0; w < 32; ++w)
    if (wk[w] > best || (wk[w] == best && wi[w] < bi)) best = wk[w], bi = wi[w];
  const float top = key_value(best);
  if (row.greedy || top == -INFINITY) {
    if (threadIdx.x == 0) {
      a.tokens[r] = top == -INFINITY ? -1 : bi;
      if (a.logprobs) a.logprobs[r] = top == -INFINITY ? -INFINITY : 0.f;
    }
    return;
  }
  Cut cut{0, ~0ull, 0};
  const bool by_k = k > 0 && k < a.vocab, by_p = p < 1.f;
  if (by_k) cut = select(row, top, false, static_cast<u64>(k), 0, hn, hm);
  if (by_p) {
    if (!by_k) {
      u64 m = 0;
      for (int i = threadIdx.x; i < a.vocab; i += blockDim.x) m += mass_of(weight(row.key(i), top));
      cta_scan(m, &cut.mass, sh);
    }
    const double goal = ceil(static_cast<double>(cut.mass) * static_cast<double>(p));
    cut = select(row, top, true, 0, goal >= 1.0 ? static_cast<u64>(goal) : 1, hn, hm);
  }
  // two walks in index order: the kept mass, then the token
  u64 total = 0;
  for (int walk = 0; walk < 2; ++walk) {
    u64 goal = 0;
    if (walk) {
      const u64 x = static_cast<u64>(fmax(floor(static_cast<double>(a.u[r]) * static_cast<double>(total)), 0.0));
      goal = x < total ? x : total - 1;
      if (threadIdx.x == 0) chosen = INT_MAX;
      __syncthreads();
    }
    u64 ties = 0, run = 0, t;
    for (int base = 0; base < a.vocab; base += blockDim.x) {
      const int i = base + threadIdx.x;
      const uint32_t key = i < a.vocab ? row.key(i) : 0;
      const bool tie = i < a.vocab && key == cut.key;
      const u64 rank = ties + cta_scan(tie ? 1 : 0, &t, sh);
      ties += t;
      u64 mass = 0;
      if (i < a.vocab && (key > cut.key || (tie && rank <= cut.ties))) {
        const float w = weight(key, top);
        if (w >= min_p) mass = mass_of(w);
      }
      const u64 upto = run + cta_scan(mass, &t, sh);
      run += t;
      if (walk && upto > goal && upto - mass <= goal) {
        chosen = i;
        chosen_mass = mass;
      }
    }
    total = run;
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    a.tokens[r] = chosen;
    if (a.logprobs)
      a.logprobs[r] = static_cast<float>(log(static_cast<double>(chosen_mass) / static_cast<double>(total)));
  }
}

}  // namespace
}  // namespace alv

using namespace alv;

extern "C" int alv_sample(alv_ctx* ctx, const alv_sample_args* s, void* stream) {
  if (!ctx || !s) return fail(ctx, ALV_ERR_ARG, "sample: bad argument");
  if (s->rows < 0 || s->vocab < 1 || !valid_dtype(s->logits_dtype) || (s->rows && (!s->logits || !s->u || !s->tokens)) ||
      s->logits_stride < s->vocab)
    return fail(ctx, ALV_ERR_ARG, "sample: bad argument");
  if (s->vocab > 1 << 20) return fail(ctx, ALV_ERR_UNSUPPORTED, "sample: at most 1,048,576 tokens");
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
  auto k = s->logits_dtype == ALV_BF16 ? sample_kernel<true> : sample_kernel<false>;
  k<<<s->rows, kSampleThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
  ALV_CUDA(ctx, cudaGetLastError());
  return ALV_OK;
}
