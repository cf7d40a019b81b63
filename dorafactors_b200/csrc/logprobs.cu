// Log probabilities of given tokens, with logsumexp, entropy and the most likely
// alternatives of each row of logits, and the gradient.
//
//   x'_j = x_j / T,  L = log sum_j exp x'_j,  log p_j = x'_j - L
//   logprob = log p_t,  entropy H = -sum_j p_j log p_j,  top = the k largest log p_j
//   dx_j = (g_lp (1[j = t] - p_j) - g_H p_j (log p_j + H) + g_L p_j) / T
//
// With M the row's maximum, d_j = x_j - M and t_j = log2(e) / T d_j, so that the largest
// term is 2^0 = 1 exactly and no logit, however large, overflows; sums are fp32, those of
// the threads are joined in fp64, and L - M / T = log1p(sum - 1) keeps what a peaked
// distribution has besides its peak.
//
// A row whose target is ignore_index is not read: its outputs are 0 (indices -1) and
// its gradient is 0.  A target outside the vocabulary gives NaN, and sets the device
// error word.  A row of -inf alone has L = -inf, log probabilities -inf, entropy 0 and
// gradient 0; a row with a NaN or +inf has no distribution: its values are NaN and its
// alternatives are columns 0 .. k-1.
#include <math_constants.h>

#include "dora_common.cuh"

namespace dora {
namespace {

constexpr int kT = 256;
constexpr int kMaxTop = 64;

constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kLog2e = 1.44269504088896340736f;
// From this size on an fp32 logsumexp has lost the part that normalises (2^-24 of it):
// the gradient then takes the row's maximum and sum anew.
constexpr float kWideLse = 256.f;

__device__ __forceinline__ float exp2_approx(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}

// Total order of a row's elements: larger value first, lower column on ties.
__device__ __forceinline__ unsigned long long order_key(float v, uint32_t col) {
  v += 0.0f;  // -0 and +0 are the same value
  const uint32_t b = __float_as_uint(v);
  const uint32_t o = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return (static_cast<unsigned long long>(o) << 32) | (0xffffffffu - col);
}
__device__ __forceinline__ float key_value(unsigned long long k) {
  const uint32_t o = uint32_t(k >> 32);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ uint32_t key_col(unsigned long long k) { return 0xffffffffu - uint32_t(k); }

template <typename V, typename Op>
__device__ __forceinline__ V block_fold(V v, V* red, Op op) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  V t = red[0];
  for (int w = 1; w < kT / 32; ++w) t = op(t, red[w]);
  __syncthreads();
  return t;
}

struct Sum {
  template <typename V> __device__ V operator()(V a, V b) const { return a + b; }
};
struct Max {
  __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
  __device__ unsigned long long operator()(unsigned long long a, unsigned long long b) const { return a > b ? a : b; }
};

template <typename T>
__global__ void __launch_bounds__(kT)
logprobs_fwd_kernel(const T* __restrict__ logits, int64_t ld, const int64_t* __restrict__ targets, int64_t ignore,
                    float s, float inv_temp, float* __restrict__ logprobs, float* __restrict__ lse,
                    float* __restrict__ entropy, int k, float* __restrict__ top_lp, int64_t* __restrict__ top_idx,
                    int64_t rows, int64_t vocab) {
  __shared__ float red[kT / 32];
  __shared__ double redd[kT / 32];
  __shared__ unsigned long long redk[kT / 32];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const int64_t target = targets[r];
    if (target == ignore) {
      if (threadIdx.x == 0) {
        logprobs[r] = 0.f;
        lse[r] = 0.f;
        if (entropy) entropy[r] = 0.f;
      }
      for (int i = threadIdx.x; i < k; i += kT) {
        top_lp[r * k + i] = 0.f;
        top_idx[r * k + i] = -1;
      }
      continue;
    }
    const T* x = logits + r * ld;
    float m = -CUDART_INF_F;
    for (int64_t c = threadIdx.x; c < vocab; c += kT) m = fmaxf(m, to_f32(x[c]));
    m = block_fold(m, red, Max());
    const float m0 = m == -CUDART_INF_F ? 0.f : m;
    float sum = 0.f, dot = 0.f;
    for (int64_t c = threadIdx.x; c < vocab; c += kT) {
      const float t = (to_f32(x[c]) - m0) * s;
      const float e = exp2_approx(t);
      sum += e;
      dot = fmaf(e, fmaxf(t, -200.f), dot);
    }
    const double total = block_fold(double(sum), redd, Sum());
    const double dots = block_fold(double(dot), redd, Sum());
    const bool none = m == -CUDART_INF_F && total == 0.0;  // every logit is -inf
    const float ln_sum = none ? -CUDART_INF_F : log1pf(float(total - 1.0));
    if (threadIdx.x == 0) {
      float lp = CUDART_NAN_F;
      if (target >= 0 && target < vocab) lp = none ? -CUDART_INF_F : fmaf(to_f32(x[target]) - m0, inv_temp, -ln_sum);
      else record_device_error(DORA_ERR_INVALID_ARGUMENT);
      logprobs[r] = lp;
      lse[r] = none ? -CUDART_INF_F : fmaf(m0, inv_temp, ln_sum);
      if (entropy) entropy[r] = none ? 0.f : ln_sum - kLn2 * float(dots / total);
    }
    unsigned long long last = ~0ull;
    const bool bad = !(total < CUDART_INF);
    for (int i = 0; i < k; ++i) {
      unsigned long long best = 0;
      if (!bad)
        for (int64_t c = threadIdx.x; c < vocab; c += kT) {
          const unsigned long long q = order_key(to_f32(x[c]), uint32_t(c));
          if (q < last && q > best) best = q;
        }
      best = block_fold(best, redk, Max());
      last = best;
      if (threadIdx.x == 0) {
        top_lp[r * k + i] = bad ? CUDART_NAN_F : none ? -CUDART_INF_F : fmaf(key_value(best) - m0, inv_temp, -ln_sum);
        top_idx[r * k + i] = bad ? i : key_col(best);
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kT)
logprobs_bwd_kernel(const T* logits, int64_t ld, const int64_t* __restrict__ targets, int64_t ignore, float s,
                    float inv_temp, const float* __restrict__ lse, const float* __restrict__ entropy,
                    const float* __restrict__ g_lp, const float* __restrict__ g_ent, const float* __restrict__ g_lse,
                    T* d, int64_t ldd, int64_t rows, int64_t vocab) {
  __shared__ float red[kT / 32];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const int64_t target = targets[r];
    const T* x = logits + r * ld;
    T* o = d + r * ldd;
    float L = lse[r];
    if (target == ignore || L == -CUDART_INF_F) {
      for (int64_t c = threadIdx.x; c < vocab; c += kT) o[c] = from_f32<T>(0.f);
      continue;
    }
    float m = 0.f;  // log p_j = (x_j - m) / T - L
    if (fabsf(L) > kWideLse) {
      m = -CUDART_INF_F;
      for (int64_t c = threadIdx.x; c < vocab; c += kT) m = fmaxf(m, to_f32(x[c]));
      m = block_fold(m, red, Max());
      float sum = 0.f;
      for (int64_t c = threadIdx.x; c < vocab; c += kT) sum += exp2_approx((to_f32(x[c]) - m) * s);
      L = logf(block_fold(sum, red, Sum()));
    }
    const float glp = g_lp ? g_lp[r] : 0.f, gl = g_lse ? g_lse[r] : 0.f, ge = g_ent ? g_ent[r] : 0.f;
    // dx_j = p_j (a + b log p_j) + 1[j = t] g_lp / T
    const float a = (gl - glp - (g_ent ? ge * entropy[r] : 0.f)) * inv_temp, b = -ge * inv_temp;
    for (int64_t c = threadIdx.x; c < vocab; c += kT) {
      const float lp = fmaf(to_f32(x[c]) - m, inv_temp, -L);
      float v = exp2_approx(lp * kLog2e) * fmaf(b, fmaxf(lp, -200.f), a);
      if (c == target) v = fmaf(glp, inv_temp, v);
      o[c] = from_f32<T>(v);
    }
  }
}

unsigned row_grid(int64_t rows) { return unsigned(rows < (1 << 20) ? rows : (1 << 20)); }

bool args_ok(int64_t rows, int64_t vocab, int64_t ld, double temperature, int dtype) {
  return rows >= 0 && vocab >= 1 && vocab < (int64_t(1) << 31) && ld >= vocab && rows <= (int64_t(1) << 40) &&
         dtype_ok(dtype) && temperature > 0 && temperature <= 1e30 && temperature >= 1e-30;
}

template <typename F> int by_type(int dtype, F f) {
  switch (dtype) {
    case DORA_DTYPE_BF16: return f(__nv_bfloat16());
    case DORA_DTYPE_F16: return f(__half());
    default: return f(float());
  }
}

}  // namespace
}  // namespace dora

using namespace dora;

extern "C" int dora_token_logprobs_fwd(const void* logits, int64_t ld, const void* targets, int64_t ignore_index,
                                       double temperature, void* logprobs, void* lse, void* entropy, int top_k,
                                       void* top_logprobs, void* top_indices, int64_t rows, int64_t vocab, int dtype,
                                       void* stream) {
  if (!args_ok(rows, vocab, ld, temperature, dtype) || top_k < 0 || top_k > vocab) return DORA_ERR_INVALID_ARGUMENT;
  if (top_k > kMaxTop) return DORA_ERR_UNSUPPORTED;
  if (rows == 0) return DORA_OK;
  if (!logits || !targets || !logprobs || !lse || (top_k && (!top_logprobs || !top_indices)))
    return DORA_ERR_INVALID_ARGUMENT;
  const float s = float(1.4426950408889634074 / temperature), inv_temp = float(1.0 / temperature);
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    logprobs_fwd_kernel<T><<<row_grid(rows), kT, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const T*>(logits), ld, static_cast<const int64_t*>(targets), ignore_index, s, inv_temp,
        static_cast<float*>(logprobs), static_cast<float*>(lse), static_cast<float*>(entropy), top_k,
        static_cast<float*>(top_logprobs), static_cast<int64_t*>(top_indices), rows, vocab);
    return check_launch();
  });
}

extern "C" int dora_token_logprobs_bwd(const void* logits, int64_t ld, const void* targets, int64_t ignore_index,
                                       double temperature, const void* lse, const void* entropy,
                                       const void* g_logprobs, const void* g_entropy, const void* g_lse,
                                       void* d_logits, int64_t ld_d, int64_t rows, int64_t vocab, int dtype,
                                       void* stream) {
  if (!args_ok(rows, vocab, ld, temperature, dtype) || ld_d < vocab) return DORA_ERR_INVALID_ARGUMENT;
  if (rows == 0) return DORA_OK;
  if (!logits || !targets || !lse || !d_logits || (g_entropy && !entropy) || (d_logits == logits && ld_d != ld))
    return DORA_ERR_INVALID_ARGUMENT;
  const float s = float(1.4426950408889634074 / temperature), inv_temp = float(1.0 / temperature);
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    logprobs_bwd_kernel<T><<<row_grid(rows), kT, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const T*>(logits), ld, static_cast<const int64_t*>(targets), ignore_index, s,
        inv_temp, static_cast<const float*>(lse), static_cast<const float*>(entropy),
        static_cast<const float*>(g_logprobs), static_cast<const float*>(g_entropy), static_cast<const float*>(g_lse),
        static_cast<T*>(d_logits), ld_d, rows, vocab);
    return check_launch();
  });
}
