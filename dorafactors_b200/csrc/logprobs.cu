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
#include <cooperative_groups.h>
#include <math_constants.h>

#include <type_traits>

#include "pair.cuh"

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

__device__ __forceinline__ uint32_t order_bits(float v) { return uint32_t(order_key(v, 0) >> 32); }

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

// A row as 16-byte units at multiples of 16 in memory, and the elements before and after them.
template <typename T> struct Row {
  static constexpr int V = Vec16<T>::N;
  const T* x;
  int vocab, head, units;
  __device__ Row(const T* x_, int vocab_) : x(x_), vocab(vocab_) {
    const int off = int(reinterpret_cast<uintptr_t>(x) & 15) / int(sizeof(T));
    head = off ? V - off : 0;
    if (head > vocab) head = vocab;
    units = (vocab - head) / V;
  }
  __device__ int col(int unit) const { return head + unit * V; }
  // The single column of this thread in the CTA that has the row's first (last) units, -1 if it has none.
  __device__ int single(bool first, bool last) const {
    const int t = threadIdx.x;
    if (first && t < head) return t;
    const int c = col(units) + t - 32;
    return last && t >= 32 && c < vocab ? c : -1;
  }
};

// ---------------------------------------------------------------------------
// Forward.  A row is one CTA's, or a cluster's whose CTAs take a part each and join over
// distributed shared memory, so that few rows are read by many SMs.  A thread keeps a
// maximum and sums relative to it, over 4 units at a time (the next 4 are on their way).
// Bound by HBM and, close behind, the exponentials (an SM makes 16 a cycle): 4096 x 128256 bf16 with
// entropy and a tenth ignored in 188 us, 0.77 of the copy rate; one row in 5 us.
//
// Alternatives: the k largest elements lie in k groups of elements at most, those with the k
// largest maxima.  While the row passes, a thread notes the maximum of each of its groups;
// the k-th largest of the threads' maxima is then a bound that all alternatives reach, and
// only groups that reach it are read again (about k of them).  Where more than kHeld elements
// reach it (many equal logits), the k are picked one by one instead.
// ---------------------------------------------------------------------------
constexpr int kU = 4;
constexpr int kGroups = 16;   // groups of a thread's elements
constexpr int kHeld = 1024;

struct Part {  // of a row, at its maximum
  float max;
  double sum, dot;
};

template <typename T> __device__ __forceinline__ uint4 no_logits() {  // -inf
  const uint32_t w = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
  return make_uint4(w, w, w, w);
}
// Distance of a smaller maximum to a larger one, in powers of two; what is there at 2^-1000 is nothing, and the
// distance stays finite for -inf and for the types' lowest values.
__device__ __forceinline__ float below(float m, float to, float s) { return fmaxf((m - to) * s, -1000.f); }
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// out[r] = the key with r larger ones among the n (all different) in `keys`, for r < k.
__device__ __forceinline__ void rank_keys(const unsigned long long* keys, int n, int k, unsigned long long* out) {
  for (int i = threadIdx.x; i < n; i += kT) {
    const unsigned long long mine = keys[i];
    int r = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) r += keys[j] > mine;
    if (r < k) out[r] = mine;
  }
}

template <typename T, bool kEntropy, bool kTop>
__global__ void __launch_bounds__(kT, 3)
logprobs_fwd_kernel(const T* __restrict__ logits, int64_t ld, const int64_t* __restrict__ targets, int64_t ignore,
                    float s, float inv_temp, float* __restrict__ logprobs, float* __restrict__ lse,
                    float* __restrict__ entropy, int k, float* __restrict__ top_lp, int64_t* __restrict__ top_idx,
                    int vocab, int ranks) {
  namespace cg = cooperative_groups;
  constexpr int V = Vec16<T>::N, N = V / 2;
  __shared__ float red[kT / 32];
  __shared__ double redd[kT / 32];
  __shared__ Part part;
  __shared__ float group_max[kTop ? kGroups + 1 : 1][kT];  // [kGroups]: the single element
  __shared__ unsigned long long held[kTop ? kHeld : 1], best[kTop ? kMaxTop : 1], redk[kT / 32];
  __shared__ int count;

  const int64_t r = blockIdx.x / ranks;
  const int rank = blockIdx.x % ranks;
  const int64_t target = targets[r];
  if (target == ignore) {
    if (rank == 0) {
      if (threadIdx.x == 0) {
        logprobs[r] = 0.f;
        lse[r] = 0.f;
        if (kEntropy) entropy[r] = 0.f;
      }
      for (int i = threadIdx.x; kTop && i < k; i += kT) {
        top_lp[r * k + i] = 0.f;
        top_idx[r * k + i] = -1;
      }
    }
    return;
  }
  const Row<T> row(logits + r * ld, vocab);
  float given = 0.f;
  if (rank == 0 && threadIdx.x == 0 && target >= 0 && target < vocab) given = to_f32(row.x[target]);
  const int u0 = int(int64_t(row.units) * rank / ranks), u1 = int(int64_t(row.units) * (rank + 1) / ranks);
  const int single = row.single(rank == 0, rank == ranks - 1);
  const uint4* units = reinterpret_cast<const uint4*>(row.x + row.head);
  const int rounds = (u1 - u0 + kT * kU - 1) / (kT * kU), per_group = (rounds + kGroups - 1) / kGroups;

  float m = -CUDART_INF_F;
  Two sum = both(0.f), dot = both(0.f);
  auto raise = [&](float to) {  // the reference of the sums, to a larger maximum
    if (to > m) {
      const float by = below(m, to, s), e = exp2_approx(by);
      if constexpr (kEntropy) dot = mul2(fma2(sum, both(by), dot), both(e));
      sum = mul2(sum, both(e));
      m = to;
    }
  };
  auto load = [&](int u, uint4 (&q)[kU]) {
    const uint4* from = units + u + threadIdx.x;
    if (u + kT * kU <= u1) {
#pragma unroll
      for (int j = 0; j < kU; ++j) q[j] = ld_stream(from + j * kT);
    } else {
#pragma unroll
      for (int j = 0; j < kU; ++j) q[j] = u + j * kT + int(threadIdx.x) < u1 ? ld_stream(from + j * kT) : no_logits<T>();
    }
  };
  float group = -CUDART_INF_F;
  int g = 0;
  auto take = [&](uint4 (&q)[kU], int i) {  // round i
    Two f[kU][N];
    float top = -CUDART_INF_F;
#pragma unroll
    for (int j = 0; j < kU; ++j) {
      Pairs<T>::unpack(q[j], f[j]);
#pragma unroll
      for (int n = 0; n < N; ++n) top = max3(top, f[j][n].a, f[j][n].b);
    }
    raise(top);
    Two these = both(0.f);  // summed up apart: beside the largest term, 1, small ones would be lost one by one
    const Two base = both(m == -CUDART_INF_F ? 0.f : -m);
#pragma unroll
    for (int j = 0; j < kU; ++j)
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const Two t = mul2(add2(f[j][n], base), both(s));
        const Two e{exp2_approx(t.a), exp2_approx(t.b)};
        these = add2(these, e);
        if constexpr (kEntropy) dot = fma2(e, Two{fmaxf(t.a, -200.f), fmaxf(t.b, -200.f)}, dot);  // t may be -inf, where e is 0
      }
    sum = add2(sum, these);
    if constexpr (kTop) {
      group = fmaxf(group, top);
      if ((i + 1) % per_group == 0 || i + 1 == rounds) {
        group_max[g++][threadIdx.x] = group;
        group = -CUDART_INF_F;
      }
    }
  };
  uint4 q[kU], next[kU];
  load(u0, q);
  for (int i = 0; i < rounds; i += 2) {
    load(u0 + (i + 1) * kT * kU, next);
    take(q, i);
    if (i + 1 == rounds) break;
    load(u0 + (i + 2) * kT * kU, q);
    take(next, i + 1);
  }
  if (single >= 0) {
    const float v = to_f32(row.x[single]);
    raise(v);
    const float t = (v - (m == -CUDART_INF_F ? 0.f : m)) * s, e = exp2_approx(t);
    sum.a += e;
    if constexpr (kEntropy) dot.a = fmaf(e, fmaxf(t, -200.f), dot.a);
    if constexpr (kTop) group_max[kGroups][threadIdx.x] = v;
  }

  // Join the threads at the CTA's maximum, in fp64.
  const float cta_max = block_fold(m, red, Max());
  {
    const float by = below(m, cta_max, s), e = exp2_approx(by);
    const double own = double(sum.a) + double(sum.b);
    const double total = block_fold(own * e, redd, Sum());
    double dots = 0.0;
    if constexpr (kEntropy)
      dots = block_fold((double(dot.a) + double(dot.b) + by * own) * e, redd, Sum());
    if (threadIdx.x == 0) part = Part{cta_max, total, dots};
  }

  if constexpr (kTop) {
    const bool any = u0 + int(threadIdx.x) < u1 || single >= 0;
    const uint32_t mine = any ? order_bits(m) : 0u;
    if (threadIdx.x == 0) count = 0;
    if (threadIdx.x < kMaxTop) best[threadIdx.x] = 0ull;
    // The largest bound of 16 leading bits that at least k threads' maxima reach, bit by bit (all 16 of a 16-bit logit).
    uint32_t least = 0u;
    for (int bit = 31; bit >= 16; --bit) {
      const uint32_t trial = least | (1u << bit);
      if (__syncthreads_count(mine >= trial) >= k) least = trial;
    }
    const float reach = least > order_bits(-CUDART_INF_F) ? key_value(static_cast<unsigned long long>(least) << 32) : -CUDART_INF_F;
    auto hold = [&](int c) {
      const int at = atomicAdd(&count, 1);  // any order: the keys are ranked
      if (at < kHeld) held[at] = order_key(to_f32(row.x[c]), uint32_t(c));
    };
    if (mine >= least) {
      uint32_t wanted = 0u;  // groups that reach the bound
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
        if (g * per_group < rounds && order_bits(group_max[g][threadIdx.x]) >= least) wanted |= 1u << g;
      for (int i = 0; i < rounds && wanted; ++i) {
        const int g = i / per_group;
        if (!(wanted >> g & 1u)) continue;
        if (i + 1 == (g + 1) * per_group) wanted &= ~(1u << g);
        const int v = u0 + i * kU * kT + threadIdx.x;
        uint4 again[kU];
#pragma unroll
        for (int j = 0; j < kU; ++j)
          again[j] = v + j * kT < u1 ? __ldg(units + v + j * kT) : no_logits<T>();
        uint32_t reached = 0u;
#pragma unroll
        for (int j = 0; j < kU; ++j) {
          float f[V];
          Vec16<T>::unpack(again[j], f);
#pragma unroll
          for (int n = 0; n < V; ++n) reached |= v + j * kT < u1 && f[n] >= reach ? 1u << (j * V + n) : 0u;
        }
        for (; reached; reached &= reached - 1) {
          const int e = __ffs(int(reached)) - 1;
          hold(row.col(v + e / V * kT) + e % V);
        }
      }
      if (single >= 0 && group_max[kGroups][threadIdx.x] >= reach) hold(single);
    }
    __syncthreads();
    if (count <= kHeld) {
      rank_keys(held, count, k, best);
    } else {
      unsigned long long last = ~0ull;
      for (int i = 0; i < k; ++i) {
        unsigned long long next = 0ull;
        auto see = [&](float v, int c) {
          const unsigned long long key = order_key(v, uint32_t(c));
          if (key < last && key > next) next = key;
        };
        for (int v = u0 + threadIdx.x; v < u1; v += kT) {
          float f[V];
          Vec16<T>::unpack(__ldg(units + v), f);
#pragma unroll
          for (int n = 0; n < V; ++n) see(f[n], row.col(v) + n);
        }
        if (single >= 0) see(to_f32(row.x[single]), single);
        last = block_fold(next, redk, Max());
        if (threadIdx.x == 0) best[i] = last;
      }
    }
  }

  Part all;
  if (ranks == 1) {
    __syncthreads();
    all = part;
  } else {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (rank == 0) {
      all = part;
      for (int j = 1; j < ranks; ++j) all.max = fmaxf(all.max, cluster.map_shared_rank(&part, j)->max);
      const float to = all.max;
      all.sum = all.dot = 0.0;
      for (int j = 0; j < ranks; ++j) {
        const Part o = *cluster.map_shared_rank(&part, j);
        const float by = below(o.max, to, s), e = exp2_approx(by);
        all.sum += o.sum * e;
        all.dot += (o.dot + by * o.sum) * e;
      }
      if constexpr (kTop)
        for (int i = threadIdx.x; i < ranks * k; i += kT) held[i] = cluster.map_shared_rank(best, i / k)[i % k];
    }
    cluster.sync();  // the other parts are read
    if (rank != 0) return;
    if constexpr (kTop) {
      // A part with fewer than k elements has zeros after them, which are no keys: they rank last.
      __syncthreads();
      rank_keys(held, ranks * k, k, best);
      __syncthreads();
    }
  }
  const bool none = all.max == -CUDART_INF_F && all.sum == 0.0;  // every logit is -inf
  const bool bad = !(all.sum < CUDART_INF);
  const float ln_sum = none ? -CUDART_INF_F : log1pf(float(all.sum - 1.0));
  const float m0 = none ? 0.f : all.max;
  if (threadIdx.x == 0) {
    float lp = CUDART_NAN_F;
    if (target >= 0 && target < vocab) lp = none ? -CUDART_INF_F : fmaf(given - m0, inv_temp, -ln_sum);
    else record_device_error(DORA_ERR_INVALID_ARGUMENT);
    logprobs[r] = lp;
    lse[r] = none ? -CUDART_INF_F : fmaf(m0, inv_temp, ln_sum);
    if constexpr (kEntropy) entropy[r] = none ? 0.f : ln_sum - kLn2 * float(all.dot / all.sum);
  }
  if constexpr (kTop)
    for (int i = threadIdx.x; i < k; i += kT) {
      top_lp[r * k + i] = bad ? CUDART_NAN_F : none ? -CUDART_INF_F : fmaf(key_value(best[i]) - m0, inv_temp, -ln_sum);
      top_idx[r * k + i] = bad ? i : key_col(best[i]);
    }
}

// ---------------------------------------------------------------------------
// Backward: one pass, a CTA to a part of a row; bound by HBM (4096 x 128256 bf16, a tenth ignored: 331 us, 0.92
// of the copy rate).  The units are those of the
// output; where the logits' rows stand differently to 16 bytes, each is cut out of two of theirs.
// ---------------------------------------------------------------------------
template <typename T, bool kEntropy>
__global__ void __launch_bounds__(kT, 4)
logprobs_bwd_kernel(const T* logits, int64_t ld, const int64_t* __restrict__ targets, int64_t ignore, float s,
                    float inv_temp, const float* __restrict__ lse, const float* __restrict__ entropy,
                    const float* __restrict__ g_lp, const float* __restrict__ g_ent, const float* __restrict__ g_lse,
                    T* d, int64_t ldd, int vocab, int parts) {
  constexpr int V = Vec16<T>::N, N = V / 2;
  __shared__ float red[kT / 32];
  const int64_t r = blockIdx.x / parts;
  const int part = blockIdx.x % parts;
  const int64_t target = targets[r];
  const T* x = logits + r * ld;
  const Row<T> out(d + r * ldd, vocab);
  T* o = d + r * ldd;
  const int u0 = int(int64_t(out.units) * part / parts), u1 = int(int64_t(out.units) * (part + 1) / parts);
  const int single = out.single(part == 0, part == parts - 1);
  float L = lse[r];
  if (target == ignore || L == -CUDART_INF_F) {
    for (int u = u0 + threadIdx.x; u < u1; u += kT) st_stream(o + out.col(u), make_uint4(0, 0, 0, 0));
    if (single >= 0) o[single] = from_f32<T>(0.f);
    return;
  }
  float m = 0.f;  // log p_j = (x_j - m) / T - L
  if (fabsf(L) > kWideLse) {
    // The row in place of which the gradient is written may be partly overwritten by now, by another CTA: the launch
    // gives rows one CTA each then.
    m = -CUDART_INF_F;
    for (int c = threadIdx.x; c < vocab; c += kT) m = fmaxf(m, to_f32(x[c]));
    m = block_fold(m, red, Max());
    float sum = 0.f;
    for (int c = threadIdx.x; c < vocab; c += kT) sum += exp2_approx((to_f32(x[c]) - m) * s);
    L = logf(block_fold(sum, red, Sum()));
  }
  const float glp = g_lp ? g_lp[r] : 0.f, gl = g_lse ? g_lse[r] : 0.f, ge = kEntropy ? g_ent[r] : 0.f;
  // dx_j = p_j (a + b log p_j) + 1[j = t] g_lp / T
  const float a = (gl - glp - (kEntropy ? ge * entropy[r] : 0.f)) * inv_temp, b = -ge * inv_temp;
  auto slope = [&](Two v) {
    const Two lp = fma2(add2(v, both(-m)), both(inv_temp), both(-L));
    const Two t = mul2(lp, both(kLog2e));
    const Two p{exp2_approx(t.a), exp2_approx(t.b)};
    if constexpr (!kEntropy) return mul2(p, both(a));
    return mul2(p, fma2(both(b), Two{fmaxf(lp.a, -200.f), fmaxf(lp.b, -200.f)}, both(a)));
  };
  const int off = int((reinterpret_cast<uintptr_t>(x + out.head) & 15) / sizeof(T));  // of the logits' row there
  auto finish = [&](int u, const uint4& q) {
    Two f[N];
    Pairs<T>::unpack(q, f);
#pragma unroll
    for (int n = 0; n < N; ++n) f[n] = slope(f[n]);
    const int64_t at = target - out.col(u);
    if (at >= 0 && at < V) {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (at == 2 * n) f[n].a = fmaf(glp, inv_temp, f[n].a);
        if (at == 2 * n + 1) f[n].b = fmaf(glp, inv_temp, f[n].b);
      }
    }
    st_stream(o + out.col(u), Pairs<T>::pack(f));
  };
  if (off == 0) {
    for (int u = u0 + threadIdx.x; u < u1; u += kT * kU) {
      uint4 q[kU];
#pragma unroll
      for (int j = 0; j < kU; ++j)
        if (u + j * kT < u1) q[j] = ld_stream_coherent(x + out.col(u + j * kT));
#pragma unroll
      for (int j = 0; j < kU; ++j)
        if (u + j * kT < u1) finish(u + j * kT, q[j]);
    }
  } else {
    auto whole = [&](int u) { return u < u1 && out.col(u) >= off && out.col(u) - off + 2 * V <= vocab; };
    for (int u = u0 + threadIdx.x; u < u1; u += kT * kU) {
      uint4 lo[kU], hi[kU];
#pragma unroll
      for (int j = 0; j < kU; ++j) {
        lo[j] = hi[j] = make_uint4(0, 0, 0, 0);
        if (whole(u + j * kT)) {
          const T* from = x + out.col(u + j * kT) - off;  // a multiple of 16
          lo[j] = __ldg(reinterpret_cast<const uint4*>(from));
          hi[j] = __ldg(reinterpret_cast<const uint4*>(from + V));
        }
      }
#pragma unroll
      for (int j = 0; j < kU; ++j) {
        const int v = u + j * kT;
        if (v >= u1) break;
        uint4 q = cut<T>(lo[j], hi[j], off);
        if (!whole(v)) {  // it reaches out of the row
          T* e = reinterpret_cast<T*>(&q);
#pragma unroll
          for (int n = 0; n < V; ++n) e[n] = x[out.col(v) + n];
        }
        finish(v, q);
      }
    }
  }
  if (single >= 0) {
    float v = slope(both(to_f32(x[single]))).a;
    if (single == target) v = fmaf(glp, inv_temp, v);
    o[single] = from_f32<T>(v);
  }
}

// Parts of a row: enough that `want` CTAs run, each with at least `least` 16-byte units; powers of two.
int row_parts(int64_t rows, int64_t units, int64_t want, int64_t least, int most) {
  int n = 1;
  while (n < most && rows * n * 2 <= want && units / (2 * n) >= least) n *= 2;
  return n;
}

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
    // A cluster of up to eight CTAs to a row while that makes no more than three CTAs an SM, each with a round of work.
    const int ranks = row_parts(rows, vocab / Vec16<T>::N, int64_t(num_sms()) * 3, kT * kU / 2, 8);
    if (rows * ranks > 0x7fffffff) return int(DORA_ERR_UNSUPPORTED);
    auto go = [&](auto kernel) {
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3(unsigned(rows * ranks));
      cfg.blockDim = dim3(kT);
      cfg.stream = static_cast<cudaStream_t>(stream);
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = unsigned(ranks);
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      count_launches(1);
      const cudaError_t e = cudaLaunchKernelEx(
          &cfg, kernel, static_cast<const T*>(logits), ld, static_cast<const int64_t*>(targets), ignore_index, s,
          inv_temp, static_cast<float*>(logprobs), static_cast<float*>(lse), static_cast<float*>(entropy), top_k,
          static_cast<float*>(top_logprobs), static_cast<int64_t*>(top_indices), int(vocab), ranks);
      return e == cudaSuccess ? int(DORA_OK) : set_cuda_error(e);
    };
    if (top_k) return entropy ? go(logprobs_fwd_kernel<T, true, true>) : go(logprobs_fwd_kernel<T, false, true>);
    return entropy ? go(logprobs_fwd_kernel<T, true, false>) : go(logprobs_fwd_kernel<T, false, false>);
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
    // Parts of at least four rounds while there are few CTAs; one in place of the logits (see the kernel).
    const int parts = logits == d_logits ? 1 : row_parts(rows, vocab / Vec16<T>::N, int64_t(num_sms()) * 8, kT * kU, 64);
    if (rows * parts > 0x7fffffff) return int(DORA_ERR_UNSUPPORTED);
    auto go = [&](auto kernel) {
      kernel<<<unsigned(rows * parts), kT, 0, static_cast<cudaStream_t>(stream)>>>(
          static_cast<const T*>(logits), ld, static_cast<const int64_t*>(targets), ignore_index, s, inv_temp,
          static_cast<const float*>(lse), static_cast<const float*>(entropy), static_cast<const float*>(g_logprobs),
          static_cast<const float*>(g_entropy), static_cast<const float*>(g_lse), static_cast<T*>(d_logits), ld_d,
          int(vocab), parts);
      return check_launch();
    };
    return g_entropy ? go(logprobs_bwd_kernel<T, true>) : go(logprobs_bwd_kernel<T, false>);
  });
}
