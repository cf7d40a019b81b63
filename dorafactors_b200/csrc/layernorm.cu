// Layer norm and RMS norm over the last dimension, forward and backward.
//
//   mean = sum x / C,  rstd = (sum (x - mean)^2 / C + eps)^-1/2          (RMS: mean = 0)
//   y    = (x - mean) * rstd * w + b
//   xh = (x - mean) * rstd,  a = dy * w
//   dx = rstd * (a - mean(a) - xh * mean(a * xh))                        (RMS: without mean(a))
//   dw = sum over rows of dy * xh,  db = sum over rows of dy
//
// Statistics, row sums and the column sums are fp32 in a fixed order (no atomics), so
// results do not change from call to call; every output is rounded once.
#include <type_traits>

#include "pair.cuh"

namespace dora {
namespace {

constexpr int kT = 256;       // threads of the kernels for any width
constexpr int kBwdFill = 512;
constexpr int fwd_fill(bool params_in_shared) { return params_in_shared ? 512 : 768; }

// ---------------------------------------------------------------------------
// A row and the threads that share it.  `tpr` threads hold a row: up to 32 (a power of
// two) of a warp, whose CTA then works on several rows, or whole warps of a CTA.
// ---------------------------------------------------------------------------
struct Shape {
  int tpr, threads, groups;  // threads a row and a CTA, rows a CTA works on at a time
};
Shape share_row(int64_t units, int per, int small_cta) {
  Shape s;
  const int64_t need = (units + per - 1) / per;
  if (need > 32) {
    s.tpr = s.threads = int((need + 31) / 32 * 32);
    s.groups = 1;
  } else {
    s.tpr = 1;
    while (s.tpr < need) s.tpr *= 2;
    s.threads = small_cta;
    s.groups = small_cta / s.tpr;
  }
  return s;
}

// Sums over the threads of a row, in every one of them; the same tree each time.  kMost: threads of the
// CTA, all of one row, or 128 for rows inside a warp.  One barrier a call: `red` alternates between two
// buffers, and a buffer is written again only after the barrier of the call in between.
template <int kMost, int kValues> struct RowSum {
  static constexpr bool kWide = kMost > 128;
  static constexpr int kWarps = kWide ? kMost / 32 : 1;
  float4 (*red)[kValues][kWarps / 4 + 1];  // [2] in shared memory: a value a warp, zero for warps that are not there
  int tpr, turn;
  __device__ RowSum(float4 (*r)[kValues][kWarps / 4 + 1], int tpr_) : red(r), tpr(tpr_), turn(0) {
    if constexpr (kWide) {
      float* f = reinterpret_cast<float*>(red);
      for (int i = threadIdx.x; i < 2 * kValues * (kWarps / 4 + 1) * 4; i += blockDim.x) f[i] = 0.f;
      __syncthreads();
    }
  }
  __device__ __forceinline__ void operator()(float (&v)[kValues]) {
    if constexpr (!kWide) {
      for (int o = tpr / 2; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < kValues; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    } else {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < kValues; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
      if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int i = 0; i < kValues; ++i) reinterpret_cast<float*>(red[turn][i])[threadIdx.x / 32] = v[i];
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kValues; ++i) {
        Two t = both(0.f);
#pragma unroll
        for (int j = 0; j < kWarps / 4; ++j) {
          const float4 q = red[turn][i][j];
          t = add2(t, add2(Two{q.x, q.y}, Two{q.z, q.w}));
        }
        v[i] = t.a + t.b;
      }
      turn ^= 1;
    }
  }
};
#define DORA_ROW_SUM(name, most, values)                                                  \
  __shared__ float4 name##_red[2][values][RowSum<most, values>::kWarps / 4 + 1];          \
  RowSum<most, values> name(name##_red, tpr)

// A unit (16-byte vector of T) of the weight or bias at column c, as pairs.
template <typename T, typename TW>
__device__ __forceinline__ void load_param(const void* w, int64_t c, Two (&f)[Pairs<T>::N]) {
  if constexpr (sizeof(TW) == 4) {
#pragma unroll
    for (int i = 0; i < Pairs<T>::N; i += 2) {
      const float4 q = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(w) + c + 2 * i));
      f[i] = Two{q.x, q.y}, f[i + 1] = Two{q.z, q.w};
    }
  } else {
    Pairs<T>::unpack(__ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(w) + c)), f);
  }
}
// The same where type and presence (`none` instead) are known at run time only.
template <typename T>
__device__ __forceinline__ void load_param(const void* w, bool f32, int64_t c, float none, Two (&f)[Pairs<T>::N]) {
  if (!w) {
#pragma unroll
    for (int i = 0; i < Pairs<T>::N; ++i) f[i] = both(none);
  } else if (f32) {
    load_param<T, float>(w, c, f);
  } else {
    load_param<T, T>(w, c, f);
  }
}
template <typename T> __device__ __forceinline__ float param(const void* w, bool f32, int64_t c, float none) {
  if (!w) return none;
  return f32 ? __ldg(static_cast<const float*>(w) + c) : to_f32(static_cast<const T*>(w)[c]);
}

// ---------------------------------------------------------------------------
// Rows of 16-byte units.  A CTA walks down the rows; a thread keeps the same PER units
// of every row (and their weights in registers) and has the next S - 1 rows' units on
// their way through shared memory, which keeps HBM busy across the barriers of a row's
// sums.  A thread reads back only what it has copied itself.
// ---------------------------------------------------------------------------
struct Walk {  // this thread's part of the rows
  int t, group;        // its number among the row's threads, and the row's among the CTA's
  int64_t first, step; // row it starts with and distance to the next
  int64_t mine, rounds; // its rows, and rounds of the CTA
};
__device__ __forceinline__ Walk walk(int64_t rows, int tpr, int groups) {
  Walk w;
  w.t = groups > 1 ? threadIdx.x & (tpr - 1) : threadIdx.x;
  w.group = groups > 1 ? threadIdx.x / tpr : 0;
  w.step = int64_t(gridDim.x) * groups;
  const int64_t r0 = int64_t(blockIdx.x) * groups;
  w.first = r0 + w.group;
  w.rounds = r0 < rows ? (rows - r0 + w.step - 1) / w.step : 0;
  w.mine = w.first < rows ? (rows - w.first + w.step - 1) / w.step : 0;
  return w;
}

// Forward: the variance is taken around the mean, from the registers.
// kParams: 0 none, 1 a weight, 2 a weight and a bias, of type TW.  They stand in shared memory, each thread's units in
// places of its own, so two CTAs of 128 registers a thread run on an SM; fp32 ones of 16-bit rows, which would take twice
// the room, come from L1 for each row, with three CTAs of 80.  (bf16, 16384 x 8192, with weight and bias: 90 us; from L1
// with three CTAs 101 us, with two 112 us; in registers 109 us.)
template <typename TA, typename TW, bool kRms, int kParams, int PER, int S, int kMax>
__global__ void __launch_bounds__(kMax, fwd_fill(sizeof(TW) == sizeof(TA)) / kMax)
ln_fwd_kernel(const TA* __restrict__ x, int64_t ldx, const void* __restrict__ w, const void* __restrict__ b, float eps, TA* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd, int64_t rows,
              int cols, int tpr, int groups) {
  using P = Pairs<TA>;
  constexpr int N = P::N, V = 2 * N;
  constexpr bool kShared = sizeof(TW) == sizeof(TA);
  extern __shared__ uint4 ring[];  // [S][PER][threads], then the parameters: [kParams][PER][threads]
  DORA_ROW_SUM(sum, kMax, 1);
  const Walk at = walk(rows, tpr, groups);
  const float inv = 1.0f / float(cols);
  bool has[PER];
#pragma unroll
  for (int p = 0; p < PER; ++p) has[p] = p == 0 || (p * tpr + at.t) * V < cols;  // every thread has a first unit
  const TA* from = x + at.first * ldx + at.t * V;
  TA* to = y + at.first * cols + at.t * V;
  const uint32_t slots = shared_addr(ring + threadIdx.x), part = blockDim.x * 16;
  int64_t fetched = 0;
  int into = 0;
  auto fetch = [&] {
    if (fetched < at.mine) {
#pragma unroll
      for (int p = 0; p < PER; ++p)
        if (has[p]) copy_async16(slots + (into * PER + p) * part, from + p * tpr * V);
      from += at.step * ldx;
      ++fetched;
    }
    copies_commit();
    into = into == S - 1 ? 0 : into + 1;
  };
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch();
  uint4* held = ring + S * PER * blockDim.x + threadIdx.x;
  if constexpr (kShared && kParams > 0) {
#pragma unroll
    for (int p = 0; p < PER; ++p)
      if (has[p]) {
        const int c = (p * tpr + at.t) * V;
        held[p * blockDim.x] = __ldg(reinterpret_cast<const uint4*>(static_cast<const TA*>(w) + c));
        if constexpr (kParams > 1)
          held[(PER + p) * blockDim.x] = __ldg(reinterpret_cast<const uint4*>(static_cast<const TA*>(b) + c));
      }
  }
  int s = 0;
  for (int64_t k = 0; k < at.rounds; ++k) {
    fetch();
    copies_done<S - 1>();
    const bool live = kMax > 128 || k < at.mine;  // rows inside a warp: all its threads take part in the sums
    Two f[PER][N];
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      if (live && has[p]) P::unpack(ring[(s * PER + p) * blockDim.x + threadIdx.x], f[p]);
      else
#pragma unroll
        for (int i = 0; i < N; ++i) f[p][i] = both(0.f);
    }
    s = s == S - 1 ? 0 : s + 1;
    float mu[1] = {0.f}, var[1];
    if constexpr (!kRms) {
      Two a = both(0.f);
#pragma unroll
      for (int p = 0; p < PER; ++p)
#pragma unroll
        for (int i = 0; i < N; ++i) a = add2(a, f[p][i]);
      mu[0] = a.a + a.b;
      sum(mu);
      mu[0] *= inv;
    }
    Two q = both(0.f);
#pragma unroll
    for (int p = 0; p < PER; ++p)
      if (has[p]) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if constexpr (!kRms) f[p][i] = add2(f[p][i], both(-mu[0]));
          q = fma2(f[p][i], f[p][i], q);
        }
      }
    var[0] = q.a + q.b;
    sum(var);
    const float rs = rsqrtf(var[0] * inv + eps);
    if (live) {
#pragma unroll
      for (int p = 0; p < PER; ++p)
        if (has[p]) {
          Two o[N], v[N];
#pragma unroll
          for (int i = 0; i < N; ++i) o[i] = mul2(f[p][i], both(rs));
          if constexpr (kParams > 0) {
            if constexpr (kShared) P::unpack(held[p * blockDim.x], v);
            else load_param<TA, TW>(w, (p * tpr + at.t) * V, v);
#pragma unroll
            for (int i = 0; i < N; ++i) o[i] = mul2(o[i], v[i]);
          }
          if constexpr (kParams > 1) {
            if constexpr (kShared) P::unpack(held[(PER + p) * blockDim.x], v);
            else load_param<TA, TW>(b, (p * tpr + at.t) * V, v);
#pragma unroll
            for (int i = 0; i < N; ++i) o[i] = add2(o[i], v[i]);
          }
          st_stream(to + p * tpr * V, P::pack(o));
        }
      if (at.t == 0) {
        const int64_t r = at.first + k * at.step;
        if (!kRms && mean) mean[r] = mu[0];
        if (rstd) rstd[r] = rs;
      }
    }
    to += at.step * cols;
  }
}

// Backward: one pass over dy and x, with the columns' sums for d_weight and d_bias in
// registers; they cost no traffic but one partial row a CTA.  bf16: RMS norm at 32768 x 4096
// 135 us (HBM, 0.91 of the copy rate), layer norm at 16384 x 8192 176 us (0.70: issue slots, with
// the 16 warps an SM that 128 registers leave).
template <typename TA, bool kRms, int PER, int S, int kMax, bool kCols>
__global__ void __launch_bounds__(kMax)
ln_bwd_kernel(const TA* __restrict__ dy, int64_t lddy, const TA* __restrict__ x, int64_t ldx,
              const void* __restrict__ w, bool f32, const float* __restrict__ mean, const float* __restrict__ rstd,
              TA* __restrict__ dx, float* __restrict__ partial, int64_t rows, int cols, int tpr, int groups,
              float one_) {
  using P = Pairs<TA>;
  constexpr int N = P::N, V = 2 * N;
  constexpr bool kHold = kMax <= 512;  // registers for the weight
  extern __shared__ uint4 ring[];  // [S][PER][2][threads]
  constexpr int kSums = kRms ? 1 : 2;
  DORA_ROW_SUM(sum, kMax, kSums);
  const Walk at = walk(rows, tpr, groups);
  const float inv = 1.0f / float(cols);
  const Two one = both(one_);
  bool has[PER];
#pragma unroll
  for (int p = 0; p < PER; ++p) has[p] = p == 0 || (p * tpr + at.t) * V < cols;  // every thread has a first unit
  const TA *dfrom = dy + at.first * lddy + at.t * V, *xfrom = x + at.first * ldx + at.t * V;
  TA* to = dx + at.first * cols + at.t * V;
  const uint32_t slots = shared_addr(ring + threadIdx.x), part = blockDim.x * 16;
  int64_t fetched = 0;
  int into = 0;
  auto fetch = [&] {
    if (fetched < at.mine) {
#pragma unroll
      for (int p = 0; p < PER; ++p)
        if (has[p]) {
          copy_async16(slots + (into * PER + p) * 2 * part, dfrom + p * tpr * V);
          copy_async16(slots + (into * PER + p) * 2 * part + part, xfrom + p * tpr * V);
        }
      dfrom += at.step * lddy;
      xfrom += at.step * ldx;
      ++fetched;
    }
    copies_commit();
    into = into == S - 1 ? 0 : into + 1;
  };
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch();
  Two wf[kHold ? PER : 1][N], dw[kCols ? PER : 1][N], db[kCols && !kRms ? PER : 1][N];
#pragma unroll
  for (int p = 0; p < PER; ++p) {
    if (kHold && has[p]) load_param<TA>(w, f32, (p * tpr + at.t) * V, 1.f, wf[p]);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (kCols) dw[p][i] = both(0.f);
      if constexpr (kCols && !kRms) db[p][i] = both(0.f);
    }
  }
  const float *mnext = kRms ? nullptr : mean + at.first, *rnext = rstd + at.first;
  float mu1 = 0.f, rs1 = 0.f;  // of the next row
  if (at.mine) {
    if constexpr (!kRms) mu1 = *mnext;
    rs1 = *rnext;
  }
  int s = 0;
  for (int64_t k = 0; k < at.rounds; ++k) {
    const float mu = mu1, rs = rs1;
    if (k + 1 < at.mine) {
      if constexpr (!kRms) mu1 = *(mnext += at.step);
      rs1 = *(rnext += at.step);
    }
    fetch();
    copies_done<S - 1>();
    const bool live = kMax > 128 || k < at.mine;
    uint4 dq[PER], xq[PER];
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      dq[p] = ring[(s * PER + p) * 2 * blockDim.x + threadIdx.x];
      xq[p] = ring[((s * PER + p) * 2 + 1) * blockDim.x + threadIdx.x];
    }
    s = s == S - 1 ? 0 : s + 1;
    auto take = [&](int p, Two (&d)[N], Two (&h)[N], Two (&a)[N]) {  // dy, xh and dy w
      P::unpack(dq[p], d);
      P::unpack(xq[p], h);
      if constexpr (!kHold) load_param<TA>(w, f32, (p * tpr + at.t) * V, 1.f, a);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        a[i] = mul2(d[i], kHold ? wf[p][i] : a[i]);
        if constexpr (!kRms) h[i] = add2(h[i], both(-mu));
        h[i] = mul2(h[i], both(rs));
      }
    };
    Two s0 = both(0.f), s1 = both(0.f);
#pragma unroll
    for (int p = 0; p < PER; ++p)
      if (live && has[p]) {
        Two d[N], h[N], a[N];
        take(p, d, h, a);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if constexpr (!kRms) s0 = add2_apart(a[i], s0, one);
          s1 = fma2(a[i], h[i], s1);
          if constexpr (kCols) dw[p][i] = fma2(d[i], h[i], dw[p][i]);
          if constexpr (kCols && !kRms) db[p][i] = add2(db[p][i], d[i]);
        }
      }
    if (dx) {  // the same for all threads
      float c[kSums];
      c[0] = s1.a + s1.b;
      if constexpr (!kRms) c[1] = s0.a + s0.b;
      sum(c);
      const Two c0 = both(kRms ? 0.f : -c[kSums - 1] * inv), c1 = both(-c[0] * inv);
#pragma unroll
      for (int p = 0; p < PER; ++p)
        if (live && has[p]) {
          Two d[N], h[N], a[N];
          take(p, d, h, a);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            if constexpr (!kRms) a[i] = add2_apart(a[i], c0, one);
            a[i] = mul2(fma2(h[i], c1, a[i]), both(rs));
          }
          st_stream(to + p * tpr * V, P::pack(a));
        }
      to += at.step * cols;
    }
  }
  if constexpr (kCols) {
    copies_done<0>();
    float* out = partial + int64_t(blockIdx.x) * 2 * cols;
    float* acc = groups > 1 ? reinterpret_cast<float*>(ring) : out;  // the groups add up in shared memory, one by one
    for (int g = 0; g < groups; ++g) {
      if (groups > 1) __syncthreads();
      if (at.group == g)
#pragma unroll
        for (int p = 0; p < PER; ++p)
          if (has[p]) {
            float2* o = reinterpret_cast<float2*>(acc + (p * tpr + at.t) * V);
#pragma unroll
            for (int i = 0; i < N; ++i) {
              const float2 q = g ? o[i] : make_float2(0.f, 0.f);
              o[i] = make_float2(dw[p][i].a + q.x, dw[p][i].b + q.y);
              if constexpr (!kRms) {
                float2* ob = o + i + cols / 2;
                const float2 v = g ? *ob : make_float2(0.f, 0.f);
                *ob = make_float2(db[p][i].a + v.x, db[p][i].b + v.y);
              }
            }
          }
    }
    if (groups > 1) {
      __syncthreads();
      for (int c = threadIdx.x; c < (kRms ? 1 : 2) * cols; c += blockDim.x) out[c] = acc[c];
    }
  }
}

// ---------------------------------------------------------------------------
// Rows that start or end off a 16-byte boundary.  They come and go in 16-byte pieces all the
// same, cut at multiples of 16 in memory, and stand in shared memory as they stand there;
// a thread takes every tpr-th element.  (Loads and stores of single elements from and to memory
// took 2.8 times as long at 16384 x 5003 in bf16.)
// ---------------------------------------------------------------------------
__host__ __device__ constexpr int row_pieces(int cols, int size) { return (cols * size + 30) / 16; }

template <bool kWide> __device__ __forceinline__ void row_sync() {
  if constexpr (kWide) __syncthreads();
  else __syncwarp();
}

// Copies `cols` elements at `from` to shared memory, piece by piece, the way they stand in memory.  The first piece
// may start in the row before (of the same buffer, from `base` on); where that would be outside, and at the
// row's end, only what belongs to the row is read.
template <typename T>
__device__ __forceinline__ void fetch_pieces(uint4* to, const T* from, const T* base, int cols, int t, int tpr) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(from), end = a + cols * sizeof(T);
  const uintptr_t a0 = a & ~uintptr_t(15);
  const uint32_t dst = shared_addr(to);
  for (int u = t; a0 + u * 16 < end; u += tpr) {
    const uintptr_t src = a0 + u * 16;
    if (src < reinterpret_cast<uintptr_t>(base)) {
      T* e = reinterpret_cast<T*>(to + u);
      for (int i = 0; i < int(16 / sizeof(T)); ++i) {
        const uintptr_t q = src + i * sizeof(T);
        if (q >= a && q < end) e[i] = *reinterpret_cast<const T*>(q);
      }
    } else {
      const int bytes = end - src < 16 ? int(end - src) : 16;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + u * 16), "l"(src), "r"(bytes) : "memory");
    }
  }
}
// The other way: `cols` elements that stand in shared memory the way they are to stand at `to`.
template <typename T>
__device__ __forceinline__ void store_pieces(T* to, const uint4* from, int cols, int t, int tpr) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(to), end = a + cols * sizeof(T);
  const uintptr_t a0 = a & ~uintptr_t(15);
  for (int u = t; a0 + u * 16 < end; u += tpr) {
    const uintptr_t dst = a0 + u * 16;
    if (dst >= a && dst + 16 <= end) {
      st_stream(reinterpret_cast<void*>(dst), from[u]);
    } else {
      const T* e = reinterpret_cast<const T*>(from + u);
      for (int i = 0; i < int(16 / sizeof(T)); ++i) {
        const uintptr_t q = dst + i * sizeof(T);
        if (q >= a && q < end) *reinterpret_cast<T*>(q) = e[i];
      }
    }
  }
}
// Where element 0 of the row at p stands in its first piece.
template <typename T> __device__ __forceinline__ int in_piece(const T* p) {
  return int(reinterpret_cast<uintptr_t>(p) & 15) / int(sizeof(T));
}
// f = f * w, or f + w, for this thread's elements of a row.
template <typename TA, int PER, bool kAdd>
__device__ __forceinline__ void with_param(const void* w, bool f32, int t, int tpr, int cols, float (&f)[PER]) {
  if (!w) return;
  float v[PER];
  if (f32) {
#pragma unroll
    for (int p = 0; p < PER; ++p) v[p] = p * tpr + t < cols ? __ldg(static_cast<const float*>(w) + p * tpr + t) : 0.f;
  } else {
#pragma unroll
    for (int p = 0; p < PER; ++p) v[p] = p * tpr + t < cols ? to_f32(static_cast<const TA*>(w)[p * tpr + t]) : 0.f;
  }
#pragma unroll
  for (int p = 0; p < PER; ++p) f[p] = kAdd ? f[p] + v[p] : __fmul_rn(f[p], v[p]);
}

constexpr int kPieceStages = 3;
constexpr int kPieceFill = 768;  // threads of these kernels an SM holds (1024 of those for the widest rows)

template <typename TA, bool kRms, int PER, int kMax>
__global__ void __launch_bounds__(kMax, kPieceFill / kMax)
ln_fwd_pieces_kernel(const TA* __restrict__ x, int64_t ldx, const void* __restrict__ w, const void* __restrict__ b,
                     bool f32, float eps, TA* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd,
                     int64_t rows, int cols, int tpr, int groups) {
  constexpr bool kWide = kMax > 128;
  constexpr int S = kPieceStages;
  extern __shared__ uint4 ring[];  // [groups][S + 1][pieces]: S rows coming, one going
  DORA_ROW_SUM(sum, kMax, 1);
  const Walk at = walk(rows, tpr, groups);
  const int pieces = row_pieces(cols, sizeof(TA));
  uint4* mine = ring + at.group * (S + 1) * pieces;
  uint4* out = mine + S * pieces;
  const float inv = 1.0f / float(cols);
  const TA* from = x + at.first * ldx;
  auto fetch = [&](int64_t k, int s) {
    if (k < at.mine) fetch_pieces(mine + s * pieces, from + k * at.step * ldx, x, cols, at.t, tpr);
    copies_commit();
  };
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch(s, s);
  int s = 0;
  for (int64_t k = 0; k < at.rounds; ++k) {
    copies_done<S - 2>();
    row_sync<kWide>();  // the row is there, and everybody is done with the one before
    fetch(k + S - 1, s == 0 ? S - 1 : s - 1);
    const bool live = kWide || k < at.mine;
    const int64_t r = at.first + k * at.step;
    const TA* row = reinterpret_cast<const TA*>(mine + s * pieces) + in_piece(x + r * ldx);
    s = s == S - 1 ? 0 : s + 1;
    float f[PER], one[1] = {0.f};
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int c = p * tpr + at.t;
      f[p] = live && c < cols ? to_f32(row[c]) : 0.f;
      one[0] += f[p];
    }
    if constexpr (!kRms) sum(one);
    const float mu = kRms ? 0.f : one[0] * inv;
    one[0] = 0.f;
#pragma unroll
    for (int p = 0; p < PER; ++p)
      if (p * tpr + at.t < cols) {
        f[p] -= mu;
        one[0] = fmaf(f[p], f[p], one[0]);
      }
    sum(one);
    const float rs = rsqrtf(one[0] * inv + eps);
#pragma unroll
    for (int p = 0; p < PER; ++p) f[p] *= rs;
    with_param<TA, PER, false>(w, f32, at.t, tpr, cols, f);
    with_param<TA, PER, true>(b, f32, at.t, tpr, cols, f);
    TA* to = reinterpret_cast<TA*>(out) + in_piece(y + r * cols);
#pragma unroll
    for (int p = 0; p < PER; ++p)
      if (live && p * tpr + at.t < cols) to[p * tpr + at.t] = from_f32<TA>(f[p]);
    row_sync<kWide>();
    if (live) {
      store_pieces(y + r * cols, out, cols, at.t, tpr);
      if (at.t == 0) {
        if (!kRms && mean) mean[r] = mu;
        if (rstd) rstd[r] = rs;
      }
    }
  }
}

template <typename TA, bool kRms, int PER, int kMax, bool kCols>
__global__ void __launch_bounds__(kMax, kPieceFill / kMax)
ln_bwd_pieces_kernel(const TA* __restrict__ dy, int64_t lddy, const TA* __restrict__ x, int64_t ldx,
                     const void* __restrict__ w, bool f32, const float* __restrict__ mean,
                     const float* __restrict__ rstd, TA* __restrict__ dx, float* __restrict__ partial, int64_t rows,
                     int cols, int tpr, int groups) {
  constexpr bool kWide = kMax > 128;
  constexpr int S = kPieceStages;
  extern __shared__ uint4 ring[];  // [groups][2 S + 1][pieces]: S rows of dy and x coming, one of dx going
  DORA_ROW_SUM(sum, kMax, 2);
  const Walk at = walk(rows, tpr, groups);
  const int pieces = row_pieces(cols, sizeof(TA));
  uint4* mine = ring + at.group * (2 * S + 1) * pieces;
  uint4* out = mine + 2 * S * pieces;
  const float inv = 1.0f / float(cols);
  float dw[kCols ? PER : 1] = {}, db[kCols && !kRms ? PER : 1] = {};
  auto fetch = [&](int64_t k, int s) {
    if (k < at.mine) {
      const int64_t r = at.first + k * at.step;
      fetch_pieces(mine + 2 * s * pieces, dy + r * lddy, dy, cols, at.t, tpr);
      fetch_pieces(mine + (2 * s + 1) * pieces, x + r * ldx, x, cols, at.t, tpr);
    }
    copies_commit();
  };
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch(s, s);
  int s = 0;
  for (int64_t k = 0; k < at.rounds; ++k) {
    const bool live = kWide || k < at.mine;
    const int64_t r = at.first + k * at.step;
    float mu = 0.f, rs = 0.f;
    if (live) {
      if constexpr (!kRms) mu = mean[r];
      rs = rstd[r];
    }
    copies_done<S - 2>();
    row_sync<kWide>();  // the row is there, and everybody is done with the one before
    fetch(k + S - 1, s == 0 ? S - 1 : s - 1);
    const TA* dr = reinterpret_cast<const TA*>(mine + 2 * s * pieces) + in_piece(dy + r * lddy);
    const TA* xr = reinterpret_cast<const TA*>(mine + (2 * s + 1) * pieces) + in_piece(x + r * ldx);
    s = s == S - 1 ? 0 : s + 1;
    float a[PER];
#pragma unroll
    for (int p = 0; p < PER; ++p) a[p] = live && p * tpr + at.t < cols ? to_f32(dr[p * tpr + at.t]) : 0.f;
    with_param<TA, PER, false>(w, f32, at.t, tpr, cols, a);
    float c01[2] = {0.f, 0.f};
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int c = p * tpr + at.t;
      if (live && c < cols) {
        const float h = (to_f32(xr[c]) - mu) * rs;
        c01[0] += a[p];
        c01[1] = fmaf(a[p], h, c01[1]);
        if constexpr (kCols) {
          const float d = to_f32(dr[c]);
          dw[p] = fmaf(d, h, dw[p]);
          if constexpr (!kRms) db[p] += d;
        }
      }
    }
    if (!dx) continue;  // the same for all threads
    sum(c01);
    const float c0 = kRms ? 0.f : c01[0] * inv, c1 = c01[1] * inv;
    TA* to = reinterpret_cast<TA*>(out) + in_piece(dx + r * cols);
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int c = p * tpr + at.t;
      if (live && c < cols) to[c] = from_f32<TA>((a[p] - c0 - (to_f32(xr[c]) - mu) * rs * c1) * rs);
    }
    row_sync<kWide>();
    if (live) store_pieces(dx + r * cols, out, cols, at.t, tpr);
  }
  if constexpr (kCols) {
    copies_done<0>();
    float* to = partial + int64_t(blockIdx.x) * 2 * cols;
    float* acc = groups > 1 ? reinterpret_cast<float*>(ring) : to;  // the groups add up in shared memory, one by one
    for (int g = 0; g < groups; ++g) {
      if (groups > 1) __syncthreads();
      if (at.group == g)
#pragma unroll
        for (int p = 0; p < PER; ++p) {
          const int c = p * tpr + at.t;
          if (c < cols) {
            acc[c] = dw[p] + (g ? acc[c] : 0.f);
            if constexpr (!kRms) acc[cols + c] = db[p] + (g ? acc[cols + c] : 0.f);
          }
        }
    }
    if (groups > 1) {
      __syncthreads();
      for (int c = threadIdx.x; c < (kRms ? 1 : 2) * cols; c += blockDim.x) to[c] = acc[c];
    }
  }
}

// ---------------------------------------------------------------------------
// The same for rows of more than a warp's worth, by 16-byte units of the columns as in the aligned kernels: a unit
// is cut out of two pieces where it stands in shared memory, and a piece of the output out of two units.
// (16384 x 5003 in bf16, against single elements from shared memory: forward 268 -> 134 us, layer norm backward 447 -> 207 us.)
// ---------------------------------------------------------------------------
template <typename TA> __device__ __forceinline__ uint4 unit_at(const uint4* pieces, int unit, int off) {
  return off ? cut<TA>(pieces[unit], pieces[unit + 1], off) : pieces[unit];
}
// Elements of f from `left` on become zero.
template <int N> __device__ __forceinline__ void keep_first(Two (&f)[N], int left) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (2 * i >= left) f[i].a = 0.f;
    if (2 * i + 1 >= left) f[i].b = 0.f;
  }
}
// The row's units, which stand in `units`, to global memory.
template <typename TA> __device__ __forceinline__ void store_units(TA* to, const uint4* units, int cols) {
  constexpr int V = Vec16<TA>::N;
  const int off = in_piece(to);
  TA* start = to - off;  // a multiple of 16
  for (int u = threadIdx.x; u * V < cols + off; u += blockDim.x) {
    const int c = u * V - off;
    if (c >= 0 && c + V <= cols) {
      st_stream(start + u * V, off ? cut<TA>(units[u - 1], units[u], V - off) : units[u]);
    } else {
      const TA* e = reinterpret_cast<const TA*>(units);
      for (int i = 0; i < V; ++i)
        if (c + i >= 0 && c + i < cols) to[c + i] = e[c + i];
    }
  }
}
// A parameter in fp32 in places of this thread's own, PER units of V elements, for any type and alignment.
template <typename TA, int PER>
__device__ __forceinline__ void hold_param(float4* held, const void* w, bool f32, float none, int cols) {
  constexpr int V = Vec16<TA>::N;
  for (int p = 0; p < PER; ++p)
    for (int h = 0; h < V / 4; ++h) {
      float v[4];
      for (int i = 0; i < 4; ++i) {
        const int c = (p * blockDim.x + threadIdx.x) * V + 4 * h + i;
        v[i] = c < cols ? param<TA>(w, f32, c, none) : 0.f;
      }
      held[(p * (V / 4) + h) * blockDim.x] = make_float4(v[0], v[1], v[2], v[3]);
    }
}
template <typename TA> __device__ __forceinline__ void held_unit(const float4* held, int p, Two (&f)[Pairs<TA>::N]) {
  constexpr int V = Vec16<TA>::N;
#pragma unroll
  for (int h = 0; h < V / 4; ++h) {
    const float4 q = held[(p * (V / 4) + h) * blockDim.x];
    f[2 * h] = Two{q.x, q.y}, f[2 * h + 1] = Two{q.z, q.w};
  }
}

template <typename TA, bool kRms, int PER, int kMax, int kCtas>
__global__ void __launch_bounds__(kMax, kCtas)
ln_fwd_shift_kernel(const TA* __restrict__ x, int64_t ldx, const void* __restrict__ w, const void* __restrict__ b,
                    bool f32, float eps, TA* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd,
                    int64_t rows, int cols) {
  using P = Pairs<TA>;
  constexpr int N = P::N, V = 2 * N, S = kPieceStages;
  const int tpr = blockDim.x, t = threadIdx.x, pieces = row_pieces(cols, sizeof(TA)) + 1;
  extern __shared__ uint4 ring[];  // [S][pieces], the output's units [PER tpr + 1], weight and bias [PER][V / 4][tpr]
  uint4* out = ring + S * pieces;
  float4* wheld = reinterpret_cast<float4*>(out + PER * tpr + 1) + t;
  float4* bheld = wheld + PER * (V / 4) * tpr;
  DORA_ROW_SUM(sum, kMax, 1);
  const float inv = 1.0f / float(cols);
  if (w) hold_param<TA, PER>(wheld, w, f32, 1.f, cols);
  if (b) hold_param<TA, PER>(bheld, b, f32, 0.f, cols);
  auto fetch = [&](int64_t r, int s) {
    if (r < rows) fetch_pieces(ring + s * pieces, x + r * ldx, x, cols, t, tpr);
    copies_commit();
  };
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch(blockIdx.x + int64_t(s) * gridDim.x, s);
  int s = 0;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    copies_done<S - 2>();
    __syncthreads();  // the row is there, and everybody is done with the one before
    fetch(r + int64_t(S - 1) * gridDim.x, s == 0 ? S - 1 : s - 1);
    const uint4* row = ring + s * pieces;
    s = s == S - 1 ? 0 : s + 1;
    const int off = in_piece(x + r * ldx);
    Two f[PER][N];
    float one[1];
    Two a = both(0.f);
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int u = p * tpr + t, left = cols - u * V;
      if (left > 0) P::unpack(unit_at<TA>(row, u, off), f[p]);
      if (left < V) keep_first(f[p], left);
#pragma unroll
      for (int i = 0; i < N; ++i) a = add2(a, f[p][i]);
    }
    one[0] = a.a + a.b;
    if constexpr (!kRms) sum(one);
    const float mu = kRms ? 0.f : one[0] * inv;
    Two q = both(0.f);
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int left = cols - (p * tpr + t) * V;
      if constexpr (!kRms) {
#pragma unroll
        for (int i = 0; i < N; ++i) f[p][i] = add2(f[p][i], both(-mu));
        if (left < V) keep_first(f[p], left);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) q = fma2(f[p][i], f[p][i], q);
    }
    one[0] = q.a + q.b;
    sum(one);
    const float rs = rsqrtf(one[0] * inv + eps);
#pragma unroll
    for (int p = 0; p < PER; ++p)
      if ((p * tpr + t) * V < cols) {
        Two v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) f[p][i] = mul2(f[p][i], both(rs));
        if (w) {
          held_unit<TA>(wheld, p, v);
#pragma unroll
          for (int i = 0; i < N; ++i) f[p][i] = mul2(f[p][i], v[i]);
        }
        if (b) {
          held_unit<TA>(bheld, p, v);
#pragma unroll
          for (int i = 0; i < N; ++i) f[p][i] = add2(f[p][i], v[i]);
        }
        out[p * tpr + t] = P::pack(f[p]);
      }
    __syncthreads();
    store_units(y + r * cols, out, cols);
    if (t == 0) {
      if (!kRms && mean) mean[r] = mu;
      if (rstd) rstd[r] = rs;
    }
  }
}

template <typename TA, bool kRms, int PER, int kMax, int kCtas, bool kCols>
__global__ void __launch_bounds__(kMax, kCtas)
ln_bwd_shift_kernel(const TA* __restrict__ dy, int64_t lddy, const TA* __restrict__ x, int64_t ldx,
                    const void* __restrict__ w, bool f32, const float* __restrict__ mean,
                    const float* __restrict__ rstd, TA* __restrict__ dx, float* __restrict__ partial, int64_t rows,
                    int cols, float one_) {
  using P = Pairs<TA>;
  constexpr int N = P::N, V = 2 * N, S = kPieceStages, kSums = kRms ? 1 : 2;
  const int tpr = blockDim.x, t = threadIdx.x, pieces = row_pieces(cols, sizeof(TA)) + 1;
  extern __shared__ uint4 ring[];  // [S][2][pieces], the output's units [PER tpr + 1], the weight [PER][V / 4][tpr]
  uint4* out = ring + 2 * S * pieces;
  float4* wheld = reinterpret_cast<float4*>(out + PER * tpr + 1) + t;
  DORA_ROW_SUM(sum, kMax, kSums);
  const float inv = 1.0f / float(cols);
  const Two one = both(one_);
  hold_param<TA, PER>(wheld, w, f32, 1.f, cols);
  auto fetch = [&](int64_t r, int s) {
    if (r < rows) {
      fetch_pieces(ring + 2 * s * pieces, dy + r * lddy, dy, cols, t, tpr);
      fetch_pieces(ring + (2 * s + 1) * pieces, x + r * ldx, x, cols, t, tpr);
    }
    copies_commit();
  };
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch(blockIdx.x + int64_t(s) * gridDim.x, s);
  Two dw[kCols ? PER : 1][N], db[kCols && !kRms ? PER : 1][N];
#pragma unroll
  for (int p = 0; p < PER; ++p)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (kCols) dw[p][i] = both(0.f);
      if constexpr (kCols && !kRms) db[p][i] = both(0.f);
    }
  int s = 0;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float mu = kRms ? 0.f : mean[r], rs = rstd[r];
    copies_done<S - 2>();
    __syncthreads();  // the row is there, and everybody is done with the one before
    fetch(r + int64_t(S - 1) * gridDim.x, s == 0 ? S - 1 : s - 1);
    const uint4 *drow = ring + 2 * s * pieces, *xrow = drow + pieces;
    s = s == S - 1 ? 0 : s + 1;
    const int doff = in_piece(dy + r * lddy), xoff = in_piece(x + r * ldx);
    uint4 dq[PER], xq[PER];
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int u = p * tpr + t;
      dq[p] = xq[p] = make_uint4(0, 0, 0, 0);
      if (u * V < cols) {
        dq[p] = unit_at<TA>(drow, u, doff);
        xq[p] = unit_at<TA>(xrow, u, xoff);
      }
    }
    auto take = [&](int p, Two (&d)[N], Two (&h)[N], Two (&a)[N]) {  // dy, xh and dy w
      const int left = cols - (p * tpr + t) * V;
      P::unpack(dq[p], d);
      P::unpack(xq[p], h);
      if (left < V) {
        keep_first(d, left);
        keep_first(h, left);
      }
      held_unit<TA>(wheld, p, a);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        a[i] = mul2(d[i], a[i]);
        if constexpr (!kRms) h[i] = add2(h[i], both(-mu));
        h[i] = mul2(h[i], both(rs));
      }
    };
    Two s0 = both(0.f), s1 = both(0.f);
#pragma unroll
    for (int p = 0; p < PER; ++p)
      if ((p * tpr + t) * V < cols) {
        Two d[N], h[N], a[N];
        take(p, d, h, a);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if constexpr (!kRms) s0 = add2_apart(a[i], s0, one);
          s1 = fma2(a[i], h[i], s1);
          if constexpr (kCols) dw[p][i] = fma2(d[i], h[i], dw[p][i]);
          if constexpr (kCols && !kRms) db[p][i] = add2(db[p][i], d[i]);
        }
      }
    if (!dx) continue;  // the same for all threads
    float c[kSums];
    c[0] = s1.a + s1.b;
    if constexpr (!kRms) c[kSums - 1] = s0.a + s0.b;
    sum(c);
    const Two c0 = both(kRms ? 0.f : -c[kSums - 1] * inv), c1 = both(-c[0] * inv);
#pragma unroll
    for (int p = 0; p < PER; ++p)
      if ((p * tpr + t) * V < cols) {
        Two d[N], h[N], a[N];
        take(p, d, h, a);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if constexpr (!kRms) a[i] = add2_apart(a[i], c0, one);
          a[i] = mul2(fma2(h[i], c1, a[i]), both(rs));
        }
        out[p * tpr + t] = P::pack(a);
      }
    __syncthreads();
    store_units(dx + r * cols, out, cols);
  }
  if constexpr (kCols) {
    float* to = partial + int64_t(blockIdx.x) * 2 * cols;
#pragma unroll
    for (int p = 0; p < PER; ++p)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int c = (p * tpr + t) * V + 2 * i;
        if (c < cols) to[c] = dw[p][i].a;
        if (c + 1 < cols) to[c + 1] = dw[p][i].b;
        if constexpr (!kRms) {
          if (c < cols) to[cols + c] = db[p][i].a;
          if (c + 1 < cols) to[cols + c + 1] = db[p][i].b;
        }
      }
    copies_done<0>();
  }
}

// Sums the Z partial rows of dw (and db, `halves` 2): a CTA 32 columns, 8 slices of Z, joined in order.
template <typename TW>
__global__ void __launch_bounds__(kT)
ln_col_finish_kernel(const float* __restrict__ partial, int Z, TW* __restrict__ dw, TW* __restrict__ db, int cols) {
  __shared__ float part[8][33];
  const int half = blockIdx.y;
  TW* out = half ? db : dw;
  if (!out) return;
  const int64_t c = int64_t(blockIdx.x) * 32 + (threadIdx.x & 31);
  const int slice = threadIdx.x / 32;
  float a = 0.f;
  if (c < cols) {
    const float* p = partial + int64_t(half) * cols + c;
    const int z1 = Z * (slice + 1) / 8;
    int z = Z * slice / 8;
    for (; z + 4 <= z1; z += 4) {
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __ldcg(p + int64_t(z + i) * 2 * cols);
#pragma unroll
      for (int i = 0; i < 4; ++i) a += v[i];
    }
    for (; z < z1; ++z) a += __ldcg(p + int64_t(z) * 2 * cols);
  }
  part[slice][threadIdx.x & 31] = a;
  __syncthreads();
  if (slice == 0 && c < cols) {
    for (int i = 1; i < 8; ++i) a += part[i][threadIdx.x & 31];
    out[c] = from_f32<TW>(a);
  }
}

// ---------------------------------------------------------------------------
// Rows wider than the kernels above hold: one CTA a row, which is read again for
// each sum (from L2 after the first time).
// ---------------------------------------------------------------------------
__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  float t = 0.f;
  for (int w = 0; w < kT / 32; ++w) t += red[w];
  __syncthreads();
  return t;
}
template <typename TA, bool kRms>
__global__ void __launch_bounds__(kT)
ln_fwd_wide_kernel(const TA* __restrict__ x, int64_t ldx, const void* __restrict__ w, const void* __restrict__ b,
                   bool f32, float eps, TA* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd,
                   int64_t rows, int64_t cols) {
  __shared__ float red[kT / 32];
  const float inv = 1.0f / float(cols);
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const TA* xr = x + r * ldx;
    float mu = 0.f;
    if constexpr (!kRms) {
      float s = 0.f;
      for (int64_t c = threadIdx.x; c < cols; c += kT) s += to_f32(xr[c]);
      mu = block_sum(s, red) * inv;
    }
    float q = 0.f;
    for (int64_t c = threadIdx.x; c < cols; c += kT) {
      const float d = to_f32(xr[c]) - mu;
      q = fmaf(d, d, q);
    }
    const float rs = rsqrtf(block_sum(q, red) * inv + eps);
    for (int64_t c = threadIdx.x; c < cols; c += kT)
      y[r * cols + c] = from_f32<TA>(fmaf((to_f32(xr[c]) - mu) * rs, param<TA>(w, f32, c, 1.f), param<TA>(b, f32, c, 0.f)));
    if (threadIdx.x == 0) {
      if (!kRms && mean) mean[r] = mu;
      if (rstd) rstd[r] = rs;
    }
  }
}

template <typename TA, bool kRms>
__global__ void __launch_bounds__(kT)
ln_bwd_wide_kernel(const TA* __restrict__ dy, int64_t lddy, const TA* __restrict__ x, int64_t ldx,
                   const void* __restrict__ w, bool f32, const float* __restrict__ mean,
                   const float* __restrict__ rstd, TA* __restrict__ dx, int64_t rows, int64_t cols) {
  __shared__ float red[kT / 32];
  const float inv = 1.0f / float(cols);
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const TA *xr = x + r * ldx, *dr = dy + r * lddy;
    const float mu = kRms ? 0.f : mean[r], rs = rstd[r];
    float s0 = 0.f, s1 = 0.f;
    for (int64_t c = threadIdx.x; c < cols; c += kT) {
      const float a = __fmul_rn(to_f32(dr[c]), param<TA>(w, f32, c, 1.f));
      s0 += a;
      s1 = fmaf(a, (to_f32(xr[c]) - mu) * rs, s1);
    }
    const float c0 = kRms ? 0.f : block_sum(s0, red) * inv;
    const float c1 = block_sum(s1, red) * inv;
    for (int64_t c = threadIdx.x; c < cols; c += kT) {
      const float a = __fmul_rn(to_f32(dr[c]), param<TA>(w, f32, c, 1.f));
      dx[r * cols + c] = from_f32<TA>((a - c0 - (to_f32(xr[c]) - mu) * rs * c1) * rs);
    }
  }
}

// Column sums of one slab of rows.
template <typename TA, bool kRms>
__global__ void __launch_bounds__(kT)
ln_col_wide_kernel(const TA* __restrict__ dy, int64_t lddy, const TA* __restrict__ x, int64_t ldx,
                   const float* __restrict__ mean, const float* __restrict__ rstd, float* __restrict__ partial,
                   int64_t rows, int64_t cols) {
  const int64_t c = int64_t(blockIdx.x) * kT + threadIdx.x;
  if (c >= cols) return;
  const int64_t z = blockIdx.y, Z = gridDim.y;
  float dw = 0.f, db = 0.f;
  for (int64_t r = rows * z / Z; r < rows * (z + 1) / Z; ++r) {
    const float d = to_f32(dy[r * lddy + c]);
    dw = fmaf(d, (to_f32(x[r * ldx + c]) - (kRms ? 0.f : mean[r])) * rstd[r], dw);
    db += d;
  }
  partial[(2 * z) * cols + c] = dw;
  if (!kRms) partial[(2 * z + 1) * cols + c] = db;
}

// ---------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------
unsigned row_grid(int64_t rows) { return unsigned(rows < (1 << 20) ? rows : (1 << 20)); }

// How the threads of the row kernels share rows.
struct Plan {
  int per = 0, most = 0;  // units (elements) a thread holds, threads a CTA has at most; per 0: not for these rows
  Shape shape = {};
  int64_t ctas = 0;
  size_t shared = 0;
};
// CTAs that walk down the rows: as many as the SMs hold, but in the backward, whose every CTA leaves a row of partial
// sums to be read again, at least eight rows to one as long as every SM has one.
int64_t walkers(const Shape& s, int64_t rows, int per_sm, bool fwd) {
  const int64_t need = (rows + s.groups - 1) / s.groups, held = int64_t(num_sms()) * (per_sm > 1 ? per_sm : 1);
  int64_t n = need < held ? need : held;
  if (!fwd && n > num_sms() && n > need / 8) n = need / 8 > num_sms() ? need / 8 : num_sms();
  return n < 1 ? 1 : n;
}
// 16-byte units; `fill` threads an SM have the registers that the kernels take.
Plan plan_units(int64_t rows, int64_t units, bool fwd, int fill) {
  Plan p;
  p.per = fwd ? (units <= 768 * 4 ? 4 : 0) : units <= 2048 ? 2 : 0;
  if (!p.per) return p;
  p.shape = share_row(units, p.per, 128);
  if (fwd) p.most = p.shape.groups > 1 ? 128 : p.shape.threads > 256 ? 768 : 256;
  else p.most = p.shape.groups > 1 ? 128 : units > 1024 ? 1024 : 512;
  p.ctas = walkers(p.shape, rows, fill / p.shape.threads, fwd);
  return p;
}
// Elements, with `buffers` rows in shared memory (200 KB of it an SM).
Plan plan_pieces(int64_t rows, int64_t cols, int size, int buffers) {
  Plan p;
  if (cols > 16384) return p;
  p.per = cols <= 2048 ? 8 : 16;
  p.shape = share_row(cols, p.per, 128);
  p.most = p.shape.groups > 1 ? 128 : cols <= 2048 ? 256 : cols <= 6144 ? 384 : 1024;
  p.shared = size_t(p.shape.groups) * buffers * row_pieces(int(cols), size) * 16;
  if (p.shared > 220 * 1024) return Plan();
  const int fill = p.most == 1024 ? 1024 : kPieceFill;
  const int by_threads = fill / p.shape.threads, by_shared = int(200 * 1024 / (p.shared + 1024));
  p.ctas = walkers(p.shape, rows, by_threads < by_shared ? by_threads : by_shared, buffers <= kPieceStages + 1);
  return p;
}

// Units of rows off a 16-byte boundary; rows of up to 32 units a thread's share stay with plan_pieces.
Plan plan_shift(int64_t rows, int64_t cols, int V, bool fwd) {
  Plan p;
  const int64_t units = (cols + V - 1) / V;
  const int per = units <= 768 ? 2 : 4;
  if (units <= 32 * per || units > 2048 || (!fwd && per > 2)) return p;
  p.per = per;
  p.most = per == 2 ? 384 : 512;
  p.shape = share_row(units, per, 128);
  const int64_t pieces = row_pieces(int(cols), 16 / V) + 1, held = int64_t(per) * p.shape.threads;
  p.shared = size_t(kPieceStages * (fwd ? 1 : 2) * pieces + held + 1 + (fwd ? 2 : 1) * held * (V / 4)) * 16;
  if (p.shared > 220 * 1024) return Plan();
  const int by_threads = per == 2 ? 768 / p.shape.threads : 1, by_shared = int(220 * 1024 / (p.shared + 2048));
  p.ctas = walkers(p.shape, rows, by_threads < by_shared ? by_threads : by_shared, fwd);
  return p;
}

template <typename K> int allow_shared(K kernel, size_t bytes) {
  if (bytes <= 40 * 1024) return DORA_OK;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
  return e == cudaSuccess ? DORA_OK : set_cuda_error(e);
}

template <typename TA, bool kRms>
int launch_fwd(const void* x, int64_t ldx, const void* w, const void* b, bool f32, float eps, void* y, float* mean,
               float* rstd, int64_t rows, int64_t cols, cudaStream_t st) {
  constexpr int V = Vec16<TA>::N;
  const bool vec = cols % V == 0 && ldx % V == 0 && aligned16(x) && aligned16(y) && aligned16(w) && aligned16(b);
  const Plan p = vec ? plan_units(rows, cols / V, true, fwd_fill(f32 == (sizeof(TA) == 4))) : Plan();
  auto X = static_cast<const TA*>(x);
  auto Y = static_cast<TA*>(y);
  if (p.per && vec && (w || !b)) {
    auto go = [&](auto kernel, int buffers) {
      const size_t smem = size_t(buffers) * p.per * p.shape.threads * 16;
      const int e = allow_shared(kernel, smem);
      if (e) return e;
      kernel<<<unsigned(p.ctas), p.shape.threads, smem, st>>>(X, ldx, w, b, eps, Y, mean, rstd, rows, int(cols),
                                                              p.shape.tpr, p.shape.groups);
      return check_launch();
    };
    auto sized = [&](auto tw, auto kind) {
      using TW = decltype(tw);
      constexpr int K = decltype(kind)::value, more = sizeof(TW) == sizeof(TA) ? K : 0;
      constexpr int S = sizeof(TW) == sizeof(TA) ? 4 : 3;
      if (p.most == 128) return go(ln_fwd_kernel<TA, TW, kRms, K, 4, S, 128>, S + more);
      return p.most == 256 ? go(ln_fwd_kernel<TA, TW, kRms, K, 4, S, 256>, S + more)
                           : go(ln_fwd_kernel<TA, TW, kRms, K, 4, 2, 768>, 2 + more);
    };
    auto typed = [&](auto tw) {
      if constexpr (!kRms)
        if (b) return sized(tw, std::integral_constant<int, 2>());
      return sized(tw, std::integral_constant<int, 1>());
    };
    if (!w) return sized(TA(), std::integral_constant<int, 0>());
    if (f32) return typed(float());
    return typed(TA());
  }
  const Plan h = plan_shift(rows, cols, V, true);
  if (h.per) {
    auto go = [&](auto kernel) {
      const int e = allow_shared(kernel, h.shared);
      if (e) return e;
      kernel<<<unsigned(h.ctas), h.shape.threads, h.shared, st>>>(X, ldx, w, b, f32, eps, Y, mean, rstd, rows, int(cols));
      return check_launch();
    };
    return h.per == 2 ? go(ln_fwd_shift_kernel<TA, kRms, 2, 384, 2>) : go(ln_fwd_shift_kernel<TA, kRms, 4, 512, 1>);
  }
  const Plan q = plan_pieces(rows, cols, int(sizeof(TA)), kPieceStages + 1);
  if (q.per) {
    auto go = [&](auto kernel) {
      const int e = allow_shared(kernel, q.shared);
      if (e) return e;
      kernel<<<unsigned(q.ctas), q.shape.threads, q.shared, st>>>(X, ldx, w, b, f32, eps, Y, mean, rstd, rows, int(cols),
                                                                  q.shape.tpr, q.shape.groups);
      return check_launch();
    };
    if (q.most == 128) return go(ln_fwd_pieces_kernel<TA, kRms, 8, 128>);
    if (q.most == 256) return go(ln_fwd_pieces_kernel<TA, kRms, 8, 256>);
    return q.most == 384 ? go(ln_fwd_pieces_kernel<TA, kRms, 16, 384>) : go(ln_fwd_pieces_kernel<TA, kRms, 16, 1024>);
  }
  ln_fwd_wide_kernel<TA, kRms><<<row_grid(rows), kT, 0, st>>>(X, ldx, w, b, f32, eps, Y, mean, rstd, rows, cols);
  return check_launch();
}

// Slabs of rows that the column kernel for wide rows works on.
int slabs_wide(int64_t rows, int64_t cols) {
  const int64_t tiles = (cols + kT - 1) / kT;
  int64_t z = (int64_t(num_sms()) * 8 + tiles - 1) / tiles;
  if (z > rows) z = rows;
  return int(z < 1 ? 1 : z > 1024 ? 1024 : z);
}

template <typename TA, bool kRms, bool kCols>
int launch_bwd_rows(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w, bool f32,
                    const float* mean, const float* rstd, void* dx, float* part, int64_t rows, int64_t cols, int* Z,
                    cudaStream_t st) {
  constexpr int V = Vec16<TA>::N;
  const bool vec = cols % V == 0 && ldx % V == 0 && lddy % V == 0 && aligned16(x) && aligned16(dy) && aligned16(dx) &&
                   aligned16(w);
  const Plan p = vec ? plan_units(rows, cols / V, false, kBwdFill) : Plan();
  auto D = static_cast<const TA*>(dy);
  auto X = static_cast<const TA*>(x);
  auto DX = static_cast<TA*>(dx);
  *Z = int(p.ctas);
  if (p.per) {
    const int S = p.most < 1024 ? 4 : 3;  // 1024 threads' rows fit shared memory three times
    size_t smem = size_t(S) * 4 * p.shape.threads * 16;
    if (smem < size_t(cols) * 8 && p.shape.groups > 1) smem = size_t(cols) * 8;
    auto go = [&](auto kernel) {
      const int e = allow_shared(kernel, smem);
      if (e) return e;
      kernel<<<unsigned(p.ctas), p.shape.threads, smem, st>>>(D, lddy, X, ldx, w, f32, mean, rstd, DX, part, rows,
                                                              int(cols), p.shape.tpr, p.shape.groups, 1.0f);
      return check_launch();
    };
    if (p.most == 128) return go(ln_bwd_kernel<TA, kRms, 2, 4, 128, kCols>);
    return p.most == 512 ? go(ln_bwd_kernel<TA, kRms, 2, 4, 512, kCols>) : go(ln_bwd_kernel<TA, kRms, 2, 3, 1024, kCols>);
  }
  const Plan h = plan_shift(rows, cols, V, false);
  if (h.per) {
    auto kernel = ln_bwd_shift_kernel<TA, kRms, 2, 384, 2, kCols>;
    const int e = allow_shared(kernel, h.shared);
    if (e) return e;
    *Z = int(h.ctas);
    kernel<<<unsigned(h.ctas), h.shape.threads, h.shared, st>>>(D, lddy, X, ldx, w, f32, mean, rstd, DX, part, rows,
                                                                int(cols), 1.0f);
    return check_launch();
  }
  const Plan q = plan_pieces(rows, cols, int(sizeof(TA)), 2 * kPieceStages + 1);
  if (q.per) {
    const size_t smem = kCols && q.shape.groups > 1 && q.shared < size_t(cols) * 8 ? size_t(cols) * 8 : q.shared;
    *Z = int(q.ctas);
    auto go = [&](auto kernel) {
      const int e = allow_shared(kernel, smem);
      if (e) return e;
      kernel<<<unsigned(q.ctas), q.shape.threads, smem, st>>>(D, lddy, X, ldx, w, f32, mean, rstd, DX, part, rows,
                                                              int(cols), q.shape.tpr, q.shape.groups);
      return check_launch();
    };
    if (q.most == 128) return go(ln_bwd_pieces_kernel<TA, kRms, 8, 128, kCols>);
    if (q.most == 256) return go(ln_bwd_pieces_kernel<TA, kRms, 8, 256, kCols>);
    return q.most == 384 ? go(ln_bwd_pieces_kernel<TA, kRms, 16, 384, kCols>)
                         : go(ln_bwd_pieces_kernel<TA, kRms, 16, 1024, kCols>);
  }
  if (dx && rows) {
    ln_bwd_wide_kernel<TA, kRms><<<row_grid(rows), kT, 0, st>>>(D, lddy, X, ldx, w, f32, mean, rstd, DX, rows, cols);
    const int e = check_launch();
    if (e) return e;
  }
  if (!kCols) return DORA_OK;
  *Z = slabs_wide(rows, cols);
  ln_col_wide_kernel<TA, kRms><<<dim3(unsigned((cols + kT - 1) / kT), unsigned(*Z)), kT, 0, st>>>(
      D, lddy, X, ldx, mean, rstd, part, rows, cols);
  return check_launch();
}

size_t bwd_workspace(int64_t rows, int64_t cols) {  // of any type and alignment
  int64_t z = 1;
  for (int V : {4, 8}) {
    const Plan p = plan_units(rows, (cols + V - 1) / V, false, kBwdFill);
    const Plan h = plan_shift(rows, cols, V, false), q = plan_pieces(rows, cols, 16 / V, 2 * kPieceStages + 1);
    for (const int64_t n : {p.ctas, h.ctas, q.ctas, int64_t(p.per && (h.per || q.per) ? 0 : slabs_wide(rows, cols))})
      if (n > z) z = n;
  }
  return size_t(z) * 2 * size_t(cols) * 4;
}

template <typename TA, bool kRms>
int launch_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w, bool f32, const float* mean,
               const float* rstd, void* dx, void* dw, void* db, void* ws, size_t ws_bytes, int64_t rows, int64_t cols,
               cudaStream_t st) {
  const bool sums = dw || db;
  if (sums && (!ws || ws_bytes < bwd_workspace(rows, cols) || !aligned16(ws))) return DORA_ERR_WORKSPACE;
  auto part = static_cast<float*>(ws);
  int Z = 0;
  const int e = sums ? launch_bwd_rows<TA, kRms, true>(dy, lddy, x, ldx, w, f32, mean, rstd, dx, part, rows, cols, &Z, st)
                     : launch_bwd_rows<TA, kRms, false>(dy, lddy, x, ldx, w, f32, mean, rstd, dx, part, rows, cols, &Z, st);
  if (e || !sums) return e;
  const dim3 grid(unsigned((cols + 31) / 32), db ? 2 : 1);
  if (f32) ln_col_finish_kernel<float><<<grid, kT, 0, st>>>(part, Z, static_cast<float*>(dw), static_cast<float*>(db), int(cols));
  else ln_col_finish_kernel<TA><<<grid, kT, 0, st>>>(part, Z, static_cast<TA*>(dw), static_cast<TA*>(db), int(cols));
  return check_launch();
}

bool shape_ok(int64_t rows, int64_t cols, int64_t ld) {
  return rows >= 0 && cols >= 0 && ld >= cols && cols <= (int64_t(1) << 30) && rows <= (int64_t(1) << 40);
}
bool types_ok(int act_dtype, int w_dtype) {
  return dtype_ok(act_dtype) && (w_dtype == act_dtype || w_dtype == DORA_DTYPE_F32);
}

template <typename F>
int by_type(int act_dtype, F f) {
  switch (act_dtype) {
    case DORA_DTYPE_BF16: return f(__nv_bfloat16());
    case DORA_DTYPE_F16: return f(__half());
    default: return f(float());
  }
}

template <bool kRms>
int norm_fwd(const void* x, int64_t ldx, const void* w, const void* b, int w_dtype, double eps, void* y, void* mean,
             void* rstd, int64_t rows, int64_t cols, int act_dtype, void* stream) {
  if (!shape_ok(rows, cols, ldx) || !types_ok(act_dtype, w_dtype) || !(eps >= 0)) return DORA_ERR_INVALID_ARGUMENT;
  if (rows == 0 || cols == 0) return DORA_OK;
  if (!x || !y || x == y) return DORA_ERR_INVALID_ARGUMENT;
  return by_type(act_dtype, [&](auto t) {
    return launch_fwd<decltype(t), kRms>(x, ldx, w, b, w_dtype == DORA_DTYPE_F32, float(eps), y,
                                         static_cast<float*>(mean), static_cast<float*>(rstd), rows, cols,
                                         static_cast<cudaStream_t>(stream));
  });
}

template <bool kRms>
int norm_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w, int w_dtype, const void* mean,
             const void* rstd, void* dx, void* dw, void* db, void* ws, size_t ws_bytes, int64_t rows, int64_t cols,
             int act_dtype, void* stream) {
  if (!shape_ok(rows, cols, ldx) || lddy < cols || !types_ok(act_dtype, w_dtype)) return DORA_ERR_INVALID_ARGUMENT;
  if (cols == 0 || (!dx && !dw && !db)) return DORA_OK;
  if (rows && (!dy || !x || !rstd || (!kRms && !mean) || (dx && (dx == dy || dx == x)))) return DORA_ERR_INVALID_ARGUMENT;
  if (rows == 0 && !dw && !db) return DORA_OK;
  return by_type(act_dtype, [&](auto t) {
    return launch_bwd<decltype(t), kRms>(dy, lddy, x, ldx, w, w_dtype == DORA_DTYPE_F32,
                                         static_cast<const float*>(mean), static_cast<const float*>(rstd), dx, dw, db,
                                         ws, ws_bytes, rows, cols, static_cast<cudaStream_t>(stream));
  });
}

}  // namespace
}  // namespace dora

using namespace dora;

extern "C" int dora_layer_norm_fwd(const void* x, int64_t ldx, const void* weight, const void* bias, int w_dtype,
                                   double eps, void* y, void* mean, void* rstd, int64_t rows, int64_t cols,
                                   int act_dtype, void* stream) {
  return norm_fwd<false>(x, ldx, weight, bias, w_dtype, eps, y, mean, rstd, rows, cols, act_dtype, stream);
}

extern "C" int dora_rms_norm_fwd(const void* x, int64_t ldx, const void* weight, int w_dtype, double eps, void* y,
                                 void* rstd, int64_t rows, int64_t cols, int act_dtype, void* stream) {
  return norm_fwd<true>(x, ldx, weight, nullptr, w_dtype, eps, y, nullptr, rstd, rows, cols, act_dtype, stream);
}

extern "C" size_t dora_layer_norm_bwd_workspace_size(int64_t rows, int64_t cols) {
  if (!shape_ok(rows, cols, cols) || cols == 0) return 0;
  return bwd_workspace(rows, cols);
}

extern "C" int dora_layer_norm_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* weight,
                                   int w_dtype, const void* mean, const void* rstd, void* dx, void* d_weight,
                                   void* d_bias, void* workspace, size_t workspace_bytes, int64_t rows, int64_t cols,
                                   int act_dtype, void* stream) {
  return norm_bwd<false>(dy, lddy, x, ldx, weight, w_dtype, mean, rstd, dx, d_weight, d_bias, workspace,
                         workspace_bytes, rows, cols, act_dtype, stream);
}

extern "C" int dora_rms_norm_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* weight,
                                 int w_dtype, const void* rstd, void* dx, void* d_weight, void* workspace,
                                 size_t workspace_bytes, int64_t rows, int64_t cols, int act_dtype, void* stream) {
  return norm_bwd<true>(dy, lddy, x, ldx, weight, w_dtype, nullptr, rstd, dx, d_weight, nullptr, workspace,
                        workspace_bytes, rows, cols, act_dtype, stream);
}
