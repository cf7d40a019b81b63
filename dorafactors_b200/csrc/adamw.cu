// AdamW over many tensors in one launch, with fp32 moments or moments of 8 bits.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g g
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// The tensors' addresses travel as kernel parameters (no table in device memory, so
// nothing of an earlier call is kept and a launch can be captured).  m and v are
// evaluated with one rounding per operation (no FMA), so that a value that lies
// between two 8-bit codes is rounded the same way by any implementation.
//
// 8-bit moments: a warp owns a block of 256 elements, eight a lane; the block's scale is
// its largest magnitude / 1.875 and a code holds the upper bits of the scaled fp32 number:
//   m: sign, 4 exponent and 3 mantissa bits, round to nearest: |m| down to 2^-15 of the
//      largest keeps a relative error of 1/16, and m moves by tenths a step;
//   v: 5 exponent and 3 mantissa bits (2^-31 of the largest), rounded up or down by 16
//      hashed bits: with b2 = 0.999 a step changes v by less than half a code, which
//      rounding to nearest would lose every time.  A v > 0 never becomes 0, since
//      sqrt(v) = 0 would leave only eps in the denominator.
//
// Measured over 672 tensors, 337M elements: fp32 1459 us (HBM, 0.99 of the copy rate); bf16 with 8-bit moments
// 783 us (the ALU pipe, 75 % busy; HBM alone would take 517 us), their values 508 us (HBM).
#include <cfloat>
#include <type_traits>

#include "pair.cuh"

namespace dora {
namespace {

constexpr int kT = 256;
constexpr int kBlock = 256;               // elements of one 8-bit scale: a warp's eight a lane
constexpr int kChunk = 4 * kBlock * (kT / 32);  // elements a CTA works on
// Kernel parameters hold up to 32764 bytes.
constexpr int kMaxTensors = 420;
constexpr int kFewTensors = 12;

template <int N> struct Table {
  dora_adamw_tensor_t t[N];
  uint32_t first[N + 1];  // chunk that each tensor starts at
  int count;
};
struct Scalars {
  float b1, omb1, b2, omb2, rbc2, eps, step, decay;
  float rbc2_step, eps_step;  // rbc2 and eps over -step: their reciprocal has the step in it
  float one;  // 1, as a value that the compiler does not know
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, int n, bool vec, float (&f)[8]) {
  if (vec && n == 8) {
    if constexpr (sizeof(T) == 4) {
      float lo[4], hi[4];
      Vec16<T>::unpack(ld_stream_coherent(p), lo);
      Vec16<T>::unpack(ld_stream_coherent(p + 4), hi);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = lo[i], f[4 + i] = hi[i];
    } else {
      Vec16<T>::unpack(ld_stream_coherent(p), f);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < n ? to_f32(p[i]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int n, bool vec, const float (&f)[8]) {
  if (vec && n == 8) {
    if constexpr (sizeof(T) == 4) {
      const float lo[4] = {f[0], f[1], f[2], f[3]}, hi[4] = {f[4], f[5], f[6], f[7]};
      st_global(p, Vec16<T>::pack(lo));
      st_global(p + 4, Vec16<T>::pack(hi));
    } else {
      st_global(p, Vec16<T>::pack(f));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = from_f32<T>(f[i]);
  }
}
__device__ __forceinline__ uint64_t load_codes(const uint8_t* p, int n, bool vec) {
  if (vec && n == 8) return *reinterpret_cast<const uint64_t*>(p);
  uint64_t c = 0;
  for (int i = 0; i < n; ++i) c |= uint64_t(p[i]) << (8 * i);
  return c;
}
__device__ __forceinline__ void store_codes(uint8_t* p, int n, bool vec, uint64_t c) {
  if (vec && n == 8) *reinterpret_cast<uint64_t*>(p) = c;
  else
    for (int i = 0; i < n; ++i) p[i] = uint8_t(c >> (8 * i));
}

// The work on codes is what bounds the 8-bit step (the ALU pipe: shifts, logic, minima), so it is laid
// out in few such operations.  A code is bits 27..20 of the scaled number's fp32 pattern, the sign in
// place of bit 27 for the first moment: the rest of the exponent is constant and its lower bits are
// zero, so it is masked off and OR-ed on rather than subtracted and added.  `top`: the code in bits 31..24.
__device__ __forceinline__ float decode_m(uint32_t top) {  // unscaled, code 0 as 2^-15
  return __uint_as_float(uint32_t(int(top) >> 4) & 0x87f00000u | (112u << 23));
}
__device__ __forceinline__ float decode_v(uint32_t top) {  // unscaled, code 0 as 2^-31
  return __uint_as_float((top >> 4) & 0x0ff00000u | (96u << 23));
}
__device__ __forceinline__ bool zero_m(uint32_t w) {  // is one of four codes +-0?
  return (((w & 0x7f7f7f7fu) + 0x7f7f7f7fu) & 0x80808080u) != 0x80808080u;
}
__device__ __forceinline__ bool zero_v(uint32_t w) { return ((w - 0x01010101u) & ~w & 0x80808080u) != 0; }

// The code comes back in bits 31..24 (others are not zero).  y: the scaled moment.  The patterns of
// the values below 2^-15 (1.125 2^-31) of a block round to the codes' lower end.
__device__ __forceinline__ uint32_t encode_m(float y) {
  const uint32_t z = __float_as_uint(fmaxf(fabsf(y), 0x1p-15f)) * 16u + (1u << 23);
  return z & 0x7fffffffu | __float_as_uint(y) & 0x80000000u;
}
__device__ __forceinline__ uint32_t encode_v(float y, uint32_t tail) {
  return __float_as_uint(fmaxf(y, 0x1.2p-31f)) * 16u + tail;
}
__device__ __forceinline__ uint32_t tops(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0073), __byte_perm(c, d, 0x0073), 0x5410);
}
// 16 hashed bits for each element of a pair, in bits 23..8: the halves of a hash x ^ (x >> 16).
__device__ __forceinline__ void hash_pair(uint32_t pair, uint32_t key, uint32_t& even, uint32_t& odd) {
  uint32_t x = pair * 0x85EBCA77u + key;
  x = (x ^ (x >> 15)) * 0xA2C79B4Du;
  x = (x ^ (x >> 13)) * 0x5BD0E6A7u;
  odd = __byte_perm(x, 0, 0x4324);
  even = __byte_perm(x, 0, 0x4104) ^ odd;
}
// The largest of three, NaN if there is one.
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float sqrt_fast(float x) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__host__ __device__ __forceinline__ bool al(const void* p, unsigned bytes) {
  return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

// What a lane works on: eight elements, as they came from memory.
template <bool k8> struct Lane {
  float g[8], p[8];
  float m[k8 ? 1 : 8], v[k8 ? 1 : 8];
  uint64_t mc, vc;  // codes
  float ms, vs;     // their scales
};

// One warp's 256 elements from b on, n of this lane's eight.  kFull: all are there and aligned.
template <typename TP, bool k8, bool kMaster, bool kFull>
__device__ __forceinline__ void step_block(const dora_adamw_tensor_t& d, const Scalars& s, int64_t b, int n,
                                           Lane<k8>& x) {
  const int lane = threadIdx.x & 31;
  const int64_t i = b + lane * 8;
  float (&gf)[8] = x.g, (&pf)[8] = x.p;
  Two m[4], v[4];
  bool zeros = false;  // may a v be 0?  Only where its code was, or in a block that counts as zero
  if constexpr (k8) {
    const uint64_t mc = x.mc, vc = x.vc;
    const Two ms = both(x.ms), vs = both(x.vs);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t mw = uint32_t(mc >> (32 * h)), vw = uint32_t(vc >> (32 * h));
      Two *mh = m + 2 * h, *vh = v + 2 * h;
      mh[0] = Two{decode_m(mw << 24), decode_m(mw << 16)}, mh[1] = Two{decode_m(mw << 8), decode_m(mw)};
      vh[0] = Two{decode_v(vw << 24), decode_v(vw << 16)}, vh[1] = Two{decode_v(vw << 8), decode_v(vw)};
      if (zero_m(mw)) {  // seldom, once a tensor has seen gradients
        if (!(mw & 0x7fu)) mh[0].a = 0.f;
        if (!(mw & 0x7f00u)) mh[0].b = 0.f;
        if (!(mw & 0x7f0000u)) mh[1].a = 0.f;
        if (!(mw & 0x7f000000u)) mh[1].b = 0.f;
      }
      if (zero_v(vw)) {
        zeros = true;
        if (!(vw & 0xffu)) vh[0].a = 0.f;
        if (!(vw & 0xff00u)) vh[0].b = 0.f;
        if (!(vw & 0xff0000u)) vh[1].a = 0.f;
        if (!(vw & 0xff000000u)) vh[1].b = 0.f;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) mh[j] = mul2(mh[j], ms), vh[j] = mul2(vh[j], vs);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) m[j] = Two{x.m[2 * j], x.m[2 * j + 1]}, v[j] = Two{x.v[2 * j], x.v[2 * j + 1]};
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const Two g{gf[2 * j], gf[2 * j + 1]};
    m[j] = add2_apart(mul2(m[j], both(s.b1)), mul2(g, both(s.omb1)), both(s.one));
    v[j] = add2_apart(mul2(v[j], both(s.b2)), mul2(mul2(g, g), both(s.omb2)), both(s.one));
    Two q;
    if constexpr (k8) {
      // Two units in the last place of the step are far below the codes' own rounding.  2^-126 is
      // nothing beside any other v, but keeps the root of one below the normal range from flushing to 0.
      const Two w = fma2(v[j], both(s.one), both(0x1p-126f));
      const Two root{sqrt_fast(w.a), sqrt_fast(w.b)};
      const Two denom = fma2(root, both(s.rbc2_step), both(s.eps_step));
      q = mul2(m[j], Two{rcp_fast(denom.a), rcp_fast(denom.b)});
    } else {
      const Two denom = fma2(Two{sqrtf(v[j].a), sqrtf(v[j].b)}, both(s.rbc2), both(s.eps));
      q = mul2(Two{m[j].a / denom.a, m[j].b / denom.b}, both(-s.step));
    }
    const Two r = fma2(Two{pf[2 * j], pf[2 * j + 1]}, both(s.decay), q);
    pf[2 * j] = r.a;
    pf[2 * j + 1] = r.b;
  }
  if constexpr (kMaster) store8(static_cast<float*>(d.master) + i, n, kFull, pf);
  store8(static_cast<TP*>(d.param) + i, n, kFull, pf);
  if constexpr (k8) {
    float tm = 0.f, tv = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      tm = max_nan(tm, fabsf(m[j].a), fabsf(m[j].b));
      tv = max_nan(tv, v[j].a, v[j].b);
    }
    // Magnitudes' bits order like unsigned integers, NaN above infinity.  Even lanes work out the first
    // moment's scale, odd ones the second's; below 2^-100 a block counts as zero (1.875 / top stays finite).
    const uint32_t um = __reduce_max_sync(0xffffffffu, __float_as_uint(tm));
    const uint32_t uv = __reduce_max_sync(0xffffffffu, __float_as_uint(tv));
    const float top = __uint_as_float((lane & 1) ? uv : um);
    const bool live = !(top < 0x1p-100f);
    const float inverse = live ? __fdiv_rn(1.875f, top) : 0.f;
    const Two mi = both(__shfl_sync(0xffffffffu, inverse, 0));
    const Two vi = both(__shfl_sync(0xffffffffu, inverse, 1));
    if (lane < 2)
      static_cast<float*>(lane ? d.exp_avg_sq_scale : d.exp_avg_scale)[b / kBlock] =
          live ? __fmul_rn(top, float(8.0 / 15.0)) : 0.f;
    zeros |= x.vs == 0.f;
    uint32_t mc[2], vc[2];
    const uint32_t pair = uint32_t(i >> 1);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const Two *mh = m + 2 * h, *vh = v + 2 * h;
      uint32_t c[4], t[4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        // A moment of -0 takes the code of +0.
        const Two y = fma2(mh[j], mi, both(0.f));
        c[2 * j] = encode_m(y.a), c[2 * j + 1] = encode_m(y.b);
      }
      mc[h] = tops(c[0], c[1], c[2], c[3]);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const Two y = mul2(vh[j], vi);
        hash_pair(pair + 2 * h + j, d.key, t[0], t[1]);
        c[2 * j] = encode_v(y.a, t[0]), c[2 * j + 1] = encode_v(y.b, t[1]);
      }
      vc[h] = tops(c[0], c[1], c[2], c[3]);
      if (zeros) {  // only a v of 0 has code 0
        if (!(vh[0].a > 0.f)) vc[h] &= 0xffffff00u;
        if (!(vh[0].b > 0.f)) vc[h] &= 0xffff00ffu;
        if (!(vh[1].a > 0.f)) vc[h] &= 0xff00ffffu;
        if (!(vh[1].b > 0.f)) vc[h] &= 0x00ffffffu;
      }
    }
    store_codes(static_cast<uint8_t*>(d.exp_avg) + i, n, kFull, uint64_t(mc[1]) << 32 | mc[0]);
    store_codes(static_cast<uint8_t*>(d.exp_avg_sq) + i, n, kFull, uint64_t(vc[1]) << 32 | vc[0]);
  } else {
    float f[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) f[2 * j] = m[j].a, f[2 * j + 1] = m[j].b;
    store8(static_cast<float*>(d.exp_avg) + i, n, kFull, f);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[2 * j] = v[j].a, f[2 * j + 1] = v[j].b;
    store8(static_cast<float*>(d.exp_avg_sq) + i, n, kFull, f);
  }
}

template <typename TP, bool k8, bool kMaster, bool kFull>
__device__ __forceinline__ void load_block(const dora_adamw_tensor_t& d, int64_t b, int n, Lane<k8>& x) {
  const int64_t i = b + (threadIdx.x & 31) * 8;
  load8(static_cast<const TP*>(d.grad) + i, n, kFull, x.g);
  if constexpr (kMaster) load8(static_cast<const float*>(d.master) + i, n, kFull, x.p);
  else load8(static_cast<const TP*>(d.param) + i, n, kFull, x.p);
  if constexpr (k8) {
    x.mc = load_codes(static_cast<const uint8_t*>(d.exp_avg) + i, n, kFull);
    x.vc = load_codes(static_cast<const uint8_t*>(d.exp_avg_sq) + i, n, kFull);
    x.ms = static_cast<const float*>(d.exp_avg_scale)[b / kBlock];
    x.vs = static_cast<const float*>(d.exp_avg_sq_scale)[b / kBlock];
  } else {
    load8(static_cast<const float*>(d.exp_avg) + i, n, kFull, x.m);
    load8(static_cast<const float*>(d.exp_avg_sq) + i, n, kFull, x.v);
  }
}

// A tensor's last block, and blocks of misaligned tensors.
template <typename TP, bool k8, bool kMaster>
__device__ __noinline__ void step_part(const dora_adamw_tensor_t& d, const Scalars& s, int64_t b) {
  const int64_t i = b + (threadIdx.x & 31) * 8;
  const int n = d.numel - i >= 8 ? 8 : d.numel > i ? int(d.numel - i) : 0;
  Lane<k8> x;
  load_block<TP, k8, kMaster, false>(d, b, n, x);
  step_block<TP, k8, kMaster, false>(d, s, b, n, x);
}

// A lane's inputs of the 8-bit step on their way through shared memory: the copies of the next blocks run while
// one is worked on, without registers for them.  A lane reads only what it has copied itself.
template <int kWords, int kGradWords> struct Stage {
  uint4 g[kGradWords][32], p[kWords][32];
  uint2 m[32], v[32];
};
template <typename T> __device__ __forceinline__ void unstage(const uint4 (*w)[32], int lane, float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    float lo[4], hi[4];
    Vec16<T>::unpack(w[0][lane], lo);
    Vec16<T>::unpack(w[1][lane], hi);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = lo[i], f[4 + i] = hi[i];
  } else {
    Vec16<T>::unpack(w[0][lane], f);
  }
}

template <typename TP, bool k8, bool kMaster, int N>
__global__ void __launch_bounds__(kT, k8 ? 4 : 3)
adamw_kernel(const __grid_constant__ Table<N> tab, const __grid_constant__ Scalars s) {
  int lo = 0, hi = tab.count;  // the tensor with first[lo] <= chunk < first[lo + 1]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (tab.first[mid] <= blockIdx.x) lo = mid;
    else hi = mid;
  }
  const dora_adamw_tensor_t& d = tab.t[lo];
  const bool aligned = al(d.param, 16) && al(d.grad, 16) && (!kMaster || al(d.master, 16)) &&
                       al(d.exp_avg, k8 ? 8 : 16) && al(d.exp_avg_sq, k8 ? 8 : 16);
  constexpr int kStride = kBlock * (kT / 32);
  const int64_t base = int64_t(blockIdx.x - tab.first[lo]) * kChunk;
  const int64_t end = base + kChunk < d.numel ? base + kChunk : d.numel;
  int64_t b = base + (threadIdx.x / 32) * kBlock;
  if constexpr (k8) {
    using TM = typename std::conditional<kMaster, float, TP>::type;  // what the step is taken on
    constexpr int kWords = sizeof(TM) / 2, kGradWords = sizeof(TP) / 2;
    constexpr int kAhead = kGradWords == 2 ? 1 : 2;  // blocks on their way; 48 KB of shared memory are the limit
    using Staged = Stage<kWords, kGradWords>;
    __shared__ Staged ring[kT / 32][kAhead + 1];
    Staged* st = ring[threadIdx.x / 32];
    const int lane = threadIdx.x & 31;
    const int full = aligned && end - b >= kBlock ? int((end - b - kBlock) / kStride) + 1 : 0;
    const TP* g = static_cast<const TP*>(d.grad) + b + lane * 8;
    const TM* p = static_cast<const TM*>(kMaster ? d.master : d.param) + b + lane * 8;
    const uint8_t *mc = static_cast<const uint8_t*>(d.exp_avg) + b + lane * 8,
                  *vc = static_cast<const uint8_t*>(d.exp_avg_sq) + b + lane * 8;
    auto fetch = [&](int k) {  // block k of this warp, if there is one
      if (k < full) {
        Staged& to = st[k % (kAhead + 1)];
        const int64_t o = int64_t(k) * kStride;
#pragma unroll
        for (int w = 0; w < kGradWords; ++w) copy_async16(shared_addr(&to.g[w][lane]), g + o + w * 4);
#pragma unroll
        for (int w = 0; w < kWords; ++w) copy_async16(shared_addr(&to.p[w][lane]), p + o + w * 4);
        copy_async8(shared_addr(&to.m[lane]), mc + o);
        copy_async8(shared_addr(&to.v[lane]), vc + o);
      }
      copies_commit();
    };
    const float *ms = static_cast<const float*>(d.exp_avg_scale), *vs = static_cast<const float*>(d.exp_avg_sq_scale);
    float ms0 = 0.f, vs0 = 0.f;
    if (full) ms0 = ms[b / kBlock], vs0 = vs[b / kBlock];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) fetch(k);
#pragma unroll 1
    for (int k = 0; k < full; ++k, b += kStride) {
      fetch(k + kAhead);
      copies_done<kAhead>();
      const Staged& from = st[k % (kAhead + 1)];
      Lane<true> x;
      unstage<TP>(from.g, lane, x.g);
      unstage<TM>(from.p, lane, x.p);
      const uint2 m2 = from.m[lane], v2 = from.v[lane];
      x.mc = uint64_t(m2.y) << 32 | m2.x;
      x.vc = uint64_t(v2.y) << 32 | v2.x;
      x.ms = ms0;
      x.vs = vs0;
      if (k + 1 < full) ms0 = ms[b / kBlock + kT / 32], vs0 = vs[b / kBlock + kT / 32];
      step_block<TP, true, kMaster, true>(d, s, b, 8, x);
    }
    for (; b < end; b += kStride) step_part<TP, true, kMaster>(d, s, b);
  } else {
    for (; b < end; b += kStride) {
      if (aligned && b + kBlock <= d.numel) {
        Lane<false> x;
        load_block<TP, false, kMaster, true>(d, b, 8, x);
        step_block<TP, false, kMaster, true>(d, s, b, 8, x);
      } else {
        step_part<TP, false, kMaster>(d, s, b);
      }
    }
  }
}

__device__ __forceinline__ float value_m(uint32_t c, float scale) {  // of the code in bits 7..0
  return __fmul_rn((c & 127u) ? decode_m(c << 24) : 0.f, scale);
}
__device__ __forceinline__ float value_v(uint32_t c, float scale) {
  return __fmul_rn((c & 255u) ? decode_v(c << 24) : 0.f, scale);
}

// The values that a flat run of 8-bit moments stands for (blocks of 256 from its start).  A warp
// decodes a block, lane l elements 4 l .. 4 l + 3 of each half, so that every store is 512 contiguous bytes.
__global__ void __launch_bounds__(kT)
adamw_decode_kernel(const uint8_t* __restrict__ mc, const float* __restrict__ ms, const uint8_t* __restrict__ vc,
                    const float* __restrict__ vs, float* __restrict__ m, float* __restrict__ v, int64_t n, bool vec) {
  const int64_t block = (int64_t(blockIdx.x) * kT + threadIdx.x) / 32;
  const int64_t b = block * kBlock;
  if (b >= n) return;
  const int lane = threadIdx.x & 31;
  const float sa = ms[block], sb = vs[block];
  if (vec && b + kBlock <= n) {
    uint32_t a[2], c[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      a[h] = __ldcs(reinterpret_cast<const uint32_t*>(mc + b) + 32 * h + lane);
      c[h] = __ldcs(reinterpret_cast<const uint32_t*>(vc + b) + 32 * h + lane);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float fm[4], fv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        fm[j] = value_m(a[h] >> (8 * j), sa);
        fv[j] = value_v(c[h] >> (8 * j), sb);
      }
      st_stream(m + b + 128 * h + 4 * lane, Vec16<float>::pack(fm));
      st_stream(v + b + 128 * h + 4 * lane, Vec16<float>::pack(fv));
    }
  } else {
    for (int64_t i = b + lane; i < b + kBlock && i < n; i += 32) {
      m[i] = value_m(mc[i], sa);
      v[i] = value_v(vc[i], sb);
    }
  }
}

template <typename TP, bool k8, bool kMaster, int N>
int run_step(const dora_adamw_tensor_t* t, int64_t count, const Scalars& s, cudaStream_t st) {
  Table<N> tab;
  int64_t i = 0;
  while (i < count) {
    int n = 0;
    uint64_t chunks = 0;
    for (; i < count && n < N; ++i) {
      const uint64_t c = (uint64_t(t[i].numel) + kChunk - 1) / kChunk;
      if (c == 0) continue;
      if (chunks + c > 0x7fffffffu) break;
      tab.t[n] = t[i];
      tab.first[n++] = uint32_t(chunks);
      chunks += c;
    }
    if (n == 0) break;
    tab.first[n] = uint32_t(chunks);
    tab.count = n;
    adamw_kernel<TP, k8, kMaster, N><<<unsigned(chunks), kT, 0, st>>>(tab, s);
    const int e = check_launch();
    if (e) return e;
  }
  return DORA_OK;
}

// A launch with 32 KB of parameters takes the host longer than one with 1 KB.
template <typename TP, bool k8, bool kMaster>
int run_sized(const dora_adamw_tensor_t* t, int64_t count, const Scalars& s, cudaStream_t st) {
  return count <= kFewTensors ? run_step<TP, k8, kMaster, kFewTensors>(t, count, s, st)
                              : run_step<TP, k8, kMaster, kMaxTensors>(t, count, s, st);
}

template <typename TP>
int run_type(const dora_adamw_tensor_t* t, int64_t count, const Scalars& s, int bits, bool master, cudaStream_t st) {
  if constexpr (sizeof(TP) == 4) {
    return bits == 8 ? run_sized<TP, true, false>(t, count, s, st) : run_sized<TP, false, false>(t, count, s, st);
  } else {
    if (master) return bits == 8 ? run_sized<TP, true, true>(t, count, s, st) : run_sized<TP, false, true>(t, count, s, st);
    return bits == 8 ? run_sized<TP, true, false>(t, count, s, st) : run_sized<TP, false, false>(t, count, s, st);
  }
}

}  // namespace
}  // namespace dora

using namespace dora;

extern "C" int dora_adamw_step(const dora_adamw_tensor_t* tensors, int64_t count, int param_dtype, int state_bits,
                               double lr, double beta1, double beta2, double eps, double weight_decay, int64_t step,
                               void* stream) {
  if (count < 0 || !dtype_ok(param_dtype) || (state_bits != 8 && state_bits != 32) || step < 1 || !(lr >= 0) ||
      !(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1) || !(eps >= 0) || !(weight_decay >= 0))
    return DORA_ERR_INVALID_ARGUMENT;
  if (count == 0) return DORA_OK;
  if (!tensors) return DORA_ERR_INVALID_ARGUMENT;
  const bool master = tensors[0].master != nullptr;
  if (master && param_dtype == DORA_DTYPE_F32) return DORA_ERR_INVALID_ARGUMENT;
  for (int64_t i = 0; i < count; ++i) {
    const dora_adamw_tensor_t& t = tensors[i];
    if (t.numel < 0 || t.numel > (int64_t(1) << 40)) return DORA_ERR_INVALID_ARGUMENT;
    if (t.numel == 0) continue;
    if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq || (t.master != nullptr) != master ||
        (state_bits == 8 && (!t.exp_avg_scale || !t.exp_avg_sq_scale)))
      return DORA_ERR_INVALID_ARGUMENT;
  }
  Scalars s;
  s.b1 = float(beta1);
  s.omb1 = float(1.0 - beta1);
  s.b2 = float(beta2);
  s.omb2 = float(1.0 - beta2);
  s.rbc2 = float(1.0 / sqrt(1.0 - pow(beta2, double(step))));
  s.eps = float(eps);
  s.step = float(lr / (1.0 - pow(beta1, double(step))));
  s.decay = float(1.0 - lr * weight_decay);
  // A step of 0 divides by the largest number there is: m over it is nothing.
  s.rbc2_step = s.step > 0.f ? -s.rbc2 / s.step : -FLT_MAX;
  s.eps_step = s.step > 0.f ? -s.eps / s.step : 0.f;
  s.one = 1.0f;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (param_dtype) {
    case DORA_DTYPE_BF16: return run_type<__nv_bfloat16>(tensors, count, s, state_bits, master, st);
    case DORA_DTYPE_F16: return run_type<__half>(tensors, count, s, state_bits, master, st);
    default: return run_type<float>(tensors, count, s, state_bits, master, st);
  }
}

extern "C" int dora_adamw_decode(const void* exp_avg_codes, const void* exp_avg_scale, const void* exp_avg_sq_codes,
                                 const void* exp_avg_sq_scale, void* exp_avg, void* exp_avg_sq, int64_t numel,
                                 void* stream) {
  if (numel < 0 || numel > (int64_t(1) << 40)) return DORA_ERR_INVALID_ARGUMENT;
  if (numel == 0) return DORA_OK;
  if (!exp_avg_codes || !exp_avg_scale || !exp_avg_sq_codes || !exp_avg_sq_scale || !exp_avg || !exp_avg_sq)
    return DORA_ERR_INVALID_ARGUMENT;
  const int64_t grid = (numel + 8 * kT - 1) / (8 * kT);
  adamw_decode_kernel<<<unsigned(grid), kT, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint8_t*>(exp_avg_codes), static_cast<const float*>(exp_avg_scale),
      static_cast<const uint8_t*>(exp_avg_sq_codes), static_cast<const float*>(exp_avg_sq_scale),
      static_cast<float*>(exp_avg), static_cast<float*>(exp_avg_sq), numel,
      al(exp_avg_codes, 4) && al(exp_avg_sq_codes, 4) && al(exp_avg, 16) && al(exp_avg_sq, 16));
  return check_launch();
}
