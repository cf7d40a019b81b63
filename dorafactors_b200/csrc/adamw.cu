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
#include "dora_common.cuh"

namespace dora {
namespace {

constexpr int kT = 256;
constexpr int kBlock = 256;               // elements of one 8-bit scale: a warp's eight a lane
constexpr int kChunk = 4 * kBlock * (kT / 32);  // elements a CTA works on
// Kernel parameters hold up to 32764 bytes.
constexpr int kMaxTensors = 420;

struct Table {
  dora_adamw_tensor_t t[kMaxTensors];
  uint32_t first[kMaxTensors + 1];  // chunk that each tensor starts at
  int count;
};
struct Scalars {
  float b1, omb1, b2, omb2, rbc2, eps, step, decay;
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

__device__ __forceinline__ float decode_m(uint32_t c, float scale) {
  const float u = (c & 127u) ? __uint_as_float(((c & 127u) + (112u << 3)) << 20) : 0.f;
  return __fmul_rn((c & 128u) ? -u : u, scale);
}
__device__ __forceinline__ float decode_v(uint32_t c, float scale) {
  return __fmul_rn(c ? __uint_as_float((c + (96u << 3)) << 20) : 0.f, scale);
}
__device__ __forceinline__ uint32_t encode_m(float m, float inverse) {
  const int y = __float_as_int(__fmul_rn(fabsf(m), inverse));
  const int c = ((y + (1 << 19)) >> 20) - (112 << 3);
  return uint32_t(c < 0 ? 0 : c > 127 ? 127 : c) | (m < 0.f ? 128u : 0u);
}
__device__ __forceinline__ uint32_t encode_v(float v, float inverse, uint32_t bits16) {
  const int y = __float_as_int(__fmul_rn(v, inverse));
  const int c = ((y + int(bits16 << 4)) >> 20) - (96 << 3);
  return v > 0.f ? uint32_t(c < 1 ? 1 : c > 255 ? 255 : c) : 0u;
}
// Largest magnitude of the block, NaN if there is one.
__device__ __forceinline__ float block_top(const float (&f)[8]) {
  uint32_t top = 0;  // |f|'s bits order like unsigned integers, NaN above infinity
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
  return __uint_as_float(__reduce_max_sync(0xffffffffu, top));
}
// Scale and its inverse; below 2^-100 the block counts as zero (1.875 / top stays finite).
__device__ __forceinline__ void block_scale(float top, float& scale, float& inverse) {
  const bool live = !(top < 0x1p-100f);
  scale = live ? __fmul_rn(top, float(8.0 / 15.0)) : 0.f;
  inverse = live ? __fdiv_rn(1.875f, top) : 0.f;
}
// 32 hashed bits for a pair of elements.
__device__ __forceinline__ uint32_t hash_pair(uint32_t pair, uint32_t key) {
  uint32_t x = pair * 0x85EBCA77u + key;
  x = (x ^ (x >> 15)) * 0xA2C79B4Du;
  x = (x ^ (x >> 13)) * 0x5BD0E6A7u;
  return x ^ (x >> 16);
}

__device__ __forceinline__ bool al(const void* p, unsigned bytes) {
  return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

template <typename TP, bool k8, bool kMaster>
__global__ void __launch_bounds__(kT)
adamw_kernel(const __grid_constant__ Table tab, const Scalars s) {
  int lo = 0, hi = tab.count;  // the tensor with first[lo] <= chunk < first[lo + 1]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (tab.first[mid] <= blockIdx.x) lo = mid;
    else hi = mid;
  }
  const dora_adamw_tensor_t& d = tab.t[lo];
  TP* p = static_cast<TP*>(d.param);
  const TP* g = static_cast<const TP*>(d.grad);
  float* master = static_cast<float*>(d.master);
  const bool vp = al(p, 16), vg = al(g, 16), vw = kMaster && al(master, 16);
  const bool vm = al(d.exp_avg, k8 ? 8 : 16), vv = al(d.exp_avg_sq, k8 ? 8 : 16);
  const int lane = threadIdx.x & 31;
  const int64_t base = int64_t(blockIdx.x - tab.first[lo]) * kChunk;
  for (int64_t b = base + (threadIdx.x / 32) * kBlock; b < base + kChunk && b < d.numel; b += kBlock * (kT / 32)) {
    const int64_t i = b + lane * 8;
    const int n = d.numel - i >= 8 ? 8 : d.numel > i ? int(d.numel - i) : 0;
    float gf[8], pf[8], m[8], v[8];
    load8(g + i, n, vg, gf);
    if constexpr (kMaster) load8(master + i, n, vw, pf);
    else load8(p + i, n, vp, pf);
    if constexpr (k8) {
      const uint64_t mc = load_codes(static_cast<const uint8_t*>(d.exp_avg) + i, n, vm);
      const uint64_t vc = load_codes(static_cast<const uint8_t*>(d.exp_avg_sq) + i, n, vv);
      const float ms = static_cast<const float*>(d.exp_avg_scale)[b / kBlock];
      const float vs = static_cast<const float*>(d.exp_avg_sq_scale)[b / kBlock];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        m[j] = decode_m(uint32_t(mc >> (8 * j)) & 255u, ms);
        v[j] = decode_v(uint32_t(vc >> (8 * j)) & 255u, vs);
      }
    } else {
      load8(static_cast<const float*>(d.exp_avg) + i, n, vm, m);
      load8(static_cast<const float*>(d.exp_avg_sq) + i, n, vv, v);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      m[j] = __fadd_rn(__fmul_rn(m[j], s.b1), __fmul_rn(gf[j], s.omb1));
      v[j] = __fadd_rn(__fmul_rn(v[j], s.b2), __fmul_rn(__fmul_rn(gf[j], gf[j]), s.omb2));
      const float denom = fmaf(sqrtf(v[j]), s.rbc2, s.eps);
      pf[j] = fmaf(pf[j], s.decay, -s.step * (m[j] / denom));
    }
    if constexpr (k8) {
      float ms, mi, vs, vi;
      block_scale(block_top(m), ms, mi);
      block_scale(block_top(v), vs, vi);
      uint64_t mc = 0, vc = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t h = hash_pair(uint32_t(i >> 1) + (j >> 1), d.key);
        mc |= uint64_t(encode_m(m[j], mi)) << (8 * j);
        vc |= uint64_t(encode_v(v[j], vi, (j & 1) ? h >> 16 : h & 0xffffu)) << (8 * j);
      }
      store_codes(static_cast<uint8_t*>(d.exp_avg) + i, n, vm, mc);
      store_codes(static_cast<uint8_t*>(d.exp_avg_sq) + i, n, vv, vc);
      if (lane == 0) {
        static_cast<float*>(d.exp_avg_scale)[b / kBlock] = ms;
        static_cast<float*>(d.exp_avg_sq_scale)[b / kBlock] = vs;
      }
    } else {
      store8(static_cast<float*>(d.exp_avg) + i, n, vm, m);
      store8(static_cast<float*>(d.exp_avg_sq) + i, n, vv, v);
    }
    if constexpr (kMaster) store8(master + i, n, vw, pf);
    store8(p + i, n, vp, pf);
  }
}

// The values that a flat run of 8-bit moments stands for (blocks of 256 from its start).
__global__ void __launch_bounds__(kT)
adamw_decode_kernel(const uint8_t* __restrict__ mc, const float* __restrict__ ms, const uint8_t* __restrict__ vc,
                    const float* __restrict__ vs, float* __restrict__ m, float* __restrict__ v, int64_t n) {
  const int64_t i = (int64_t(blockIdx.x) * kT + threadIdx.x) * 8;
  if (i >= n) return;
  const int c = n - i >= 8 ? 8 : int(n - i);
  const uint64_t a = load_codes(mc + i, c, al(mc, 8)), b = load_codes(vc + i, c, al(vc, 8));
  const float sa = ms[i / kBlock], sb = vs[i / kBlock];
  float fm[8], fv[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    fm[j] = decode_m(uint32_t(a >> (8 * j)) & 255u, sa);
    fv[j] = decode_v(uint32_t(b >> (8 * j)) & 255u, sb);
  }
  store8(m + i, c, al(m, 16), fm);
  store8(v + i, c, al(v, 16), fv);
}

template <typename TP, bool k8, bool kMaster>
int run_step(const dora_adamw_tensor_t* t, int64_t count, const Scalars& s, cudaStream_t st) {
  Table tab;
  int64_t i = 0;
  while (i < count) {
    int n = 0;
    uint64_t chunks = 0;
    for (; i < count && n < kMaxTensors; ++i) {
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
    adamw_kernel<TP, k8, kMaster><<<unsigned(chunks), kT, 0, st>>>(tab, s);
    const int e = check_launch();
    if (e) return e;
  }
  return DORA_OK;
}

template <typename TP>
int run_type(const dora_adamw_tensor_t* t, int64_t count, const Scalars& s, int bits, bool master, cudaStream_t st) {
  if constexpr (sizeof(TP) == 4) {
    return bits == 8 ? run_step<TP, true, false>(t, count, s, st) : run_step<TP, false, false>(t, count, s, st);
  } else {
    if (master) return bits == 8 ? run_step<TP, true, true>(t, count, s, st) : run_step<TP, false, true>(t, count, s, st);
    return bits == 8 ? run_step<TP, true, false>(t, count, s, st) : run_step<TP, false, false>(t, count, s, st);
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
      static_cast<float*>(exp_avg), static_cast<float*>(exp_avg_sq), numel);
  return check_launch();
}
