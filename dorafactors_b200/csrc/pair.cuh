// Two fp32 numbers in one instruction (sm_100's packed forms), each rounded like its scalar form.
#pragma once

#include "dora_common.cuh"

namespace dora {

struct Two {
  float a, b;
};
__device__ __forceinline__ unsigned long long bits2(Two x) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x.a), "f"(x.b));
  return r;
}
__device__ __forceinline__ Two two(unsigned long long r) {
  Two x;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x.a), "=f"(x.b) : "l"(r));
  return x;
}
__device__ __forceinline__ Two both(float x) { return Two{x, x}; }
__device__ __forceinline__ Two mul2(Two x, Two y) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(x)), "l"(bits2(y)));
  return two(r);
}
__device__ __forceinline__ Two fma2(Two x, Two y, Two z) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits2(x)), "l"(bits2(y)), "l"(bits2(z)));
  return two(r);
}
// A sum.  Where x or y is a product, the compiler may join the two into an FMA with one rounding.
__device__ __forceinline__ Two add2(Two x, Two y) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(x)), "l"(bits2(y)));
  return two(r);
}
// A sum of rounded operands, whatever they are: an FMA by a 1 that the compiler does not know.
__device__ __forceinline__ Two add2_apart(Two x, Two y, Two one) { return fma2(x, one, y); }

// A 16-byte vector as pairs.
template <typename T> struct Pairs {
  static constexpr int N = Vec16<T>::N / 2;
  __device__ __forceinline__ static void unpack(const uint4& v, Two (&f)[N]) {
    if constexpr (sizeof(T) == 4) {
      f[0] = Two{__uint_as_float(v.x), __uint_as_float(v.y)};
      f[1] = Two{__uint_as_float(v.z), __uint_as_float(v.w)};
    } else {
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = unpack_word(w[i], T());
    }
  }
  __device__ __forceinline__ static uint4 pack(const Two (&f)[N]) {
    if constexpr (sizeof(T) == 4) {
      return make_uint4(__float_as_uint(f[0].a), __float_as_uint(f[0].b), __float_as_uint(f[1].a),
                        __float_as_uint(f[1].b));
    } else {
      return make_uint4(pack_word(f[0], T()), pack_word(f[1], T()), pack_word(f[2], T()), pack_word(f[3], T()));
    }
  }

 private:
  __device__ __forceinline__ static Two unpack_word(uint32_t w, __nv_bfloat16) {
    return Two{__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
  }
  __device__ __forceinline__ static Two unpack_word(uint32_t w, __half) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return Two{f.x, f.y};
  }
  __device__ __forceinline__ static uint32_t pack_word(Two f, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f.a, f.b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ __forceinline__ static uint32_t pack_word(Two f, __half) {
    const __half2 h = __floats2half2_rn(f.a, f.b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

// The 16 bytes that start `off` elements of T (0 .. a vector less one; the same for all threads) after a's first, of a and
// the vector b after it.
template <typename T> __device__ __forceinline__ uint4 cut(const uint4& a, const uint4& b, int off) {
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  uint32_t o[5];
  switch (sizeof(T) == 4 ? off : off / 2) {
    case 0: for (int i = 0; i < 5; ++i) o[i] = w[i]; break;
    case 1: for (int i = 0; i < 5; ++i) o[i] = w[i + 1]; break;
    case 2: for (int i = 0; i < 5; ++i) o[i] = w[i + 2]; break;
    default: for (int i = 0; i < 5; ++i) o[i] = w[i + 3]; break;
  }
  if (sizeof(T) == 2 && (off & 1))
    for (int i = 0; i < 4; ++i) o[i] = __byte_perm(o[i], o[i + 1], 0x5432);
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// A 16-byte copy to shared memory that runs on its own; a thread that reads back only what it has copied
// itself needs no barrier, just copies_done.
__device__ __forceinline__ void copy_async16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_async8(uint32_t to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLater> __device__ __forceinline__ void copies_done() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kLater) : "memory");
}
__device__ __forceinline__ uint32_t shared_addr(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }

}  // namespace dora
