// f32x2.cuh -- two floats an instruction, and 16-byte chunks as floats.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

namespace nl {

using Pair = unsigned long long;

__device__ __forceinline__ Pair pair(float x, float y) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpair(Pair v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// A 16-byte chunk of N values as N / 2 pairs, and back.
template <typename T> struct Chunk;
template <> struct Chunk<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void get(const uint4 &w, Pair *v) {
    v[0] = pair(__uint_as_float(w.x), __uint_as_float(w.y));
    v[1] = pair(__uint_as_float(w.z), __uint_as_float(w.w));
  }
  static __device__ __forceinline__ uint4 put(const Pair *v) {
    const float2 a = unpair(v[0]), b = unpair(v[1]);
    return make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x),
                      __float_as_uint(b.y));
  }
};
template <> struct Chunk<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ Pair word(uint32_t u) {
    return pair(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t word(Pair v) {
    const float2 f = unpair(v);
    const __nv_bfloat162 p = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t *>(&p);
  }
  static __device__ __forceinline__ void get(const uint4 &w, Pair *v) {
    v[0] = word(w.x); v[1] = word(w.y); v[2] = word(w.z); v[3] = word(w.w);
  }
  static __device__ __forceinline__ uint4 put(const Pair *v) {
    return make_uint4(word(v[0]), word(v[1]), word(v[2]), word(v[3]));
  }
};

}  // namespace nl
