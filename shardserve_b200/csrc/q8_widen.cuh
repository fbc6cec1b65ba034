// From 8-bit codes to the operand types of the tensor cores: fp16 for Q.K, fp32 (read as tf32) for
// P.V.  Both hold every code exactly.
#pragma once

#include <cuda_fp16.h>

#include "ptx.cuh"
#include "q8.cuh"

namespace ss {

constexpr float kMinVs = 0x1p-80f;  // smaller V scales count as 0

// Four int8 codes as two fp16 pairs: byte u + 128 under exponent 2^10 reads 1152 + u.
__device__ __forceinline__ uint32_t sub_1152(uint32_t h) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(h), "r"(0x64806480u));
  return r;
}
template <int FMT>
__device__ __forceinline__ void widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (FMT == SS_CODE_INT8) {
    w ^= 0x80808080u;
    lo = sub_1152(__byte_perm(w, 0x64646464u, 0x4140));
    hi = sub_1152(__byte_perm(w, 0x64646464u, 0x4342));
  } else {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  }
}
// Four codes of a word as fp32 (tf32 holds them exactly).  2^23 + u is the integer u's fp32
// pattern under exponent 2^23.
template <int FMT>
__device__ __forceinline__ void widen_f32(uint32_t w, uint32_t (&f)[4]) {
  if constexpr (FMT == SS_CODE_INT8) {
    w ^= 0x80808080u;
    const uint64_t off = f2pack(-8388736.f, -8388736.f);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint64_t v = add2(f2pack(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + 2 * i)),
                                     __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7441 + 2 * i))),
                              off);
      f[2 * i] = static_cast<uint32_t>(v);
      f[2 * i + 1] = static_cast<uint32_t>(v >> 32);
    }
  } else {
    uint32_t h[2];
    widen<FMT>(w, h[0], h[1]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
      f[2 * i] = __float_as_uint(v.x);
      f[2 * i + 1] = __float_as_uint(v.y);
    }
  }
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace ss
