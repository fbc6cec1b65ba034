// Base-2 exponential of pairs on the FMA pipe, for softmax loops that the MUFU unit would bound.
#pragma once

#include "ptx.cuh"

namespace ss {

// 2^x for a pair of fp32 values on the FMA pipe, offloading the MUFU unit (which computes
// 16 exponentials per clock per SM, as many as the tensor core needs here at full rate).
// Method: Cody-Waite range reduction 2^x = 2^n * 2^f with n = rint(x) (the 1.5 * 2^23
// addition trick, round-to-nearest), f in [-1/2, 1/2], and a cubic for 2^f whose
// coefficients are a minimax fit for relative error made for this kernel by iteratively
// reweighted least squares (Lawson's algorithm) on 4001 Chebyshev nodes: fit error
// 7.5e-5, measured 1.3e-4 in fp32 evaluation (bf16 P keeps 2^-9 = 2.0e-3).  Inputs are
// clamped to >= -126 so 2^n stays a normal power of two; the result for x < -126 is
// below 1.2e-38 instead of 0, which no sum of P notices.  2^n is applied by adding
// n << 23 to the exponent field: the low 9 bits of rint's float pattern hold n mod 512.
__device__ __forceinline__ uint64_t exp2_poly2(uint64_t x2) {
  float x0, x1;
  f2unpack(x2, x0, x1);
  x2 = f2pack(fmaxf(x0, -126.f), fmaxf(x1, -126.f));
  const uint64_t magic = f2pack(12582912.f, 12582912.f), nmagic = f2pack(-12582912.f, -12582912.f);
  const uint64_t j2 = add2(x2, magic);
  const uint64_t r2 = add2(j2, nmagic);                       // rint(x), exact
  const uint64_t f2 = fma2(r2, f2pack(-1.f, -1.f), x2);       // x - rint(x), exact
  uint64_t p2 = fma2(f2pack(0x1.c3f76p-5f, 0x1.c3f76p-5f), f2, f2pack(0x1.f0de1cp-3f, 0x1.f0de1cp-3f));
  p2 = fma2(p2, f2, f2pack(0x1.62f31ap-1f, 0x1.62f31ap-1f));
  p2 = fma2(p2, f2, f2pack(0x1.fff692p-1f, 0x1.fff692p-1f));
  float p0, p1, j0, j1;
  f2unpack(p2, p0, p1);
  f2unpack(j2, j0, j1);
  return f2pack(__int_as_float(__float_as_int(p0) + (__float_as_int(j0) << 23)),
                __int_as_float(__float_as_int(p1) + (__float_as_int(j1) << 23)));
}

}  // namespace ss
