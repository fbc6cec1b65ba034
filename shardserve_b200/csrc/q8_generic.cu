// Ragged paged attention over the 8-bit pool, one warp per (query token, head): the plainest
// correct form.  It serves the layouts that the split-K kernel cannot address (codes whose rows
// are not 16-byte addressable, more than 16 query heads per KV head) and is not tuned: codes are
// read byte by byte and every query head reads its KV head's codes itself.
//
//   x_i = (q . K_i) * (K scale * sm_scale * log2(e)),   m, l, acc: base-2 online softmax in fp32,
//   acc += 2^(x_i - m) * V scale * V_i
#include <cuda_bf16.h>
#include <math_constants.h>

#include "ptx.cuh"
#include "q8.cuh"

namespace ss {

namespace {

constexpr int kWarpsPerBlock = 4;

template <int D, int FMT>
__global__ void __launch_bounds__(32 * kWarpsPerBlock) q8_generic_kernel(const Q8AttnArgs g) {
  griddep_wait();
  const AttnArgs& a = g.a;
  const long long w = static_cast<long long>(blockIdx.x) * kWarpsPerBlock + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (w >= a.T * a.H) return;
  const long long t = w / a.H;
  const int h = static_cast<int>(w % a.H), kvh = h / a.group;
  const TokInfo ti = q8_token_info(a, t, h == 0 && lane == 0);
  constexpr int PER = D / 32;
  float qv[PER], acc[PER];
  const __nv_bfloat16* qp = a.q + t * a.q_st + h * a.q_sh;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    qv[i] = __bfloat162float(qp[(lane + 32 * i) * a.q_sd]);
    acc[i] = 0.f;
  }
  // The row's power of two is taken out of q: products with codes neither overflow nor lose bits where
  // the scores themselves do not.
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) top = fmaxf(top, fabsf(qv[i]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -126), 126);
#pragma unroll
  for (int i = 0; i < PER; ++i) qv[i] *= __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
  const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23) * a.scale_log2;
  float m = -CUDART_INF_F, l = 0.f;
  for (int pg = 0; pg < ti.npages; ++pg) {
    const long long pid = ld_index(a.bt, a.bt64, ti.seq * a.bt_sb + pg * a.bt_sn);
    const bool valid = pid >= 0 && pid < g.p.N;
    if (!valid && lane == 0) atomicOr(a.err, SS_DEVERR_PAGE);
    const float* sp = g.p.scales + pid * g.p.s_sn + kvh * g.p.s_sh;
    const float ks = valid ? sp[0] : 0.f, vs = valid ? sp[g.p.s_sw] : 0.f;
    const float f = ks * up;
    const int nk = min(kPage, ti.L - pg * kPage);
    for (int s = 0; s < nk; ++s) {
      float part = 0.f, vv[PER];
      const uint8_t* kr = g.p.k + pid * g.p.k_sn + s * g.p.k_ss + kvh * g.p.k_sh;
      const uint8_t* vr = g.p.v + pid * g.p.v_sn + s * g.p.v_ss + kvh * g.p.v_sh;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        vv[i] = 0.f;
        if (valid) {
          const long long d = lane + 32 * i;
          part += qv[i] * q8_decode(FMT, kr[d * g.p.k_sd]);
          vv[i] = q8_decode(FMT, vr[d * g.p.v_sd]);
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
      const float x = part * f;
      const float mn = fmaxf(m, x), ref = mn == -CUDART_INF_F ? 0.f : mn;
      const float alpha = ex2(m - ref), p = ex2(x - ref), pv = p * vs;
      l = l * alpha + p;
#pragma unroll
      for (int i = 0; i < PER; ++i) acc[i] = acc[i] * alpha + pv * vv[i];
      m = mn;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;  // no key: zeros
  __nv_bfloat16* op = a.out + t * a.o_st + h * a.o_sh;
#pragma unroll
  for (int i = 0; i < PER; ++i) op[(lane + 32 * i) * a.o_sd] = __float2bfloat16(acc[i] * inv);
}

}  // namespace

cudaError_t launch_q8_generic(const Q8AttnArgs& g, cudaStream_t stream) {
  const long long blocks = (g.a.T * g.a.H + kWarpsPerBlock - 1) / kWarpsPerBlock;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  const dim3 grid(static_cast<unsigned>(blocks)), block(32 * kWarpsPerBlock);
  if (g.p.D == 128) {
    if (g.p.fmt == SS_CODE_INT8) q8_generic_kernel<128, SS_CODE_INT8><<<grid, block, 0, stream>>>(g);
    else q8_generic_kernel<128, SS_CODE_E4M3><<<grid, block, 0, stream>>>(g);
  } else {
    if (g.p.fmt == SS_CODE_INT8) q8_generic_kernel<64, SS_CODE_INT8><<<grid, block, 0, stream>>>(g);
    else q8_generic_kernel<64, SS_CODE_E4M3><<<grid, block, 0, stream>>>(g);
  }
  return cudaGetLastError();
}

}  // namespace ss
