// Quantising slot-mapped append into the 8-bit paged pool, and the read-back.
//
// Append.  Token t's K / V row goes to row slot % 16 of page slot / 16.  Per page, KV head and
// tensor the codes share one scale, so a call computes, over the rows R it writes to a page,
//     s   = max |x| over R and head_dim / qmax     (finite values; 0 below 2^-100)
//     new = max(old, s)     old = the page's scale, or 0 where the call writes row 0 of the page
//     codes held by the page <- round(c * (old / new)),  new rows <- round(x * (1 / new))
// A call that writes row 0 starts the page anew: what a former request left there becomes zeros.
// The result does not depend on the order of the call's tokens (a maximum does not), except that
// of two tokens with the same slot the later one is kept.
//
// Every page must be handled once, by one warp per (head, tensor), wherever its tokens stand in
// the call.  CTA c owns the pages first met in its window of tokens: it puts the window's pages
// into a hash table in shared memory, then reads all T slots (from L2) to find the pages' rows
// and the pages that an earlier window owns.  T slots per CTA cost little while a window holds
// 1/148 of the call: 8192 tokens are 64 KB per SM, ~1 us.
//
// A warp handles a (page, head, tensor): one pass finds the largest |x|, and the rows, kept in
// registers, are encoded in the second; lane = eight consecutive values.
//
// Bound: HBM for prompts (3 bytes per value), latency for decode steps.  With the read-back that
// follows it, 16,000 prompt tokens of 8 KV heads of 128: 58.5 us for 196 MB (30 at the copy's rate).  Of the
// append's 27 us the page lists take 5 (1 the hash, 4 the pass over all slots) and the blocks 22, four to
// five one after another per warp, 4.4 TB/s.  64 decode rows: 9.4 us the two calls, two launches and four
// dependent trips to memory each.
#include <cuda_bf16.h>

#include <algorithm>

#include "ptx.cuh"
#include "q8.cuh"
#include "q8_widen.cuh"

namespace ss {

namespace {

constexpr int kMaxWindow = 512;          // tokens of one CTA
constexpr int kHash = 2 * kMaxWindow;    // hash slots at most (at most half full)

struct AppendSmem {
  int key[kHash];              // page of a hash slot, -1: empty
  int idx[kHash];              // its index in the lists below
  int page[kMaxWindow];
  int earlier[kMaxWindow];     // an earlier window owns the page
  int row[kMaxWindow][kPage];  // last token that writes each row, -1: none
  int n;
};

__device__ __forceinline__ unsigned hash_page(int page) {
  return (static_cast<unsigned>(page) * 2654435769u) >> 22;
}

// Eight consecutive values of a row, where the row is 16-byte addressable (vec) or anyhow.
__device__ __forceinline__ uint4 load_values(const __nv_bfloat16* p, long long sd, int vec) {
  if (vec) return __ldg(reinterpret_cast<const uint4*>(p));
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = static_cast<uint32_t>(__bfloat16_as_ushort(p[2 * i * sd])) |
           static_cast<uint32_t>(__bfloat16_as_ushort(p[(2 * i + 1) * sd])) << 16;
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint2 load_codes(const uint8_t* p, long long sd, int vec) {
  if (vec) return *reinterpret_cast<const uint2*>(p);
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i >> 2] |= static_cast<uint32_t>(p[i * sd]) << (8 * (i & 3));
  return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ void store_codes(uint8_t* p, long long sd, int vec, uint2 c) {
  if (vec) {
    *reinterpret_cast<uint2*>(p) = c;
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) p[i * sd] = static_cast<uint8_t>((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
}
// Four codes of four numbers.  FINITE: none of them lies past the largest code, so the integer can
// be read off the low byte of x + 1.5 * 2^23 (rounded to nearest even by that addition).
template <int FMT, bool FINITE>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  if constexpr (FMT == SS_CODE_INT8 && FINITE) {
    const uint32_t ua = __float_as_uint(__fadd_rn(a, 12582912.f)), ub = __float_as_uint(__fadd_rn(b, 12582912.f));
    const uint32_t uc = __float_as_uint(__fadd_rn(c, 12582912.f)), ud = __float_as_uint(__fadd_rn(d, 12582912.f));
    return __byte_perm(__byte_perm(ua, ub, 0x0040), __byte_perm(uc, ud, 0x0040), 0x5410);
  } else if constexpr (FMT == SS_CODE_E4M3) {
    const float2 lo = make_float2(a, b), hi = make_float2(c, d);
    return static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(lo, __NV_SATFINITE, __NV_E4M3)) |
           static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(hi, __NV_SATFINITE, __NV_E4M3)) << 16;
  } else {
    return q8_encode(FMT, a) | q8_encode(FMT, b) << 8 | q8_encode(FMT, c) << 16 |
           static_cast<uint32_t>(q8_encode(FMT, d)) << 24;
  }
}
template <int FMT, bool FINITE>
__device__ __forceinline__ uint2 encode_row(const uint4& v, float f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __fmul_rn(__uint_as_float(w[i] << 16), f);
    x[2 * i + 1] = __fmul_rn(__uint_as_float(w[i] & 0xffff0000u), f);
  }
  return make_uint2(encode4<FMT, FINITE>(x[0], x[1], x[2], x[3]), encode4<FMT, FINITE>(x[4], x[5], x[6], x[7]));
}
template <int FMT>
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float f) {
  float x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = __fmul_rn(q8_decode(FMT, static_cast<uint8_t>(w >> (8 * i))), f);
  return encode4<FMT, false>(x[0], x[1], x[2], x[3]);
}

// One page, head and tensor by one warp; `rows` = last token per row of the page.  D / 8 lanes hold
// a row's values, eight each; step s holds rows RP s .. RP s + RP - 1.
template <int D, int FMT>
__device__ __forceinline__ void append_block(const int* rows, const __nv_bfloat16* x, long long x_st,
                                             long long x_sd, int xvec, uint8_t* codes,
                                             long long c_ss, long long c_sd, int cvec,
                                             float* scale, int lane) {
  constexpr int LR = D / 8, RP = 32 / LR, ST = kPage / RP;
  const int r0 = lane / LR, c8 = lane % LR * 8;
  uint4 v[ST];
  unsigned has = 0;  // steps whose row this lane's row group writes
  unsigned top = 0;  // largest magnitude bits, in both halves
  const bool fresh = rows[0] >= 0;
  const float was = *scale;
#pragma unroll
  for (int s = 0; s < ST; ++s) {
    const int t = rows[s * RP + r0];
    v[s] = make_uint4(0, 0, 0, 0);
    if (t >= 0) {
      has |= 1u << s;
      v[s] = load_values(x + t * x_st + c8 * x_sd, x_sd, xvec);
    }
  }
#pragma unroll
  for (int s = 0; s < ST; ++s) {
    top = __vmaxu2(top, __vmaxu2(v[s].x & 0x7fff7fffu, v[s].y & 0x7fff7fffu));
    top = __vmaxu2(top, __vmaxu2(v[s].z & 0x7fff7fffu, v[s].w & 0x7fff7fffu));
  }
  top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
  const bool finite = top < 0x7f80u;
  float amax = __uint_as_float(top << 16);
  if (!finite) {  // the scale comes from the finite values
    amax = 0.f;
#pragma unroll
    for (int s = 0; s < ST; ++s) {
      const uint32_t w[4] = {v[s].x, v[s].y, v[s].z, v[s].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a = fabsf(__uint_as_float(w[i] << 16)), b = fabsf(__uint_as_float(w[i] & 0xffff0000u));
        if (a < __int_as_float(0x7f800000)) amax = fmaxf(amax, a);  // false for inf and NaN
        if (b < __int_as_float(0x7f800000)) amax = fmaxf(amax, b);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  }
  const float old = fresh ? 0.f : was;
  float s = __fdiv_rn(amax, q8_max(FMT));
  if (s < kQ8Tiny) s = 0.f;
  const float now = fmaxf(old, s);
  // Where the scale is 0 every finite value is so small that its product with 2^-126 is code 0; an
  // infinity still takes the largest code (of value 0) instead of NaN, which 0 would make of it.
  const float recip = now > 0.f ? __fdiv_rn(1.f, now) : 0x1p-126f;
  uint8_t* const base = codes + r0 * c_ss + c8 * c_sd;
  if (fresh || now != old || now == 0.f) {  // the page's other rows follow the new scale
    const float ratio = now > 0.f ? __fdiv_rn(old, now) : 0.f;
#pragma unroll
    for (int st = 0; st < ST; ++st) {
      if (has >> st & 1) continue;
      uint8_t* p = base + st * RP * c_ss;
      uint2 c = make_uint2(0, 0);
      if (!fresh) {
        c = load_codes(p, c_sd, cvec);
        c = make_uint2(rescale4<FMT>(c.x, ratio), rescale4<FMT>(c.y, ratio));
      }
      store_codes(p, c_sd, cvec, c);
    }
    if (lane == 0) *scale = now;
  }
#pragma unroll
  for (int st = 0; st < ST; ++st) {
    if (!(has >> st & 1)) continue;
    store_codes(base + st * RP * c_ss, c_sd, cvec,
                finite ? encode_row<FMT, true>(v[st], recip) : encode_row<FMT, false>(v[st], recip));
  }
}

template <int D, int FMT>
__global__ void __launch_bounds__(1024, 1)
    q8_append_kernel(const Q8AppendArgs a, int window, int hash_shift, int kvec, int vvec, int kcvec, int vcvec) {
  griddep_wait();  // k / v, the slots and the pool may come from the preceding kernel
  extern __shared__ uint8_t smem_raw[];
  AppendSmem& sm = *reinterpret_cast<AppendSmem*>(smem_raw);
  const int tid = threadIdx.x, nt = blockDim.x;
  const long long w0 = static_cast<long long>(blockIdx.x) * window;
  const long long w1 = min(w0 + window, a.T);
  const unsigned mask = (kHash >> hash_shift) - 1;
  // This thread's first slot, for both passes below.
  const long long limit = a.p.N * kPage;
  auto slot_at = [&](long long t) { return ld_index(a.slots, a.slots64, t); };
  const long long mine = tid < a.T ? slot_at(tid) : -1;
  for (int i = tid; i <= static_cast<int>(mask); i += nt) sm.key[i] = -1;
  for (int i = tid; i < window; i += nt) sm.earlier[i] = 0;
  for (int i = tid; i < window * kPage; i += nt) (&sm.row[0][0])[i] = -1;
  if (tid == 0) sm.n = 0;
  __syncthreads();
  for (long long t = w0 + tid; t < w1; t += nt) {
    const long long slot = slot_at(t);
    if (slot < 0 || slot >= limit) {
      if (a.err && slot != -1) atomicOr(a.err, SS_DEVERR_SLOT);
      continue;
    }
    const int page = static_cast<int>(slot / kPage);
    for (unsigned h = hash_page(page) >> hash_shift;; h = (h + 1) & mask) {
      const int was = atomicCAS(&sm.key[h], -1, page);
      if (was == -1) {
        const int i = atomicAdd(&sm.n, 1);
        sm.idx[h] = i;
        sm.page[i] = page;
        break;
      }
      if (was == page) break;
    }
  }
  __syncthreads();
  const int n = sm.n;
  if (n == 0) return;
  auto take = [&](long long t, long long slot) {
    if (slot < 0 || slot >= limit) return;
    const int page = static_cast<int>(slot / kPage);
    for (unsigned h = hash_page(page) >> hash_shift;; h = (h + 1) & mask) {
      const int key = sm.key[h];
      if (key == -1) break;
      if (key == page) {
        const int i = sm.idx[h];
        if (t < w0)
          sm.earlier[i] = 1;
        else
          atomicMax(&sm.row[i][slot % kPage], static_cast<int>(t));
        break;
      }
    }
  };
  take(tid, mine);
  constexpr int U = 4;  // slots in flight
  for (long long t = tid + nt; t < a.T; t += U * nt) {
    long long s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) s[u] = t + u * nt < a.T ? slot_at(t + u * nt) : -1;
#pragma unroll
    for (int u = 0; u < U; ++u) take(t + u * nt, s[u]);
  }
  __syncthreads();
  const int warp = tid >> 5, lane = tid & 31, warps = nt >> 5;
  const int per_page = 2 * a.p.KVH;
  for (int item = warp; item < n * per_page; item += warps) {
    const int i = item / per_page, rest = item % per_page, h = rest >> 1;
    if (sm.earlier[i]) continue;
    const long long page = sm.page[i];
    float* scale = a.p.scales + page * a.p.s_sn + h * a.p.s_sh + (rest & 1) * a.p.s_sw;
    if ((rest & 1) == 0)
      append_block<D, FMT>(sm.row[i], a.k + h * a.k_sh, a.k_st, a.k_sd, kvec,
                           a.p.k + page * a.p.k_sn + h * a.p.k_sh, a.p.k_ss, a.p.k_sd, kcvec, scale,
                           lane);
    else
      append_block<D, FMT>(sm.row[i], a.v + h * a.v_sh, a.v_st, a.v_sd, vvec,
                           a.p.v + page * a.p.v_sn + h * a.p.v_sh, a.p.v_ss, a.p.v_sd, vcvec, scale,
                           lane);
  }
}

// Pieces of 8 values of a K row and of the V row (or one value where rows are not 8-byte addressable),
// two of a thread in flight.  A CTA takes `rows` whole rows, so that a piece's row is a 32-bit product
// away (magic = ceil(2^32 / pieces of a row), exact for the few thousand pieces of a CTA that holds more
// than one row).
template <int D, int FMT, bool VEC>
__global__ void __launch_bounds__(256) q8_read_kernel(const Q8ReadArgs a, int rows, unsigned magic) {
  griddep_wait();
  constexpr int E = VEC ? 8 : 1, U = 2;
  const int per_row = a.p.KVH * (D / E);
  const long long limit = a.p.N * kPage;
  const long long t0 = static_cast<long long>(blockIdx.x) * rows;
  const int pieces = static_cast<int>(min(static_cast<long long>(rows), a.T - t0)) * per_row;
  for (int i0 = threadIdx.x; i0 < pieces; i0 += U * 256) {
    long long t[U], slot[U];
    int e[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(i0 + u * 256, pieces - 1);
      const int r = rows == 1 ? 0 : static_cast<int>(__umulhi(static_cast<unsigned>(i), magic));
      t[u] = t0 + r;
      e[u] = (i - r * per_row) * E;
      slot[u] = ld_index(a.slots, a.slots64, t[u]);
    }
    float sk[U], sv[U];
    uint2 kc[U], vc[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool ok = slot[u] >= 0 && slot[u] < limit;
      if (!ok && slot[u] != -1 && a.err && e[u] == 0) atomicOr(a.err, SS_DEVERR_SLOT);
      const long long page = ok ? slot[u] / kPage : 0;
      const int row = ok ? static_cast<int>(slot[u] % kPage) : 0, h = e[u] / D, d = e[u] % D;
      const float* sp = a.p.scales + page * a.p.s_sn + h * a.p.s_sh;
      const uint8_t* ks = a.p.k + page * a.p.k_sn + row * a.p.k_ss + h * a.p.k_sh + d * a.p.k_sd;
      const uint8_t* vs = a.p.v + page * a.p.v_sn + row * a.p.v_ss + h * a.p.v_sh + d * a.p.v_sd;
      sk[u] = sv[u] = 0.f;
      kc[u] = vc[u] = make_uint2(0, 0);
      if (ok) {
        sk[u] = sp[0];
        sv[u] = sp[a.p.s_sw];
        if constexpr (VEC) {
          kc[u] = *reinterpret_cast<const uint2*>(ks);
          vc[u] = *reinterpret_cast<const uint2*>(vs);
        } else {
          kc[u].x = *ks;
          vc[u].x = *vs;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u * 256 >= pieces) break;
      const int h = e[u] / D, d = e[u] % D;
      __nv_bfloat16* kd = a.k + t[u] * a.k_st + h * a.k_sh + d * a.k_sd;
      __nv_bfloat16* vd = a.v + t[u] * a.v_st + h * a.v_sh + d * a.v_sd;
      if constexpr (VEC) {
        auto four = [](uint32_t w, float s, uint32_t& lo, uint32_t& hi) {
          uint32_t f[4];
          widen_f32<FMT>(w, f);
          lo = pack_bf16(__uint_as_float(f[0]) * s, __uint_as_float(f[1]) * s);
          hi = pack_bf16(__uint_as_float(f[2]) * s, __uint_as_float(f[3]) * s);
        };
        uint4 o;
        four(kc[u].x, sk[u], o.x, o.y);
        four(kc[u].y, sk[u], o.z, o.w);
        *reinterpret_cast<uint4*>(kd) = o;
        four(vc[u].x, sv[u], o.x, o.y);
        four(vc[u].y, sv[u], o.z, o.w);
        *reinterpret_cast<uint4*>(vd) = o;
      } else {
        *kd = __float2bfloat16(q8_decode(FMT, static_cast<uint8_t>(kc[u].x)) * sk[u]);
        *vd = __float2bfloat16(q8_decode(FMT, static_cast<uint8_t>(vc[u].x)) * sv[u]);
      }
    }
  }
}

// Rows of `align` bytes: unit head_dim stride, base and the other strides multiples of it.
bool rows_ok(const void* p, long long esize, long long align, long long s0, long long s1,
             long long s2, long long sd) {
  return sd == 1 && reinterpret_cast<uintptr_t>(p) % align == 0 && s0 * esize % align == 0 &&
         s1 * esize % align == 0 && s2 * esize % align == 0;
}

void one_after_another(cudaLaunchConfig_t& cfg, cudaLaunchAttribute* attr) {
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
}

}  // namespace

cudaError_t launch_q8_append(const Q8AppendArgs& a, cudaStream_t stream) {
  // One window per SM, so that T slots are read once per SM; small calls get one page each.
  const long long window = std::min<long long>(std::max<long long>((a.T + 147) / 148, 1), kMaxWindow);
  long long warps = 4;
  while (warps < 32 && warps < window * 2 * a.p.KVH) warps *= 2;
  const int D = a.p.D;
  const int kvec = rows_ok(a.k, 2, 16, a.k_st, a.k_sh, 0, a.k_sd);
  const int vvec = rows_ok(a.v, 2, 16, a.v_st, a.v_sh, 0, a.v_sd);
  const int kcvec = rows_ok(a.p.k, 1, 8, a.p.k_sn, a.p.k_ss, a.p.k_sh, a.p.k_sd);
  const int vcvec = rows_ok(a.p.v, 1, 8, a.p.v_sn, a.p.v_ss, a.p.v_sh, a.p.v_sd);
  int shift = 0;  // a hash of four slots per token of the window, at least 32
  while ((kHash >> (shift + 1)) >= std::max<long long>(4 * window, 32)) ++shift;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((a.T + window - 1) / window));
  cfg.blockDim = dim3(static_cast<unsigned>(32 * warps));
  cfg.dynamicSmemBytes = sizeof(AppendSmem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  one_after_another(cfg, attr);
  const int w = static_cast<int>(window);
  if (D == 128)
    return a.p.fmt == SS_CODE_INT8
               ? cudaLaunchKernelEx(&cfg, q8_append_kernel<128, SS_CODE_INT8>, a, w, shift, kvec, vvec, kcvec, vcvec)
               : cudaLaunchKernelEx(&cfg, q8_append_kernel<128, SS_CODE_E4M3>, a, w, shift, kvec, vvec, kcvec, vcvec);
  return a.p.fmt == SS_CODE_INT8
             ? cudaLaunchKernelEx(&cfg, q8_append_kernel<64, SS_CODE_INT8>, a, w, shift, kvec, vvec, kcvec, vcvec)
             : cudaLaunchKernelEx(&cfg, q8_append_kernel<64, SS_CODE_E4M3>, a, w, shift, kvec, vvec, kcvec, vcvec);
}

cudaError_t launch_q8_read(const Q8ReadArgs& a, cudaStream_t stream) {
  const bool vec = rows_ok(a.k, 2, 16, a.k_st, a.k_sh, 0, a.k_sd) &&
                   rows_ok(a.v, 2, 16, a.v_st, a.v_sh, 0, a.v_sd) &&
                   rows_ok(a.p.k, 1, 8, a.p.k_sn, a.p.k_ss, a.p.k_sh, a.p.k_sd) &&
                   rows_ok(a.p.v, 1, 8, a.p.v_sn, a.p.v_ss, a.p.v_sh, a.p.v_sd);
  // Two pieces per thread once the CTAs fill the SMs with one.
  const long long per_row = static_cast<long long>(a.p.KVH) * a.p.D / (vec ? 8 : 1);
  const long long pieces = a.T * per_row > 148ll * 8 * 256 ? 512 : 256;
  const int rows = static_cast<int>(std::max<long long>(pieces / per_row, 1));
  const unsigned magic = static_cast<unsigned>(((1ull << 32) + per_row - 1) / per_row);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((a.T + rows - 1) / rows));
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  one_after_another(cfg, attr);
#define SS_Q8_READ(D, FMT)                                                                         \
  return vec ? cudaLaunchKernelEx(&cfg, q8_read_kernel<D, FMT, true>, a, rows, magic)              \
             : cudaLaunchKernelEx(&cfg, q8_read_kernel<D, FMT, false>, a, rows, magic)
  if (a.p.D == 128) {
    if (a.p.fmt == SS_CODE_INT8) SS_Q8_READ(128, SS_CODE_INT8);
    SS_Q8_READ(128, SS_CODE_E4M3);
  }
  if (a.p.fmt == SS_CODE_INT8) SS_Q8_READ(64, SS_CODE_INT8);
  SS_Q8_READ(64, SS_CODE_E4M3);
#undef SS_Q8_READ
}

}  // namespace ss
