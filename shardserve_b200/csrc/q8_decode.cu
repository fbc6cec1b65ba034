// Split-K ragged paged attention over the 8-bit pool for decode-style query tokens.
//
// Mathematics, per query token and KV head (G query heads share the head's codes):
//   x_ih = (q_h . Kc_i) * ks_page * sm_scale * log2 e + log2(vs_page),   w_ih = 2^(x_ih - r_h)
//   O_h  = sum_i w_ih Vc_i,   l_h = sum_i w_ih / vs_page,   out_h = O_h / l_h
// with Kc / Vc the codes and ks / vs their page's scales: the V scale rides in the exponent, so
// the products see the codes themselves and no page's scale costs another page precision.  r_h is
// raised only when a weight would pass 2^20, found by a vote: most pages need no warp reduction.
//
// Q.K.  The row's power of two is taken out of q.  Integer codes of up to 8 query heads per KV head:
// q is rounded to 21 bits below it and written as three signed digits of base 256, and the product
// of each digit with the codes is an integer MMA on the bytes as they stand (exact; widening them
// costs two ALU instructions per pair of codes more than the third digit's products).  Two of the
// digits share one MMA: rows 0-7 and 8-15 of its A operand.  Else (e4m3 codes, more heads, whose rows
// fill A): an fp16 product, which holds the codes exactly, and q but for the last bits of elements 2^17
// and more below their row's largest (2^-25 of it).
// P.V.  tf32: the weights keep 11 bits as in fp16, but over fp32's range (fp16 would flush weights
// 2^30 below the row's largest, which are all there is of an output dimension whose leading keys hold
// code 0; bf16 has the range and three bits less).  The codes are exact.  Everything else is fp32.
//
// What bounds it: HBM (2 * head_dim bytes per key and KV head) for what a call adds in length, 5.4 TB/s
// (6.8 where the codes stand in L2: 680 cycles a page and scheduler), and a fixed 18 us.  64 rows of
// context U[128, 4096], 16 query and 2 KV heads of 128, int8: 71 MB, 28.7 us a call, of which copying
// takes 10.9; 32 rows of 16 k to 32 k keys, 8 query heads and 1 KV head: 196 MB, 55 us (29.9).  The
// fixed part, from the last CTA of the call before: the start until its successor has its shares, up to 4 us
// until its first pages are in, 2 in each of the two joins, the rest the spread of the CTAs' ends.
// (Ids and positions read before the wait for the kernel before took 3 us off the start, and are not sound
// where that kernel writes them.  Those arrays or the first pages fetched into L2 before the wait moved a call
// by -1 to +1 us, case by case; whole 128-byte lines of K per copy, exchanged between lanes, by less than 1 %;
// codes widened with fp32 additions of fp16 operands instead of byte permutations, by nothing.)
//
// Data path.  A warp streams its own pages: every lane copies (cp.async) the 16-byte pieces that it
// will use itself into slots of its own, three pages ahead, and loads them back in fragment order;
// no other lane reads them, so nothing synchronises but the lane's own copy groups.  (With the next
// page in registers instead, issued piece by piece as registers came free, about 32 KiB per SM were
// in flight and a page took a warp 4,400 cycles: 31 us for the 64 rows.)  The order of head_dim and
// of the keys inside a product is free as long as both operands agree.  Lane (g, t) = (lane / 4,
// lane % 4):
//   S = Q K^T       M = query heads (of one KV head), N = 8 keys.  The lane loads bytes
//                   [64 c + 16 t, +16) of keys g and g + 8 (16-byte loads); Q is loaded to match.
//   O^T = V^T P^T   m16n8k8, M = 16 values of head_dim, N = 8 heads, K = 8 keys.  The lane loads
//                   bytes [D/8 g, +D/8) of keys 2t, 2t+1, 2t+8, 2t+9, which are the keys whose
//                   weights for head g it already holds: S's accumulators are P^T's operand.
// A lane's V bytes are consecutive, so its outputs are 32 consecutive bytes of an output row.
//
// Work split.  Unit = (row, page), row = (token, KV head).  One CTA per SM takes an equal run of
// units and every warp a run of the CTA's, cut at the rows' ends where that costs no warp more than
// two units.  A row inside a warp's run goes straight to the output.  Rows cut by warp boundaries leave
// fp32 partial states in shared memory, combined by the CTA; rows cut by CTA boundaries leave one
// state per CTA in the workspace, and the CTA that arrives last at the row's counter combines them in
// CTA order (no CTA waits for another one, and the bits do not depend on who arrives last).
#include <cuda_bf16.h>
#include <math_constants.h>

#include <algorithm>
#include <mutex>

#include "ptx.cuh"
#include "q8.cuh"
#include "q8_widen.cuh"

namespace ss {

namespace {

constexpr int kMaxTok = 6144;     // query tokens per launch (row lists in shared memory)
constexpr int kMaxCtas = 1024;    // counters in the workspace
constexpr int kCounterBytes = 4 * kMaxCtas;
constexpr float kSlack = 20.f;    // weights stay below 2^20 (of the reference they started with)

template <int D, int NG>
struct DecTraits {
  static constexpr int kWarps = NG == 1 ? 16 : 8;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int KT = 128 / D;         // 16-key tiles (pages) per step
  static constexpr int C = D / 64;           // 64-byte chunks of a K row
  static constexpr int MT = D / 16;          // 16-value tiles of the output
  static constexpr int VW = D / 32;          // 32-bit words a lane holds of a V row
  static constexpr int kRows = 8 * NG;       // query heads of a row (padded)
  static constexpr int kState = kRows * D + 2 * kRows;  // floats of a partial state: O, r, l
  static constexpr int kStages = 48 / kWarps;            // steps in flight per warp, 4 KiB each
  static constexpr int kRing = kStages * 4096;           // bytes of a warp's slots
  static_assert(kState * 4 <= kRing, "a warp's state fits its idle slots");
};

struct Piece {  // a warp's part of a row that others share
  int row;      // -1: none
  int first;    // the row's first page is inside
  int last;     // the row's last page is inside
  int mid;      // its state stands in the workspace (the warp went on to another row), not in its slots
};

// a / b for 0 <= a, 0 < b: an fp32 quotient, put right by its remainder.
__device__ __forceinline__ int quotient(int a, int b) {
  int q = __float2int_rz(__fdividef(static_cast<float>(a), static_cast<float>(b)));
  int r = static_cast<int>(static_cast<unsigned>(a) - static_cast<unsigned>(q) * static_cast<unsigned>(b));
  while (r < 0) { --q; r += b; }
  while (r >= b) { ++q; r -= b; }
  return q;
}
__device__ __forceinline__ uint32_t to_tf32(float x) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Integer product of 8-bit digits and codes, 32 deep.
__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                       uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Copies into the lane's own slots, and back.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int N>
__device__ __forceinline__ void copy_some(uint32_t dst, const void* src, int bytes) {  // the rest: zeros
  if constexpr (N == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(bytes) : "memory");
}
template <int VW>
__device__ __forceinline__ void copy_v(uint32_t dst, const void* src) {
  if constexpr (VW == 4)
    copy16(dst, src);
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ uint4 load_slot16(uint32_t src) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(src) : "memory");
  return v;
}
template <int VW>
__device__ __forceinline__ void load_v(uint32_t src, uint32_t (&w)[VW]) {
  if constexpr (VW == 4) {
    const uint4 v = load_slot16(src);
    w[0] = v.x; w[1] = v.y; w[VW - 2] = v.z; w[VW - 1] = v.w;
  } else {
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(src) : "memory");
  }
}

struct DecParams {
  Q8AttnArgs g;
  int t0, tn;          // tokens of this launch
  int skip_runs;       // tokens of runs belong to the tile kernel
  int split;           // the tile kernel comes next and takes the SMs that q8_split leaves it
  int min_chunk;       // fewest units of a CTA
  int sms;
  unsigned* counter;   // [kMaxCtas], zero between calls
  float* part;         // [2 * grid] partial states
  float* mid;          // [grid][warps] states of rows that a warp ends before its run does
};

// Folds `n` states, state i at `at(i)`, into one, U at a time; a thread of the group handles float4
// e.  CG: the states were written by other CTAs during this launch (read past L1).
template <int D, int NG, int U, bool CG, typename At>
__device__ __forceinline__ void fold(At at, int n, int e, float4& o, float& r, float& l) {
  using Tr = DecTraits<D, NG>;
  const int head = e / (D / 4);
  o = make_float4(0.f, 0.f, 0.f, 0.f);
  r = -CUDART_INF_F;
  l = 0.f;
  for (int i0 = 0; i0 < n; i0 += U) {
    float rv[U], lv[U];
    float4 ov[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      rv[u] = -CUDART_INF_F;
      lv[u] = 0.f;
      ov[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i0 + u < n) {
        const float* s = at(i0 + u);
        if (CG) {
          rv[u] = __ldcg(s + Tr::kRows * D + head);
          lv[u] = __ldcg(s + Tr::kRows * D + Tr::kRows + head);
          ov[u] = __ldcg(reinterpret_cast<const float4*>(s) + e);
        } else {
          rv[u] = s[Tr::kRows * D + head];
          lv[u] = s[Tr::kRows * D + Tr::kRows + head];
          ov[u] = reinterpret_cast<const float4*>(s)[e];
        }
      }
    }
    float rn = r;
#pragma unroll
    for (int u = 0; u < U; ++u) rn = fmaxf(rn, rv[u]);
    const float ref = rn == -CUDART_INF_F ? 0.f : rn;
    const float f = ex2(r - ref);
    o.x *= f; o.y *= f; o.z *= f; o.w *= f;
    l *= f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float w = ex2(rv[u] - ref);
      o.x += ov[u].x * w; o.y += ov[u].y * w; o.z += ov[u].z * w; o.w += ov[u].w * w;
      l += lv[u] * w;
    }
    r = rn;
  }
}

template <int D, int NG>
struct DecSmem {
  using Tr = DecTraits<D, NG>;
  // Slots of the warps; before the stream, the staged ids and lengths; after it, states.
  alignas(16) uint8_t ring[Tr::kWarps][Tr::kRing];
  float2 scale[Tr::kWarps][Tr::kStages][Tr::KT];
  Piece piece[Tr::kWarps][2];
  int pre[kMaxTok + 1];  // units before each token
  int scan[Tr::kWarps], keys[2][Tr::kWarps];
  int arrived[2];
};
static_assert((2 * kMaxTok + 2 * kQ8Pad) * 4 <= 48 * 4096, "the staged tokens fit the slots");

template <int D, int FMT, int NG, bool PK>
__global__ void __launch_bounds__(DecTraits<D, NG>::kThreads, 1)
    q8_decode_kernel(const __grid_constant__ DecParams P) {
  using Tr = DecTraits<D, NG>;
  constexpr int NW = Tr::kWarps, NT = Tr::kThreads, KT = Tr::KT, C = Tr::C, MT = Tr::MT, VW = Tr::VW;
  constexpr bool kDigits = FMT == SS_CODE_INT8 && NG == 1;  // Q.K as integer products
  extern __shared__ __align__(16) uint8_t smem_raw[];
  DecSmem<D, NG>& sm = *reinterpret_cast<DecSmem<D, NG>*>(smem_raw);
  const AttnArgs& a = P.g.a;
  const Q8Pool& pool = P.g.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // Nothing is read before the kernel before has ended: its index arrays, like its pool rows, may come
  // from that kernel, and what it wrote is seen only after the wait.  The next kernel is let go at once: the
  // tile kernel, which reads nothing that this one writes, starts on the SMs that this one leaves.
  griddep_wait();
  griddep_launch_dependents();

  // ---- units before every token ----------------------------------------------------------
  int* const seq = reinterpret_cast<int*>(sm.ring) + kQ8Pad;
  int* const len = seq + kMaxTok + kQ8Pad;
  stage_tokens(a, P.t0, P.tn, seq, len, blockIdx.x == 0);
  __syncthreads();
  const int per = (P.tn + NT - 1) / NT;
  const int b0 = min(tid * per, P.tn), b1 = min(b0 + per, P.tn);
  int sum = 0, rows_keys = 0, run_keys = 0;
  for (int i = b0; i < b1; ++i) {
    sm.pre[i] = sum;  // within this thread's run
    if (P.skip_runs && in_staged_run(seq, i)) {
      run_keys += q8_clamped(len[i]);
      len[i] = -1;
    } else {
      rows_keys += q8_clamped(len[i]);
      sum += (len[i] + kPage - 1) / kPage * a.KVH;
    }
  }
  int inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += x;
  }
  if (P.split) {
    rows_keys = __reduce_add_sync(0xffffffffu, rows_keys);
    run_keys = __reduce_add_sync(0xffffffffu, run_keys);
    if (lane == 0) {
      sm.keys[0][warp] = rows_keys;
      sm.keys[1][warp] = run_keys;
    }
  }
  if (lane == 31) sm.scan[warp] = inc;
  if (tid < 2 * NW) sm.piece[tid >> 1][tid & 1].row = -1;  // (ordered by the barriers below)
  __syncthreads();
  const int part_sum = sm.scan[lane % NW];
  const int before = inc - sum + __reduce_add_sync(0xffffffffu, lane < warp ? part_sum : 0);
  const int U = __reduce_add_sync(0xffffffffu, lane < NW ? part_sum : 0);
  int G = gridDim.x;
  if (P.split) {
    rows_keys = run_keys = 0;
    for (int w = 0; w < NW; ++w) {
      rows_keys += sm.keys[0][w];
      run_keys += sm.keys[1][w];
    }
    G = max(q8_split(rows_keys, run_keys, P.sms), 1);
  }
  for (int i = b0; i < b1; ++i) sm.pre[i] += before;
  if (tid == 0) sm.pre[P.tn] = U;
  __syncthreads();
  // Tokens of this launch without keys: zero rows, spread over the CTAs.
  for (int i = blockIdx.x; i < P.tn; i += gridDim.x) {
    if (len[i] != 0) continue;
    for (int e = tid; e < a.H * D; e += NT)
      a.out[(P.t0 + i) * a.o_st + static_cast<long long>(e / D) * a.o_sh + e % D] = __float2bfloat16(0.f);
  }
  const int chunk = max(U == 0 ? 0 : quotient(U - 1, G) + 1, P.min_chunk);
  const long long c0 = static_cast<long long>(blockIdx.x) * chunk;
  if (c0 >= U) return;
  const int n_cta = static_cast<int>(min(static_cast<long long>(chunk), U - c0));
  // Shares of the warps, in unit order.  A row's end inside a warp's share costs it more than two units
  // (its copies run dry and its queries change: 4 us), and the CTA waits for its slowest warp; so rows
  // get warps of their own, as long as no warp then holds more than two units above an even share (64
  // rows 27.5 -> 25.9 us, 250 rows of head_dim 64 40.0 -> 37.6).
  auto token_of = [&](int unit, int lo) {  // the last token that begins at or before the unit
    for (int hi = P.tn; hi - lo > 1;) {
      const int step = (hi - lo + 31) / 32, i = lo + (lane + 1) * step;
      const int n = __popc(__ballot_sync(0xffffffffu, i < hi && sm.pre[min(i, P.tn)] <= unit));
      lo += n * step;
      hi = min(hi, lo + step);
    }
    return lo;
  };
  int u, u1, tok;  // this warp's units, and the token of the first
  {
    const int even = (n_cta + NW - 1) / NW, first_tok = token_of(static_cast<int>(c0), 0);
    // Lane i: units that the CTA holds of the i-th row from the token's first one on.
    const int ahead = quotient(lane, a.KVH), tk = min(first_tok + ahead, P.tn - 1);
    const int np = (len[tk] + kPage - 1) / kPage, r0 = sm.pre[tk] + (lane - ahead * a.KVH) * np;
    const int e0 = max(r0, static_cast<int>(c0)), e1 = min(r0 + np, static_cast<int>(c0) + n_cta);
    const int mine = first_tok + ahead < P.tn ? max(e1 - e0, 0) : 0;
    int size = 0, parts = 0;  // most units of a warp, the row's warps
    // (With one unit per warp, or more rows than lanes, the shares are even.)
    if (even > 1 && static_cast<int>(__reduce_add_sync(0xffffffffu, mine)) == n_cta)
      for (int s = even; s <= even + 2 && size == 0; ++s) {
        parts = mine == 0 ? 0 : quotient(mine - 1, s) + 1;
        if (static_cast<int>(__reduce_add_sync(0xffffffffu, parts)) <= NW) size = s;
      }
    if (size != 0) {
      int upto = parts;  // warps up to and with this row's
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
      }
      const unsigned after = __ballot_sync(0xffffffffu, upto > warp);
      const int row = after ? __ffs(after) - 1 : 31;
      const int n = __shfl_sync(0xffffffffu, mine, row), k = max(__shfl_sync(0xffffffffu, parts, row), 1);
      const int i = warp - (__shfl_sync(0xffffffffu, upto, row) - k), q = quotient(n, k), rest = n - q * k;
      u = __shfl_sync(0xffffffffu, e0, row) + i * q + min(i, rest);
      u1 = after ? u + q + (i < rest ? 1 : 0) : u;
      tok = first_tok + __shfl_sync(0xffffffffu, ahead, row);
    } else {  // even shares; warps 0 .. nwa - 1 hold at least one unit each
      const int nwa = min(NW, n_cta), wq = quotient(n_cta, nwa), wr = n_cta - wq * nwa;
      u = static_cast<int>(c0) + warp * wq + min(warp, wr);
      u1 = warp < nwa ? u + wq + (warp < wr ? 1 : 0) : u;
      tok = u < u1 ? token_of(u, first_tok) : 0;
    }
  }

  const int g = lane >> 2, t4 = lane & 3;
  int seq_now = 0, L = 0, tok_now = -1;  // of the token whose row is streamed
  if (u < u1) {
    tok_now = tok;
    seq_now = seq[tok];
    L = len[tok];
  }
  __syncthreads();  // the staged tokens have been read: the slots are free
  const uint32_t slot = smem_u32(sm.ring[warp]) + lane * 16;
  const uint32_t slot_sc = smem_u32(sm.scale[warp]);
  const long long k_ss = PK ? D : pool.k_ss, v_ss = PK ? D : pool.v_ss;

  while (u < u1) {
    while (sm.pre[tok + 1] <= u) ++tok;
    if (tok != tok_now) {
      const TokInfo ti = q8_token_info(a, P.t0 + tok, false);
      tok_now = tok;
      seq_now = static_cast<int>(ti.seq);
      L = ti.L;
    }
    const int np = (L + kPage - 1) / kPage;
    const int rem = u - sm.pre[tok];
    const int h = quotient(rem, np), p0 = rem - h * np;
    const int cnt = min(np - p0, u1 - u);  // pages of this segment
    const long long btrow = static_cast<long long>(seq_now) * a.bt_sb;
    const long long t = P.t0 + tok;

    // Page ids, 32 at a time (lane i: page p0 + base + i).
    auto load_ids = [&](int base) -> int {
      const int i = base + lane;
      int id = -1;
      if (i < cnt) {
        const long long pid = ld_index(a.bt, a.bt64, btrow + static_cast<long long>(p0 + i) * a.bt_sn);
        if (pid >= 0 && pid < pool.N)
          id = static_cast<int>(pid);
        else
          atomicOr(a.err, SS_DEVERR_PAGE);
      }
      return id;
    };
    int ids = load_ids(0), ids_next = load_ids(32);

    // Lane pointers into page 0; the strides are constants where the rows of a head's page are one
    // run of memory (PK), which makes every piece but a page's first an immediate offset.
    const uint8_t* kbase = pool.k + static_cast<long long>(h) * pool.k_sh + 16 * t4 + g * k_ss;
    const uint8_t* vbase = pool.v + static_cast<long long>(h) * pool.v_sh + (D / 8) * g + 2 * t4 * v_ss;
    const float* sbase = pool.scales + static_cast<long long>(h) * pool.s_sh;
    const int nfull = min(cnt, L / kPage - p0);  // pages of the segment that are attended whole
    auto keys_of = [&](int i) { return i < cnt ? min(kPage, L - (p0 + i) * kPage) : 0; };
    // Copies pages i .. i + KT - 1 into a stage.  K pieces stand at slots (k, r, c), V's after them.
    int fetched = 0;
    auto fetch = [&](int stage) {
      const int i = fetched;
      fetched += KT;
      if (i < cnt) {
        if (i > 0 && (i & 31) == 0) {
          ids = ids_next;
          ids_next = load_ids(i + 32);
        }
        const uint32_t dst = slot + stage * 4096;
#pragma unroll
        for (int k = 0; k < KT; ++k) {
          const int pg = i + k < cnt ? __shfl_sync(0xffffffffu, ids, (i + k) & 31) : -1;
          const uint8_t* ks = kbase + pg * pool.k_sn;
          const uint8_t* vs = vbase + pg * pool.v_sn;
          const uint32_t kd = dst + k * (2 * C * 512);
          const uint32_t vd = dst + 2048 + k * (C * 1024) - (VW == 2 ? lane * 8 : 0);
          const uint32_t sd = slot_sc + (stage * KT + k) * 8;
          if (i + k < nfull && pg >= 0) {
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
              for (int c = 0; c < C; ++c) copy16(kd + (r * C + c) * 512, ks + 8 * r * k_ss + 64 * c);
#pragma unroll
            for (int j = 0; j < 4; ++j) copy_v<VW>(vd + j * (VW * 128), vs + ((j & 1) + 8 * (j >> 1)) * v_ss);
            if (lane == 0) {
              const float* s = sbase + pg * pool.s_sn;
              if (PK) {
                copy_some<8>(sd, s, 8);
              } else {
                copy_some<4>(sd, s, 4);
                copy_some<4>(sd + 4, s + pool.s_sw, 4);
              }
            }
          } else {  // the row's last page, a page outside the pool, or past the segment
            const int n = pg < 0 ? 0 : keys_of(i + k);
            const uint8_t* none = pool.k;
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
              for (int c = 0; c < C; ++c) {
                const bool on = g + 8 * r < n;
                copy_some<16>(kd + (r * C + c) * 512, on ? ks + 8 * r * k_ss + 64 * c : none, on ? 16 : 0);
              }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int row = (j & 1) + 8 * (j >> 1);  // key 2 t + row
              const bool on = 2 * t4 + row < n;
              copy_some<4 * VW>(vd + j * (VW * 128), on ? vs + row * v_ss : none, on ? 4 * VW : 0);
            }
            if (lane == 0) {
              const float* s = sbase + pg * pool.s_sn;
              float2 sc = make_float2(0.f, 1.f);
              if (n > 0) sc = make_float2(__ldg(s), __ldg(s + pool.s_sw));
              asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(sd), "f"(sc.x), "f"(sc.y) : "memory");
            }
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // The queries are asked for before the first pages: behind them they would wait for 28 MB.
    // Lane (g, t) holds head g's values [64 c + 16 t, +16), the order of the K bytes.
    uint32_t raw[NG][C][8];
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const int hd = 8 * n + g;
          uint4 v = make_uint4(0, 0, 0, 0);
          if (hd < a.group)
            v = __ldg(reinterpret_cast<const uint4*>(
                a.q + t * a.q_st + static_cast<long long>(h * a.group + hd) * a.q_sh + 64 * c + 16 * t4 + 8 * w));
          raw[n][c][4 * w] = v.x; raw[n][c][4 * w + 1] = v.y; raw[n][c][4 * w + 2] = v.z; raw[n][c][4 * w + 3] = v.w;
        }
#pragma unroll
    for (int st = 0; st < Tr::kStages; ++st) fetch(st);

    // Queries as fp16 with the row's power of two taken out.
    uint32_t qf[NG][C][4][2];
    // The same as three signed digits of base 256: digits [64 c + 16 t + 8 p, +8), two words each.
    uint32_t qd[3][C][2][2];
    float qs[NG];  // of head 8 n + g: 2^e * sm_scale * log2 e (for digits 2^-21 of it)
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      unsigned top = 0;  // largest magnitude bits (NaN and infinity on top) of either half
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int w = 0; w < 8; ++w) top = __vmaxu2(top, raw[n][c][w] & 0x7fff7fffu);
      top = max(top & 0xffffu, top >> 16);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // Rows below 2^-63 are raised by 2^64 (exact, subnormals too), so that their power of two has a
      // normal reciprocal.
      const bool tiny = top < 64u << 7;
      if (tiny) {
        const __nv_bfloat162 grow = __float2bfloat162_rn(0x1p64f);
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int w = 0; w < 8; ++w) {
            const __nv_bfloat162 v = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&raw[n][c][w]), grow);
            raw[n][c][w] = *reinterpret_cast<const uint32_t*>(&v);
          }
        top = __float_as_uint(__uint_as_float(top << 16) * 0x1p64f) >> 16;
      }
      // bf16's largest exponent is 127, which the digits need as it is: with one less, 21 bits would not hold
      // the values.  As fp16 they may reach 4, and with 126 the reciprocal below stays normal.
      const int e = min(max(static_cast<int>(top >> 7) - 127, -104), kDigits ? 127 : 126);
      // 2^(e - 21), which is a normal number where 2^e times the factor may not be.
      float up = __uint_as_float(static_cast<uint32_t>(127 + e - 21) << 23) * a.scale_log2;
      if (tiny) up *= 0x1p-64f;
      if constexpr (kDigits) {
        // round(q 2^(21 - e)) + 0x808080 by an addition whose sum's low bits are that integer; its
        // bytes, each less 128, are the digits.
        const float grow = __uint_as_float(static_cast<uint32_t>(127 + 21 - e) << 23);
        auto whole = [&](uint32_t v) {
          return __float_as_uint(fmaf(__uint_as_float(v), grow, 12582912.f)) - 0x4b400000u + 0x808080u;
        };
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int w = 0; w < 4; ++w) {  // values 4 w .. 4 w + 3
            const uint32_t f0 = whole(raw[n][c][2 * w] << 16), f1 = whole(raw[n][c][2 * w] & 0xffff0000u);
            const uint32_t f2 = whole(raw[n][c][2 * w + 1] << 16), f3 = whole(raw[n][c][2 * w + 1] & 0xffff0000u);
            const uint32_t l01 = __byte_perm(f0, f1, 0x5140), l23 = __byte_perm(f2, f3, 0x5140);
            const uint32_t h01 = __byte_perm(f0, f1, 0x0062), h23 = __byte_perm(f2, f3, 0x0062);
            qd[0][c][w >> 1][w & 1] = __byte_perm(h01, h23, 0x5410) ^ 0x80808080u;
            qd[1][c][w >> 1][w & 1] = __byte_perm(l01, l23, 0x7632) ^ 0x80808080u;
            qd[2][c][w >> 1][w & 1] = __byte_perm(l01, l23, 0x5410) ^ 0x80808080u;
          }
        qs[n] = top >= 0x7f80u ? CUDART_NAN_F : up;
      } else {
        const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int w = 0; w < 8; ++w)
            qf[n][c][w >> 1][w & 1] = pack_f16(__uint_as_float(raw[n][c][w] << 16) * down,
                                               __uint_as_float(raw[n][c][w] & 0xffff0000u) * down);
        qs[n] = up * 0x1p21f;
      }
    }

    // Of head 8 n + g: the reference (0 before the first score), how far a score may pass it (-inf
    // before the first one), and the sum of weights.
    float acc[NG][MT][4], base[NG], limit[NG], lsum[NG];
#pragma unroll
    for (int n = 0; n < NG; ++n) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[n][i][j] = 0.f;
      base[n] = 0.f;
      limit[n] = -CUDART_INF_F;
      lsum[n] = 0.f;
    }

    int stage = 0;
    for (int i = 0; i < cnt; i += KT) {
      asm volatile("cp.async.wait_group %0;" ::"n"(Tr::kStages - 1) : "memory");
      __syncwarp();  // lane 0's copies of the scales
      const uint32_t src = slot + stage * 4096;
      // ---- scores: x[k][r][j + 2 n] of key 8 r + 2 t + j, head 8 n + g ----------------------
      float x[KT][2][4];
      float2 sc[KT];
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        sc[k] = sm.scale[warp][stage][k];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          if constexpr (kDigits) {
            int hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < C; ++c) {
              const uint4 kv = load_slot16(src + (k * 2 * C + r * C + c) * 512);
              mma_s8(hi, qd[0][c][0][0], qd[1][c][0][0], qd[0][c][0][1], qd[1][c][0][1], kv.x, kv.y);
              mma_s8(lo, qd[2][c][0][0], 0u, qd[2][c][0][1], 0u, kv.x, kv.y);
              mma_s8(hi, qd[0][c][1][0], qd[1][c][1][0], qd[0][c][1][1], qd[1][c][1][1], kv.z, kv.w);
              mma_s8(lo, qd[2][c][1][0], 0u, qd[2][c][1][1], 0u, kv.z, kv.w);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
              x[k][r][j] = fmaf(static_cast<float>(hi[j] * 256 + hi[j + 2]), 256.f, static_cast<float>(lo[j]));
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) x[k][r][j] = 0.f;
#pragma unroll
            for (int c = 0; c < C; ++c) {
              const uint4 kv = load_slot16(src + (k * 2 * C + r * C + c) * 512);
              const uint32_t kw[4] = {kv.x, kv.y, kv.z, kv.w};
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                uint32_t b0, b1;
                widen<FMT>(kw[w], b0, b1);
                mma_f16(x[k][r], qf[0][c][w][0], NG == 2 ? qf[NG - 1][c][w][0] : 0u, qf[0][c][w][1],
                        NG == 2 ? qf[NG - 1][c][w][1] : 0u, b0, b1);
              }
            }
          }
        }
      }
      // ---- weights: x becomes its distance from the row's reference -----------------------
      bool raise = false;
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        const float lv = lg2(fmaxf(sc[k].y, kMinVs));
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          const float f = sc[k].x * qs[n], b = lv - base[n];
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int j = 0; j < 2; ++j) x[k][r][2 * n + j] = fmaf(x[k][r][2 * n + j], f, b);
        }
        if (i + k >= nfull) {  // keys past the row
          const int n = keys_of(i + k);
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int j = 0; j < 2; ++j)
              if (8 * r + 2 * t4 + j >= n)
#pragma unroll
                for (int m = 0; m < NG; ++m) x[k][r][2 * m + j] = -CUDART_INF_F;
        }
#pragma unroll
        for (int n = 0; n < NG; ++n)
          raise |= fmaxf(max3(x[k][0][2 * n], x[k][0][2 * n + 1], x[k][1][2 * n]), x[k][1][2 * n + 1]) > limit[n];
      }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          // How far the reference moves: to the largest of these scores, never down.
          float m = limit[n] == -CUDART_INF_F ? -CUDART_INF_F : 0.f;
#pragma unroll
          for (int k = 0; k < KT; ++k)
#pragma unroll
            for (int r = 0; r < 2; ++r) m = max3(m, x[k][r][2 * n], x[k][r][2 * n + 1]);
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
          const bool some = m != -CUDART_INF_F;  // a score has been seen
          const float up = some ? m : 0.f;
          // Before the first score there is nothing to scale.
          const float f = limit[n] == -CUDART_INF_F ? 0.f : ex2(-up);
          base[n] += up;
          if (some) limit[n] = kSlack;
          lsum[n] *= f;
          const float f0 = __shfl_sync(0xffffffffu, f, 8 * t4), f1 = __shfl_sync(0xffffffffu, f, 8 * t4 + 4);
#pragma unroll
          for (int q = 0; q < MT; ++q) {
            acc[n][q][0] *= f0;
            acc[n][q][1] *= f1;
            acc[n][q][2] *= f0;
            acc[n][q][3] *= f1;
          }
#pragma unroll
          for (int k = 0; k < KT; ++k)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              x[k][r][2 * n] -= up;
              x[k][r][2 * n + 1] -= up;
            }
        }
      }
      uint32_t pb[KT][NG][2][2];
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        const float iv = __frcp_rn(fmaxf(sc[k].y, kMinVs));
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          float sum = 0.f;
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float w = ex2(x[k][r][2 * n + j]);
              sum += w;
              pb[k][n][r][j] = to_tf32(w);
            }
          lsum[n] = fmaf(sum, iv, lsum[n]);
        }
        if (!(sc[k].y >= kMinVs)) {  // a page whose V scale is 0 holds zeros
#pragma unroll
          for (int n = 0; n < NG; ++n) pb[k][n][0][0] = pb[k][n][0][1] = pb[k][n][1][0] = pb[k][n][1][1] = 0u;
        }
      }
      // ---- values ---------------------------------------------------------------------------
#pragma unroll
      for (int k = 0; k < KT; ++k)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          uint32_t w0[VW], w1[VW];  // keys 8 r + 2 t and the one after
          const uint32_t vsrc = src + 2048 + k * (C * 1024) - (VW == 2 ? lane * 8 : 0) + 2 * r * (VW * 128);
          load_v<VW>(vsrc, w0);
          load_v<VW>(vsrc + VW * 128, w1);
#pragma unroll
          for (int w = 0; w < VW; ++w) {
            uint32_t v0[4], v1[4];
            widen_f32<FMT>(w0[w], v0);
            widen_f32<FMT>(w1[w], v1);
#pragma unroll
            for (int n = 0; n < NG; ++n) {
              mma_tf32(acc[n][2 * w], v0[0], v0[1], v1[0], v1[1], pb[k][n][r][0], pb[k][n][r][1]);
              mma_tf32(acc[n][2 * w + 1], v0[2], v0[3], v1[2], v1[3], pb[k][n][r][0], pb[k][n][r][1]);
            }
          }
        }
      __syncwarp();  // the stage's scales have been read
      fetch(stage);
      stage = stage + 1 == Tr::kStages ? 0 : stage + 1;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    // ---- the segment's end ----------------------------------------------------------------
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      lsum[n] += __shfl_xor_sync(0xffffffffu, lsum[n], 1);
      lsum[n] += __shfl_xor_sync(0xffffffffu, lsum[n], 2);
    }
    const bool first = p0 == 0, last = p0 + cnt == np;
    if (first && last) {
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int hd = 8 * n + 2 * t4 + j;
          const float l = __shfl_sync(0xffffffffu, lsum[n], 8 * t4 + 4 * j);
          if (hd >= a.group) continue;
          const float inv = l == 0.f ? 0.f : 1.f / l;
          uint32_t o[MT];
#pragma unroll
          for (int q = 0; q < MT; ++q) o[q] = pack_bf16(acc[n][q][j] * inv, acc[n][q][j + 2] * inv);
          uint4* dst = reinterpret_cast<uint4*>(a.out + t * a.o_st + static_cast<long long>(h * a.group + hd) * a.o_sh + (D / 8) * g);
#pragma unroll
          for (int q = 0; q < MT / 4; ++q) dst[q] = make_uint4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
        }
    } else {
      const int which = first ? 1 : 0;
      const bool mid = u + cnt < u1;
      __syncwarp();
      float* st = mid ? P.mid + (static_cast<long long>(blockIdx.x) * NW + warp) * Tr::kState
                      : reinterpret_cast<float*>(sm.ring[warp]);
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int hd = 8 * n + 2 * t4 + j;
          float4* dst = reinterpret_cast<float4*>(st + hd * D + (D / 8) * g);
#pragma unroll
          for (int q = 0; q < MT / 2; ++q)
            dst[q] = make_float4(acc[n][2 * q][j], acc[n][2 * q][j + 2], acc[n][2 * q + 1][j], acc[n][2 * q + 1][j + 2]);
        }
      if (t4 == 0)
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          st[Tr::kRows * D + 8 * n + g] = limit[n] == -CUDART_INF_F ? -CUDART_INF_F : base[n];
          st[Tr::kRows * D + Tr::kRows + 8 * n + g] = lsum[n];
        }
      if (lane == 0) sm.piece[warp][which] = Piece{tok * a.KVH + h, first, last, mid};
    }
    u += cnt;
  }
  __syncthreads();

  // ---- rows cut by warp boundaries --------------------------------------------------------
  // Pieces stand in unit order: slot 0 (goes on from the warp before), then slot 1 (begins here).
  // Several groups of kRows * D / 4 threads each take a row at a time.
  constexpr int GT = Tr::kRows * D / 4;         // threads that hold a state as float4
  constexpr int NGR = NT >= GT ? NT / GT : 1;   // groups
  constexpr int ER = GT > NT ? GT / NT : 1;     // float4 per thread where a state is larger
  const int grp = tid / GT;
  auto write_row = [&](int row, int e, const float4& o, float l) {
    const int hd = e / (D / 4), d = (e % (D / 4)) * 4;
    if (hd >= a.group) return;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int tk = quotient(row, a.KVH);
    const long long t = P.t0 + tk;
    *reinterpret_cast<uint2*>(a.out + t * a.o_st + static_cast<long long>((row - tk * a.KVH) * a.group + hd) * a.o_sh + d) =
        make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
  };
  static_assert(2 * NW <= 32, "a warp's lanes hold the pieces");
  Piece mine{-1, 0, 0, 0};
  if (lane < 2 * NW) mine = sm.piece[lane >> 1][lane & 1];
  const unsigned valid = __ballot_sync(0xffffffffu, mine.row >= 0);
  const unsigned firsts = __ballot_sync(0xffffffffu, mine.row >= 0 && mine.first);
  const unsigned lasts = __ballot_sync(0xffffffffu, mine.row >= 0 && mine.last);
  int open_row[2] = {-1, -1};  // rows that other CTAs share (0: begun earlier, 1: begun here)
  int idx = 0;
  for (unsigned todo = firsts | (valid & (0u - valid)); todo; todo &= todo - 1, ++idx) {
    const int i = __ffs(todo) - 1;
    // Its pieces: this one and the slots 0 of the following warps, up to the row's last.
    const unsigned from = ~0u << i, fin = lasts & from;
    const unsigned span = valid & from & (fin ? (fin & (0u - fin)) * 2 - 1 : ~0u);
    const int n = __popc(span), row = __shfl_sync(0xffffffffu, mine.row, i);
    const bool begins = firsts >> i & 1, whole = begins && fin;
    if (!whole) open_row[begins ? 1 : 0] = row;
    if (idx % NGR != grp) continue;
    // Only a row's last piece can have been left behind by its warp.
    const int w0 = i >> 1, end = n == 1 ? i : 2 * (w0 + n - 1);
    const float* tail = sm.piece[end >> 1][end & 1].mid
                            ? P.mid + (static_cast<long long>(blockIdx.x) * NW + (end >> 1)) * Tr::kState
                            : reinterpret_cast<const float*>(sm.ring[end >> 1]);
    for (int r = 0; r < ER; ++r) {
      const int e = (tid % GT) + r * NT, head = e / (D / 4);
      float4 o;
      float rr, l;
      fold<D, NG, 4, false>(
          [&](int k) { return k == n - 1 ? tail : reinterpret_cast<const float*>(sm.ring[w0 + k]); }, n, e, o, rr, l);
      if (whole) {
        write_row(row, e, o, l);
      } else {
        float* dst = P.part + (2ll * blockIdx.x + (begins ? 1 : 0)) * Tr::kState;
        __stcg(reinterpret_cast<float4*>(dst) + e, o);
        if (e % (D / 4) == 0) {
          __stcg(dst + Tr::kRows * D + head, rr);
          __stcg(dst + Tr::kRows * D + Tr::kRows + head, l);
        }
      }
    }
  }

  // ---- rows cut by CTA boundaries: at most one begun earlier and one begun here -------------
  if (open_row[0] >= 0 || open_row[1] >= 0) {  // uniform: every thread walked the same pieces
    int cf[2] = {0, 0}, parts[2] = {0, 0};
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (open_row[s] < 0) continue;
      const int tk = quotient(open_row[s], a.KVH), h = open_row[s] - tk * a.KVH;
      const int np = quotient(sm.pre[tk + 1] - sm.pre[tk], a.KVH);
      const int first_unit = sm.pre[tk] + h * np;
      cf[s] = quotient(first_unit, chunk);
      parts[s] = quotient(first_unit + np - 1, chunk) - cf[s] + 1;
    }
    __syncthreads();  // the CTA's partial states are written
    if (tid == 0 && open_row[0] >= 0) sm.arrived[0] = static_cast<int>(atom_add_acq_rel_gpu_u32(P.counter + cf[0], 1u));
    if (tid == 32 && open_row[1] >= 0) sm.arrived[1] = static_cast<int>(atom_add_acq_rel_gpu_u32(P.counter + cf[1], 1u));
    __syncthreads();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (open_row[s] < 0 || sm.arrived[s] != parts[s] - 1) continue;
      if (tid == 32 * s) P.counter[cf[s]] = 0;
      if (grp != s % NGR) continue;  // a group each
      fence_acq_rel_gpu();
      for (int r = 0; r < ER; ++r) {
        const int e = (tid % GT) + r * NT;
        float4 o;
        float rr, l;
        fold<D, NG, 8, true>([&](int k) { return P.part + (2ll * (cf[s] + k) + (k == 0 ? 1 : 0)) * Tr::kState; },
                             parts[s], e, o, rr, l);
        write_row(open_row[s], e, o, l);
      }
    }
  }
}

int decode_sms(int device) {
  static std::mutex mu;
  static int cache[64] = {0};
  if (device < 0 || device >= 64) return 148;
  std::lock_guard<std::mutex> lock(mu);
  if (cache[device] == 0 &&
      cudaDeviceGetAttribute(&cache[device], cudaDevAttrMultiProcessorCount, device) != cudaSuccess)
    cache[device] = 148;
  return std::min(cache[device], kMaxCtas);
}

template <int D, int FMT, int NG, bool PK>
cudaError_t launch_one(const DecParams& p, int grid, cudaStream_t stream) {
  using Tr = DecTraits<D, NG>;
  static std::once_flag once[64];
  static cudaError_t err[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  std::call_once(once[dev], [&] {
    err[dev] = cudaFuncSetAttribute(q8_decode_kernel<D, FMT, NG, PK>,
                                    cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    static_cast<int>(sizeof(DecSmem<D, NG>)));
  });
  if (err[dev] != cudaSuccess) return err[dev];
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(Tr::kThreads);
  cfg.dynamicSmemBytes = sizeof(DecSmem<D, NG>);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, q8_decode_kernel<D, FMT, NG, PK>, p);
}

}  // namespace

size_t q8_decode_workspace(int device) {
  static_assert(16 * DecTraits<128, 1>::kState >= 8 * DecTraits<128, 2>::kState, "largest states of a CTA");
  return kWsHeader + kCounterBytes +
         static_cast<size_t>(decode_sms(device)) * (2 * DecTraits<128, 2>::kState + 16 * DecTraits<128, 1>::kState) *
             sizeof(float);
}

bool q8_decode_supported(const Q8AttnArgs& g) {
  const AttnArgs& a = g.a;
  const Q8Pool& p = g.p;
  auto codes16 = [](const void* base, long long sn, long long ss, long long sh, long long sd) {
    return sd == 1 && sn % 16 == 0 && ss % 16 == 0 && sh % 16 == 0 &&
           (reinterpret_cast<uintptr_t>(base) & 15) == 0;
  };
  auto rows16 = [](const void* base, long long st, long long sh, long long sd) {
    return sd == 1 && st % 8 == 0 && sh % 8 == 0 && (reinterpret_cast<uintptr_t>(base) & 15) == 0;
  };
  return a.group <= 16 && codes16(p.k, p.k_sn, p.k_ss, p.k_sh, p.k_sd) &&
         codes16(p.v, p.v_sn, p.v_ss, p.v_sh, p.v_sd) && rows16(a.q, a.q_st, a.q_sh, a.q_sd) &&
         rows16(a.out, a.o_st, a.o_sh, a.o_sd);
}

cudaError_t launch_q8_decode(const Q8AttnArgs& g, bool skip_runs, bool split, int device,
                             void* workspace, cudaStream_t stream, int* launches) {
  DecParams p;
  p.g = g;
  p.skip_runs = skip_runs;
  p.split = split;
  p.counter = reinterpret_cast<unsigned*>(static_cast<uint8_t*>(workspace) + kWsHeader);
  p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kWsHeader + kCounterBytes);
  const int sms = decode_sms(device);
  p.sms = sms;
  p.mid = p.part + 2ll * sms * DecTraits<128, 2>::kState;
  const bool packed = g.p.k_ss == g.p.D && g.p.v_ss == g.p.D && g.p.s_sw == 1 && g.p.s_sn % 2 == 0 &&
                      g.p.s_sh % 2 == 0 && (reinterpret_cast<uintptr_t>(g.p.scales) & 7) == 0;
  // Tokens per launch: the row lists' room, and units that fit 31 bits.
  const long long per_token = g.a.W * g.a.KVH;
  const long long most = std::max<long long>(1, std::min<long long>(kMaxTok, 0x7fffffffLL / per_token));
  *launches = 0;
  for (long long t0 = 0; t0 < g.a.T; t0 += most) {
    p.t0 = static_cast<int>(t0);
    p.tn = static_cast<int>(std::min(most, g.a.T - t0));
    const bool wide = g.a.group > 8;
    p.min_chunk = wide ? 8 : 16;
    // No more CTAs than the table could fill (the lengths are on the device).
    const long long bound = std::max<long long>(1, (per_token * p.tn + p.min_chunk - 1) / p.min_chunk);
    const int grid = split ? sms : static_cast<int>(std::min<long long>(sms, bound));
    cudaError_t e;
#define SS_Q8_DECODE_PK(D, FMT, NG) \
  e = packed ? launch_one<D, FMT, NG, true>(p, grid, stream) : launch_one<D, FMT, NG, false>(p, grid, stream)
#define SS_Q8_DECODE(D, NG)                              \
  if (g.p.fmt == SS_CODE_INT8) {                         \
    SS_Q8_DECODE_PK(D, SS_CODE_INT8, NG);                \
  } else {                                               \
    SS_Q8_DECODE_PK(D, SS_CODE_E4M3, NG);                \
  }
    if (g.p.D == 128) {
      if (wide) { SS_Q8_DECODE(128, 2) } else { SS_Q8_DECODE(128, 1) }
    } else {
      if (wide) { SS_Q8_DECODE(64, 2) } else { SS_Q8_DECODE(64, 1) }
    }
#undef SS_Q8_DECODE_PK
#undef SS_Q8_DECODE
    if (e != cudaSuccess) return e;
    ++*launches;
  }
  return cudaSuccess;
}

}  // namespace ss
