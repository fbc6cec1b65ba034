// Prompt chunks over the 8-bit pool as tcgen05 tiles.
//
// Tokens of runs of at least kQ8MinRun consecutive query tokens of one sequence are computed here,
// all others by the split-K kernel (q8_decode.cu).  The mathematics is that kernel's:
//   x_ij = (q_i . Kc_j) * ks_page * sm_scale * log2 e + log2(vs_page),   w_ij = 2^(x_ij - r_i)
//   O_i  = sum_j w_ij Vc_j,   l_i = sum_j w_ij / vs_page,   out_i = O_i / l_i
// K codes and q (its row's power of two taken out) are fp16, which holds the codes exactly, and q but for the
// last bits of elements 2^17 and more below their row's largest (2^-25 of it); the weights
// and the V codes are tf32: fp16 has the bits but not the range (weights 2^30 below the row's
// largest would vanish where the leading keys hold code 0), bf16 the range but not the bits.  The weights are
// rounded to nearest, by an integer addition (96.7 us for the prompt below; cut off, as the product does by
// itself, they made outputs 3e-4 too small at 95; with cvt.rna 101).
//
// What bounds it: the tensor pipe's issue rate.  A 128 x 128 x 16 fp16 product took 107 cycles and a
// 128 x 128 x 8 tf32 product with A in TMEM 75 (measured alone), so a pair of tiles needs 2 * (8 * 107
// + 16 * 75) = 4,100 cycles per key block of 128; the loop runs at 6,300, the rest being waits of the
// four products and two softmaxes on one another.  A 3001-token prompt (16 query and 2 KV heads of
// 128; 37 GFLOP) takes 97 us, of which about 6 are the start, 8 the join of cut windows.
//
// A window is up to 2 * (128 / group) tokens of one run: two tiles of 128 rows (token, query head
// of the KV head) that share every K / V block.  A work item is (window, KV head, range of
// 128-key blocks).  Per block j, tile t:
//   S_t = Q_t K_j^T      kind::f16, A, B in shared memory, fp32 in TMEM columns [128 t, +128)
//   softmax              one thread per row; P overwrites S_t in TMEM; O_t is rescaled only when a
//                        weight would pass 2^20
//   O_t += P_t V_j       kind::tf32, A = P_t from TMEM, B = V_j^T in shared memory
// in the order S_0(j+1), O_1(j), S_1(j+1), O_0(j+1): each softmax has two products' time.
// The codes are widened on their way into shared memory: K rows to 128-byte swizzled fp16 lines by
// three warps, V transposed (lane = key) to lines of 32 keys in fp32 by eight (a page of a block
// each); a page's registers are loaded for the next block as soon as it is stored.
//
// The roles' loops are kept rolled and small: with everything unrolled each warp ran at about one
// instruction in five cycles, the rate at which instructions came from the cache, a key block took
// 10,000 cycles whatever was taken out of it, and the prompt took 123 us.
//
// Scheduling.  Every CTA lists the launch's windows (a scan over its tokens) and takes an equal run
// of the units (window, KV head, block; beginning a window counts as two blocks), so that all finish
// together; a window that a run's end cuts leaves fp32 states in the workspace, joined by
// q8_merge_kernel.  (Whole windows taken from a counter, long ones first and the longest cut in two,
// left 12 to 19 blocks per CTA in that prompt: 110 us.)  The roles walk the CTA's run on their own: a
// producer is in the next window while the softmax warps finish the last.  A call that also has
// tokens outside runs launches the split-K kernel first, and the two share out the SMs by their work
// (q8_split): 56 decode rows beside 8 chunks of 512 tokens 136 -> 126 us.
//
// Warps: 0 MMA issuer, 1-3 K, 4-11 V, 12-15 softmax of tile 0, 16-19 of tile 1 (TMEM lane quadrant =
// warp % 4), up to 96 registers a thread.
#include <cuda_bf16.h>
#include <math_constants.h>

#include <algorithm>
#include <climits>
#include <mutex>

#include "exp2.cuh"
#include "ptx.cuh"
#include "q8.cuh"
#include "q8_widen.cuh"

namespace ss {

namespace {

constexpr int kThreads = 640;
constexpr int kVWarp = 4, kSoftmaxWarp = 12;  // first V and softmax warps
constexpr int kRows = 128;         // rows of a tile
constexpr int kNB = 128;           // keys of a block
constexpr int kPages = kNB / kPage;
constexpr int kMaxTokP = 8192;     // tokens per launch
static_assert((kMaxTokP + kThreads - 1) / kThreads <= 32, "a thread's tokens fit a mask");
// Windows per launch.  A run that lies inside the launch has kQ8MinRun tokens or more for each of its
// windows (the shortest windows take 16 tokens).  The run cut by the launch's beginning and the one cut by
// its end may hold a single token here: x of them, y of the other and 8-token runs between, x + y = 8,
// list one window more than the launch has eighths.
constexpr int kMaxWin = kMaxTokP / kQ8MinRun + 1;
constexpr int kMinPart = 4;        // units: smallest share of a CTA
constexpr int kHead = 2;           // units that beginning a window costs (Q, first and last waits)
constexpr float kSlackP = 20.f;
constexpr int kPolyEvery = 3;      // one exponential pair in 3 on the FMA pipe

template <int D>
struct Lay {
  static constexpr int kHalves = D / 64;
  static constexpr int kQ = kHalves * kRows * 128;   // Q tile, fp16
  static constexpr int kK = kHalves * kNB * 128;     // K block, fp16
  static constexpr int kV = 2 * D * 128;             // V^T of 64 keys, fp32: 2 atoms of 32 keys
  static constexpr int kOffK = 2 * kQ;
  static constexpr int kOffV = kOffK + 2 * kK;
  static constexpr int kOffCtl = kOffV + 2 * kV;
};

enum : int { kBarQ = 0, kBarS = 2, kBarPH = 4, kBarP = 6, kBarPV = 8, kBarKF = 10, kBarKE = 12,
             kBarVF = 14, kBarVE = 16, kBarEnd = 18, kNumBars = 19 };

struct CtlQ {
  unsigned long long bar[kNumBars];
  float4 sc[4][kPages];   // per block (mod 4) and page: K scale, log2 and reciprocal of V's
  uint32_t tmem;
  int red[kThreads / 32];
  int run_keys;
  int v_nan;              // a NaN code of V (e4m3) has been met
  int walk[3];            // the CTA's units [0], [1] and the window of the first
  unsigned short first[kMaxWin], count[kMaxWin];
  int keys[kMaxWin], seq[kMaxWin];
  int pre[kMaxWin + 1];   // units before each window
};

// Bit 7 of every byte that is an e4m3 NaN.
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return (w & 0x7f7f7f7fu) + 0x01010101u & 0x80808080u; }

struct PrefillParams {
  Q8AttnArgs g;
  int t0, tn;
  int split;          // the split-K kernel of the call runs beside this one, on q8_split's SMs
  int tpt;            // tokens per tile
  unsigned magic;     // ceil(2^32 / window): x / window = (x * magic) >> 32 for x < 2^13
  unsigned magic_group;  // the same for the group (0: of one head)
  float* part;        // [2 * grid] states: of the window begun before the CTA's run, and in it
  int4* cuts;         // [grid] {first token, tokens, KV head, parts} of the window that the CTA
                      // begins and leaves unfinished (parts 0: none)
};

template <int D>
struct State {  // a cut window's state: O as [D / 4][256 rows] float4, then r and l of 256 rows
  static constexpr int kFloats = 256 * D + 512;
};

__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity));
}
__device__ __forceinline__ void tc_mma_tf32_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc,
                                               uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::tf32 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
constexpr uint32_t idesc_of(int fmt, int N) {  // fp32 accumulators, M = 128, both K-major
  return (1u << 4) | (static_cast<uint32_t>(fmt) << 7) | (static_cast<uint32_t>(fmt) << 10) |
         (static_cast<uint32_t>(N >> 3) << 17) | (128u >> 4 << 24);
}
__device__ __forceinline__ void st_shared16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void st_shared4(uint32_t addr, uint32_t a) {
  asm volatile("st.shared.b32 [%0], %1;" ::"r"(addr), "r"(a) : "memory");
}

__device__ __forceinline__ uint4 ld_shared16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
// 16 bytes from global to shared memory, or 16 zeros (bytes = 0).
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Writes NaN over the outputs (or, of a cut window, the state: row r of State<D>) of the calling thread's
// query row where a row of V that it attends (keys below lim of k0 .. k1 - 1) holds NaN.  A warp looks a
// page over at once.  Out of line: inlined, it made the loops that never come here 4 % slower.
template <int D>
__device__ __noinline__ void put_nan(const AttnArgs& a, const Q8Pool& pool, long long bt_row, int kvh, int k0,
                                     int k1, int lim, __nv_bfloat16* out, float* state) {
  const int lane = threadIdx.x & 31;
  for (int k = k0; k < k1; k += kPage) {
    const long long id = ld_index(a.bt, a.bt64, bt_row + k / kPage * a.bt_sn);
    if (id < 0 || id >= pool.N) continue;
    const uint8_t* page = pool.v + id * pool.v_sn + kvh * pool.v_sh;
    const uint4* part = reinterpret_cast<const uint4*>(page + (lane >> 1) * pool.v_ss + (lane & 1) * (D / 2));
    uint32_t any = 0;
    for (int i = 0; i < D / 32; ++i) {
      const uint4 v = __ldg(part + i);
      any |= nan_codes(v.x) | nan_codes(v.y) | nan_codes(v.z) | nan_codes(v.w);
    }
    for (unsigned hit = __ballot_sync(0xffffffffu, any != 0); hit != 0;) {
      const int key = (__ffs(hit) - 1) >> 1;
      hit &= ~(3u << 2 * key);
      if (k + key >= min(k1, lim)) continue;
      const uint8_t* codes = page + key * pool.v_ss;
      for (int d = 0; d < D; ++d) {
        if ((__ldg(codes + d) & 0x7f) != 0x7f) continue;
        if (state != nullptr)
          __stcg(state + d / 4 * 1024 + d % 4, CUDART_NAN_F);
        else
          out[d] = __ushort_as_bfloat16(0x7fff);
      }
    }
  }
}

// Sum and (exclusive) maximum scans over the CTA.
__device__ __forceinline__ int scan_sum(int v, int* red, int warp, int lane, int& total) {
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += x;
  }
  __syncthreads();
  if (lane == 31) red[warp] = inc;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += red[w];
    total += red[w];
  }
  return before + inc - v;
}
__device__ __forceinline__ int scan_max(int v, int* red, int warp, int lane) {
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc = max(inc, x);
  }
  __syncthreads();
  if (lane == 31) red[warp] = inc;
  __syncthreads();
  int before = -1;
  for (int w = 0; w < warp; ++w) before = max(before, red[w]);
  const int up = __shfl_up_sync(0xffffffffu, inc, 1);
  return lane == 0 ? before : max(before, up);
}

template <int D, int FMT>
__global__ void __launch_bounds__(kThreads, 1)
    q8_prefill_kernel(const __grid_constant__ PrefillParams P) {
  using L = Lay<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  const uint32_t sb = smem_u32(smem);
  CtlQ* ctl = reinterpret_cast<CtlQ*>(smem + L::kOffCtl);
  const uint32_t bars = smem_u32(ctl->bar);
  auto bar = [&](int i) { return bars + 8 * i; };
  const AttnArgs& a = P.g.a;
  const Q8Pool& pool = P.g.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int tw = 2 * P.tpt;  // tokens of a window

  if (tid == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(bar(kBarQ + t), 128);
      mbar_init(bar(kBarS + t), 1);
      mbar_init(bar(kBarPH + t), 128);
      mbar_init(bar(kBarP + t), 128);
      mbar_init(bar(kBarPV + t), 1);
      mbar_init(bar(kBarKF + t), 3);
      mbar_init(bar(kBarKE + t), 1);
      mbar_init(bar(kBarVF + t), 4);
      mbar_init(bar(kBarVE + t), 1);
    }
    mbar_init(bar(kBarEnd), 1);
    ctl->run_keys = 0;
    ctl->v_nan = 0;
    fence_mbar_init();
  }
  if (warp == 0) {
    tmem_alloc(smem_u32(&ctl->tmem), 512);
    tmem_relinquish();
  }
  // After the split-K kernel of the same call, which waited for what came before it, nothing is
  // waited for until the end.
  if (!P.split) griddep_wait();
  griddep_launch_dependents();

  // ---- the windows of this launch ----------------------------------------------------------
  int nwin, units, ctas = gridDim.x;  // CTAs that take units
  {
    // The operand buffers are idle: the staged ids and lengths stand there.
    int* const seq = reinterpret_cast<int*>(smem) + kQ8Pad;
    int* const len = seq + kMaxTokP + kQ8Pad;
    stage_tokens(a, P.t0, P.tn, seq, len, blockIdx.x == 0);
    __syncthreads();
    const int per = (P.tn + kThreads - 1) / kThreads;
    const int b0 = min(tid * per, P.tn), b1 = min(b0 + per, P.tn);
    auto starts = [&](int i) { return i == 0 || seq[i - 1] != seq[i]; };
    // Token i of the run that starts at `start` (as far as this launch sees).
    auto in_run = [&](int i, int start) { return i - start >= kQ8Pad || in_staged_run(seq, i); };
    auto place = [&](int x) { return x - tw * static_cast<int>(__umulhi(static_cast<unsigned>(x), P.magic)); };
    int start = -1;  // last run start at or before a token
    for (int i = b0; i < b1; ++i)
      if (starts(i)) start = i;
    const int before = scan_max(start, ctl->red, warp, lane);
    start = before;
    int all_keys = 0;     // of this thread's tokens
    unsigned begins = 0;  // tokens of this thread that begin a window (at most 13 tokens a thread)
    for (int i = b0; i < b1; ++i) {
      if (starts(i)) start = i;
      if (place(i - start) == 0 && in_run(i, start)) begins |= 1u << (i - b0);
      all_keys += q8_clamped(len[i]);
    }
    int idx = scan_sum(__popc(begins), ctl->red, warp, lane, nwin);
    for (; begins; begins &= begins - 1) ctl->first[idx++] = static_cast<unsigned short>(b0 + __ffs(begins) - 1);
    __syncthreads();
    // One warp per window: its tokens, and the keys that they attend.
    for (int w = warp; w < nwin; w += kThreads / 32) {
      const int f = ctl->first[w], id = seq[f];
      int count = 0, keys = 0, sum = 0;
      for (int k = 0; k < tw; k += 32) {
        const int i = f + k + lane;
        const bool on = k + lane < tw && i < P.tn && seq[i] == id;
        const unsigned m = __ballot_sync(0xffffffffu, on);
        const int n = m == ~0u ? 32 : __ffs(~m) - 1;  // up to the run's end
        keys = max(keys, lane < n ? len[i] : 0);
        sum += lane < n ? q8_clamped(len[i]) : 0;
        count += n;
        if (n < 32) break;
      }
      keys = __reduce_max_sync(0xffffffffu, keys);
      sum = __reduce_add_sync(0xffffffffu, sum);
      if (lane == 0) {
        if (P.split) atomicAdd(&ctl->run_keys, sum);
        ctl->count[w] = static_cast<unsigned short>(count);
        ctl->keys[w] = keys;
        ctl->seq[w] = id;
      }
    }
    __syncthreads();
    auto units_of = [](int keys) { return keys > 0 ? (keys + kNB - 1) / kNB + kHead : 0; };
    constexpr int kPer = (kMaxWin + kThreads - 1) / kThreads;
    int blocks = 0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int w = tid * kPer + k;
      if (w < nwin) blocks += units_of(ctl->keys[w]);
    }
    int run = scan_sum(blocks * a.KVH, ctl->red, warp, lane, units);
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int w = tid * kPer + k;
      if (w < nwin) {
        ctl->pre[w] = run;
        run += units_of(ctl->keys[w]) * a.KVH;
      }
    }
    if (tid == 0) ctl->pre[nwin] = units;
    if (P.split) {
      int total;
      scan_sum(all_keys, ctl->red, warp, lane, total);
      ctas -= q8_split(total - ctl->run_keys, ctl->run_keys, ctas);
      ctas = max(ctas, 1);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl->tmem;
  const int share = max((units + ctas - 1) / ctas, kMinPart);
  const int u0 = min(static_cast<long long>(blockIdx.x) * share, static_cast<long long>(units));
  const int u1 = min(u0 + static_cast<long long>(share), static_cast<long long>(units));

  int jg = 0;      // blocks processed so far by this CTA (phases of the K and V barriers)
  // Phases of a tile's own barriers: tile 1 sits out windows that fill one tile only.
  int jt[2] = {0, 0}, qt[2] = {0, 0};  // blocks and windows of each tile so far
  bool ok = true;
  struct Item {
    int win, first, count, kvh, j0, j1, keys, nb, len;
  };
  // The part of a window and KV head that unit u stands in, as far as this CTA's run goes.
  auto item_at = [&](int u, int win) -> Item {
    Item it;
    while (ctl->pre[win + 1] <= u) ++win;
    it.win = win;
    it.first = ctl->first[win];
    it.count = ctl->count[win];
    it.keys = ctl->keys[win];
    it.nb = (it.keys + kNB - 1) / kNB;
    const int n = it.nb + kHead, rest = u - ctl->pre[win];
    it.kvh = rest / n;
    const int x0 = rest - it.kvh * n, x1 = min(n, x0 + u1 - u);
    it.len = x1 - x0;
    it.j0 = max(x0 - kHead, 0);
    it.j1 = max(x1 - kHead, 0);
    return it;
  };
  int win0 = 0;  // window of the run's first unit
  if (u0 < u1) {
    int hi = nwin;
    while (hi - win0 > 1) {
      const int mid = (win0 + hi) >> 1;
      if (ctl->pre[mid] <= u0) win0 = mid; else hi = mid;
    }
  }
  if (tid == 0) {
    ctl->walk[0] = u0;
    ctl->walk[1] = u1;
    ctl->walk[2] = win0;
  }
  auto timed_out = [&]() {
    if (lane == 0) atomicOr(a.err, SS_DEVERR_TIMEOUT);
  };

  if (warp < kSoftmaxWarp) {
    if (warp == 0) {
      // ================================= MMA issuer ====================================
      constexpr uint32_t id_qk = idesc_of(0, kNB), id_pv = idesc_of(2, D);
      const bool leader = elect_one();
      for (int u = u0, win = win0; u < u1 && ok;) {
        const Item it = item_at(u, win);
        const int nblk = it.j1 - it.j0;
        u += it.len;
        win = it.win;
        if (nblk == 0) continue;
        const bool two = it.count > P.tpt;  // both tiles hold tokens
        auto qk = [&](int t, int st) {
          if (leader) {
            uint64_t qd = smem_desc_sw128(sb + t * L::kQ, 16, 1024);
            uint64_t kd = smem_desc_sw128(sb + L::kOffK + st * L::kK, 16, 1024);
#pragma unroll 1
            for (int i = 0; i < L::kHalves; ++i) {
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                tc_mma_f16(tmem + t * kNB, qd + kk * 2, kd + kk * 2, id_qk, (i | kk) ? 1u : 0u);
              qd += kRows * 128 / 16;
              kd += kNB * 128 / 16;
            }
            tc_commit(bar(kBarS + t));
          }
          __syncwarp();
        };
        auto pv = [&](int t, int j, bool release) -> bool {  // block j of this item
#pragma unroll 1
          for (int half = 0; half < 2; ++half) {
            if (!wait_warp(bar(kBarVF + half), (jg + j) & 1)) return false;
            if (!wait_warp(bar((half ? kBarP : kBarPH) + t), (jt[t] + j) & 1)) return false;
            tc_fence_after();
            if (leader) {
              uint64_t vd = smem_desc_sw128(sb + L::kOffV + half * L::kV, 16, 1024);
              uint32_t pa = tmem + t * kNB + half * 64;
#pragma unroll 1
              for (int i = 0; i < 2; ++i) {  // 32 keys each
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                  tc_mma_tf32_ts(tmem + 256 + t * 128, pa + kk * 8, vd + kk * 2, id_pv,
                                 (j | half | i | kk) ? 1u : 0u);
                vd += D * 128 / 16;
                pa += 32;
              }
              if (release) tc_commit(bar(kBarVE + half));
            }
            __syncwarp();
          }
          if (leader) tc_commit(bar(kBarPV + t));
          __syncwarp();
          return true;
        };
        {
          ok = wait_warp(bar(kBarQ), qt[0] & 1);
          if (ok && two) ok = wait_warp(bar(kBarQ + 1), qt[1] & 1);
          for (int j = 0; j < nblk && ok; ++j) {
            const int jb = jg + j, st = jb & 1;
            ok = wait_warp(bar(kBarKF + st), (jb >> 1) & 1);
            if (!ok) break;
            tc_fence_after();
            qk(0, st);
            if (two) {
              if (j > 0 && !(ok = pv(1, j - 1, true))) break;
              qk(1, st);
            }
            if (leader) tc_commit(bar(kBarKE + st));
            __syncwarp();
            ok = pv(0, j, !two);
          }
          if (ok && two) ok = pv(1, nblk - 1, true);
          if (!ok) timed_out();
          jg += nblk;
          jt[0] += nblk;
          ++qt[0];
          if (two) {
            jt[1] += nblk;
            ++qt[1];
          }
        }
        tc_fence_before();
      }
      if (leader) tc_commit(bar(kBarEnd));  // every product issued has completed before TMEM is freed
      __syncwarp();
      if (!wait_warp(bar(kBarEnd), 0)) timed_out();
    } else {
      // ================================== producers ====================================
      const bool is_v = warp >= kVWarp;
      // Page ids and scales of a block's 8 pages: lanes 0-7.  id -1: past the keys or outside the
      // pool.
      for (int u = u0, win = win0; u < u1 && ok;) {
        const Item it = item_at(u, win);
        const int nblk = it.j1 - it.j0;
        u += it.len;
        win = it.win;
        if (nblk == 0) continue;
        const long long bt_row = static_cast<long long>(ctl->seq[it.win]) * a.bt_sb;
        const float* sbase = pool.scales + static_cast<long long>(it.kvh) * pool.s_sh;
        auto load_id = [&](int j) -> int {
          const int pi = (it.j0 + j) * kPages + lane;
          if (j >= nblk || lane >= kPages || pi * kPage >= it.keys) return -1;
          const long long id = ld_index(a.bt, a.bt64, bt_row + pi * a.bt_sn);
          if (id >= 0 && id < pool.N) return static_cast<int>(id);
          atomicOr(a.err, SS_DEVERR_PAGE);
          return -1;
        };
        auto load_scale = [&](int id) -> float2 {
          if (id < 0) return make_float2(0.f, 1.f);
          const float* s = sbase + id * pool.s_sn;
          return make_float2(__ldg(s), __ldg(s + pool.s_sw));
        };
        int id = load_id(0), id_next = load_id(1);
        float2 scl = load_scale(id);
        if (!is_v) {
          // Warp 1 + r widens pages r, r + 3, r + 6.  Load (i, k) of a page: 8 keys (8 k + lane % 8) x
          // 64 values (64 i + 16 (lane / 8)).
          const int r = warp - 1, key = lane & 7;
          const uint8_t* base = pool.k + static_cast<long long>(it.kvh) * pool.k_sh + key * pool.k_ss + 16 * (lane >> 3);
          // 16-byte chunk 2 (lane / 8) + q of a line of 64 values, swizzled by the key.
          uint32_t at[2];
#pragma unroll
          for (int q = 0; q < 2; ++q)
            at[q] = sb + L::kOffK + key * 128 + (((2 * (lane >> 3) + q) ^ key) << 4);
          auto load = [&](int j, int p, uint4 (&v)[L::kHalves][2]) {
            const int pid = __shfl_sync(0xffffffffu, id, p & 31);
            const int left = pid < 0 || p >= kPages ? 0 : it.keys - ((it.j0 + j) * kPages + p) * kPage;
            const uint8_t* src = base + static_cast<long long>(max(pid, 0)) * pool.k_sn;
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
              for (int i = 0; i < L::kHalves; ++i) {
                v[i][k] = make_uint4(0, 0, 0, 0);
                if (key + 8 * k < left) v[i][k] = __ldg(reinterpret_cast<const uint4*>(src + 8 * k * pool.k_ss + 64 * i));
              }
          };
          uint4 buf[3][L::kHalves][2];
#pragma unroll
          for (int n = 0; n < 3; ++n) load(0, r + 3 * n, buf[n]);
          for (int j = 0; j < nblk; ++j) {
            const int jb = jg + j, st = jb & 1;
            const float2 now = scl;
            id = id_next;
            id_next = load_id(j + 2);
            scl = load_scale(id);
            ok = wait_warp(bar(kBarKE + st), ((jb >> 1) & 1) ^ 1);
            if (!ok) break;
            if (r == 0 && lane < kPages) {
              const float vs = fmaxf(now.y, kMinVs);
              ctl->sc[jb & 3][lane] = make_float4(now.x, lg2(vs), __frcp_rn(vs), 0.f);
            }
#pragma unroll
            for (int n = 0; n < 3; ++n) {
              if (r + 3 * n < kPages) {
                const uint32_t off = st * L::kK + (r + 3 * n) * (16 * 128);
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                  for (int i = 0; i < L::kHalves; ++i) {
                    const uint4 v = buf[n][i][k];
                    uint32_t w[8];
                    widen<FMT>(v.x, w[0], w[1]);
                    widen<FMT>(v.y, w[2], w[3]);
                    widen<FMT>(v.z, w[4], w[5]);
                    widen<FMT>(v.w, w[6], w[7]);
                    st_shared16(at[0] + off + i * (kNB * 128) + 8 * k * 128, w[0], w[1], w[2], w[3]);
                    st_shared16(at[1] + off + i * (kNB * 128) + 8 * k * 128, w[4], w[5], w[6], w[7]);
                  }
              }
              load(j + 1, r + 3 * n, buf[n]);  // in flight until the next block
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(kBarKF + st));
          }
        } else {
          // Warp 4 + 4 h + u widens page u of half h of every block.  Load i: 16 keys (lane % 16) x
          // 32 values (32 i + 16 (lane / 16)).
          const int h = (warp - kVWarp) >> 2, u = warp & 3, key = lane & 15, hi = lane >> 4;
          const uint8_t* base = pool.v + static_cast<long long>(it.kvh) * pool.v_sh + key * pool.v_ss + 16 * hi;
          // Line of value 16 hi + k (k = 0 .. 15), this lane's key.  The upper lanes take their values
          // in the order k ^ 4, which puts the two half-warps' stores into different banks.
          uint32_t at[8];
#pragma unroll
          for (int m = 0; m < 8; ++m)
            at[m] = sb + L::kOffV + h * L::kV + (u >> 1) * (D * 128) + 16 * hi * 128 + (m < 4 ? 512 : -512) * hi +
                    ((((u & 1) * 4 + (key >> 2)) ^ (4 * hi) ^ m) << 4) + (key & 3) * 4;
          uint4 buf[D / 32];
          bool dead = false;  // the page's V scale counts as 0: its codes are no part of the product, but for NaN
          auto load = [&](int j) {
            const int pid = __shfl_sync(0xffffffffu, id, 4 * h + u);
            const float vs = __shfl_sync(0xffffffffu, scl.y, 4 * h + u);
            dead = !(vs >= kMinVs);
            const int left = pid < 0 || (FMT == SS_CODE_INT8 && dead) ? 0 : it.keys - ((it.j0 + j) * kPages + 4 * h + u) * kPage;
            const uint8_t* src = base + static_cast<long long>(max(pid, 0)) * pool.v_sn;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
              buf[i] = make_uint4(0, 0, 0, 0);
              if (key < left) buf[i] = __ldg(reinterpret_cast<const uint4*>(src + 32 * i));
            }
          };
          load(0);
          for (int j = 0; j < nblk; ++j) {
            const int jb = jg + j;
            id = id_next;
            id_next = load_id(j + 2);
            scl = load_scale(id);
            ok = wait_warp(bar(kBarVE + h), (jb & 1) ^ 1);
            if (!ok) break;
            if constexpr (FMT == SS_CODE_E4M3) {
              // A NaN would reach the tile's rows that do not attend its key too (0 * NaN): the product sees
              // zeros, and the softmax warps see to the rows that do at the end.
              uint32_t any = 0;
#pragma unroll
              for (int i = 0; i < D / 32; ++i)
                any |= nan_codes(buf[i].x) | nan_codes(buf[i].y) | nan_codes(buf[i].z) | nan_codes(buf[i].w);
              const unsigned lanes = __ballot_sync(0xffffffffu, any != 0);
              if (dead) {
#pragma unroll
                for (int i = 0; i < D / 32; ++i) buf[i] = make_uint4(0, 0, 0, 0);
              }
              if (lanes != 0) {
                ctl->v_nan = 1;
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                  buf[i].x &= ~((nan_codes(buf[i].x) >> 7) * 0xffu);
                  buf[i].y &= ~((nan_codes(buf[i].y) >> 7) * 0xffu);
                  buf[i].z &= ~((nan_codes(buf[i].z) >> 7) * 0xffu);
                  buf[i].w &= ~((nan_codes(buf[i].w) >> 7) * 0xffu);
                }
              }
            }
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
              const uint4 v = buf[i];
              const uint32_t w[4] = {hi ? v.y : v.x, hi ? v.x : v.y, hi ? v.w : v.z, hi ? v.z : v.w};
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                uint32_t f[4];
                widen_f32<FMT>(w[q], f);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  st_shared4(at[(4 * q + e) & 7] + i * (32 * 128) + (4 * q + e) * 128, f[e]);
              }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(kBarVF + h));
            load(j + 1);  // in flight until the next block
          }
        }
        if (!ok) timed_out();
        jg += nblk;
      }
    }
  } else {
    const int tt = (warp - kSoftmaxWarp) >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + tt * kNB + lane_off, tO = tmem + 256 + tt * 128 + lane_off;
    const int rt = row / a.group, rh = row - rt * a.group;  // token inside the tile, head
    // Windows without keys: zero rows.
    for (int w = blockIdx.x; w < nwin; w += gridDim.x) {
      if (ctl->keys[w] != 0) continue;
      for (int e = tid - 32 * kSoftmaxWarp; e < ctl->count[w] * a.H * (D / 8); e += 256) {
        const int d = e % (D / 8) * 8, h = e / (D / 8) % a.H, i = e / (D / 8) / a.H;
        *reinterpret_cast<uint4*>(a.out + (P.t0 + ctl->first[w] + i) * a.o_st + h * a.o_sh + d) = make_uint4(0, 0, 0, 0);
      }
    }
    if (warp == kSoftmaxWarp && lane == 0) {  // the window that this run begins and does not finish
      int4 cut = make_int4(0, 0, 0, 0);
      if (u0 < u1) {
        int win = win0;
        while (ctl->pre[win + 1] < u1) ++win;
        const int n = (ctl->keys[win] + kNB - 1) / kNB + kHead, kvh = (u1 - 1 - ctl->pre[win]) / n;
        const int begin = ctl->pre[win] + kvh * n + kHead, end = begin + n - kHead;  // its blocks
        if (begin >= u0 && begin < u1 && end > u1)
          cut = make_int4(P.t0 + ctl->first[win], ctl->count[win], kvh, (end - 1) / share - static_cast<int>(blockIdx.x) + 1);
      }
      P.cuts[blockIdx.x] = cut;
    }
    // An item's Q is loaded before the epilogue of the one before it: the product of its first block
    // then runs beside that epilogue.
    Item it, cur;
    bool have = false;  // cur's blocks are done, its epilogue is not
    float ref = 0.f, lsum = 0.f, f_row = 0.f;
    auto takes = [&](const Item& i) { return tt == 0 || i.count > P.tpt; };  // this tile holds tokens
    auto is_mine = [&](const Item& i) { return rt < P.tpt && tt * P.tpt + rt < i.count; };
    for (int u = u0, win = win0; ok;) {
      bool more = false;
      while (u < u1 && !more) {
        it = item_at(u, win);
        u += it.len;
        win = it.win;
        more = it.j1 > it.j0;
      }
      long long my_seq = 0, my_pos = 0;
      float f_next = 0.f;
      if (more && takes(it)) {
        const long long tc = P.t0 + it.first + (is_mine(it) ? tt * P.tpt + rt : 0);
        my_seq = ld_index(a.seq, a.seq64, tc);
        my_pos = ld_index(a.pos, a.pos64, tc);
        // ---- 32 rows of Q per warp, D / 8 lanes each 16 bytes of a row: copied to their place, then
        // turned there into fp16 with the row's power of two taken out.
        constexpr int LR = D / 8, RP = 32 / LR;  // lanes of a row, rows of a step
        const int c = lane % LR, r0 = (warp & 3) * 32 + lane / LR;
        const __nv_bfloat16* qb = a.q + (P.t0 + it.first + tt * P.tpt) * a.q_st +
                                  static_cast<long long>(it.kvh * a.group) * a.q_sh + 8 * c;
        const int left = min(it.count - tt * P.tpt, P.tpt);  // tokens of this tile
        const uint32_t dst = sb + tt * L::kQ + (c >> 3) * (kRows * 128);
        auto at = [&](int r) { return dst + r * 128 + (((c & 7) ^ (r & 7)) << 4); };
#pragma unroll 1
        for (int r = r0; r < r0 + 32; r += RP) {
          const int tok = a.group == 1 ? r : static_cast<int>(__umulhi(static_cast<unsigned>(r), P.magic_group));
          const int hd = r - tok * a.group;
          cp_async16(at(r), tok < left ? qb + tok * a.q_st + hd * a.q_sh : a.q, tok < left ? 16 : 0);
        }
        cp_async_wait_all();
#pragma unroll 1
        for (int n0 = 0; n0 < 32 / RP; n0 += 4) {
          uint4 v[4];
          float amax[4];
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            v[n] = ld_shared16(at(r0 + (n0 + n) * RP));
            const uint32_t w[4] = {v[n].x, v[n].y, v[n].z, v[n].w};
            amax[n] = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k)
              amax[n] = fmaxf(amax[n], fmaxf(fabsf(__uint_as_float(w[k] << 16)), fabsf(__uint_as_float(w[k] & 0xffff0000u))));
          }
#pragma unroll
          for (int o = 1; o < LR; o <<= 1)
#pragma unroll
            for (int n = 0; n < 4; ++n) amax[n] = fmaxf(amax[n], __shfl_xor_sync(0xffffffffu, amax[n], o));
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const uint32_t w[4] = {v[n].x, v[n].y, v[n].z, v[n].w};
            const int e = min(max(static_cast<int>(__float_as_uint(amax[n]) >> 23) - 127, -126), 126);
            // A negative sm_scale changes q's sign, so that the factor of the scores is >= 0.
            const float down = copysignf(__uint_as_float(static_cast<uint32_t>(127 - e) << 23), a.scale_log2);
            uint32_t h[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              h[k] = pack_f16(__uint_as_float(w[k] << 16) * down, __uint_as_float(w[k] & 0xffff0000u) * down);
            st_shared16(at(r0 + (n0 + n) * RP), h[0], h[1], h[2], h[3]);
            const float f = __shfl_sync(0xffffffffu, __uint_as_float(static_cast<uint32_t>(127 + e) << 23), (lane % RP) * LR);
            if (lane / RP == n0 + n) f_next = f * fabsf(a.scale_log2);  // the row this lane computes
          }
        }
        fence_proxy_async_smem();
        mbar_arrive(bar(kBarQ + tt));
      }
      if (have) {
        // ---- O_t / l of the item before, or the state of a cut window ---------------------
        const bool whole = cur.j1 - cur.j0 == cur.nb, mine = is_mine(cur);
        float* const state = P.part + (2ll * blockIdx.x + (cur.j0 == 0 ? 1 : 0)) * State<D>::kFloats;
        __nv_bfloat16* op = a.out + (P.t0 + cur.first + tt * P.tpt + rt) * a.o_st +
                            static_cast<long long>(cur.kvh * a.group + rh) * a.o_sh;
        ok = wait_warp(bar(kBarPV + tt), (jt[0] - 1) & 1);
        if (ok) {
          tc_fence_after();
          // A row whose keys are all masked never got a reference (and its weights are not sums of
          // exact zeros where the polynomial made them).
          if (ref == -CUDART_INF_F && lsum == lsum) lsum = 0.f;
          const float inv = lsum == 0.f ? 0.f : 1.f / lsum;
          float4* st = reinterpret_cast<float4*>(state) + tt * kRows + row;
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(tO + c * 32, o);
            tmem_wait_ld();
            if (!whole) {
#pragma unroll
              for (int i = 0; i < 8; ++i)
                __stcg(st + (c * 8 + i) * 256,
                       make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]),
                                   __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3])));
            } else if (mine) {
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                uint4 v;
                v.x = pack_bf16(__uint_as_float(o[q * 8 + 0]) * inv, __uint_as_float(o[q * 8 + 1]) * inv);
                v.y = pack_bf16(__uint_as_float(o[q * 8 + 2]) * inv, __uint_as_float(o[q * 8 + 3]) * inv);
                v.z = pack_bf16(__uint_as_float(o[q * 8 + 4]) * inv, __uint_as_float(o[q * 8 + 5]) * inv);
                v.w = pack_bf16(__uint_as_float(o[q * 8 + 6]) * inv, __uint_as_float(o[q * 8 + 7]) * inv);
                *reinterpret_cast<uint4*>(op + c * 32 + q * 8) = v;
              }
            }
          }
          if (!whole) {
            float* rl = state + 256 * D + tt * kRows + row;
            __stcg(rl, ref);
            __stcg(rl + 256, lsum);
          }
        }
        if (!ok) break;
        tc_fence_before();
      }
      if (!more) break;
      cur = it;
      have = takes(it);
      const int nblk = it.j1 - it.j0;
      if (have) {
        // Rows past the window compute unmasked.
        const int lim = !is_mine(it) ? INT_MAX : my_seq == -1 ? 0 : token_info_from(a, my_seq, my_pos, false).L;
        f_row = f_next;
        ref = -CUDART_INF_F;
        lsum = 0.f;
        for (int j = 0; j < nblk; ++j) {
          const int jb = jt[0] + j;  // this tile's blocks so far
          ok = wait_warp(bar(kBarS + tt), jb & 1);
          if (!ok) break;
          tc_fence_after();
          // The scores are read twice, 32 at a time, for the row's maximum and for the weights: the
          // loops stay rolled.  (Straight-line code for 128 scores runs at the rate at which the
          // instruction cache refills, about one instruction in five cycles.)
          const int nv = lim - (it.j0 + j) * kNB;
          const bool partial = !__all_sync(0xffffffffu, nv >= kNB);
          const float4* sc = ctl->sc[(jg + j) & 3];
          // The factor is kept above 0 so that a masked score stays -inf under a zero scale.
          auto factor = [&](const float4& c) { return fmaxf(c.x * f_row, 1e-37f); };
          uint32_t x[32];
          auto read = [&](int c) {
            tmem_ld32(tS + c * 32, x);
            tmem_wait_ld();
            if (partial) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (c * 32 + i >= nv) x[i] = __float_as_uint(-CUDART_INF_F);
            }
          };
          float top = -CUDART_INF_F;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            read(c);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float m = max_nan(__uint_as_float(x[16 * h]), __uint_as_float(x[16 * h + 1]));
#pragma unroll
              for (int i = 2; i < 16; i += 2)
                m = max3_nan(m, __uint_as_float(x[16 * h + i]), __uint_as_float(x[16 * h + i + 1]));
              const float4 pc = sc[2 * c + h];
              top = max_nan(top, fmaf(m, factor(pc), pc.y));
            }
          }
          const bool raise = top > ref + kSlackP;
          const float ref_new = raise ? top : ref;
          const float alpha = raise ? ex2(ref - ref_new) : 1.f;
          if (j > 0 && __any_sync(0xffffffffu, raise)) {
            ok = wait_warp(bar(kBarPV + tt), (jb - 1) & 1);  // complete: S_t(j) was issued after it
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(tO + c * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st32(tO + c * 32, o);
            }
          }
          ref = ref_new;
          const float base = ref == -CUDART_INF_F ? 0.f : ref;
          // A score that is NaN or infinity makes the row NaN.  (Not every weight would: the polynomial's
          // clamp turns NaN into a number.)
          float part = top < CUDART_INF_F ? 0.f : CUDART_NAN_F;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            read(c);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float4 pc = sc[2 * c + h];
              const float f = factor(pc), b = pc.y - base;
              const uint64_t f2 = f2pack(f, f), b2 = f2pack(b, b);
              uint64_t acc[2] = {0, 0};
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                uint32_t& s0 = x[h * 16 + 2 * i];
                uint32_t& s1 = x[h * 16 + 2 * i + 1];
                const uint64_t x2 = fma2(f2pack(__uint_as_float(s0), __uint_as_float(s1)), f2, b2);
                uint64_t w2;
                if ((h * 8 + i) % kPolyEvery == kPolyEvery - 1) {
                  w2 = exp2_poly2(x2);
                } else {
                  float x0, x1;
                  f2unpack(x2, x0, x1);
                  w2 = f2pack(ex2(x0), ex2(x1));
                }
                acc[i & 1] = add2(acc[i & 1], w2);
                // Half of the lowest of tf32's bits: the product ignores the 13 bits below, which would
                // make every output 2^-11 * 0.7 too small on average.
                s0 = static_cast<uint32_t>(w2) + 0x1000u;
                s1 = static_cast<uint32_t>(w2 >> 32) + 0x1000u;
              }
              float a0, a1;
              f2unpack(add2(acc[0], acc[1]), a0, a1);
              part = fmaf(a0 + a1, pc.z, part);
            }
            tmem_st32(tS + c * 32, x);
            if (c & 1) {
              tmem_wait_st();
              tc_fence_before();
              mbar_arrive(bar((c == 1 ? kBarPH : kBarP) + tt));
            }
          }
          lsum = lsum * alpha + part;
        }
        jt[0] += nblk;
      }
      jg += nblk;
    }
    if (!ok) timed_out();
  }
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (FMT == SS_CODE_E4M3 && ctl->v_nan && warp >= kSoftmaxWarp) {
    // NaN codes of V stood as zeros in the products: the rows that attend them are put right here, each by
    // the thread that wrote it, in a second walk over the CTA's items.  (Its state comes from shared memory:
    // no registers are kept for it in the loops above.)
    const int t = (warp - kSoftmaxWarp) >> 2, row = (warp & 3) * 32 + lane, rt = row / a.group;
    int u = ctl->walk[0], win = ctl->walk[2];
    const int end = ctl->walk[1];
    while (u < end) {
      while (ctl->pre[win + 1] <= u) ++win;
      const int keys = ctl->keys[win], nb = (keys + kNB - 1) / kNB, n = nb + kHead;
      const int kvh = (u - ctl->pre[win]) / n, x0 = u - ctl->pre[win] - kvh * n, x1 = min(n, x0 + end - u);
      const int j0 = max(x0 - kHead, 0), j1 = max(x1 - kHead, 0), wt = t * P.tpt + rt;
      u += x1 - x0;
      if (j1 == j0 || ctl->count[win] <= t * P.tpt) continue;
      const long long tok = P.t0 + ctl->first[win] + wt;
      const bool mine = rt < P.tpt && wt < ctl->count[win];
      put_nan<D>(a, pool, static_cast<long long>(ctl->seq[win]) * a.bt_sb, kvh, j0 * kNB, min(j1 * kNB, keys),
                 mine ? q8_token_info(a, tok, false).L : 0,
                 a.out + tok * a.o_st + static_cast<long long>(kvh * a.group + row - rt * a.group) * a.o_sh,
                 j1 - j0 == nb ? nullptr
                               : P.part + (2ll * blockIdx.x + (j0 == 0 ? 1 : 0)) * State<D>::kFloats + 4 * (t * kRows + row));
    }
  }
  if (P.split) griddep_wait();  // this grid ends after the split-K kernel
}

// Joins the states of cut windows: one thread per (row, 16 values).  (Joined by the CTA that ends last,
// from TMEM and the other part's state: 2 us slower, on the tail of the launch.)
template <int D>
__global__ void __launch_bounds__(256) q8_merge_kernel(const PrefillParams P) {
  griddep_wait();
  const AttnArgs& a = P.g.a;
  const int cta = blockIdx.x / (D / 16), c = blockIdx.x % (D / 16);
  const int4 cut = P.cuts[cta];
  {
    const int parts = cut.w;
    if (parts == 0) return;
    const int row = threadIdx.x, tile = row / kRows, r = row % kRows;
    const int rt = r / a.group, rh = r - rt * a.group, wt = tile * P.tpt + rt;
    if (rt >= P.tpt || wt >= cut.y) return;
    // Part 0 is the state of the window that the CTA begins, the others those that the following
    // CTAs found begun.
    auto state = [&](int p) { return P.part + (2ll * (cta + p) + (p == 0 ? 1 : 0)) * State<D>::kFloats; };
    float ref = -CUDART_INF_F, l = 0.f;
    for (int p = 0; p < parts; ++p) ref = fmaxf(ref, __ldcg(state(p) + 256 * D + row));
    const float base = ref == -CUDART_INF_F ? 0.f : ref;
    float4 o[4] = {};
    for (int p = 0; p < parts; ++p) {
      const float* s = state(p);
      const float w = ex2(__ldcg(s + 256 * D + row) - base);
      l += w * __ldcg(s + 256 * D + 256 + row);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float4 v = __ldcg(reinterpret_cast<const float4*>(s) + (c * 4 + k) * 256 + row);
        o[k].x += w * v.x; o[k].y += w * v.y; o[k].z += w * v.z; o[k].w += w * v.w;
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint4* dst = reinterpret_cast<uint4*>(a.out + static_cast<long long>(cut.x + wt) * a.o_st +
                                          static_cast<long long>(cut.z * a.group + rh) * a.o_sh + c * 16);
#pragma unroll
    for (int k = 0; k < 2; ++k)
      dst[k] = make_uint4(pack_bf16(o[2 * k].x * inv, o[2 * k].y * inv), pack_bf16(o[2 * k].z * inv, o[2 * k].w * inv),
                          pack_bf16(o[2 * k + 1].x * inv, o[2 * k + 1].y * inv), pack_bf16(o[2 * k + 1].z * inv, o[2 * k + 1].w * inv));
  }
}

int prefill_sms(int device) {
  static std::mutex mu;
  static int cache[64] = {0};
  if (device < 0 || device >= 64) return 148;
  std::lock_guard<std::mutex> lock(mu);
  if (cache[device] == 0 &&
      cudaDeviceGetAttribute(&cache[device], cudaDevAttrMultiProcessorCount, device) != cudaSuccess)
    cache[device] = 148;
  return cache[device];
}

template <int D>
constexpr size_t prefill_smem() {
  return Lay<D>::kOffCtl + sizeof(CtlQ) + 1024;
}
static_assert(prefill_smem<128>() <= 227 * 1024, "shared memory");

template <int D, int FMT>
bool prepare_one(int device) {
  static std::once_flag once[64];
  static bool fine[64];
  std::call_once(once[device], [&] {
    fine[device] = cudaFuncSetAttribute(q8_prefill_kernel<D, FMT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        static_cast<int>(prefill_smem<D>())) == cudaSuccess;
  });
  return fine[device];
}

template <typename... Args>
cudaError_t launch_chained(void (*kernel)(Args...), int grid, int threads, size_t smem,
                           cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace

size_t q8_prefill_workspace(int device) {
  return static_cast<size_t>(prefill_sms(device)) * (2 * State<128>::kFloats * sizeof(float) + sizeof(int4));
}

bool q8_prefill_supported(const Q8AttnArgs& g, int device) {
  if (device < 0 || device >= 64 || !q8_decode_supported(g)) return false;
  // A launch counts its units (up to W / 8 + 1 blocks and kHead per window and KV head) in 31 bits.
  if (g.a.W / (kNB / kPage) + 1 + kHead > INT_MAX / kMaxWin / g.a.KVH) return false;
  const bool i8 = g.p.fmt == SS_CODE_INT8;
  return g.p.D == 128 ? (i8 ? prepare_one<128, SS_CODE_INT8>(device) : prepare_one<128, SS_CODE_E4M3>(device))
                      : (i8 ? prepare_one<64, SS_CODE_INT8>(device) : prepare_one<64, SS_CODE_E4M3>(device));
}

cudaError_t launch_q8_prefill(const Q8AttnArgs& g, long long t0, long long tn, bool split, int device,
                              void* states, cudaStream_t stream) {
  PrefillParams p;
  p.g = g;
  p.split = split;
  p.t0 = static_cast<int>(t0);
  p.tn = static_cast<int>(tn);
  p.tpt = kRows / g.a.group;
  const int grid = prefill_sms(device);
  p.magic = static_cast<unsigned>(((1ull << 32) + 2 * p.tpt - 1) / (2 * p.tpt));
  p.magic_group = static_cast<unsigned>(((1ull << 32) + g.a.group - 1) / g.a.group);
  p.part = static_cast<float*>(states);
  p.cuts = reinterpret_cast<int4*>(p.part + 2ll * grid * State<128>::kFloats);
  const bool i8 = g.p.fmt == SS_CODE_INT8;
  if (g.p.D == 128)
    return i8 ? launch_chained(q8_prefill_kernel<128, SS_CODE_INT8>, grid, kThreads, prefill_smem<128>(), stream, p)
              : launch_chained(q8_prefill_kernel<128, SS_CODE_E4M3>, grid, kThreads, prefill_smem<128>(), stream, p);
  return i8 ? launch_chained(q8_prefill_kernel<64, SS_CODE_INT8>, grid, kThreads, prefill_smem<64>(), stream, p)
            : launch_chained(q8_prefill_kernel<64, SS_CODE_E4M3>, grid, kThreads, prefill_smem<64>(), stream, p);
}

cudaError_t launch_q8_merge(const Q8AttnArgs& g, int device, void* states,
                            cudaStream_t stream) {
  PrefillParams p;
  p.g = g;
  p.t0 = p.tn = p.split = 0;
  p.tpt = kRows / g.a.group;
  p.magic = p.magic_group = 0;
  const int ctas = prefill_sms(device), grid = ctas * (g.p.D / 16);
  p.part = static_cast<float*>(states);
  p.cuts = reinterpret_cast<int4*>(p.part + 2ll * ctas * State<128>::kFloats);
  return g.p.D == 128 ? launch_chained(q8_merge_kernel<128>, grid, 256, 0, stream, p)
                      : launch_chained(q8_merge_kernel<64>, grid, 256, 0, stream, p);
}

int q8_prefill_window() { return kMaxTokP; }

}  // namespace ss
