// 8-bit paged KV pool: shared declarations of the quantising append, the read-back and the
// attention kernels.
//
// A pool holds codes [pages, 16, kv_heads, head_dim], one byte each, for K and for V, and fp32
// scales [pages, kv_heads, 2] (K, V): code c of a page and head stands for c * scale.  Codes are
// signed 8-bit integers in [-127, 127] (SS_CODE_INT8) or e4m3 numbers (SS_CODE_E4M3, largest
// 448).  Scales are finite and >= 0.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "attention.cuh"

namespace ss {

// A pool and the scales of its pages; strides in elements (bytes for the codes).
struct Q8Pool {
  uint8_t* k;
  long long k_sn, k_ss, k_sh, k_sd;
  uint8_t* v;
  long long v_sn, v_ss, v_sh, v_sd;
  float* scales;
  long long s_sn, s_sh, s_sw;
  long long N;  // pages
  int KVH, D;
  int fmt;  // SS_CODE_*
};

struct Q8AttnArgs {
  AttnArgs a;  // queries, tables, output (its pool pointers are unused)
  Q8Pool p;
};

struct Q8AppendArgs {
  Q8Pool p;
  const __nv_bfloat16* k;
  long long k_st, k_sh, k_sd;
  const __nv_bfloat16* v;
  long long v_st, v_sh, v_sd;
  const void* slots;
  int slots64;
  long long T;
  unsigned* err;  // may be null
};

struct Q8ReadArgs {
  Q8Pool p;
  __nv_bfloat16* k;
  long long k_st, k_sh, k_sd;
  __nv_bfloat16* v;
  long long v_st, v_sh, v_sd;
  const void* slots;
  int slots64;
  long long T;
  unsigned* err;  // may be null
};

struct BlockTablesArgs {
  const void* cached;
  int cached64;
  const void* fresh;  // new tokens of each row
  int fresh64;
  long long B;  // rows
  void* tables;
  long long t_sb, t_sn, W;
  int tables64;
  const void* free_pages;
  int free64;
  long long F;  // entries of the free list
  const int* head;
  int* head_out;
  long long T;
  int* seqs;
  long long* positions;
  long long* slots;
  long long* last;
  int* lens;
  unsigned* err;     // workspace word 0
  unsigned* ticket;  // workspace word 20: zero between calls
};

// Largest magnitude a code stands for before its scale.
__host__ __device__ constexpr float q8_max(int fmt) { return fmt == SS_CODE_INT8 ? 127.f : 448.f; }
// Blocks whose scale would fall below this hold zeros: 1 / scale stays finite, and no bf16 value
// of a model is that small.
constexpr float kQ8Tiny = 0x1p-100f;

__device__ __forceinline__ float q8_decode(int fmt, uint8_t c) {
  if (fmt == SS_CODE_INT8) return static_cast<float>(static_cast<int8_t>(c));
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}
// Nearest code, ties to even; values past the largest code (infinities among them) saturate.
// NaN becomes 0 as an integer code and stays NaN as an e4m3 code.
__device__ __forceinline__ uint8_t q8_encode(int fmt, float x) {
  if (fmt == SS_CODE_INT8) {
    const float r = rintf(x);
    return static_cast<uint8_t>(static_cast<int8_t>(
        static_cast<int>(r != r ? 0.f : fminf(fmaxf(r, -127.f), 127.f))));
  }
  return static_cast<uint8_t>(__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3));
}

// As token_info, but sequence id -1 marks a padding token: no keys, and no error bit.
__device__ __forceinline__ TokInfo q8_token_info(const AttnArgs& a, long long t, bool report) {
  const long long seq = ld_index(a.seq, a.seq64, t);
  if (seq == -1) return TokInfo{-1, 0, 0};
  return token_info_from(a, seq, ld_index(a.pos, a.pos64, t), report);
}

// Tokens t0 .. t0 + tn - 1 into shared memory: seq[i] (32 bits of the id; kQ8MinRun - 1 neighbours
// on either side too) and len[i] (keys).  Both attention kernels tell runs from these.
constexpr int kQ8MinRun = 8;   // tokens of shorter runs belong to the split-K kernel
constexpr int kQ8Pad = kQ8MinRun - 1;
__device__ __forceinline__ void stage_tokens(const AttnArgs& a, long long t0, int tn, int* seq,
                                             int* len, bool report) {
  // The neighbours first: their loads are in flight with the others.  Past the batch's ends stands
  // anything but the id of the token at the end.
  int at = 0, neighbour = 0;
  if (threadIdx.x < 2 * kQ8Pad) {
    const int k = threadIdx.x;
    at = k < kQ8Pad ? -1 - k : tn + k - kQ8Pad;
    const long long t = t0 + at, in = t < 0 ? 0 : min(t, a.T - 1);
    const int id = static_cast<int>(ld_index(a.seq, a.seq64, in));
    neighbour = in == t ? id : ~id;
  }
  auto put = [&](int i, long long s, long long p) {
    seq[i] = static_cast<int>(s);
    len[i] = s == -1 ? 0 : token_info_from(a, s, p, report).L;
  };
  if (tn <= static_cast<int>(blockDim.x)) {
    const int i = threadIdx.x;
    if (i < tn) put(i, ld_index(a.seq, a.seq64, t0 + i), ld_index(a.pos, a.pos64, t0 + i));
  } else {
    constexpr int U = 8;  // loads in flight: every one is a round trip to L2 or beyond
    for (int i0 = threadIdx.x; i0 < tn; i0 += U * blockDim.x) {
      long long s[U], p[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = min(i0 + u * static_cast<int>(blockDim.x), tn - 1);
        s[u] = ld_index(a.seq, a.seq64, t0 + i);
        p[u] = ld_index(a.pos, a.pos64, t0 + i);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * static_cast<int>(blockDim.x);
        if (i < tn) put(i, s[u], p[u]);
      }
    }
  }
  if (threadIdx.x < 2 * kQ8Pad) seq[at] = neighbour;
}
// Token i of staged ids lies in a run of at least kQ8MinRun tokens of one sequence.
__device__ __forceinline__ bool in_staged_run(const int* seq, int i) {
  const int s = seq[i];
  int n = 1;
#pragma unroll
  for (int k = 1, on = 1; k <= kQ8Pad; ++k) n += (on = on && seq[i - k] == s);
#pragma unroll
  for (int k = 1, on = 1; k <= kQ8Pad; ++k) n += (on = on && seq[i + k] == s);
  return n >= kQ8MinRun;
}

// CTAs of `all` that the split-K kernel takes beside the tiles, by the work of the two: the keys that
// tokens outside runs attend cost it `7.7` units each, the tiles `0.9` per key and run token (ns per
// SM and KV head, both measured alone at 8 query heads per KV head of 128, int8).  Other groups,
// head_dim 64 and e4m3 use the same two numbers, unmeasured: a wrong share only makes one side end after
// the other.  Both kernels compute it from the same sums, of lengths clamped so that they fit 31 bits.
constexpr int kQ8SplitTokens = 6144;  // both kernels list a call of up to so many tokens at once
__host__ __device__ __forceinline__ int q8_clamped(int len) { return len < 262143 ? len : 262143; }
__device__ __forceinline__ int q8_split(int rows_keys, int run_keys, int all) {
  if (rows_keys == 0) return 0;
  if (run_keys == 0) return all;
  const float a = 7.7f * static_cast<float>(rows_keys), b = 0.9f * static_cast<float>(run_keys);
  return min(max(__float2int_rn(static_cast<float>(all) * a / (a + b)), 4), all - 4);
}

cudaError_t launch_q8_append(const Q8AppendArgs& a, cudaStream_t stream);
cudaError_t launch_q8_read(const Q8ReadArgs& a, cudaStream_t stream);
cudaError_t launch_q8_generic(const Q8AttnArgs& a, cudaStream_t stream);
// Split-K kernel (q8_decode.cu): workspace bytes, the layouts it addresses, and the launch
// (*launches: kernels enqueued).  skip_runs: tokens of runs belong to the tiles; split: the tiles come
// right after and take the SMs that q8_split leaves them.
size_t q8_decode_workspace(int device);
bool q8_decode_supported(const Q8AttnArgs& g);
cudaError_t launch_q8_decode(const Q8AttnArgs& g, bool skip_runs, bool split, int device,
                             void* workspace, cudaStream_t stream, int* launches);
// tcgen05 tiles of prompt chunks (q8_prefill.cu), for runs of at least kQ8MinRun tokens: workspace
// bytes of the cut windows' states, the layouts it takes, tokens per launch, and the launches of
// the tiles and of the join of the cut windows.
size_t q8_prefill_workspace(int device);
bool q8_prefill_supported(const Q8AttnArgs& g, int device);
int q8_prefill_window();
cudaError_t launch_q8_prefill(const Q8AttnArgs& g, long long t0, long long tn, bool split, int device,
                              void* states, cudaStream_t stream);
cudaError_t launch_q8_merge(const Q8AttnArgs& g, int device, void* states, cudaStream_t stream);
cudaError_t launch_block_tables(const BlockTablesArgs& a, cudaStream_t stream);
int block_tables_max_rows();

// Bookkeeping of the C-ABI layer (capi.cu).
void count_launches(unsigned n);
void set_last_path(int path);

}  // namespace ss
