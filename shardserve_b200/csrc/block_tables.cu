// Block tables and slot maps of a step, built from request lengths alone.
//
// Row r holds c_r cached tokens and gets n_r new ones.  With have_r = ceil(c_r / 16) and
// want_r = ceil((c_r + n_r) / 16), row r takes want_r - have_r pages from the free list, in row
// order:
//     tables[r, j] = free[head + sum_{i < r}(want_i - have_i) + j - have_r]   have_r <= j < want_r
// and its new tokens stand at offset sum_{i < r} n_i of the step's flat batch:
//     seqs = r, positions = c_r + j, slots = tables[r, position / 16] * 16 + position % 16
//
// Every CTA scans all rows (two 64-bit prefix sums, 4 bytes a row read from L2) into shared
// memory and then takes its share of the table entries, rows and tokens, found by binary search;
// no CTA reads what another one writes (a new token's page comes from the free list itself where
// the call takes it).  The new lengths and the new head may be written over the old ones, so the
// CTA that arrives last at a counter writes them.  Latency bound: one pass over a few KB.  64 rows take
// 4.0 us on the GPU, 1000 decode rows with 24 chunks of 512 tokens 9.8; a call from Python takes the
// host about 11 us (six output tensors), which is what a loop of calls runs at.
#include <cuda_runtime.h>

#include <algorithm>

#include "ptx.cuh"
#include "q8.cuh"

namespace ss {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxRows = 12288;

struct RowSpan {
  long long cached, fresh, have, want;
  bool bad;
};

__device__ __forceinline__ RowSpan row_span(const BlockTablesArgs& a, long long r) {
  RowSpan s;
  s.cached = ld_index(a.cached, a.cached64, r);
  s.fresh = ld_index(a.fresh, a.fresh64, r);
  s.bad = s.cached < 0 || s.fresh < 0;
  // (At most 2^62 and 2^40, either past any table, so that no sum of them overflows 64 bits.)
  s.cached = min(max(s.cached, 0ll), 1ll << 62);
  s.fresh = min(max(s.fresh, 0ll), 1ll << 40);
  const long long room = a.W * kPage;
  s.bad |= s.cached > room || s.fresh > room - s.cached;
  // A row past its table keeps its tokens' places in the batch; they get no slot.
  s.have = (min(s.cached, room) + kPage - 1) / kPage;
  s.want = min((min(s.cached, room) + min(s.fresh, room) + kPage - 1) / kPage, a.W);
  return s;
}

__device__ __forceinline__ void put_index(void* p, int is64, long long i, long long v) {
  if (is64)
    static_cast<long long*>(p)[i] = v;
  else
    static_cast<int*>(p)[i] = static_cast<int>(v);
}

// Largest r with off[r] <= x, for off[0] = 0 <= x < off[n].
__device__ __forceinline__ int find_row(const int* off, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (off[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kThreads) block_tables_kernel(const BlockTablesArgs a) {
  extern __shared__ int smem[];
  const int B = static_cast<int>(a.B), tid = threadIdx.x;
  int* tok = smem;          // [B + 1] first token of each row
  int* pag = smem + B + 1;  // [B + 1] first taken page of each row
  __shared__ long long red[2][kWarps];
  __shared__ int is_last;
  const int per = (B + kThreads - 1) / kThreads;
  const int r0 = min(tid * per, B), r1 = min(r0 + per, B);
  long long st = 0, sp = 0;
  unsigned e = 0;
  for (int r = r0; r < r1; ++r) {
    const RowSpan s = row_span(a, r);
    st += s.fresh;
    sp += s.want - s.have;
    if (s.bad) e |= SS_DEVERR_POS;
  }
  const int w = tid >> 5, lane = tid & 31;
  long long it = st, ip = sp;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, it, o), y = __shfl_up_sync(0xffffffffu, ip, o);
    if (lane >= o) {
      it += x;
      ip += y;
    }
  }
  if (lane == 31) {
    red[0][w] = it;
    red[1][w] = ip;
  }
  __syncthreads();
  long long bt = 0, bp = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    if (i < w) {
      bt += red[0][i];
      bp += red[1][i];
    }
  }
  long long t = bt + it - st, p = bp + ip - sp;
  for (int r = r0; r < r1; ++r) {
    const RowSpan s = row_span(a, r);
    tok[r] = static_cast<int>(min(t, a.T));
    pag[r] = static_cast<int>(min(p, 0x7fffffffll));
    t += s.fresh;
    p += s.want - s.have;
  }
  if (B == 0 ? tid == 0 : (r1 == B && r0 < r1)) {
    tok[B] = static_cast<int>(min(t, a.T));
    pag[B] = static_cast<int>(min(p, 0x7fffffffll));
    if (t > a.T) e |= SS_DEVERR_POS;  // more new tokens than the batch holds
  }
  const long long head = max(*a.head, 0);
  __syncthreads();
  const int taken = pag[B], placed = tok[B];
  if (tid == 0 && blockIdx.x == 0 && head + taken > a.F) e |= SS_DEVERR_PAGE;
  auto free_page = [&](long long k) -> long long {
    return k < a.F ? ld_index(a.free_pages, a.free64, k) : -1;
  };
  const long long gid = static_cast<long long>(blockIdx.x) * kThreads + tid;
  const long long step = static_cast<long long>(gridDim.x) * kThreads;
  for (long long i = gid; i < a.T; i += step) {
    if (i >= placed) {  // padding
      a.seqs[i] = -1;
      a.positions[i] = -1;
      a.slots[i] = -1;
      continue;
    }
    const int r = find_row(tok, B, static_cast<int>(i));
    const RowSpan s = row_span(a, r);
    const long long pos = s.cached + (i - tok[r]), col = pos / kPage;
    long long page = -1;
    if (col < s.have)
      page = ld_index(a.tables, a.tables64, r * a.t_sb + col * a.t_sn);
    else if (col < s.want)
      page = free_page(head + pag[r] + col - s.have);
    a.seqs[i] = r;
    a.positions[i] = pos;
    a.slots[i] = page >= 0 ? page * kPage + pos % kPage : -1;
  }
  for (long long i = gid; i < taken; i += step) {
    const int r = find_row(pag, B, static_cast<int>(i));
    const RowSpan s = row_span(a, r);
    put_index(a.tables, a.tables64, r * a.t_sb + (s.have + i - pag[r]) * a.t_sn, free_page(head + i));
  }
  for (long long r = gid; r < B; r += step) a.last[r] = tok[r + 1] > tok[r] ? tok[r + 1] - 1 : -1;
  if (e && blockIdx.x == 0) atomicOr(a.err, e);
  if (gridDim.x > 1) {
    __syncthreads();
    if (tid == 0) is_last = atom_add_acq_rel_gpu_u32(a.ticket, 1u) == gridDim.x - 1;
    __syncthreads();
    if (!is_last) return;
    if (tid == 0) *a.ticket = 0;
  } else {
    __syncthreads();
  }
  for (int r = tid; r < B; r += kThreads) {
    const RowSpan s = row_span(a, r);
    a.lens[r] = static_cast<int>(min(s.cached + s.fresh, 0x7fffffffll));
  }
  if (tid == 0) *a.head_out = static_cast<int>(min(head + taken, max(head, a.F)));
}

}  // namespace

int block_tables_max_rows() { return kMaxRows; }

cudaError_t launch_block_tables(const BlockTablesArgs& a, cudaStream_t stream) {
  const size_t smem = 2 * (static_cast<size_t>(a.B) + 1) * sizeof(int);
  if (smem > 47 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(block_tables_kernel,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>(2 * (kMaxRows + 1) * sizeof(int)));
    if (e != cudaSuccess) return e;
  }
  // About four entries a thread; one CTA needs no counter.
  const long long items = a.T + 2 * a.B;
  const unsigned grid = static_cast<unsigned>(std::min<long long>(std::max<long long>(items / (4 * kThreads), 1), 148));
  block_tables_kernel<<<grid, kThreads, smem, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace ss
