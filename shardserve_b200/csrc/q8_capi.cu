// C ABI of the 8-bit KV pool and of the block tables (include/shardserve_b200.h): argument
// checks and dispatch.
#include <cuda_runtime.h>

#include <cmath>

#include "q8.cuh"

namespace {

int invalid(const char* what) {
  ss::set_error_message("%s", what);
  return SS_ERR_INVALID;
}
int cuda_failed(cudaError_t e, const char* what) {
  ss::set_error_message("%s: %s", what, cudaGetErrorString(e));
  return SS_ERR_CUDA;
}
bool nonneg(const int64_t* st, int n) {
  for (int i = 0; i < n; ++i)
    if (st[i] < 0) return false;
  return true;
}

// Fills the pool description; returns SS_OK or the error.
int take_pool(ss::Q8Pool* p, const void* k_pool, const int64_t* ks, const void* v_pool,
              const int64_t* vs, int fmt, const float* scales, const int64_t* sst,
              int64_t num_pages, int kv_heads, int head_dim) {
  if (!k_pool || !v_pool || !scales || !ks || !vs || !sst) return invalid("null pointer argument");
  if (fmt != SS_CODE_INT8 && fmt != SS_CODE_E4M3)
    return invalid("code_format must be SS_CODE_INT8 or SS_CODE_E4M3");
  if (head_dim != 64 && head_dim != 128) return invalid("head_dim must be 64 or 128");
  if (kv_heads < 1 || num_pages < 1) return invalid("kv_heads and num_pages must be positive");
  if (num_pages > (1LL << 31) - 1) return invalid("num_pages must be below 2^31");
  if (!nonneg(ks, 4) || !nonneg(vs, 4) || !nonneg(sst, 3))
    return invalid("negative strides are not supported");
  p->k = static_cast<uint8_t*>(const_cast<void*>(k_pool));
  p->k_sn = ks[0]; p->k_ss = ks[1]; p->k_sh = ks[2]; p->k_sd = ks[3];
  p->v = static_cast<uint8_t*>(const_cast<void*>(v_pool));
  p->v_sn = vs[0]; p->v_ss = vs[1]; p->v_sh = vs[2]; p->v_sd = vs[3];
  p->scales = const_cast<float*>(scales);
  p->s_sn = sst[0]; p->s_sh = sst[1]; p->s_sw = sst[2];
  p->N = num_pages;
  p->KVH = kv_heads;
  p->D = head_dim;
  p->fmt = fmt;
  return SS_OK;
}

}  // namespace

extern "C" {

int ss_kv_append_q8(const void* k, const int64_t k_strides[3], const void* v,
                    const int64_t v_strides[3], void* k_pool, const int64_t k_pool_strides[4],
                    void* v_pool, const int64_t v_pool_strides[4], int code_format, float* scales,
                    const int64_t scale_strides[3], const void* slots, int slots_is_int64,
                    int64_t tokens, int64_t num_pages, int kv_heads, int head_dim, void* workspace,
                    void* stream) {
  if (tokens < 0 || tokens > (1LL << 31) - 1) return invalid("tokens must be in [0, 2^31)");
  ss::Q8AppendArgs a;
  const int rc = take_pool(&a.p, k_pool, k_pool_strides, v_pool, v_pool_strides, code_format, scales,
                           scale_strides, num_pages, kv_heads, head_dim);
  if (rc != SS_OK) return rc;
  if (tokens == 0) return SS_OK;
  if (!k || !v || !slots || !k_strides || !v_strides) return invalid("null pointer argument");
  if (!nonneg(k_strides, 3) || !nonneg(v_strides, 3))
    return invalid("negative strides are not supported");
  a.k = static_cast<const __nv_bfloat16*>(k);
  a.k_st = k_strides[0]; a.k_sh = k_strides[1]; a.k_sd = k_strides[2];
  a.v = static_cast<const __nv_bfloat16*>(v);
  a.v_st = v_strides[0]; a.v_sh = v_strides[1]; a.v_sd = v_strides[2];
  a.slots = slots;
  a.slots64 = slots_is_int64 ? 1 : 0;
  a.T = tokens;
  a.err = static_cast<unsigned*>(workspace);
  const cudaError_t e = ss::launch_q8_append(a, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_failed(e, "kv_append_q8 launch");
  ss::count_launches(1);
  return SS_OK;
}

int ss_kv_read_q8(const void* k_pool, const int64_t k_pool_strides[4], const void* v_pool,
                  const int64_t v_pool_strides[4], int code_format, const float* scales,
                  const int64_t scale_strides[3], const void* slots, int slots_is_int64,
                  void* k_out, const int64_t k_out_strides[3], void* v_out,
                  const int64_t v_out_strides[3], int64_t tokens, int64_t num_pages, int kv_heads,
                  int head_dim, void* workspace, void* stream) {
  if (tokens < 0 || tokens > (1LL << 31) - 1) return invalid("tokens must be in [0, 2^31)");
  ss::Q8ReadArgs a;
  const int rc = take_pool(&a.p, k_pool, k_pool_strides, v_pool, v_pool_strides, code_format, scales,
                           scale_strides, num_pages, kv_heads, head_dim);
  if (rc != SS_OK) return rc;
  if (tokens == 0) return SS_OK;
  if (!k_out || !v_out || !slots || !k_out_strides || !v_out_strides)
    return invalid("null pointer argument");
  if (!nonneg(k_out_strides, 3) || !nonneg(v_out_strides, 3))
    return invalid("negative strides are not supported");
  a.k = static_cast<__nv_bfloat16*>(k_out);
  a.k_st = k_out_strides[0]; a.k_sh = k_out_strides[1]; a.k_sd = k_out_strides[2];
  a.v = static_cast<__nv_bfloat16*>(v_out);
  a.v_st = v_out_strides[0]; a.v_sh = v_out_strides[1]; a.v_sd = v_out_strides[2];
  a.slots = slots;
  a.slots64 = slots_is_int64 ? 1 : 0;
  a.T = tokens;
  a.err = static_cast<unsigned*>(workspace);
  const cudaError_t e = ss::launch_q8_read(a, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_failed(e, "kv_read_q8 launch");
  ss::count_launches(1);
  return SS_OK;
}

int ss_q8_workspace_bytes(int device, int heads, int kv_heads, int head_dim, size_t* bytes) {
  if (!bytes) return invalid("null pointer argument");
  if (head_dim != 64 && head_dim != 128) return invalid("head_dim must be 64 or 128");
  if (heads < 1 || kv_heads < 1 || heads % kv_heads)
    return invalid("query heads must be divisible by KV heads");
  *bytes = ss::q8_decode_workspace(device) + ss::q8_prefill_workspace(device);
  return SS_OK;
}

int ss_ragged_paged_attention_q8(
    const void* q, const int64_t q_strides[3], const void* k_pool, const int64_t k_pool_strides[4],
    const void* v_pool, const int64_t v_pool_strides[4], int code_format, const float* scales,
    const int64_t scale_strides[3], const void* block_tables, const int64_t bt_strides[2],
    int64_t bt_rows, int64_t bt_cols, int bt_is_int64, const void* query_seq_ids,
    int seq_ids_is_int64, const void* positions, int positions_is_int64, void* out,
    const int64_t out_strides[3], int64_t tokens, int heads, int kv_heads, int head_dim,
    int64_t num_pages, float sm_scale, void* workspace, size_t workspace_bytes, void* stream) {
  ss::Q8AttnArgs g;
  const int rc = take_pool(&g.p, k_pool, k_pool_strides, v_pool, v_pool_strides, code_format, scales,
                           scale_strides, num_pages, kv_heads, head_dim);
  if (rc != SS_OK) return rc;
  if (tokens < 1) return invalid("ragged batch cannot be empty");
  if (tokens > (1LL << 31) - 1) return invalid("tokens must be below 2^31");
  if (heads < 1 || heads % kv_heads) return invalid("query heads must be divisible by KV heads");
  if (bt_rows < 1 || bt_cols < 1) return invalid("block_tables must be non-empty");
  if (bt_cols > (1LL << 27) - 1) return invalid("block_tables must have fewer than 2^27 columns");
  if (bt_cols > ((1LL << 31) - 1) / kv_heads)  // the kernels count a token's pages of all heads in 31 bits
    return invalid("block_tables columns times kv_heads must be below 2^31");
  if (!q || !block_tables || !query_seq_ids || !positions || !out || !q_strides || !bt_strides ||
      !out_strides)
    return invalid("null pointer argument");
  if (!nonneg(q_strides, 3) || !nonneg(bt_strides, 2) || !nonneg(out_strides, 3))
    return invalid("negative strides are not supported");
  if (!std::isfinite(sm_scale)) return invalid("sm_scale must be finite");
  if (!workspace) {
    ss::set_error_message("a workspace is required");
    return SS_ERR_WORKSPACE;
  }
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return cuda_failed(e, "cudaGetDevice");
  const size_t need = ss::q8_decode_workspace(device) + ss::q8_prefill_workspace(device);
  if (workspace_bytes < need) {
    ss::set_error_message("a workspace of at least %zu bytes is required", need);
    return SS_ERR_WORKSPACE;
  }
  ss::AttnArgs& a = g.a;
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.q_st = q_strides[0]; a.q_sh = q_strides[1]; a.q_sd = q_strides[2];
  a.bt = block_tables;
  a.bt_sb = bt_strides[0]; a.bt_sn = bt_strides[1];
  a.bt64 = bt_is_int64 ? 1 : 0;
  a.seq = query_seq_ids; a.seq64 = seq_ids_is_int64 ? 1 : 0;
  a.pos = positions; a.pos64 = positions_is_int64 ? 1 : 0;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.o_st = out_strides[0]; a.o_sh = out_strides[1]; a.o_sd = out_strides[2];
  a.kp = a.vp = nullptr;
  a.k_sn = a.k_ss = a.k_sh = a.k_sd = a.v_sn = a.v_ss = a.v_sh = a.v_sd = 0;
  a.T = tokens; a.B = bt_rows; a.W = bt_cols; a.N = num_pages;
  a.H = heads; a.KVH = kv_heads; a.D = head_dim; a.group = heads / kv_heads;
  a.sm_scale = sm_scale;
  a.scale_log2 = sm_scale * 1.4426950408889634f;
  a.err = static_cast<unsigned*>(workspace);
  if (ss::q8_decode_supported(g)) {
    // A batch with more tokens than rows holds a prompt chunk.
    const bool tiles = tokens > bt_rows && ss::q8_prefill_supported(g, device);
    void* states = static_cast<uint8_t*>(workspace) + ss::q8_decode_workspace(device);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    // A batch that both kernels list at once runs them side by side; a larger one runs the tiles
    // launch by launch, each with the join of its cut windows, and then the split-K kernel.
    const bool split = tiles && tokens <= ss::kQ8SplitTokens;
    const int64_t per = ss::q8_prefill_window();
    int launches = 0;
    auto rows = [&]() {
      e = ss::launch_q8_decode(g, tiles, split, device, workspace, s, &launches);
      ss::count_launches(static_cast<unsigned>(launches));
      return e == cudaSuccess ? SS_OK : cuda_failed(e, "q8 split-K attention launch");
    };
    if (split && rows() != SS_OK) return SS_ERR_CUDA;
    for (int64_t t0 = 0; tiles && t0 < tokens; t0 += per) {
      e = ss::launch_q8_prefill(g, t0, tokens - t0 < per ? tokens - t0 : per, split, device, states, s);
      if (e == cudaSuccess) e = ss::launch_q8_merge(g, device, states, s);
      if (e != cudaSuccess) return cuda_failed(e, "q8 tile attention launch");
      ss::count_launches(2);
    }
    if (!split && rows() != SS_OK) return SS_ERR_CUDA;
    ss::set_last_path(tiles ? 7 : 5);
    return SS_OK;
  }
  e = ss::launch_q8_generic(g, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_failed(e, "q8 attention launch");
  ss::count_launches(1);
  ss::set_last_path(6);
  return SS_OK;
}

int ss_build_block_tables(const void* cached_lens, int cached_is_int64, const void* new_lens,
                          int new_is_int64, void* block_tables, const int64_t bt_strides[2],
                          int64_t rows, int64_t cols, int bt_is_int64, const void* free_pages,
                          int free_is_int64, int64_t num_free, const int32_t* free_head,
                          int64_t tokens, int32_t* seqs, int64_t* positions, int64_t* slots,
                          int64_t* last, int32_t* lens, int32_t* free_head_out, void* workspace,
                          void* stream) {
  if (rows < 0 || tokens < 0 || num_free < 0) return invalid("negative size");
  if (rows > ss::block_tables_max_rows()) {
    ss::set_error_message("block tables are built for at most %d rows", ss::block_tables_max_rows());
    return SS_ERR_INVALID;
  }
  if (tokens > (1LL << 31) - 1 || num_free > (1LL << 31) - 1)
    return invalid("tokens and num_free must be below 2^31");
  if (rows > 0 && (cols < 1 || cols > (1LL << 27) - 1))
    return invalid("block_tables must have 1 to 2^27 - 1 columns");
  if (!free_head || !free_head_out || !workspace || (num_free > 0 && !free_pages) ||
      (tokens > 0 && (!seqs || !positions || !slots)) ||
      (rows > 0 && (!cached_lens || !new_lens || !block_tables || !bt_strides || !last || !lens)))
    return invalid("null pointer argument");
  if (rows > 0 && !nonneg(bt_strides, 2)) return invalid("negative strides are not supported");
  ss::BlockTablesArgs a;
  a.cached = cached_lens; a.cached64 = cached_is_int64 ? 1 : 0;
  a.fresh = new_lens; a.fresh64 = new_is_int64 ? 1 : 0;
  a.B = rows;
  a.tables = block_tables;
  a.t_sb = rows > 0 ? bt_strides[0] : 0;
  a.t_sn = rows > 0 ? bt_strides[1] : 0;
  a.W = rows > 0 ? cols : 1;
  a.tables64 = bt_is_int64 ? 1 : 0;
  a.free_pages = free_pages; a.free64 = free_is_int64 ? 1 : 0;
  a.F = num_free;
  a.head = free_head;
  a.head_out = free_head_out;
  a.T = tokens;
  a.seqs = seqs;
  a.positions = reinterpret_cast<long long*>(positions);
  a.slots = reinterpret_cast<long long*>(slots);
  a.last = reinterpret_cast<long long*>(last);
  a.lens = lens;
  a.err = static_cast<unsigned*>(workspace);
  a.ticket = static_cast<unsigned*>(workspace) + 20;
  const cudaError_t e = ss::launch_block_tables(a, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_failed(e, "build_block_tables launch");
  ss::count_launches(1);
  return SS_OK;
}

}  // extern "C"
