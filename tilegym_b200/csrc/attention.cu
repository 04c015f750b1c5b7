// Attention over the paged e4m3 key / value cache.
//
//   o_i = sum_j softmax_j(scale * q_i . k_j) v_j,  j <= pos_i  and  (j > pos_i - window  or  j < sinks)
//
// The C entry point: checks, tensor maps of the pages, and the choice between the kernel for few rows of a (sequence, cache
// head), where reading the cache is the work, and the one for many, where the products are.
#include <cstdio>

#include "tg_attention.cuh"

using namespace tg;

// Rows of a unit in the kernel for few rows, 0 where the batch has too many for it.
static int few_rows_of(int64_t q_heads, int64_t kv_heads, int32_t max_q_len) {
  if (q_heads < 1 || kv_heads < 1 || max_q_len < 1) return 0;
  const int64_t rows = q_heads / kv_heads * max_q_len;
  return rows <= kFewRowsMax ? few_rows_padded(static_cast<int>(rows)) : 0;
}

extern "C" TG_API uint64_t tg_paged_attention_workspace_bytes(int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                                              int32_t max_q_len, int64_t tokens, int64_t seqs, int64_t pages_per_seq,
                                                              int32_t num_sms) {
  if (q_heads < 1 || kv_heads < 1 || q_heads % kv_heads != 0 || q_heads / kv_heads > 64 || max_q_len < 1) return 0;
  const int rows = few_rows_of(q_heads, kv_heads, max_q_len);
  const int dim = head_dim == 64 ? 64 : 128;
  if (rows == 0) {
    if (tokens < 1 || seqs < 1 || tokens > (1 << 28) || seqs > (1 << 20)) return 0;
    const int group = static_cast<int>(q_heads / kv_heads);
    return many_rows_workspace(dim, many_rows_tiles(tokens, seqs, group) * kv_heads, many_rows_splits(tokens, seqs, kv_heads, group, pages_per_seq, num_sms));
  }
  // the larger of the two types' block counts
  return few_rows_workspace(dim, rows, few_rows_blocks(dim, rows, true, num_sms));
}

extern "C" TG_API int32_t tg_paged_attention(const TgTensorDesc* O, const TgTensorDesc* Q, const TgTensorDesc* Kc, const TgTensorDesc* Vc,
                                             const TgTensorDesc* Ks, const TgTensorDesc* Vs, const TgTensorDesc* block_table,
                                             const TgTensorDesc* seq_lens, const TgTensorDesc* cu_seqlens, int32_t max_q_len, float scale,
                                             int32_t window, int32_t sinks, uint64_t workspace, uint64_t workspace_bytes, int32_t device_id,
                                             uint64_t stream) {
  AttentionParams p = {};
  int32_t rc;
  if ((rc = check_cache(&p.c, Kc, Vc, Ks, Vs, block_table, seq_lens, cu_seqlens)) != TG_OK) return rc;
  if (Q == nullptr || O == nullptr) return api_fail(TG_ERR_NULL, "q or output descriptor is null");
  if (!is_16bit(Q->dtype)) return api_fail(TG_ERR_DTYPE, "q must be bf16 or f16");
  if (Q->ndim != 3) return api_fail(TG_ERR_ARGS, "q must be [tokens, heads, head_dim]");
  const int64_t T = Q->shape[0], heads = Q->shape[1], D = p.c.dim;
  if (T > (1 << 28)) return api_fail(TG_ERR_ARGS, "too many tokens");
  if (cu_seqlens == nullptr && T != p.c.seqs) return api_fail(TG_ERR_ARGS, "without cu_seqlens there is one new token per sequence");
  if (heads < 1 || heads % p.c.heads != 0 || heads / p.c.heads > 64)
    return api_fail(TG_ERR_ARGS, "the query heads must be a multiple of the cache's heads, at most 64 times as many");
  if ((rc = check_heads(Q, "q: [tokens, heads, head_dim of the cache], 16-byte aligned", T, heads, D, Q->dtype)) != TG_OK) return rc;
  if ((rc = check_heads_out(O, "output: shape and type of q, 16-byte aligned", T, heads, D, Q->dtype)) != TG_OK) return rc;
  if ((rc = check_heads_place(O, Q)) != TG_OK) return rc;
  if (max_q_len < 1) return api_fail(TG_ERR_ARGS, "max_q_len must be at least 1");
  if (window < 0 || sinks < 0) return api_fail(TG_ERR_ARGS, "window and sinks must not be negative");
  if (sinks > 0 && window == 0) return api_fail(TG_ERR_ARGS, "sinks only mean something under a window");
  if (!(scale > 0.f) || scale > 3.0e38f) return api_fail(TG_ERR_ARGS, "scale must be positive and finite");
  if (T == 0 || p.c.seqs == 0) return TG_OK;
  if (p.c.pages < 1) return api_fail(TG_ERR_ARGS, "the cache has no page");
  ScopedDevice guard(device_id);
  if (guard.err != cudaSuccess) {
    cudaGetLastError();
    return api_fail(TG_ERR_DEVICE, "cannot select the CUDA device");
  }
  int num_sms = 0;
  int32_t* status = nullptr;
  if ((rc = api_init_device(device_id, &num_sms, &status)) != TG_OK) return rc;
  p.q = reinterpret_cast<const void*>(Q->ptr);
  p.o = reinterpret_cast<void*>(O->ptr);
  p.q_tok = Q->strides[0];
  p.q_head = Q->strides[1];
  p.o_tok = O->strides[0];
  p.o_head = O->strides[1];
  p.tokens = static_cast<int32_t>(T);
  p.q_heads = static_cast<int32_t>(heads);
  p.group = static_cast<int32_t>(heads / p.c.heads);
  p.scale = scale;
  p.window = window;
  p.sinks = sinks;
  p.max_q_len = max_q_len;
  p.status = status;
  p.wait_limit_us = api_wait_limit_us();
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  CUtensorMap tmK, tmV;
  const int64_t page_heads = static_cast<int64_t>(p.c.pages) * p.c.heads;
  if ((rc = api_make_page_map(&tmK, Kc->ptr, page_heads * kPage, p.c.dim, kPage)) != TG_OK) return rc;
  if ((rc = api_make_page_map(&tmV, Vc->ptr, page_heads * p.c.dim, kPage, p.c.dim)) != TG_OK) return rc;
  if (const int rows = few_rows_of(heads, p.c.heads, max_q_len); rows > 0) {
    const int blocks = few_rows_blocks(p.c.dim, rows, Q->dtype == TG_BF16, num_sms);
    if (workspace == 0) return api_fail(TG_ERR_NULL, "the workspace is null");
    if (workspace & 15u) return api_fail(TG_ERR_ALIGN, "the workspace must be 16-byte aligned");
    if (workspace_bytes < few_rows_workspace(p.c.dim, rows, blocks)) return api_fail(TG_ERR_ARGS, "the workspace is too small");
    const uint64_t parts = 2ull * blocks * rows;
    p.part_o = reinterpret_cast<float*>(workspace);
    p.part_ml = reinterpret_cast<float2*>(workspace + parts * p.c.dim * 4);
    p.record = reinterpret_cast<int4*>(workspace + parts * p.c.dim * 4 + parts * 8);
    const cudaError_t e = launch_attention_few_rows(tmK, tmV, p, rows, blocks, Q->dtype == TG_BF16, st);
    if (e == cudaSuccess) return TG_OK;
    char msg[160];
    snprintf(msg, sizeof(msg), "paged_attention launch failed: %s", cudaGetErrorString(e));
    return api_fail(TG_ERR_LAUNCH, msg);
  }
  p.splits = many_rows_splits(T, p.c.seqs, p.c.heads, p.group, p.c.max_pages, num_sms);
  if (p.splits > 1) {
    const int64_t blocks = many_rows_tiles(T, p.c.seqs, p.group) * p.c.heads;
    if (workspace == 0) return api_fail(TG_ERR_NULL, "the workspace is null");
    if (workspace & 15u) return api_fail(TG_ERR_ALIGN, "the workspace must be 16-byte aligned");
    if (workspace_bytes < many_rows_workspace(p.c.dim, blocks, p.splits)) return api_fail(TG_ERR_ARGS, "the workspace is too small");
    p.part_o = reinterpret_cast<float*>(workspace);
    p.part_ml = reinterpret_cast<float2*>(workspace + 256ull * blocks * p.splits * p.c.dim * 4);
  }
  const cudaError_t e = launch_attention_many_rows(tmK, tmV, p, Q->dtype == TG_BF16, st);
  if (e != cudaSuccess) {
    char msg[160];
    snprintf(msg, sizeof(msg), "paged_attention launch failed: %s", cudaGetErrorString(e));
    return api_fail(TG_ERR_LAUNCH, msg);
  }
  return TG_OK;
}
