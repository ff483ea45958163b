// Record forms of the entry points an eager program calls most
// (include/litelang_amd.h, "record calls"): host code only.
#include "ll_common.h"

namespace {
template <typename T> T* ptr(int64_t v) { return (T*)(uintptr_t)v; }
}  // namespace

extern "C" int64_t ll_call_rmsnorm(const LLRmsnormCall* c) {
  LL_CHECK_ARG(c, "ll_call_rmsnorm: null record");
  return ll_rmsnorm(ptr<void>(c->x), c->x_row_stride, ptr<const void>(c->residual),
                    c->residual_row_stride, ptr<const void>(c->gamma), ptr<void>(c->out),
                    c->out_row_stride, c->M, c->N, (float)c->eps, (int)c->dtype,
                    ptr<ihipStream_t>(c->stream));
}

extern "C" int64_t ll_call_decode_attention(const LLDecodeAttentionCall* c) {
  LL_CHECK_ARG(c, "ll_call_decode_attention: null record");
  // (shapes the entry point refuses go to it for its error)
  if (c->batch > 0 && c->kv_heads > 0 && c->head_dim > 0 && c->max_len_in_batch >= 0) {
    const int64_t need = ll_decode_attention_workspace_size(c->batch, c->q_heads, c->kv_heads,
                                                            c->head_dim, c->max_len_in_batch);
    if (need > c->workspace_bytes) return need;
  }
  return ll_decode_attention(
      ptr<const void>(c->q), c->q_stride_b, c->q_stride_h, ptr<const void>(c->k_cache),
      c->k_stride_tok, c->k_stride_head, ptr<const void>(c->v_cache), c->v_stride_tok,
      c->v_stride_head, ptr<const int32_t>(c->req_to_tokens), c->req_to_tokens_stride,
      ptr<const void>(c->b_req_idx), (int)c->req_idx_i64, ptr<const void>(c->b_seq_len),
      (int)c->seq_len_i64, ptr<void>(c->out), c->out_stride_b, c->out_stride_h, c->batch,
      c->q_heads, c->kv_heads, c->head_dim, c->max_len_in_batch, (float)c->sm_scale, (int)c->dtype,
      ptr<void>(c->workspace), c->workspace_bytes, ptr<ihipStream_t>(c->stream));
}

extern "C" int64_t ll_call_prefill_attention(const LLPrefillAttentionCall* c) {
  LL_CHECK_ARG(c, "ll_call_prefill_attention: null record");
  return ll_prefill_attention(
      ptr<const void>(c->q), c->q_stride_tok, c->q_stride_h, ptr<const void>(c->k_cache),
      c->k_stride_tok, c->k_stride_head, ptr<const void>(c->v_cache), c->v_stride_tok,
      c->v_stride_head, ptr<void>(c->out), c->out_stride_tok, c->out_stride_h,
      ptr<const int32_t>(c->req_to_tokens), c->req_to_tokens_stride, ptr<const void>(c->b_req_idx),
      (int)c->req_idx_i64, ptr<const void>(c->b_start_loc), (int)c->start_loc_i64,
      ptr<const void>(c->b_seq_len), (int)c->seq_len_i64, ptr<const void>(c->b_shared_seq_len),
      (int)c->shared_i64, c->batch, c->q_heads, c->kv_heads, c->head_dim, c->max_input_len,
      (float)c->sm_scale, (int)c->dtype, ptr<ihipStream_t>(c->stream));
}

extern "C" int64_t ll_call_gemm(const LLGemmCall* c) {
  LL_CHECK_ARG(c, "ll_call_gemm: null record");
  int64_t need = 0;
  if (c->M > 64) {
    if (!c->any_workspace && c->dtype != LL_F32)
      need = ll_gemm_tiles_workspace_size(c->M, c->N, c->K, 2);
  } else if (c->M > 0 && c->N > 0 && c->K > 0) {
    need = ll_gemm_workspace_size(c->M, c->N, c->K);
  }
  if (need > c->workspace_bytes) return need;
  return ll_gemm(ptr<const void>(c->X), c->ldx, ptr<const void>(c->W), c->ldw,
                 ptr<const void>(c->bias), ptr<void>(c->Y), c->ldy, c->M, c->N, c->K,
                 (int)c->dtype, ptr<void>(c->workspace), c->workspace_bytes,
                 ptr<ihipStream_t>(c->stream));
}

extern "C" int64_t ll_call_window_prefill_attention(const LLWindowPrefillAttentionCall* c) {
  LL_CHECK_ARG(c, "ll_call_window_prefill_attention: null record");
  return ll_window_prefill_attention(
      ptr<const void>(c->q), c->q_stride_tok, c->q_stride_h, ptr<const void>(c->k_cache),
      c->k_stride_tok, c->k_stride_head, ptr<const void>(c->v_cache), c->v_stride_tok,
      c->v_stride_head, ptr<void>(c->out), c->out_stride_tok, c->out_stride_h,
      ptr<const int32_t>(c->req_to_tokens), c->req_to_tokens_stride, ptr<const void>(c->b_req_idx),
      (int)c->req_idx_i64, ptr<const void>(c->b_start_loc), (int)c->start_loc_i64,
      ptr<const void>(c->b_seq_len), (int)c->seq_len_i64, ptr<const void>(c->b_shared_seq_len),
      (int)c->shared_i64, c->batch, c->q_heads, c->kv_heads, c->head_dim, c->max_input_len,
      c->window, c->sinks, (float)c->sm_scale, (int)c->dtype, ptr<ihipStream_t>(c->stream));
}

extern "C" int64_t ll_call_window_decode_attention(const LLWindowDecodeAttentionCall* c) {
  LL_CHECK_ARG(c, "ll_call_window_decode_attention: null record");
  const int64_t need = ll_window_decode_attention_workspace_size(
      c->batch, c->q_heads, c->kv_heads, c->head_dim, c->max_len_in_batch, c->window, c->sinks);
  if (need > c->workspace_bytes) return need;
  return ll_window_decode_attention(
      ptr<const void>(c->q), c->q_stride_b, c->q_stride_h, ptr<const void>(c->k_cache),
      c->k_stride_tok, c->k_stride_head, ptr<const void>(c->v_cache), c->v_stride_tok,
      c->v_stride_head, ptr<const int32_t>(c->req_to_tokens), c->req_to_tokens_stride,
      ptr<const void>(c->b_req_idx), (int)c->req_idx_i64, ptr<const void>(c->b_seq_len),
      (int)c->seq_len_i64, ptr<void>(c->out), c->out_stride_b, c->out_stride_h, c->batch,
      c->q_heads, c->kv_heads, c->head_dim, c->max_len_in_batch, c->window, c->sinks,
      (float)c->sm_scale, (int)c->dtype, ptr<void>(c->workspace), c->workspace_bytes,
      ptr<ihipStream_t>(c->stream));
}

extern "C" int64_t ll_call_rope_positions(const LLRopePositionsCall* c) {
  LL_CHECK_ARG(c, "ll_call_rope_positions: null record");
  return ll_rope_positions(
      ptr<const void>(c->q), c->q_stride_tok, c->q_stride_h, ptr<void>(c->q_out),
      c->q_out_stride_tok, c->q_out_stride_h, c->q_heads, ptr<const void>(c->k), c->k_stride_tok,
      c->k_stride_h, ptr<void>(c->k_out), c->k_out_stride_tok, c->k_out_stride_h, c->k_heads,
      ptr<const void>(c->positions), (int)c->positions_i64, ptr<const float>(c->inv_freq),
      c->rotary_dim, (int)c->interleaved, (float)c->factor, c->ntok, c->head_dim, (int)c->dtype,
      ptr<ihipStream_t>(c->stream));
}

extern "C" int64_t ll_call_qk_norm_rope_kv_scatter(const LLQkNormRopeKvScatterCall* c) {
  LL_CHECK_ARG(c, "ll_call_qk_norm_rope_kv_scatter: null record");
  return ll_qk_norm_rope_kv_scatter(
      ptr<const void>(c->qkv), c->qkv_row_stride, c->ntok, c->q_heads, c->kv_heads, c->head_dim,
      ptr<void>(c->q_out), c->q_out_stride_tok, c->q_out_stride_h, ptr<const void>(c->q_gamma),
      ptr<const void>(c->k_gamma), (float)c->eps, ptr<const void>(c->positions),
      (int)c->positions_i64, ptr<const float>(c->inv_freq), c->rotary_dim, (int)c->interleaved,
      (float)c->factor, ptr<const int32_t>(c->slots), ptr<void>(c->pool_layer),
      c->pool_slot_stride, c->pool_head_stride, c->pool_slots, (int)c->dtype,
      ptr<ihipStream_t>(c->stream));
}

extern "C" int64_t ll_call_build_slot_maps(const LLBuildSlotMapsCall* c) {
  LL_CHECK_ARG(c, "ll_call_build_slot_maps: null record");
  return ll_build_slot_maps(
      ptr<const void>(c->b_req_idx), (int)c->req_idx_i64, ptr<const void>(c->b_seq_len),
      (int)c->seq_len_i64, ptr<const void>(c->b_cached_len), (int)c->cached_len_i64, c->batch,
      ptr<const int32_t>(c->free_pages), c->n_free, c->page_size, ptr<int32_t>(c->block_table),
      c->block_table_stride, c->block_table_cols, ptr<int32_t>(c->req_to_tokens),
      c->req_to_tokens_stride, c->req_rows, c->max_len, ptr<int32_t>(c->slots),
      ptr<int32_t>(c->positions), c->max_tokens, ptr<int32_t>(c->b_start_loc),
      ptr<int32_t>(c->last_rows), ptr<int32_t>(c->counts), ptr<ihipStream_t>(c->stream));
}

extern "C" int64_t ll_call_kv8_store(const LLKv8StoreCall* c) {
  LL_CHECK_ARG(c, "ll_call_kv8_store: null record");
  return ll_kv8_store(
      ptr<const void>(c->k), c->k_stride_tok, c->k_stride_h, ptr<const void>(c->v),
      c->v_stride_tok, c->v_stride_h, ptr<const int32_t>(c->slots), c->ntok, c->kv_heads,
      c->head_dim, ptr<void>(c->k_codes), c->kc_stride_tok, c->kc_stride_h,
      ptr<void>(c->v_codes), c->vc_stride_tok, c->vc_stride_h, ptr<float>(c->k_scale),
      c->ks_stride_block, c->ks_stride_h, ptr<float>(c->v_scale), c->vs_stride_block,
      c->vs_stride_h, c->slots_n, c->block, (int)c->code, (int)c->dtype,
      ptr<ihipStream_t>(c->stream));
}

extern "C" int64_t ll_call_kv8_load(const LLKv8LoadCall* c) {
  LL_CHECK_ARG(c, "ll_call_kv8_load: null record");
  return ll_kv8_load(
      ptr<const void>(c->k_codes), c->kc_stride_tok, c->kc_stride_h,
      ptr<const void>(c->v_codes), c->vc_stride_tok, c->vc_stride_h, ptr<const float>(c->k_scale),
      c->ks_stride_block, c->ks_stride_h, ptr<const float>(c->v_scale), c->vs_stride_block,
      c->vs_stride_h, c->slots_n, c->block, (int)c->code, ptr<const int32_t>(c->req_to_tokens),
      c->req_to_tokens_stride, c->req_rows, ptr<const void>(c->b_req_idx), (int)c->req_idx_i64,
      ptr<const void>(c->b_start_loc), (int)c->start_loc_i64, ptr<const void>(c->b_seq_len),
      (int)c->seq_len_i64, c->batch, c->max_len_in_batch, ptr<void>(c->k_out), c->ko_stride_tok,
      c->ko_stride_h, ptr<void>(c->v_out), c->vo_stride_tok, c->vo_stride_h, c->out_rows,
      c->kv_heads, c->head_dim, (int)c->dtype, ptr<ihipStream_t>(c->stream));
}

extern "C" int64_t ll_call_kv8_decode_attention(const LLKv8DecodeAttentionCall* c) {
  LL_CHECK_ARG(c, "ll_call_kv8_decode_attention: null record");
  const int64_t need = ll_kv8_decode_attention_workspace_size(c->batch, c->q_heads, c->kv_heads,
                                                              c->head_dim, c->max_len_in_batch);
  if (need > c->workspace_bytes) return need;
  return ll_kv8_decode_attention(
      ptr<const void>(c->q), c->q_stride_b, c->q_stride_h, ptr<const void>(c->k_codes),
      c->kc_stride_tok, c->kc_stride_h, ptr<const void>(c->v_codes), c->vc_stride_tok,
      c->vc_stride_h, ptr<const float>(c->k_scale), c->ks_stride_block, c->ks_stride_h,
      ptr<const float>(c->v_scale), c->vs_stride_block, c->vs_stride_h, c->slots_n, c->block,
      (int)c->code, ptr<const int32_t>(c->req_to_tokens), c->req_to_tokens_stride, c->req_rows,
      ptr<const void>(c->b_req_idx), (int)c->req_idx_i64, ptr<const void>(c->b_seq_len),
      (int)c->seq_len_i64, ptr<void>(c->out), c->out_stride_b, c->out_stride_h, c->batch,
      c->q_heads, c->kv_heads, c->head_dim, c->max_len_in_batch, (float)c->sm_scale,
      (int)c->dtype, ptr<void>(c->workspace), c->workspace_bytes, ptr<ihipStream_t>(c->stream));
}

extern "C" int64_t ll_call_linear_w4(const LLLinearW4Call* c) {
  LL_CHECK_ARG(c, "ll_call_linear_w4: null record");
  const int64_t need = ll_linear_w4_workspace_size(c->M, c->N, c->K);
  if (need > c->workspace_bytes) return need;
  return ll_linear_w4(ptr<const void>(c->x), c->ldx, ptr<const void>(c->packed), (int)c->has_zero,
                      c->group, ptr<const void>(c->bias), ptr<void>(c->y), c->ldy, c->M, c->N, c->K,
                      (int)c->dtype, ptr<void>(c->workspace), c->workspace_bytes,
                      ptr<ihipStream_t>(c->stream));
}

extern "C" int64_t ll_call_adjust_logits(const LLAdjustLogitsCall* c) {
  LL_CHECK_ARG(c, "ll_call_adjust_logits: null record");
  return ll_adjust_logits(
      ptr<const void>(c->logits), c->ld_logits, ptr<void>(c->out), c->ld_out, c->batch,
      c->vocab, ptr<const int32_t>(c->tokens), c->tokens_stride, c->tokens_rows, c->tokens_cols,
      ptr<const void>(c->b_req_idx), (int)c->req_idx_i64, ptr<const void>(c->b_prompt_len),
      (int)c->prompt_len_i64, ptr<const void>(c->b_seq_len), (int)c->seq_len_i64,
      ptr<const float>(c->repetition), ptr<const float>(c->frequency), ptr<const float>(c->presence),
      ptr<const int32_t>(c->bias_ids), c->bias_ids_stride, ptr<const float>(c->bias_values),
      c->bias_values_stride, c->n_bias, ptr<const uint32_t>(c->mask), c->mask_stride,
      (int)c->dtype, ptr<ihipStream_t>(c->stream));
}
