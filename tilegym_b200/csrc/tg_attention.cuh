// Arguments of the attention kernels.
#pragma once
#include "tg_decoder_common.cuh"

namespace tg {

struct AttentionParams {
  CacheView c;
  const void* q;  // [tokens, q_heads, dim]
  void* o;
  int64_t q_tok, q_head, o_tok, o_head;  // pitches in elements
  int32_t tokens, q_heads, group;        // group: query heads of one cache head
  float scale;
  int32_t window, sinks;
};

}  // namespace tg
