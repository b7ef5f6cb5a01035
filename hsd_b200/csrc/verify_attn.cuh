// The verification attention's launch, shared with the attention over the 8-bit
// cache (kv8_attn.cu).
#pragma once

#include "common.cuh"

namespace hsd {
namespace attn {

// Scales of 64 columns of one KV head: scores times k; V (held in fp16) times v.
struct __align__(16) ColumnScale {
  float score;   // k * softmax scale * log2 e
  float log2_v;  // log2 v
  float inv_v;   // 1 / v
  float pad;
};

}  // namespace attn
}  // namespace hsd

namespace hsd_host {

// Checked arguments of hsd_verify_attention; partials, flags and sync are the
// stream-K scratch (all null: one CTA per item); with
// col_scale [num_kv_heads][2 ceil(kv_len / 128)], k (bf16) and v (fp16) hold values
// that the scales multiply, `scale` and sync are not used, and the kernel launched
// just before, which has waited for all before it, clears the flags.
struct AttentionArgs {
  const void *q, *k, *v;
  int64_t q_row_stride, q_head_stride, k_row_stride, k_head_stride, v_row_stride, v_head_stride;
  void* out;
  float* lse;
  int32_t q_len, kv_len, num_q_heads, num_kv_heads;
  float scale;
  const hsd_plan_t* plan;
  void* partials;   // attention_partials_bytes()
  uint32_t* flags;  // attention_flags_bytes(), zero before the first use
  uint32_t* sync;   // two words, likewise
  int32_t* status;
  hsd_stream_t stream;
  const hsd::attn::ColumnScale* col_scale;
};
int attention_launch(const AttentionArgs& a);
// HSD_OK, or HSD_ERR_TOO_LARGE for more query tiles than a launch takes.
int attention_check_tiles(const hsd_plan_t& plan, const char* what);
size_t attention_partials_bytes();  // with col_scale's part
size_t attention_flags_bytes();

}  // namespace hsd_host
