// Packed verification attention over a cache whose first columns are held in
// 8 bits: argument checks and the choice of kernel.
#include "kv8_attn.cuh"

namespace {

bool strides_ok(const void* p, int64_t rs, int64_t hs) {
  return p && (reinterpret_cast<uintptr_t>(p) & 15) == 0 && rs > 0 && hs > 0 && (rs % 8) == 0 &&
         (hs % 8) == 0;
}

}  // namespace

extern "C" size_t hsd_kv8_attention_workspace_bytes(int32_t q_len, int32_t kv_len,
                                                    int32_t num_q_heads, int32_t num_kv_heads) {
  if (q_len <= 0 || kv_len <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 ||
      num_q_heads % num_kv_heads)
    return 0;
  return hsd_host::kv8_rows_workspace_bytes(q_len, kv_len, num_q_heads, num_kv_heads);
}

extern "C" int hsd_verify_attention_kv8(
    const void* q, int64_t q_row_stride, int64_t q_head_stride, const int8_t* k8,
    int64_t k8_head_stride, const int8_t* v8, int64_t v8_head_stride, const float* k_scale,
    const float* v_scale, int64_t scale_head_stride, int32_t sealed, const void* k_tail,
    int64_t kt_row_stride, int64_t kt_head_stride, const void* v_tail, int64_t vt_row_stride,
    int64_t vt_head_stride, int32_t tail_row0, void* out, float* lse, int32_t q_len,
    int32_t kv_len, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, float scale,
    const hsd_plan_t* plan, void* workspace, size_t workspace_bytes, int32_t* status,
    hsd_stream_t stream) {
  if (head_dim != hsd::kv8a::HD) {
    hsd_host::set_error("hsd_verify_attention_kv8: head_dim %d unsupported (128 only)", head_dim);
    return HSD_ERR_UNSUPPORTED;
  }
  if (!(scale > 0.f) || scale > 3.0e38f) {
    hsd_host::set_error("hsd_verify_attention_kv8: scale %g must be positive and finite",
                        double(scale));
    return HSD_ERR_INVALID_ARG;
  }
  const bool has8 = sealed > 0, has_tail = sealed < kv_len;
  auto a16 = [](const void* x) { return x && (reinterpret_cast<uintptr_t>(x) & 15) == 0; };
  auto a4 = [](const void* x) { return x && (reinterpret_cast<uintptr_t>(x) & 3) == 0; };
  const int64_t need8 = num_kv_heads > 1 ? int64_t(sealed) * 128 : 16;
  if (!plan || plan->q_len != q_len || plan->kv_len != kv_len || q_len <= 0 || kv_len <= 0 ||
      num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads || !a16(out) ||
      (reinterpret_cast<uintptr_t>(lse) & 3) || !strides_ok(q, q_row_stride, q_head_stride) ||
      sealed < 0 || sealed % 64 || sealed > kv_len || tail_row0 < 0 || tail_row0 > sealed ||
      (has8 && (!a16(k8) || !a16(v8) || !a4(k_scale) || !a4(v_scale) || k8_head_stride < need8 ||
                v8_head_stride < need8 || (k8_head_stride % 16) || (v8_head_stride % 16) ||
                scale_head_stride < (num_kv_heads > 1 ? sealed / 64 : 0))) ||
      (has_tail && (!strides_ok(k_tail, kt_row_stride, kt_head_stride) ||
                    !strides_ok(v_tail, vt_row_stride, vt_head_stride)))) {
    hsd_host::set_error(
        "hsd_verify_attention_kv8: bad arguments (q_len=%d kv_len=%d heads=%d/%d, plan %d/%d, "
        "sealed=%d tail_row0=%d; pointers 16-byte aligned, strides multiples of 8 elements, "
        "sealed a multiple of 64 in [0, kv_len], tail_row0 in [0, sealed])",
        q_len, kv_len, num_q_heads, num_kv_heads, plan ? plan->q_len : -1,
        plan ? plan->kv_len : -1, sealed, tail_row0);
    return HSD_ERR_INVALID_ARG;
  }
  const size_t need =
      hsd_kv8_attention_workspace_bytes(q_len, kv_len, num_q_heads, num_kv_heads);
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) || workspace_bytes < need) {
    hsd_host::set_error(
        "hsd_verify_attention_kv8: workspace %zu bytes (need %zu, 256-byte aligned)",
        workspace_bytes, need);
    return HSD_ERR_INVALID_ARG;
  }
  hsd_host::Kv8AttnArgs a;
  hsd::kv8a::Params& p = a.p;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_row_stride = q_row_stride;
  p.q_head_stride = q_head_stride;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.scale_stride = scale_head_stride;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.lse = lse;
  p.blk_list = plan->blk_list;
  p.blk_count = plan->blk_count;
  p.mask_words = plan->mask_words;
  p.status = status;
  p.q_len = q_len;
  p.kv_len = kv_len;
  p.hq = num_q_heads;
  p.hkv = num_kv_heads;
  p.group = num_q_heads / num_kv_heads;
  p.n_kv64 = plan->n_kv64;
  p.n_kv128 = plan->n_kv128;
  p.sealed = sealed;
  p.tail_row0 = tail_row0;
  p.scale_log2 = scale * 1.4426950408889634f;
  a.k8 = k8;
  a.v8 = v8;
  a.k8_head_stride = k8_head_stride;
  a.v8_head_stride = v8_head_stride;
  a.k_tail = k_tail;
  a.v_tail = v_tail;
  a.kt_row_stride = kt_row_stride;
  a.kt_head_stride = kt_head_stride;
  a.vt_row_stride = vt_row_stride;
  a.vt_head_stride = vt_head_stride;
  a.workspace = workspace;
  a.stream = reinterpret_cast<cudaStream_t>(stream);
  return hsd_host::kv8_rows_launch(a);
}
