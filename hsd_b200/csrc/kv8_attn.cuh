// Shared by the kernels of the attention over the 8-bit cache: the launch's
// parameters, the exact int8 -> bf16 conversion, and the tensor maps.
#pragma once

#include "common.cuh"

namespace hsd {
namespace kv8a {

constexpr int HD = 128;

struct Params {
  const __nv_bfloat16* q;
  int64_t q_row_stride, q_head_stride;
  const float* k_scale;  // [Hkv][scale_stride] per 64 sealed columns
  const float* v_scale;
  int64_t scale_stride;
  __nv_bfloat16* out;
  float* lse;  // or null
  const uint32_t* blk_list;
  const int32_t* blk_count;
  const uint64_t* mask_words;
  int32_t* status;
  int q_len, kv_len, hq, hkv, group;
  int n_kv64, n_kv128;
  int sealed;     // columns held in 8 bits, a multiple of 64
  int tail_row0;  // column c >= sealed is row c - tail_row0 of the bf16 tail
  float scale_log2;
};

// A factor on sealed columns' scores, never below the smallest normal number: a block of zero keys
// (scale 2^-100 / 127) times a zero query row's unit (2^-100) is past fp32's range, and
// 0 times a masked score (-inf) would be NaN.  Scores under such a factor are below
// 2^-100, as good as 0.  NaN stays.
__device__ __forceinline__ float score_factor(float x) {
  return x < 1.1754943508222875e-38f ? 1.1754943508222875e-38f : x;
}

// Four signed bytes -> two bf16 pairs, exactly.  A byte placed under the bf16
// exponent of 128 reads 128 + (its low 7 bits); the same with only the sign
// bit kept reads 128, or 256 when it is set: their difference is the signed
// value.  8 instructions for four values, none of them a conversion.
__device__ __forceinline__ void bytes_to_bf16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t p0 = __byte_perm(w, 0x43434343u, 0x4140);
  const uint32_t p1 = __byte_perm(w, 0x43434343u, 0x4342);
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(lo) : "r"(p0 & 0xFF7FFF7Fu), "r"(p0 & 0xFF80FF80u));
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(hi) : "r"(p1 & 0xFF7FFF7Fu), "r"(p1 & 0xFF80FF80u));
}

// Bytes `sel` (two nibble pairs) of a word of n + 128 -> two exact fp16: 1024 +
// 128 + n is the byte under the exponent of 1024.
__device__ __forceinline__ uint32_t biased_to_f16(uint32_t w, uint32_t sel) {
  uint32_t r;
  const uint32_t p = __byte_perm(w, 0x64646464u, sel);
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(p), "r"(0x64806480u));
  return r;
}
// Four signed bytes -> two fp16 pairs, exactly.
__device__ __forceinline__ void bytes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t b = w ^ 0x80808080u;
  lo = biased_to_f16(b, 0x4140);
  hi = biased_to_f16(b, 0x4342);
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

}  // namespace kv8a
}  // namespace hsd

namespace hsd_host {
// The two kernels behind hsd_verify_attention_kv8.  No call relies on what the
// workspace holds when it starts.
struct Kv8AttnArgs {
  hsd::kv8a::Params p;
  const int8_t* k8;
  const int8_t* v8;
  int64_t k8_head_stride, v8_head_stride;
  const void* k_tail;
  const void* v_tail;
  int64_t kt_row_stride, kt_head_stride, vt_row_stride, vt_head_stride;
  void* workspace;
  cudaStream_t stream;
};
// The rows kernel for these sizes: CTAs per tile, whether the join kernel joins them
// (else they are a cluster), its time by its own model, and the device's SMs.
struct Kv8RowsChoice {
  int splits;
  bool join;
  bool fine;  // sealed columns 32 at a time instead of 64
  float us;
  int sms;
};
Kv8RowsChoice kv8_rows_choose(int q_len, int kv_len, int hq, int hkv);
size_t kv8_rows_workspace_bytes(int q_len, int hq, int hkv, const Kv8RowsChoice& c);
int kv8_rows_launch(const Kv8AttnArgs& a, const Kv8RowsChoice& c);
// 3-D map {128 dims, rows, heads} of int8 (box 128 x box_rows) or bf16 (box
// 64 x box_rows), 128-byte swizzle.
int kv8_map(CUtensorMap* map, const void* base, bool bf16, int64_t rows, int heads,
            int64_t row_stride, int64_t head_stride, int box_rows, const char* what);
}  // namespace hsd_host
