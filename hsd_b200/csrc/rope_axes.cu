// Rotary positions with several axes, fused with the cache update, one launch.
//
// Image and video tokens carry one position per axis (time, height, width;
// the HunYuan pipeline's position ids are [1, 4, Q], H:2033, H:2100, H:2128),
// and each of the 64 dimension pairs of a head turns with one of them:
//
//   angle(r, i) = positions[axis(i)][r] * inv_freq[i]
//   y_i = scaling (x_i cos - x_{i+64} sin),  y_{i+64} = scaling (x_{i+64} cos + x_i sin)
//
// Products and sums in fp32, one rounding to bf16 at the end.
//
// Angles.  A position of 10^5 times a frequency loses 0.004 rad in fp32, so
// the frequency is kept as turns per position in 64-bit fixed point (units of
// 2^-64 turn): position * turns modulo 2^64 is the fraction of a turn, a product
// without error for any int64 position, negative ones included (two's complement
// wraps as turns do).  The upper 32 bits, as a signed fraction of a half turn, feed
// sincospif.  Error in half turns: 2^-25 for rounding the angle to fp32, 2^-31 for
// the bits below, and |position| * 2^-64 for the frequency's rounding to 2^-64 turn,
// which is below the first up to positions of 2^39 (at 2^63 nothing is left).
//
// Work: a CTA takes a few rows; 64 threads per row compute the row's cosines
// and sines once into shared memory, and all heads use them.  The rows' first
// loads are issued before, so they run under the trigonometry.  HBM bound:
// each query, key and value row is read once and written once.  Measured: 45.3 us
// for 16640 rows of 16/8 heads (273 MB, 6.0 TB/s, 0.93 of a copy), 4.4 us for 2176
// rows of 12/2 heads, 1.9 us (a launch) for one row.
#include "common.cuh"

namespace hsd {
namespace rope_axes {

constexpr int kThreads = 256;
constexpr int kMaxRows = 4;  // rows per CTA
constexpr int kMaxAxes = 8;
constexpr int kAhead = 4;    // units per thread loaded ahead of the trigonometry

struct Params {
  const __nv_bfloat16* q;
  __nv_bfloat16* q_out;
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  const int64_t* positions;
  const uint64_t* turns;
  const int32_t* pair_axis;
  __nv_bfloat16* k_cache;
  __nv_bfloat16* v_cache;
  int64_t q_row_stride, q_out_row_stride, k_row_stride, v_row_stride;
  int64_t pos_axis_stride, pos_row_stride;
  int64_t kc_head_stride, vc_head_stride, cache_row_stride;
  int64_t dst_row0;
  int32_t* status;
  float scaling;
  int n_rows, n_axes, hq, hkv, rows_per_cta;
};

// 8 lanes of a head's first half with their partners (query / key), or 16
// lanes of a value row.
struct Unit {
  uint4 a, b;
  __nv_bfloat16* dst;
  int table;  // offset of the row's 8 angles in shared memory, < 0: value, copied
};

__device__ __forceinline__ void load_unit(const Params& p, int row0, int u, int per_row, Unit& w) {
  const int rl = u / per_row;
  const int t = u - rl * per_row;
  const int64_t row = row0 + rl;
  const int head = t >> 3, c = t & 7;
  const __nv_bfloat16* src;
  int64_t second = 64;
  if (head < p.hq) {
    src = p.q + row * p.q_row_stride + head * 128 + c * 8;
    w.dst = p.q_out + row * p.q_out_row_stride + head * 128 + c * 8;
    w.table = rl * 64 + c * 8;
  } else if (head < p.hq + p.hkv) {
    const int h = head - p.hq;
    src = p.k + row * p.k_row_stride + h * 128 + c * 8;
    w.dst = p.k_cache + h * p.kc_head_stride + (p.dst_row0 + row) * p.cache_row_stride + c * 8;
    w.table = rl * 64 + c * 8;
  } else {
    const int h = head - p.hq - p.hkv;
    src = p.v + row * p.v_row_stride + h * 128 + c * 8;
    w.dst = p.v_cache + h * p.vc_head_stride + (p.dst_row0 + row) * p.cache_row_stride + c * 8;
    w.table = -1;
  }
  w.a = *reinterpret_cast<const uint4*>(src);
  w.b = *reinterpret_cast<const uint4*>(src + second);
}

__device__ __forceinline__ float lo_f(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_f(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

__device__ __forceinline__ void store_unit(const Unit& w, const float2* cs) {
  uint4 y1 = w.a, y2 = w.b;
  if (w.table >= 0) {
    const uint32_t* A = &w.a.x;
    const uint32_t* B = &w.b.x;
    uint32_t* Y1 = &y1.x;
    uint32_t* Y2 = &y2.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // {cos, sin} of two neighbouring pairs
      const float4 t = *reinterpret_cast<const float4*>(cs + w.table + 2 * i);
      const float a0 = lo_f(A[i]), a1 = hi_f(A[i]), b0 = lo_f(B[i]), b1 = hi_f(B[i]);
      Y1[i] = pack_bf16x2(a0 * t.x - b0 * t.y, a1 * t.z - b1 * t.w);
      Y2[i] = pack_bf16x2(b0 * t.x + a0 * t.y, b1 * t.z + a1 * t.w);
    }
  }
  *reinterpret_cast<uint4*>(w.dst) = y1;
  *reinterpret_cast<uint4*>(w.dst + 64) = y2;
}

__global__ void __launch_bounds__(kThreads) rope_axes_kernel(const Params p) {
  pdl_wait_then_release();  // launched with launch_pdl
  __shared__ __align__(16) float2 cs[kMaxRows * 64];
  const int row0 = int(blockIdx.x) * p.rows_per_cta;
  const int rows = min(p.rows_per_cta, p.n_rows - row0);
  const int per_row = (p.hq + 2 * p.hkv) * 8;
  const int total = rows * per_row;
  Unit w[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int u = int(threadIdx.x) + i * kThreads;
    if (u < total) load_unit(p, row0, u, per_row, w[i]);
  }
  if (int(threadIdx.x) < rows * 64) {
    const int rl = threadIdx.x >> 6, i = threadIdx.x & 63;
    const int axis = p.pair_axis[i];
    int64_t pos = 0;
    if (axis >= 0 && axis < p.n_axes)
      pos = p.positions[axis * p.pos_axis_stride + (row0 + rl) * p.pos_row_stride];
    else
      report(p.status, HSD_DEV_BAD_INDEX | 0x601);
    const uint64_t turn = p.turns[i] * uint64_t(pos);
    float s, c;
    sincospif(float(int32_t(uint32_t(turn >> 32))) * 4.656612873077393e-10f, &s, &c);
    cs[threadIdx.x] = make_float2(c * p.scaling, s * p.scaling);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (int(threadIdx.x) + i * kThreads < total) store_unit(w[i], cs);
  for (int u = int(threadIdx.x) + kAhead * kThreads; u < total; u += kThreads) {
    load_unit(p, row0, u, per_row, w[0]);
    store_unit(w[0], cs);
  }
}

}  // namespace rope_axes
}  // namespace hsd

extern "C" int hsd_rope_append_axes(
    const void* q, int64_t q_row_stride, void* q_out, int64_t q_out_row_stride, const void* k,
    int64_t k_row_stride, const void* v, int64_t v_row_stride, const int64_t* positions,
    int64_t pos_axis_stride, int64_t pos_row_stride, int32_t n_axes, const uint64_t* turns,
    const int32_t* pair_axis, float scaling, int32_t n_rows, int32_t num_q_heads,
    int32_t num_kv_heads, int32_t head_dim, void* k_cache, int64_t k_cache_head_stride,
    void* v_cache, int64_t v_cache_head_stride, int64_t cache_row_stride, int64_t dst_row0,
    int32_t* status, hsd_stream_t stream) {
  using namespace hsd;
  if (head_dim != 128) {
    hsd_host::set_error("hsd_rope_append_axes: head_dim %d unsupported (128 only)", head_dim);
    return HSD_ERR_UNSUPPORTED;
  }
  if (n_axes < 1 || n_axes > rope_axes::kMaxAxes) {
    hsd_host::set_error("hsd_rope_append_axes: %d position axes (1 to %d)", n_axes,
                        rope_axes::kMaxAxes);
    return HSD_ERR_UNSUPPORTED;
  }
  auto a16 = [](const void* x) { return x && (reinterpret_cast<uintptr_t>(x) & 15) == 0; };
  auto a8 = [](const void* x) { return x && (reinterpret_cast<uintptr_t>(x) & 7) == 0; };
  const int64_t qw = int64_t(num_q_heads) * 128, kw = int64_t(num_kv_heads) * 128;
  // rows beyond any memory would wrap around to others
  if (n_rows < 0 || num_q_heads < 0 || num_kv_heads <= 0 || dst_row0 < 0 ||
      dst_row0 > (int64_t(1) << 48) || num_q_heads > 4096 || num_kv_heads > 4096 ||
      (num_q_heads > 0 && (!a16(q) || !a16(q_out) || q_row_stride < qw || q_out_row_stride < qw)) ||
      !a16(k) || !a16(v) || !a16(k_cache) || !a16(v_cache) || !a8(positions) || !a8(turns) ||
      !pair_axis || k_row_stride < kw || v_row_stride < kw || cache_row_stride < 128 ||
      (q_row_stride % 8) || (q_out_row_stride % 8) || (k_row_stride % 8) || (v_row_stride % 8) ||
      (cache_row_stride % 8) || (k_cache_head_stride % 8) || (v_cache_head_stride % 8)) {
    hsd_host::set_error(
        "hsd_rope_append_axes: bad arguments (rows=%d heads=%d/%d; pointers 16-byte aligned, "
        "strides multiples of 8 elements covering the heads)",
        n_rows, num_q_heads, num_kv_heads);
    return HSD_ERR_INVALID_ARG;
  }
  if (n_rows == 0) return HSD_OK;
  rope_axes::Params p;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_out = static_cast<__nv_bfloat16*>(q_out);
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.positions = positions;
  p.turns = turns;
  p.pair_axis = pair_axis;
  p.k_cache = static_cast<__nv_bfloat16*>(k_cache);
  p.v_cache = static_cast<__nv_bfloat16*>(v_cache);
  p.q_row_stride = q_row_stride;
  p.q_out_row_stride = q_out_row_stride;
  p.k_row_stride = k_row_stride;
  p.v_row_stride = v_row_stride;
  p.pos_axis_stride = pos_axis_stride;
  p.pos_row_stride = pos_row_stride;
  p.kc_head_stride = k_cache_head_stride;
  p.vc_head_stride = v_cache_head_stride;
  p.cache_row_stride = cache_row_stride;
  p.dst_row0 = dst_row0;
  p.status = status;
  p.scaling = scaling;
  p.n_rows = n_rows;
  p.n_axes = n_axes;
  p.hq = num_q_heads;
  p.hkv = num_kv_heads;
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    sms = 148;
  // more rows per CTA once every SM holds several CTAs anyway
  p.rows_per_cta = n_rows >= 8 * sms ? 4 : n_rows >= 4 * sms ? 2 : 1;
  const int grid = (n_rows + p.rows_per_cta - 1) / p.rows_per_cta;
  return hsd_host::launch_pdl(rope_axes::rope_axes_kernel, dim3(unsigned(grid)),
                              dim3(rope_axes::kThreads), 0,
                              reinterpret_cast<cudaStream_t>(stream), "rope_axes_kernel launch", 0,
                              p);
}
