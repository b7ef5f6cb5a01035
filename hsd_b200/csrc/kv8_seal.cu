// The page's KV cache in 8 bits: sealing whole 64-token blocks of every
// layer's planes, and reading sealed rows back as bf16.
//
// A plane is one layer's K or V of one KV head.  A block of 64 rows x 128
// dims shares one scale (64 columns are the mask's tile width, so a tile of
// the attention has one scale per operand):
//
//   a = max |x| over the block's finite values, at least 2^-100
//   scale = a / 127,   n = rint(127 x / a) in [-127, 127],   x ~ n * scale
//
// Rounding.  t = x * (127 / a) in fp32 is off by at most 2^-23 of itself.
// With bf16 x and a (8-bit significands), 127 x / a either is a half-integer
// or differs from every half-integer by at least 2^-17 of it; rounding t to
// 19 mantissa bits therefore restores exact ties and moves nothing else
// across a border, so n is the correctly rounded quotient, ties to even.
//
// Seal: HBM bound, 2 bytes read and 1 written per value.  One CTA per block:
// the block's 16 KB sit in registers between the maximum and the rounding, so
// the rows are read once.  Unseal: 1 byte read, 2 written.  Measured: 28 layers of
// 2 heads, 2560 rows (110 MB, partly in L2): seal 15.3 us, 7.2 TB/s; unseal 14.6 us,
// 7.6 TB/s; 8 heads, 2048 rows (352 MB): 52.7 us, 6.7 TB/s and 53.9 us, 6.5 TB/s.
#include "common.cuh"

namespace hsd {
namespace kv8 {

constexpr int kThreads = 256;
constexpr int kBlockRows = 64;
constexpr int kDim = 128;
constexpr float kMinAmax = 7.888609052210118e-31f;  // 2^-100

__device__ __forceinline__ float lo_f(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_f(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// fp32 bits of 1.5 * 2^23 + rint(x * inv): the low byte is n
__device__ __forceinline__ uint32_t quantise(float x, float inv) {
  const uint32_t t = (__float_as_uint(__fmul_rn(x, inv)) + 8u) & ~15u;
  return __float_as_uint(__fadd_rn(__uint_as_float(t), 12582912.0f));
}

// non-finite values: infinities saturate, NaN gives 0
__device__ __forceinline__ float tame(float x, float amax) {
  const float y = fminf(fmaxf(x, -amax), amax);
  return x == x ? y : 0.f;
}

__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// largest of two bf16 magnitudes at a time (as integers: the order of magnitudes)
__device__ __forceinline__ uint32_t mag_max(uint32_t m, uint32_t w) {
  return __vmaxu2(m, w & 0x7FFF7FFFu);
}
// the same over the finite ones only
__device__ __forceinline__ uint32_t finite_mag_max(uint32_t m, uint32_t w) {
  uint32_t lo = w & 0x7FFFu, hi = (w >> 16) & 0x7FFFu;
  lo = lo >= 0x7F80u ? 0u : lo;
  hi = hi >= 0x7F80u ? 0u : hi;
  return __vmaxu2(m, lo | (hi << 16));
}

__device__ __forceinline__ uint32_t block_max(uint32_t m, uint32_t* red) {
  m = max(m & 0xFFFFu, m >> 16);
  m = __reduce_max_sync(0xffffffffu, m);
  if (lane_id() == 0) red[warp_id()] = m;
  __syncthreads();
  m = red[lane_id() & (kThreads / 32 - 1)];
  return __reduce_max_sync(0xffffffffu, m);
}

// CTA (block, plane)
__global__ void __launch_bounds__(kThreads)
    seal_kernel(const uint64_t* src_planes, int64_t src_row0, int8_t* data, int64_t plane_stride,
                float* scale, int64_t scale_stride, int block0, int32_t* status) {
  pdl_wait_then_release();  // launched with launch_pdl
  __shared__ uint32_t red[2][kThreads / 32];
  const int b = blockIdx.x;
  const int64_t plane = blockIdx.y;
  const uint4* src = reinterpret_cast<const uint4*>(
      reinterpret_cast<const char*>(src_planes[plane]) +
      (src_row0 + int64_t(b) * kBlockRows) * (kDim * 2));
  // thread: 16 consecutive values at 16 (tid + 256 j), j = 0, 1
  uint4 x[4];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    x[2 * j] = __ldcs(src + 2 * (int(threadIdx.x) + kThreads * j));
    x[2 * j + 1] = __ldcs(src + 2 * (int(threadIdx.x) + kThreads * j) + 1);
  }
  uint32_t* w = &x[0].x;
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = mag_max(m, w[i]);
  m = block_max(m, red[0]);
  const bool odd = m >= 0x7F80u;  // block holds an infinity or NaN (same for all threads)
  if (odd) {
    m = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = finite_mag_max(m, w[i]);
    m = block_max(m, red[1]);
    if (threadIdx.x == 0) report(status, HSD_DEV_BAD_VALUE | 0x701);
  }
  const float amax = fmaxf(__uint_as_float(m << 16), kMinAmax);
  const float inv = __fdiv_rn(127.0f, amax);
  int4* dst = reinterpret_cast<int4*>(data + plane * plane_stride +
                                      (int64_t(block0) + b) * (kBlockRows * kDim));
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w0 = w[8 * j + 2 * i], w1 = w[8 * j + 2 * i + 1];
      float f[4] = {lo_f(w0), hi_f(w0), lo_f(w1), hi_f(w1)};
      if (odd) {
#pragma unroll
        for (int k = 0; k < 4; ++k) f[k] = tame(f[k], amax);
      }
      o[i] = low_bytes(quantise(f[0], inv), quantise(f[1], inv), quantise(f[2], inv),
                       quantise(f[3], inv));
    }
    dst[int(threadIdx.x) + kThreads * j] = make_int4(int(o[0]), int(o[1]), int(o[2]), int(o[3]));
  }
  if (threadIdx.x == 0)
    scale[plane * scale_stride + block0 + b] = __fdiv_rn(amax, 127.0f);
}

// signed byte k of w as a float
template <int k>
__device__ __forceinline__ float byte_f(uint32_t w) {
  return float(int32_t(w << (24 - 8 * k)) >> 24);
}

// CTA (64-row group, plane); thread: 8 values at a time, four in flight, so that
// a warp's loads and stores are contiguous (16 values a thread, in two stores 32
// bytes apart, took 23 us instead of 14 us for 112 planes x 2560 rows)
__global__ void __launch_bounds__(kThreads)
    unseal_kernel(const int8_t* data, int64_t plane_stride, const float* scale,
                  int64_t scale_stride, int64_t row0, int n_rows, const uint64_t* dst_planes,
                  int64_t dst_row0) {
  pdl_wait_then_release();  // launched with launch_pdl
  const int64_t plane = blockIdx.y;
  const int64_t first = int64_t(blockIdx.x) * kBlockRows;  // row of the range
  const int rows = int(min(int64_t(kBlockRows), int64_t(n_rows) - first));
  const uint2* src =
      reinterpret_cast<const uint2*>(data + plane * plane_stride + (row0 + first) * kDim);
  uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<char*>(dst_planes[plane]) +
                                        (dst_row0 + first) * (kDim * 2));
  const float* sc = scale + plane * scale_stride;
  constexpr int kUnits = kBlockRows * kDim / 8 / kThreads;
  uint2 v[kUnits];
  float s[kUnits];
#pragma unroll
  for (int j = 0; j < kUnits; ++j) {
    const int u = int(threadIdx.x) + kThreads * j;  // 16 units of 8 values per row
    const int r = u >> 4;
    if (r < rows) {
      v[j] = __ldcs(src + u);
      s[j] = __ldg(sc + (row0 + first + r) / kBlockRows);
    }
  }
#pragma unroll
  for (int j = 0; j < kUnits; ++j) {
    const int u = int(threadIdx.x) + kThreads * j;
    // streamed: the rows are read once, later, and by another kernel
    if ((u >> 4) < rows)
      __stcs(dst + u, make_uint4(pack_bf16x2(byte_f<0>(v[j].x) * s[j], byte_f<1>(v[j].x) * s[j]),
                                 pack_bf16x2(byte_f<2>(v[j].x) * s[j], byte_f<3>(v[j].x) * s[j]),
                                 pack_bf16x2(byte_f<0>(v[j].y) * s[j], byte_f<1>(v[j].y) * s[j]),
                                 pack_bf16x2(byte_f<2>(v[j].y) * s[j], byte_f<3>(v[j].y) * s[j])));
  }
}

}  // namespace kv8
}  // namespace hsd

namespace {

constexpr int kMaxPlanes = 65535;  // grid y
// Rows beyond any memory: what is below it leaves room for a launch's rows and for
// bytes (256 a row) in 64 bits.
constexpr int64_t kMaxRow = int64_t(1) << 48;

int check_kv8(const char* what, const uint64_t* planes, int32_t n_planes, const void* data,
              int64_t plane_stride, const void* scale, int64_t scale_stride, int64_t last_row) {
  if (n_planes < 0 || (n_planes > 0 && (!planes || !data || !scale)) ||
      (reinterpret_cast<uintptr_t>(data) & 15) || (reinterpret_cast<uintptr_t>(scale) & 3) ||
      (reinterpret_cast<uintptr_t>(planes) & 7) || (plane_stride % 16) || plane_stride < 0 ||
      scale_stride < 0 ||
      (n_planes > 1 && (plane_stride < last_row * 128 || scale_stride < (last_row + 63) / 64))) {
    hsd_host::set_error(
        "%s: bad arguments (planes=%d; data 16-byte aligned, plane strides covering %lld rows)",
        what, n_planes, static_cast<long long>(last_row));
    return HSD_ERR_INVALID_ARG;
  }
  if (n_planes > kMaxPlanes) {
    hsd_host::set_error("%s: %d planes exceed %d", what, n_planes, kMaxPlanes);
    return HSD_ERR_TOO_LARGE;
  }
  return HSD_OK;
}

}  // namespace

extern "C" int hsd_kv8_seal(const uint64_t* src_planes, int32_t n_planes, int64_t src_row0,
                            int8_t* data, int64_t plane_stride, float* scale, int64_t scale_stride,
                            int32_t block0, int32_t n_blocks, int32_t* status,
                            hsd_stream_t stream) {
  using namespace hsd;
  if (src_row0 < 0 || src_row0 > kMaxRow || block0 < 0 || n_blocks < 0) {
    hsd_host::set_error("hsd_kv8_seal: bad range (row %lld, blocks %d + %d)",
                        static_cast<long long>(src_row0), block0, n_blocks);
    return HSD_ERR_INVALID_ARG;
  }
  int rc = check_kv8("hsd_kv8_seal", src_planes, n_planes, data, plane_stride, scale, scale_stride,
                     (int64_t(block0) + n_blocks) * 64);
  if (rc || n_planes == 0 || n_blocks == 0) return rc;
  return hsd_host::launch_pdl(kv8::seal_kernel, dim3(unsigned(n_blocks), unsigned(n_planes)),
                              dim3(kv8::kThreads), 0, reinterpret_cast<cudaStream_t>(stream),
                              "seal_kernel launch", 0, src_planes, src_row0, data, plane_stride,
                              scale, scale_stride, int(block0), status);
}

extern "C" int hsd_kv8_unseal(const int8_t* data, int64_t plane_stride, const float* scale,
                              int64_t scale_stride, int32_t n_planes, int64_t row0, int32_t n_rows,
                              const uint64_t* dst_planes, int64_t dst_row0, hsd_stream_t stream) {
  using namespace hsd;
  if (row0 < 0 || row0 > kMaxRow || n_rows < 0 || dst_row0 < 0 || dst_row0 > kMaxRow) {
    hsd_host::set_error("hsd_kv8_unseal: bad range (rows %lld + %d to %lld)",
                        static_cast<long long>(row0), n_rows, static_cast<long long>(dst_row0));
    return HSD_ERR_INVALID_ARG;
  }
  int rc = check_kv8("hsd_kv8_unseal", dst_planes, n_planes, data, plane_stride, scale,
                     scale_stride, row0 + n_rows);
  if (rc || n_planes == 0 || n_rows == 0) return rc;
  return hsd_host::launch_pdl(kv8::unseal_kernel,
                              dim3(unsigned((n_rows + 63) / 64), unsigned(n_planes)),
                              dim3(kv8::kThreads), 0, reinterpret_cast<cudaStream_t>(stream),
                              "unseal_kernel launch", 0, data, plane_stride, scale, scale_stride,
                              row0, int(n_rows), dst_planes, dst_row0);
}
