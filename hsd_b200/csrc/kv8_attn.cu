// Packed verification attention over a cache whose first columns are held in
// 8 bits: argument checks, the choice of kernel, and the path for many rows.
//
// Many rows.  Every K and V element meets every query tile and head pair (17 x
// 3 times for a region page), so converting where it is used costs far more
// than the cache's bytes; here one launch expands the layer's columns into
// the workspace and the tcgen05 verification kernel (verify_attn.cu) reads that,
// with one score factor and one V factor per 64 columns in its softmax.  K
// becomes bf16 (int8: the same integers, exactly; the bf16 tail copied), V fp16
// (int8 exactly; 64 tail rows times the power of two that brings their largest
// value to [64, 128): exact down to 2^-21 of it, else within 2^-31 of it), so that
// P can be fp16 and keep 11 bits.  The expansion reads 1 byte and writes 2 per
// sealed value, and the attention finds it in L2; for a region step's 4800 columns of
// 2 heads it is latency (7.1 us alone from cold caches, about 3.5 in a stream of steps,
// where the attention's setup runs under it).  Both together: 51.7 us for 2176 rows,
// 12/2 heads, 4800 columns (the bf16 kernel alone 47.8), 215 us for 2049 rows and
// 18,450 columns (210) at 1965 MHz; a long stream of the latter runs into the board's
// 1000 W limit, at 1785 MHz, and takes 239 a call.
#include "kv8_attn.cuh"
#include "verify_attn.cuh"

#include <algorithm>

#include <cuda_fp16.h>

namespace hsd {
namespace kv8a {

struct ExpandParams {
  const int8_t* x8[2];  // K, V
  int64_t head_stride8[2];
  const float* scale[2];
  int64_t scale_stride;
  const __nv_bfloat16* tail[2];
  int64_t row_stride[2], head_stride[2];
  const uint8_t* tile_class;
  const uint64_t* mask_words;
  uint16_t* dst;  // [2][hkv][kv_len][128]: K bf16, V fp16
  attn::ColumnScale* col_scale;
  uint32_t* flags;  // of the attention, cleared here
  int n_flags;
  int kv_len, hkv, n_kv64, n_qtiles, sealed, tail_row0;
  float scale_log2;
};

constexpr int kExpandThreads = 256;
// Least V factor, 2^-60: what blocks of zeros take, and where smaller V keeps its bits
// in fp16 down to 2^-73.  The running maximum is that of score + log2 of the factor, so
// a factor far below the others' would lose its columns' part of the row sum in the
// exponentials that bring sums to a common maximum (below 2^-126 they are 0): beside V
// of 2^b, weights below 2^-(72 - b) of the largest are lost.
constexpr float kMinVScale = 8.673617379884035e-19f;
constexpr uint32_t kMinVExponent = 127 - 60 + 6;

// Columns of a 64-column tile that some query row sees: a warp per query tile, four
// tiles' loads in flight.
__device__ __forceinline__ uint64_t seen_columns(const ExpandParams& p, int t, uint32_t* red) {
  if (threadIdx.x < 2) red[threadIdx.x] = 0u;
  __syncthreads();
  constexpr int kWarps = kExpandThreads / 32;
  uint64_t w = 0ull;
  for (int q0 = warp_id(); q0 < p.n_qtiles; q0 += 4 * kWarps) {
    int cls[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int qt = q0 + u * kWarps;
      cls[u] = qt < p.n_qtiles ? p.tile_class[size_t(qt) * p.n_kv64 + t] : 0;
    }
    uint64_t m[4][4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        m[u][i] = cls[u] == 1 ? p.mask_words[(size_t(q0 + u * kWarps) * p.n_kv64 + t) * 128 +
                                             32 * i + lane_id()]
                              : (cls[u] == 2 ? ~0ull : 0ull);
#pragma unroll
    for (int u = 0; u < 4; ++u) w |= (m[u][0] | m[u][1]) | (m[u][2] | m[u][3]);
  }
  const uint32_t lo = __reduce_or_sync(0xffffffffu, uint32_t(w));
  const uint32_t hi = __reduce_or_sync(0xffffffffu, uint32_t(w >> 32));
  if (lane_id() == 0) {
    atomicOr(&red[0], lo);
    atomicOr(&red[1], hi);
  }
  __syncthreads();
  return uint64_t(red[0]) | (uint64_t(red[1]) << 32);
}

// CTA (64-column tile, KV head, K or V)
__global__ void __launch_bounds__(kExpandThreads) expand_kernel(const ExpandParams p) {
  pdl_wait_then_release();  // launched with launch_pdl
  __shared__ uint32_t red[2], warp_top[kExpandThreads / 32];
  const int t = blockIdx.x, h = blockIdx.y, z = blockIdx.z, tid = threadIdx.x;
  if (t == 0 && h == 0 && z == 0)
    for (int i = tid; i < p.n_flags; i += kExpandThreads) p.flags[i] = 0u;
  const int col0 = 64 * t;
  uint4* dst = reinterpret_cast<uint4*>(
      p.dst + (size_t(z * p.hkv + h) * p.kv_len + col0) * HD);
  float v_unit = 1.f;  // V: value = fp16 * v_unit
  if (col0 < p.sealed) {
    const uint4* src =
        reinterpret_cast<const uint4*>(p.x8[z] + h * p.head_stride8[z] + int64_t(col0) * HD);
    uint4 v[2];
    v[0] = __ldcs(src + tid);
    v[1] = __ldcs(src + tid + kExpandThreads);
    // A block of next to nothing (zeros are sealed with the scale 2^-100 / 127)
    // takes the least factor, so that its columns' part of the row sum, formed as
    // P / scale, does not underflow.
    bool tiny = false;
    float of_unit = 1.f;  // what is left of the scale (0: the scale is 0, and so are the values)
    if (z == 1) {
      v_unit = p.scale[1][h * p.scale_stride + t];
      tiny = v_unit < kMinVScale;
      if (tiny) {
        of_unit = v_unit / kMinVScale;
        v_unit = kMinVScale;
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      uint32_t o[8];
      const uint32_t in[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (z == 0) {
          bytes_to_bf16(in[i], o[2 * i], o[2 * i + 1]);
        } else {
          bytes_to_f16(in[i], o[2 * i], o[2 * i + 1]);
          if (tiny) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&o[2 * i + k]));
              o[2 * i + k] = pack_f16x2(x.x * of_unit, x.y * of_unit);
            }
          }
        }
      }
      const int at = 2 * (tid + u * kExpandThreads);
      dst[at] = make_uint4(o[0], o[1], o[2], o[3]);
      dst[at + 1] = make_uint4(o[4], o[5], o[6], o[7]);
    }
  } else {
    const __nv_bfloat16* src = p.tail[z] + h * p.head_stride[z] +
                               int64_t(col0 - p.tail_row0) * p.row_stride[z] + (tid & 15) * 8;
    const int rows = min(64, p.kv_len - col0);
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r = 16 * u + (tid >> 4);
      v[u] = make_uint4(0u, 0u, 0u, 0u);
      if (r < rows) v[u] = __ldg(reinterpret_cast<const uint4*>(src + r * p.row_stride[z]));
    }
    if (z == 1) {
      // what stands in columns that no row sees must not reach the sums (0 * V)
      const uint64_t seen = seen_columns(p, t, red);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (!((seen >> (16 * u + (tid >> 4))) & 1ull)) v[u] = make_uint4(0u, 0u, 0u, 0u);
    }
    if (z == 1) {
      // the block's largest finite magnitude, as bf16 bits
      uint32_t top = 0;
      const uint32_t* w = &v[0].x;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t lo = w[i] & 0x7FFFu, hi = (w[i] >> 16) & 0x7FFFu;
        top = max(top, max(lo < 0x7F80u ? lo : 0u, hi < 0x7F80u ? hi : 0u));
      }
      top = __reduce_max_sync(0xffffffffu, top);
      if (lane_id() == 0) warp_top[warp_id()] = top;
      __syncthreads();
      top = __reduce_max_sync(0xffffffffu, warp_top[lane_id() & (kExpandThreads / 32 - 1)]);
      // v_unit = 2^(e - 6) for a largest value in [2^e, 2^(e + 1)); e as a float's
      // exponent field, held where both v_unit and its inverse are normal.  A block of
      // zeros takes the least, as a sealed one does: the running maximum is that of
      // score + log2 v_unit, and a larger unit would cost the other columns' P bits.
      const uint32_t e = min(max(top >> 7, kMinVExponent), 250u);
      v_unit = __uint_as_float((e - 6u) << 23);
      const float inv = __uint_as_float((260u - e) << 23);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        uint32_t* x = &v[u].x;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[i] = pack_f16x2(__uint_as_float(x[i] << 16) * inv,
                            __uint_as_float(x[i] & 0xFFFF0000u) * inv);
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r = 16 * u + (tid >> 4);
      if (r < rows) dst[r * 16 + (tid & 15)] = v[u];
    }
  }
  // score factor by the K CTA, V factors by the V CTA
  if (tid == 0) {
    attn::ColumnScale* c = p.col_scale + size_t(h) * ((p.n_kv64 + 1) & ~1) + t;
    // the absent second half of an odd last block: any finite factors
    const bool pad = t == p.n_kv64 - 1 && (t & 1) == 0;
    if (z == 0) {
      c->score = col0 < p.sealed
                     ? score_factor(p.scale[0][h * p.scale_stride + t] * p.scale_log2)
                     : p.scale_log2;
      if (pad) c[1].score = 1.f;
    } else {
      c->log2_v = log2f(v_unit);
      c->inv_v = 1.f / v_unit;
      if (pad) {
        c[1].log2_v = 0.f;
        c[1].inv_v = 1.f;
      }
    }
  }
}

}  // namespace kv8a
}  // namespace hsd

namespace {

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

// Workspace of the path for many rows: flags, partial records, scales, rows.
struct ManyLayout {
  size_t partials, scales, rows, total;
};
ManyLayout many_layout(int32_t kv_len, int32_t hkv) {
  ManyLayout m;
  m.partials = align256(hsd_host::attention_flags_bytes());
  m.scales = m.partials + align256(hsd_host::attention_partials_bytes());
  m.rows = m.scales +
           align256(size_t(hkv) * ((kv_len + 127) / 128) * 2 * sizeof(hsd::attn::ColumnScale));
  m.total = m.rows + size_t(2) * hkv * kv_len * hsd::kv8a::HD * 2;
  return m;
}

// Rows kernel or many rows, by the time each takes over the whole cache (what the plan
// leaves visible of it is known on the device alone).  Many rows: 22 us, the expansion
// (1.3e-4 us a column and KV head), 2.05 us per SM for every 128 rows x 128 columns x
// two heads, and 1.2 us for each part of an item (128 rows, two heads) that its first
// CTA merges when all SMs share few items.  Measured (rows / many, us): 12/2 heads, 1600
// columns: 128 rows 17 / 36, 256 rows 37 / 36, 384 rows 35 / 30; 8192 columns: 64 rows
// 27 / 58, 128 rows 57 / 58, 256 rows 99 / 48; 16/8 heads, 32768 columns: 32 rows 60 /
// 111, 128 rows 206 / 111; 8/1 heads, 32768 columns: 64 rows 60 / 88, 128 rows 110 / 88.
struct Path {
  bool many;
  hsd_host::Kv8RowsChoice rows;
  size_t bytes;
};
Path choose_path(int32_t q_len, int32_t kv_len, int32_t hq, int32_t hkv) {
  const hsd_host::Kv8RowsChoice rows = hsd_host::kv8_rows_choose(q_len, kv_len, hq, hkv);
  const float sms = float(rows.sms);
  const float items = float((q_len + 127) / 128) * float((hq / hkv + 1) / 2) * float(hkv);
  const float blocks = float((kv_len + 127) / 128);
  const float merges = std::max(std::min(blocks, sms / items) - 1.f, 0.f);
  const float many = 22.f + 1.3e-4f * float(kv_len) * float(hkv) +
                     2.05f * items * blocks / sms + 1.2f * merges;
  if (rows.us <= many)
    return {false, rows, hsd_host::kv8_rows_workspace_bytes(q_len, hq, hkv, rows)};
  return {true, rows, many_layout(kv_len, hkv).total};
}

int many_launch(const hsd_host::Kv8AttnArgs& a, const hsd_plan_t& plan, float scale) {
  using namespace hsd;
  const kv8a::Params& p = a.p;
  int rc = hsd_host::attention_check_tiles(plan, "hsd_verify_attention_kv8");
  if (rc) return rc;
  if (p.hkv > 65535) {
    hsd_host::set_error("hsd_verify_attention_kv8: %d KV heads exceed the launch's range", p.hkv);
    return HSD_ERR_TOO_LARGE;
  }
  const ManyLayout m = many_layout(p.kv_len, p.hkv);
  char* ws = static_cast<char*>(a.workspace);
  kv8a::ExpandParams e;
  e.x8[0] = a.k8;
  e.x8[1] = a.v8;
  e.head_stride8[0] = a.k8_head_stride;
  e.head_stride8[1] = a.v8_head_stride;
  e.scale[0] = p.k_scale;
  e.scale[1] = p.v_scale;
  e.scale_stride = p.scale_stride;
  e.tail[0] = static_cast<const __nv_bfloat16*>(a.k_tail);
  e.tail[1] = static_cast<const __nv_bfloat16*>(a.v_tail);
  e.row_stride[0] = a.kt_row_stride;
  e.row_stride[1] = a.vt_row_stride;
  e.head_stride[0] = a.kt_head_stride;
  e.head_stride[1] = a.vt_head_stride;
  e.tile_class = plan.tile_class;
  e.mask_words = plan.mask_words;
  e.dst = reinterpret_cast<uint16_t*>(ws + m.rows);
  e.col_scale = reinterpret_cast<attn::ColumnScale*>(ws + m.scales);
  e.flags = reinterpret_cast<uint32_t*>(ws);
  e.n_flags = int(hsd_host::attention_flags_bytes() / sizeof(uint32_t));
  e.kv_len = p.kv_len;
  e.hkv = p.hkv;
  e.n_kv64 = p.n_kv64;
  e.n_qtiles = plan.n_qtiles;
  e.sealed = p.sealed;
  e.tail_row0 = p.tail_row0;
  e.scale_log2 = p.scale_log2;
  rc = hsd_host::launch_pdl(kv8a::expand_kernel,
                            dim3(unsigned(p.n_kv64), unsigned(p.hkv), 2),
                            dim3(kv8a::kExpandThreads), 0, a.stream, "expand_kernel launch", 0, e);
  if (rc) return rc;
  hsd_host::AttentionArgs v;
  v.q = p.q;
  v.q_row_stride = p.q_row_stride;
  v.q_head_stride = p.q_head_stride;
  v.k = e.dst;
  v.v = e.dst + size_t(p.hkv) * p.kv_len * kv8a::HD;
  v.k_row_stride = v.v_row_stride = kv8a::HD;
  v.k_head_stride = v.v_head_stride = int64_t(p.kv_len) * kv8a::HD;
  v.out = p.out;
  v.lse = p.lse;
  v.q_len = p.q_len;
  v.kv_len = p.kv_len;
  v.num_q_heads = p.hq;
  v.num_kv_heads = p.hkv;
  v.scale = scale;
  v.plan = &plan;
  v.sync = nullptr;
  v.flags = e.flags;
  v.partials = ws + m.partials;
  v.status = p.status;
  v.stream = reinterpret_cast<hsd_stream_t>(a.stream);
  v.col_scale = e.col_scale;
  return hsd_host::attention_launch(v);
}

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
  return choose_path(q_len, kv_len, num_q_heads, num_kv_heads).bytes;
}

extern "C" int hsd_kv8_attention_choice(int32_t q_len, int32_t kv_len, int32_t num_q_heads,
                                        int32_t num_kv_heads, int32_t choice[4]) {
  if (q_len <= 0 || kv_len <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 ||
      num_q_heads % num_kv_heads || !choice) {
    hsd_host::set_error("hsd_kv8_attention_choice: bad arguments (q_len=%d kv_len=%d heads=%d/%d)",
                        q_len, kv_len, num_q_heads, num_kv_heads);
    return HSD_ERR_INVALID_ARG;
  }
  const Path path = choose_path(q_len, kv_len, num_q_heads, num_kv_heads);
  choice[0] = path.many;
  choice[1] = path.many ? 0 : path.rows.splits;
  choice[2] = path.many ? 0 : path.rows.join;
  choice[3] = path.many ? 0 : (path.rows.fine ? 32 : 64);
  return HSD_OK;
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
  const Path path = choose_path(q_len, kv_len, num_q_heads, num_kv_heads);
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) ||
      workspace_bytes < path.bytes) {
    hsd_host::set_error(
        "hsd_verify_attention_kv8: workspace %zu bytes (need %zu, 256-byte aligned)",
        workspace_bytes, path.bytes);
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
  return path.many ? many_launch(a, *plan, scale) : hsd_host::kv8_rows_launch(a, path.rows);
}
