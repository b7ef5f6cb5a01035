// Attention over the 8-bit cache for few query rows (single tokens, normal
// rows of the verification loop).
//
// What bounds it is reading the cache once, so the rows of all query heads of
// one KV head are packed (packed row i = query row i / group, head i % group)
// into tiles of 16, and the cache's columns are split over all SMs.  A warp
// owns a running softmax of one tile and takes 64 sealed columns (or 32 bf16
// ones) at a time: one TMA copy each of K and V, 8 KB each, into its own
// two-stage ring; no warp waits for another before the join.
//
// m16n8k16 bf16 MMAs (16 rows; tcgen05's smallest tile is 64 rows x 128
// threads of softmax, mostly empty here).  The fragments come straight from
// the bytes in shared memory: the order of dims inside an MMA's K = 16 is
// free as long as Q agrees, and so is the order of columns as long as P and
// the mask agree, so each lane's 16-byte load of K holds its operands of four
// MMAs, and pairs of V rows are joined by byte permutes.  Columns 2t and
// 2t + 1 of an S tile are columns t and t + 4 of its eight, and lane group g
// holds V dims 16 perm(g)..+15, perm(n) = n / 2 + 4 (n % 2): with the 128-byte
// swizzle every 16-byte load is then free of bank conflicts.
//
// Scales: S is multiplied by the block's K scale inside the exponent; P by
// the V scale before it is rounded to bf16 (bf16 keeps fp32's range, so no
// scale underflows); the row sum takes the unrounded, unscaled P in fp32.
// P's rounding (2^-9 relative, to nearest) is that of every bf16 attention.
//
// Join: warps of a CTA through shared memory, CTAs through fp32 partial rows
// in the workspace and a second small launch.  No counters and no flags: the
// result does not depend on the order in which CTAs finish.
#include "kv8_attn.cuh"

namespace hsd {
namespace kv8r {

using kv8a::HD;
using kv8a::Params;

constexpr int kWarps = 6;
constexpr int kThreads = kWarps * 32;
constexpr int kStages = 2;
constexpr int kTile = 64 * HD;          // bytes: 64 int8 rows, or 32 bf16 rows
constexpr int kStageBytes = 2 * kTile;  // K and V
constexpr int kRows = 16;
constexpr int kRecord = kRows * HD + 2 * kRows;  // floats of a partial record
constexpr size_t kSmem = size_t(kWarps) * kStages * kStageBytes + 1024;

struct Split {
  float* partials;  // [tile][splits][kRecord], or null
  int splits, n_tiles;
};

__device__ __forceinline__ int perm(int n) { return (n >> 1) | ((n & 1) << 2); }

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                    uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// The warp's walk over its units: 64-column halves of the tile's block list,
// a bf16 half in two steps of 32 columns.
struct Cursor {
  int u;        // half of the list, -1 before the first
  int col;      // first column of the step
  bool tail, second, partial;
};

__device__ __forceinline__ bool next_step(const Params& p, const uint32_t* list, int n_units,
                                          int stride, Cursor& c) {
  if (c.tail && !c.second && c.col + 32 < p.kv_len) {
    c.second = true;
    c.col += 32;
    return true;
  }
  while (true) {
    c.u += stride;
    if (c.u >= n_units) return false;
    const uint32_t e = list[c.u >> 1];
    const int hf = c.u & 1;
    if (!((e >> (24 + 2 * hf)) & 1u)) continue;
    c.partial = ((e >> (25 + 2 * hf)) & 1u) != 0;
    c.col = int(e & 0xFFFFFFu) * 128 + 64 * hf;
    c.tail = c.col >= p.sealed;
    c.second = false;
    return true;
  }
}

// Running softmax of the warp's 16 rows; this lane: rows g and g + 8.
struct State {
  float m[2], l[2];
  float o[16][4];
};

// Scores of NT tiles of eight columns -> P (bf16 pairs) with the state
// updated.  bits[r]: the row's mask, bit i = column i of the step.
template <int NT>
__device__ __forceinline__ void softmax_step(float (&c)[NT][4], const uint64_t (&bits)[2],
                                             bool partial, float sc, float vs, int t, State& s,
                                             uint32_t (&pk)[NT][2]) {
  float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[j][i] *= sc;
      const int r = i >> 1;
      if (partial && !((bits[r] >> (8 * j + t + 4 * (i & 1))) & 1ull)) c[j][i] = -INFINITY;
      mx[r] = fmaxf(mx[r], c[j][i]);
    }
  float alpha[2], nm[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
    const float m_new = fmaxf(s.m[r], mx[r]);
    nm[r] = m_new == -INFINITY ? 0.f : -m_new;
    alpha[r] = ex2_approx(s.m[r] + nm[r]);  // 0 when the row had nothing yet
    s.m[r] = m_new;
  }
  float sum[2] = {0.f, 0.f};
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float a = ex2_approx(c[j][2 * r] + nm[r]);
      const float b = ex2_approx(c[j][2 * r + 1] + nm[r]);
      sum[r] += a + b;
      pk[j][r] = pack_bf16x2(a * vs, b * vs);
    }
  s.l[0] = s.l[0] * alpha[0] + sum[0];
  s.l[1] = s.l[1] * alpha[1] + sum[1];
  if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s.o[i][0] *= alpha[0];
      s.o[i][1] *= alpha[0];
      s.o[i][2] *= alpha[1];
      s.o[i][3] *= alpha[1];
    }
  }
}

__device__ __forceinline__ void sealed_step(uint32_t kb, uint32_t vb, const uint32_t (&qf)[8][4],
                                            const uint64_t (&bits)[2], bool partial, float sc,
                                            float vs, int g, int t, State& s) {
  float c[8][4];
  const int pg = perm(g);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c[j][i] = 0.f;
    const uint32_t row = kb + uint32_t(8 * j + pg) * 128u;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 w = lds128(row + (uint32_t((4 * h + t) ^ pg) << 4));
      uint32_t b0, b1;
      kv8a::bytes_to_bf16(w.x, b0, b1);
      mma(c[j], qf[4 * h], b0, b1);
      kv8a::bytes_to_bf16(w.y, b0, b1);
      mma(c[j], qf[4 * h + 1], b0, b1);
      kv8a::bytes_to_bf16(w.z, b0, b1);
      mma(c[j], qf[4 * h + 2], b0, b1);
      kv8a::bytes_to_bf16(w.w, b0, b1);
      mma(c[j], qf[4 * h + 3], b0, b1);
    }
  }
  uint32_t pk[8][2];
  softmax_step<8>(c, bits, partial, sc, vs, t, s, pk);
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) {
    const uint32_t a[4] = {pk[2 * kk][0], pk[2 * kk][1], pk[2 * kk + 1][0], pk[2 * kk + 1][1]};
    uint32_t w[4][4];  // rows t, t + 4, t + 8, t + 12 of the 16: dims 16 pg..+15
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 16 * kk + 4 * i + t;
      const uint4 v = lds128(vb + uint32_t(r) * 128u + (uint32_t(pg ^ (r & 7)) << 4));
      w[i][0] = v.x;
      w[i][1] = v.y;
      w[i][2] = v.z;
      w[i][3] = v.w;
    }
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      uint32_t x0, x1, x2, x3, y0, y1, y2, y3;
      kv8a::bytes_to_bf16(__byte_perm(w[0][d], w[1][d], 0x5140), x0, x1);
      kv8a::bytes_to_bf16(__byte_perm(w[0][d], w[1][d], 0x7362), x2, x3);
      kv8a::bytes_to_bf16(__byte_perm(w[2][d], w[3][d], 0x5140), y0, y1);
      kv8a::bytes_to_bf16(__byte_perm(w[2][d], w[3][d], 0x7362), y2, y3);
      mma(s.o[4 * d], a, x0, y0);
      mma(s.o[4 * d + 1], a, x1, y1);
      mma(s.o[4 * d + 2], a, x2, y2);
      mma(s.o[4 * d + 3], a, x3, y3);
    }
  }
}

// 32 bf16 columns: two 64-dim sub-tiles of 32 rows x 128 bytes per operand.
// V rows that no row of the tile sees (seen) read as zero, so what stands in
// masked columns never reaches the sums.
__device__ __forceinline__ void tail_step(uint32_t kb, uint32_t vb, const uint32_t (&qf)[8][4],
                                          const uint64_t (&bits)[2], bool partial, uint32_t seen,
                                          float sc, int g, int t, State& s) {
  float c[4][4];
  const int pg = perm(g);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c[j][i] = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t row = kb + uint32_t(h * (kTile / 2) + (8 * j + pg) * 128);
#pragma unroll
      for (int cc = 0; cc < 2; ++cc) {
        const uint4 w = lds128(row + (uint32_t((2 * t + cc) ^ pg) << 4));
        mma(c[j], qf[4 * h + 2 * cc], w.x, w.y);
        mma(c[j], qf[4 * h + 2 * cc + 1], w.z, w.w);
      }
    }
  }
  uint32_t pk[4][2];
  softmax_step<4>(c, bits, partial, sc, 1.f, t, s, pk);
  const uint32_t vsub = vb + uint32_t((pg >> 2) * (kTile / 2));
#pragma unroll
  for (int kk = 0; kk < 2; ++kk) {
    const uint32_t a[4] = {pk[2 * kk][0], pk[2 * kk][1], pk[2 * kk + 1][0], pk[2 * kk + 1][1]};
#pragma unroll
    for (int cc = 0; cc < 2; ++cc) {
      uint32_t w[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 16 * kk + 4 * i + t;
        uint4 v = lds128(vsub + uint32_t(r) * 128u +
                         (uint32_t((2 * (pg & 3) + cc) ^ (r & 7)) << 4));
        if (!((seen >> r) & 1u)) v = make_uint4(0u, 0u, 0u, 0u);
        w[i][0] = v.x;
        w[i][1] = v.y;
        w[i][2] = v.z;
        w[i][3] = v.w;
      }
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        mma(s.o[8 * cc + 2 * d], a, __byte_perm(w[0][d], w[1][d], 0x5410),
            __byte_perm(w[2][d], w[3][d], 0x5410));
        mma(s.o[8 * cc + 2 * d + 1], a, __byte_perm(w[0][d], w[1][d], 0x7632),
            __byte_perm(w[2][d], w[3][d], 0x7632));
      }
    }
  }
}

__device__ __forceinline__ void store_row(const Params& p, int kvh, int row, int d4, float4 v,
                                          float m, float l) {
  const int q = row / p.group, h = kvh * p.group + row - q * p.group;
  const float inv = l > 0.f ? 1.f / l : 0.f;
  *reinterpret_cast<uint2*>(p.out + (size_t(q) * p.hq + h) * HD + 4 * d4) =
      make_uint2(pack_bf16x2(v.x * inv, v.y * inv), pack_bf16x2(v.z * inv, v.w * inv));
  if (d4 == 0 && p.lse)
    p.lse[size_t(h) * p.q_len + q] =
        l > 0.f ? (m + __log2f(l)) * 0.69314718055994530942f : -INFINITY;
}

// CTA (split, KV head, tile of 16 packed rows)
__global__ void __launch_bounds__(kThreads, 1)
    rows_kernel(const __grid_constant__ CUtensorMap tm_k8, const __grid_constant__ CUtensorMap tm_v8,
                const __grid_constant__ CUtensorMap tm_kt, const __grid_constant__ CUtensorMap tm_vt,
                const Params p, const Split sp) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  __shared__ uint64_t full[kWarps][kStages];
  __shared__ float2 ml[kWarps][kRows];
  __shared__ int abort_flag;
  const int warp = warp_id(), lane = lane_id();
  const int g = lane >> 2, t = lane & 3;
  if (threadIdx.x == 0) {
    for (int w = 0; w < kWarps; ++w)
      for (int i = 0; i < kStages; ++i) mbar_init(&full[w][i], 1);
    abort_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();
  pdl_wait_then_release();  // launched with launch_pdl: nothing global is read before
  volatile int* abort = &abort_flag;
  const int kvh = blockIdx.y;
  const int row0 = int(blockIdx.z) * kRows;  // first packed row
  const int n_rows = min(kRows, p.q_len * p.group - row0);
  const int qt = (row0 / p.group) >> 7;  // a tile's rows lie in one query tile: 128 group % 16 == 0
  const uint32_t* list = p.blk_list + size_t(qt) * p.n_kv128;
  const int n_units = 2 * p.blk_count[qt];
  const int stride = sp.splits * kWarps;
  uint8_t* ring = smem + warp * (kStages * kStageBytes);

  Cursor ic;  // issued up to here
  ic.u = int(blockIdx.x) * kWarps + warp - stride;
  ic.tail = ic.second = ic.partial = false;
  ic.col = 0;
  Cursor cc = ic;  // consumed up to here
  int issued = 0, consumed = 0;
  auto issue = [&]() {
    if (!next_step(p, list, n_units, stride, ic)) return;
    if (lane == 0) {
      uint64_t* bar = &full[warp][issued % kStages];
      uint8_t* kd = ring + (issued % kStages) * kStageBytes;
      uint8_t* vd = kd + kTile;
      mbar_arrive_expect_tx(bar, kStageBytes);
      if (ic.tail) {
        const int r = ic.col - p.tail_row0;
        for (int h = 0; h < 2; ++h) {
          tma_load_3d(kd + h * (kTile / 2), &tm_kt, bar, 64 * h, r, kvh);
          tma_load_3d(vd + h * (kTile / 2), &tm_vt, bar, 64 * h, r, kvh);
        }
      } else {
        tma_load_3d(kd, &tm_k8, bar, 0, ic.col, kvh);
        tma_load_3d(vd, &tm_v8, bar, 0, ic.col, kvh);
      }
    }
    ++issued;
  };
  for (int i = 0; i < kStages; ++i) issue();

  // Q fragments: MMA (h, w) covers dims 64 h + 16 t + 4 w..+3 of lane group t
  uint32_t qf[8][4];
  int mrow[2];  // the lane's rows in the query tile, -1: no such row
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int i = row0 + g + 8 * r;
    const bool have = g + 8 * r < n_rows;
    const int q = i / p.group;
    mrow[r] = have ? (q & 127) : -1;
    const __nv_bfloat16* src = p.q + int64_t(q) * p.q_row_stride +
                               int64_t(kvh * p.group + i - q * p.group) * p.q_head_stride;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint4 a = make_uint4(0u, 0u, 0u, 0u), b = a;
      if (have) {
        a = *reinterpret_cast<const uint4*>(src + 64 * h + 16 * t);
        b = *reinterpret_cast<const uint4*>(src + 64 * h + 16 * t + 8);
      }
      qf[4 * h][r] = a.x;
      qf[4 * h][r + 2] = a.y;
      qf[4 * h + 1][r] = a.z;
      qf[4 * h + 1][r + 2] = a.w;
      qf[4 * h + 2][r] = b.x;
      qf[4 * h + 2][r + 2] = b.y;
      qf[4 * h + 3][r] = b.z;
      qf[4 * h + 3][r + 2] = b.w;
    }
  }

  State s;
  s.m[0] = s.m[1] = -INFINITY;
  s.l[0] = s.l[1] = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) s.o[i][k] = 0.f;

  bool ok = true;
  while (ok && next_step(p, list, n_units, stride, cc)) {
    const int tile64 = cc.col >> 6;
    float sc = p.scale_log2, vs = 1.f;
    if (!cc.tail) {
      sc *= p.k_scale[kvh * p.scale_stride + tile64];
      vs = p.v_scale[kvh * p.scale_stride + tile64];
    }
    uint64_t bits[2] = {~0ull, ~0ull};
    uint32_t seen = 0xffffffffu;
    if (cc.partial) {
      const uint64_t* words = p.mask_words + (size_t(qt) * p.n_kv64 + tile64) * 128;
      bits[0] = mrow[0] >= 0 ? words[mrow[0]] : 0ull;
      bits[1] = mrow[1] >= 0 ? words[mrow[1]] : 0ull;
    }
    if (cc.tail) {
      if (cc.second) {
        bits[0] >>= 32;
        bits[1] >>= 32;
      }
      seen = __reduce_or_sync(0xffffffffu, uint32_t(bits[0]) | uint32_t(bits[1]));
    }
    const int st = consumed % kStages;
    ok = __all_sync(0xffffffffu, mbar_wait(&full[warp][st], uint32_t(consumed / kStages) & 1u,
                                           abort, p.status, 0x800));
    if (!ok) break;
    const uint32_t kb = smem_u32(ring + st * kStageBytes);
    if (!cc.partial || __any_sync(0xffffffffu, (bits[0] | bits[1]) != 0ull)) {
      if (cc.tail)
        tail_step(kb, kb + kTile, qf, bits, cc.partial, seen, sc, g, t, s);
      else
        sealed_step(kb, kb + kTile, qf, bits, cc.partial, sc, vs, g, t, s);
    }
    ++consumed;
    __syncwarp();  // every lane has read the stage before it is refilled
    issue();
  }
  if (!ok)  // copies in flight must land before the CTA's memory goes
    for (int k = consumed; k < issued; ++k)
      mbar_wait(&full[warp][k % kStages], uint32_t(k / kStages) & 1u, abort, p.status, 0x801,
                false);

  // ---- join the CTA's warps
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    s.l[r] += __shfl_xor_sync(0xffffffffu, s.l[r], 1);
    s.l[r] += __shfl_xor_sync(0xffffffffu, s.l[r], 2);
    if (t == 0) ml[warp][g + 8 * r] = make_float2(s.m[r], s.l[r]);
    float* dst = reinterpret_cast<float*>(ring) + (g + 8 * r) * (HD + 4);
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *reinterpret_cast<float4*>(dst + 64 * e + 16 * t + i) =
            make_float4(s.o[i][2 * r + e], s.o[i + 1][2 * r + e], s.o[i + 2][2 * r + e],
                        s.o[i + 3][2 * r + e]);
  }
  __syncthreads();
  const size_t tile = size_t(kvh) * gridDim.z + blockIdx.z;
  float* rec = sp.partials ? sp.partials + (tile * sp.splits + blockIdx.x) * kRecord : nullptr;
  for (int idx = threadIdx.x; idx < n_rows * 32; idx += kThreads) {
    const int r = idx >> 5, d4 = idx & 31;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, ml[w][r].x);
    const float nm = m == -INFINITY ? 0.f : -m;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float2 x = ml[w][r];
      const float f = ex2_approx(x.x + nm);
      const float4 v = *reinterpret_cast<const float4*>(
          reinterpret_cast<const float*>(smem + w * (kStages * kStageBytes)) + r * (HD + 4) +
          4 * d4);
      l += x.y * f;
      acc.x += v.x * f;
      acc.y += v.y * f;
      acc.z += v.z * f;
      acc.w += v.w * f;
    }
    if (rec) {
      *reinterpret_cast<float4*>(rec + r * HD + 4 * d4) = acc;
      if (d4 == 0) reinterpret_cast<float2*>(rec + kRows * HD)[r] = make_float2(m, l);
    } else {
      store_row(p, kvh, row0 + r, d4, acc, m, l);
    }
  }
}

// Join the splits: warp (packed row, KV head), lane = 4 dims.
__global__ void __launch_bounds__(128) join_kernel(const Params p, const Split sp) {
  pdl_wait_then_release();  // launched with launch_pdl
  const int row = int(blockIdx.x) * 4 + warp_id();
  const int kvh = blockIdx.y, d4 = lane_id();
  if (row >= p.q_len * p.group) return;
  const int r = row % kRows;
  const float* rec0 =
      sp.partials + (size_t(kvh) * sp.n_tiles + row / kRows) * sp.splits * kRecord;
  float m = -INFINITY;
  for (int i = d4; i < sp.splits; i += 32)
    m = fmaxf(m, __ldcg(rec0 + size_t(i) * kRecord + kRows * HD + 2 * r));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float nm = m == -INFINITY ? 0.f : -m;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
#pragma unroll 8
  for (int i = 0; i < sp.splits; ++i) {
    const float* rec = rec0 + size_t(i) * kRecord;
    const float2 x = __ldcg(reinterpret_cast<const float2*>(rec + kRows * HD) + r);
    const float4 v = __ldcg(reinterpret_cast<const float4*>(rec + r * HD) + d4);
    const float f = ex2_approx(x.x + nm);
    l += x.y * f;
    acc.x += v.x * f;
    acc.y += v.y * f;
    acc.z += v.z * f;
    acc.w += v.w * f;
  }
  store_row(p, kvh, row, d4, acc, m, l);
}

}  // namespace kv8r
}  // namespace hsd

namespace hsd_host {

using namespace hsd;

namespace {
int n_tiles(int q_len, int group) {
  return int((int64_t(q_len) * group + kv8r::kRows - 1) / kv8r::kRows);
}
// CTAs per tile: one wave of one CTA per SM, each warp with a unit at least.
int n_splits(int q_len, int kv_len, int hq, int hkv) {
  const int64_t tiles = int64_t(n_tiles(q_len, hq / hkv)) * hkv;
  const int units = (kv_len + 63) / 64;
  const int most = (units + kv8r::kWarps - 1) / kv8r::kWarps;
  const int64_t s = kv8_sm_count() / tiles;
  return s < 1 ? 1 : s > most ? most : int(s);
}
}  // namespace

size_t kv8_rows_workspace_bytes(int q_len, int kv_len, int hq, int hkv) {
  const int s = n_splits(q_len, kv_len, hq, hkv);
  if (s == 1) return kKv8FlagBytes;
  return kKv8FlagBytes + size_t(n_tiles(q_len, hq / hkv)) * hkv * s * kv8r::kRecord * sizeof(float);
}

int kv8_map(CUtensorMap* map, const void* base, bool bf16, int64_t rows, int heads,
            int64_t row_stride, int64_t head_stride, int box_rows, const char* what) {
  EncodeTiledFn enc = tensor_map_encoder();
  if (!enc) {
    set_error("cuTensorMapEncodeTiled unavailable");
    return HSD_ERR_CUDA;
  }
  const int es = bf16 ? 2 : 1;
  cuuint64_t dims[3] = {128, cuuint64_t(rows), cuuint64_t(heads)};
  cuuint64_t strides[2] = {cuuint64_t(row_stride) * es, cuuint64_t(head_stride) * es};
  cuuint32_t box[3] = {bf16 ? 64u : 128u, cuuint32_t(box_rows), 1};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r =
      enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 3,
          const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled(%s) failed: %d", what, int(r));
    return HSD_ERR_CUDA;
  }
  return HSD_OK;
}

int kv8_sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0)
    return 148;
  return n;
}

int kv8_rows_launch(const Kv8AttnArgs& a) {
  const hsd::kv8a::Params& p = a.p;
  CUtensorMap k8, v8, kt, vt;
  const int64_t tail_rows = p.kv_len - p.tail_row0;
  const bool has8 = p.sealed > 0, has_tail = p.sealed < p.kv_len;
  // a side without columns is never loaded; its map describes the other one
  int rc = HSD_OK;
  if (has8) {
    rc = kv8_map(&k8, a.k8, false, p.sealed, p.hkv, 128, a.k8_head_stride, 64, "k8");
    if (!rc) rc = kv8_map(&v8, a.v8, false, p.sealed, p.hkv, 128, a.v8_head_stride, 64, "v8");
  }
  if (!rc && has_tail) {
    rc = kv8_map(&kt, a.k_tail, true, tail_rows, p.hkv, a.kt_row_stride, a.kt_head_stride, 32,
                 "k tail");
    if (!rc)
      rc = kv8_map(&vt, a.v_tail, true, tail_rows, p.hkv, a.vt_row_stride, a.vt_head_stride, 32,
                   "v tail");
  }
  if (rc) return rc;
  if (!has8) {
    k8 = kt;
    v8 = vt;
  }
  if (!has_tail) {
    kt = k8;
    vt = v8;
  }
  kv8r::Split sp;
  sp.n_tiles = n_tiles(p.q_len, p.group);
  sp.splits = n_splits(p.q_len, p.kv_len, p.hq, p.hkv);
  sp.partials = sp.splits > 1 ? reinterpret_cast<float*>(static_cast<char*>(a.workspace) + kKv8FlagBytes)
                               : nullptr;
  if (sp.n_tiles > 65535 || p.hkv > 65535) {
    set_error("hsd_verify_attention_kv8: %d rows x %d heads exceed the launch's range", p.q_len,
              p.hq);
    return HSD_ERR_TOO_LARGE;
  }
  rc = cuda_check(cudaFuncSetAttribute(kv8r::rows_kernel,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       int(kv8r::kSmem)),
                  "cudaFuncSetAttribute(rows_kernel)");
  if (rc) return rc;
  rc = launch_pdl(kv8r::rows_kernel,
                  dim3(unsigned(sp.splits), unsigned(p.hkv), unsigned(sp.n_tiles)),
                  dim3(kv8r::kThreads), kv8r::kSmem, a.stream, "rows_kernel launch", 0, k8, v8, kt,
                  vt, p, sp);
  if (rc || sp.splits == 1) return rc;
  return launch_pdl(kv8r::join_kernel,
                    dim3(unsigned((p.q_len * p.group + 3) / 4), unsigned(p.hkv)), dim3(128), 0,
                    a.stream, "join_kernel launch", 0, p, sp);
}

}  // namespace hsd_host
