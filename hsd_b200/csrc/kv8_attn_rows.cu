// Attention over the 8-bit cache for few query rows (single tokens, normal
// rows of the verification loop).
//
// What bounds it is reading the cache once, so the rows of all query heads of
// one KV head are packed (packed row i = query row i / group, head i % group)
// into tiles of 16, and the cache's columns are split over all SMs.  A warp
// owns a running softmax of one tile and takes 64 sealed columns (32 where that
// leaves each warp one step; 32 bf16 ones) at a time: one TMA copy each of K and V,
// 8 KB each, into its own three buffers, each refilled as soon as its tile has been
// used; no warp waits for another before the join.  At full rate a copy takes 3 to 4 us, so the SM needs
// about 150 KB in flight: eight warps with three tiles each (with two tiles a
// warp waited 870 of 6300 cycles for V).
//
// m16n8k16 MMAs (tcgen05's smallest tile is 64 rows with a thread of softmax
// each, mostly empty here), transposed: S^T = K Q^T and O^T = V^T P^T, so that
// the cache fills the 16-row side and 8 or 16 query rows (kNB = 1 or 2 blocks of
// 8) the other: with 8 rows, half the MMAs and accumulators of the upright form.
// The fragments come straight from the bytes in shared memory: the order of dims
// inside an MMA's K = 16 is free as long as Q agrees, and so is the order of
// columns as long as P and the mask agree, so each lane's 16-byte load of K holds
// its operands of four MMAs, and pairs of V rows are joined by byte permutes; P^T
// needs one 8 x 8 transpose (movmatrix) per 8 columns.  Column n of eight is
// column perm(n) = n / 2 + 4 (n % 2), and lane group g holds V dims
// 16 perm(g)..+15: with the 128-byte swizzle every 16-byte load is then free of
// bank conflicts.
//
// Types.  Sealed columns run in fp16, where an int8 becomes a number with one
// byte permute and one subtraction (1024 + 128 + n is the exponent byte above n's
// byte, sign bit flipped) and P keeps 11 bits.  Ranges: each Q row is divided by
// a power of two that brings its largest value to [1, 2) and enters the score
// factor again; P is formed as 2^15 exp(s - max), so that weights down to
// 2^-39 count; O is kept in units of the block's V scale and rescaled from
// block to block.  bf16 columns run in bf16 throughout.  Scores, sums and O are
// fp32; the row sum takes the unrounded P.
//
// Measured: one row, 16/8 heads, 131,051 columns (269 MB): 47 us and 4 us for the
// join, 5.3 TB/s over both (0.82 of a copy; a wait of 3 to 4 us for the first tiles
// and the join are what is left).  12/2 heads, 2625 columns: one row 5.3 us, forty
// 11.7 us: latency (launch, block list, tile, join), not bytes.
//
// Join: warps of a CTA through shared memory; up to sixteen CTAs of a tile as a
// cluster, each writing its rows into the shared memory of the CTA that joins them
// (reading them from there instead took a second barrier and 0.8 us); or, where
// clusters do not fit, through fp32 partial rows in the workspace and a second small
// launch.  No counters and no flags: the result does not depend on the order in which CTAs finish.
#include "kv8_attn.cuh"

#include <algorithm>
#include <atomic>
#include <mutex>

namespace hsd {
namespace kv8r {

using kv8a::HD;
using kv8a::biased_to_f16;
using kv8a::bytes_to_f16;
using kv8a::pack_f16x2;
using kv8a::Params;
using kv8a::score_factor;

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 64 * HD;  // bytes: 64 int8 rows, or 32 bf16 rows
constexpr int kBuf = 3;  // the issue order keeps exactly three tiles ahead
static_assert(kBuf == 3, "a step's K and V and the next step's K are issued before any is used");
constexpr int kRing = kBuf * kTile;  // a warp's buffers: K, V, K, V, ... in turn
constexpr int kMaxRows = 16;
constexpr int kMaxCluster = 16;  // above 8: by opt-in, where the device has room for them
constexpr int kMaxIn = 30;  // the most of s ceil(kMaxRows / s) for s <= kMaxCluster
constexpr int kRecord = kMaxRows * HD + 2 * kMaxRows;  // floats of a partial record
constexpr float kPShift = 15.0f;                 // P = 2^15 exp(s - max)

struct __align__(1024) Smem {
  uint8_t ring[kWarps][kRing];  // then each warp's O, rows HD + 4 floats apart
  uint2 q16[8][2][32];          // Q fragments [MMA][block of 8 rows]: fp16 of q / unit, bf16
  uint2 qbf[8][2][32];
  float unit[kMaxRows];  // power of two of the row
  float2 ml[kWarps][kMaxRows];
  // rows that the cluster's CTAs hand to this one: [CTA][row / CTAs]
  float4 in_rows[kMaxIn][HD / 4];
  float2 in_ml[kMaxIn];
  uint64_t full[kWarps][kBuf];
  int abort;
};
constexpr size_t kSmem = sizeof(Smem) + 1024;
static_assert(kSmem <= 232448, "shared memory budget exceeded");
static_assert(kMaxRows * (HD + 4) * 4 <= kRing, "a warp's O must fit its ring");

struct Split {
  float* partials;  // [tile][splits][kRecord], or null: one CTA or one cluster per tile
  int splits, n_tiles, rows;  // rows: packed rows of a tile
};

__device__ __forceinline__ int perm(int n) { return (n >> 1) | ((n & 1) << 2); }

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 lds128(const uint8_t* p) {
  return *reinterpret_cast<const uint4*>(p);
}

// The warp's walk over its units: 64-column halves of the tile's block list (a bf16
// half in two steps of 32 columns), or, NT = 2, 32-column quarters.  The list is read
// a unit ahead.
struct Walk {
  const uint32_t* list;
  int n_units, stride, u;
  int room;        // entries that may be read (the list's, or more than it has)
  uint32_t ahead;  // entry of unit u
};
struct Step {
  int col;  // first column, -1: none
  bool tail, second, partial;
};

template <int NT>
__device__ __forceinline__ uint32_t list_entry(const Walk& w, int u) {
  // does not wait for n_units; next_step ignores what lies behind it
  const int i = u >> (NT == 4 ? 1 : 2);
  return i < w.room ? w.list[i] : 0u;
}

template <int NT>
__device__ __forceinline__ Step next_step(const Params& p, Walk& w, const Step& last) {
  Step c;
  if (NT == 4 && last.col >= 0 && last.tail && !last.second && last.col + 32 < p.kv_len) {
    c = last;
    c.second = true;
    c.col += 32;
    return c;
  }
  c.second = false;
  while (true) {
    const uint32_t e = w.ahead;
    const int u = w.u;
    if (u >= w.n_units) {
      c.col = -1;
      c.tail = c.partial = false;
      return c;
    }
    w.u += w.stride;
    w.ahead = list_entry<NT>(w, w.u);
    const int hf = (NT == 4 ? u : u >> 1) & 1;
    if (!((e >> (24 + 2 * hf)) & 1u)) continue;
    c.partial = ((e >> (25 + 2 * hf)) & 1u) != 0;
    c.col = int(e & 0xFFFFFFu) * 128 + 64 * hf;
    if (NT == 2 && (u & 1)) {
      c.second = true;
      c.col += 32;
      if (c.col >= p.kv_len) {
        c.second = false;
        continue;
      }
    }
    c.tail = c.col >= p.sealed;
    return c;
  }
}

__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// A step's scales and mask words (this lane's rows 2 t and 2 t + 1 of each block
// of 8), loaded while the step before is at its product.
template <int kNB>
struct Aside {
  float ks, vs;
  uint64_t bits[2 * kNB];
};

template <int kNB>
__device__ __forceinline__ void load_aside(const Params& p, const Step& c, int kvh, int qt,
                                           const int (&mrow)[2 * kNB], Aside<kNB>& a) {
  const int t64 = c.col >> 6;
  a.ks = a.vs = 1.f;
  if (!c.tail) {
    a.ks = __ldg(p.k_scale + kvh * p.scale_stride + t64);
    a.vs = __ldg(p.v_scale + kvh * p.scale_stride + t64);
  }
  const uint64_t* words = p.mask_words + (size_t(qt) * p.n_kv64 + t64) * 128;
#pragma unroll
  for (int r = 0; r < 2 * kNB; ++r) {
    a.bits[r] = ~0ull;  // rows that do not exist mask nothing
    if (c.partial && mrow[r] >= 0) a.bits[r] = words[mrow[r]];
    if (c.second) a.bits[r] >>= 32;
  }
}

// Running softmax of the warp's 8 kNB rows; this lane: rows 2 t and 2 t + 1 of
// each block.  o is in units of `unit` (0 before the first block), a V scale that
// blocks down to 2^-20 of it keep, their P carrying the quotient (fp16 P has room:
// weights down to 2^-19 still count).  A block more than 2^60 below the largest
// scale so far does not lower the unit further, so that O stays finite; its own
// part is then lost.
template <int kNB>
struct State {
  float m[2 * kNB], l[2 * kNB], unit, unit_max;
  float o[kNB][8][4];  // dims 16 perm(g) + 2 i, + 1 of rows 2 t, 2 t + 1
};

// Scores of NT tiles of 16 columns (c: column perm(g), rows 2 t and 2 t + 1, then
// column 8 + perm(g)) -> P^T fragments, with the state's maximum, sum and O
// brought up to date.
template <int kNB, int NT, bool kHalf>
__device__ __forceinline__ void softmax_step(float (&c)[kNB][NT][4],
                                             const uint64_t (&bits)[2 * kNB], bool masked,
                                             const float (&sc)[2 * kNB], float vs, int pg,
                                             State<kNB>& s, uint32_t (&pk)[kNB][NT][2]) {
  s.unit_max = fmaxf(s.unit_max, vs);
  // (2^-110, below what sealing leaves: a unit for scales of 0 alone)
  const float low = fmaxf(fmaxf(vs, s.unit_max * 8.673617379884035e-19f), 7.703719777548943e-34f);
  const bool keep = vs > 0.f && vs <= s.unit && vs >= s.unit * 9.5367431640625e-07f;
  const float v_unit = keep ? s.unit : low;
  if (masked) {
#pragma unroll
    for (int b = 0; b < kNB; ++b)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!((uint32_t(bits[2 * b + (i & 1)] >> (16 * j)) >> (pg + 8 * (i >> 1))) & 1u))
            c[b][j][i] = -INFINITY;
  }
  // P with the quotient of the V scales; the row sum without it.  Held at 2^-100, where
  // fp16 P is 0 already (V then adds nothing), so that its inverse and fp32 P stay in
  // range and the weights count whatever the quotient.
  const float exact = __fdividef(vs, v_unit);
  const float quotient = exact < 7.888609052210118e-31f ? 7.888609052210118e-31f : exact;
  const float shift = kPShift + __log2f(quotient);
  const float unscale = __fdividef(1.f, quotient);
  const float f = __fdividef(s.unit, v_unit);
  s.unit = v_unit;
  float of[2 * kNB];  // factors on O
  bool any = false;
#pragma unroll
  for (int b = 0; b < kNB; ++b) {
    float nm[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = 2 * b + e;
      float mx = fmaxf(c[b][0][e], c[b][0][2 + e]);
#pragma unroll
      for (int j = 1; j < NT; ++j) mx = fmax3(mx, c[b][j][e], c[b][j][2 + e]);
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float m_new = fmaxf(s.m[r], mx * sc[r]);
      const float neg = m_new == -INFINITY ? 0.f : -m_new;
      const float alpha = ex2_approx(s.m[r] + neg);  // 0 when the row had nothing yet
      nm[e] = neg + shift;
      s.m[r] = m_new;
      of[r] = alpha * f;
      any |= of[r] != 1.f;
      s.l[r] *= alpha;
    }
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float x = ex2_approx(fmaf(c[b][j][2 * k], sc[2 * b], nm[0]));
        const float y = ex2_approx(fmaf(c[b][j][2 * k + 1], sc[2 * b + 1], nm[1]));
        sum[0] += x;
        sum[1] += y;
        pk[b][j][k] = transpose8(kHalf ? pack_f16x2(x, y) : pack_bf16x2(x, y));
      }
    s.l[2 * b] += sum[0] * unscale;
    s.l[2 * b + 1] += sum[1] * unscale;
  }
  if (__any_sync(0xffffffffu, any)) {
#pragma unroll
    for (int b = 0; b < kNB; ++b)
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) s.o[b][i][k] *= of[2 * b + (k & 1)];
  }
}

template <int kNB, int NT>
__device__ __forceinline__ void sealed_scores(const uint8_t* kb, const uint2 (*q16)[2][32], int g,
                                              int t, float (&c)[kNB][NT][4]) {
  const int pg = perm(g), lane = lane_id();
#pragma unroll
  for (int b = 0; b < kNB; ++b)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) c[b][j][i] = 0.f;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t w[2 * NT][4];  // column perm(g) of every eight
#pragma unroll
    for (int j = 0; j < 2 * NT; ++j) {
      const uint4 v = lds128(kb + (8 * j + pg) * 128 + (((4 * h + t) ^ pg) << 4));
      w[j][0] = v.x;
      w[j][1] = v.y;
      w[j][2] = v.z;
      w[j][3] = v.w;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint2 q[kNB];
#pragma unroll
      for (int b = 0; b < kNB; ++b) q[b] = q16[4 * h + k][b][lane];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        uint32_t a[4];
        bytes_to_f16(w[2 * j][k], a[0], a[2]);
        bytes_to_f16(w[2 * j + 1][k], a[1], a[3]);
#pragma unroll
        for (int b = 0; b < kNB; ++b) mma_f16(c[b][j], a, q[b].x, q[b].y);
      }
    }
  }
}

template <int kNB, int NT>
__device__ __forceinline__ void sealed_values(const uint8_t* vb, const uint32_t (&pk)[kNB][NT][2],
                                              int g, int t, State<kNB>& s) {
  const int pg = perm(g);
#pragma unroll
  for (int kk = 0; kk < NT; ++kk) {
    uint32_t w[4][4];  // rows t, t + 4, t + 8, t + 12 of the 16: dims 16 pg..+15
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 16 * kk + 4 * i + t;
      const uint4 v = lds128(vb + r * 128 + ((pg ^ (r & 7)) << 4));
      w[i][0] = v.x ^ 0x80808080u;
      w[i][1] = v.y ^ 0x80808080u;
      w[i][2] = v.z ^ 0x80808080u;
      w[i][3] = v.w ^ 0x80808080u;
    }
#pragma unroll
    for (int d = 0; d < 4; ++d) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {  // dims 4 d + 2 e, + 1
        const uint32_t lo = __byte_perm(w[0][d], w[1][d], e ? 0x7362 : 0x5140);
        const uint32_t hi = __byte_perm(w[2][d], w[3][d], e ? 0x7362 : 0x5140);
        const uint32_t a[4] = {biased_to_f16(lo, 0x4140), biased_to_f16(lo, 0x4342),
                               biased_to_f16(hi, 0x4140), biased_to_f16(hi, 0x4342)};
#pragma unroll
        for (int b = 0; b < kNB; ++b) mma_f16(s.o[b][2 * d + e], a, pk[b][kk][0], pk[b][kk][1]);
      }
    }
  }
}

// 32 bf16 columns: two 64-dim sub-tiles of 32 rows x 128 bytes per operand.
template <int kNB>
__device__ __forceinline__ void tail_scores(const uint8_t* kb, const uint2 (*qbf)[2][32], int g,
                                            int t, float (&c)[kNB][2][4]) {
  const int pg = perm(g), lane = lane_id();
#pragma unroll
  for (int b = 0; b < kNB; ++b)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) c[b][j][i] = 0.f;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int cc = 0; cc < 2; ++cc)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint8_t* row =
            kb + h * (kTile / 2) + (16 * j + pg) * 128 + (((2 * t + cc) ^ pg) << 4);
        const uint4 x = lds128(row), y = lds128(row + 8 * 128);
        const uint32_t a0[4] = {x.x, y.x, x.y, y.y}, a1[4] = {x.z, y.z, x.w, y.w};
#pragma unroll
        for (int b = 0; b < kNB; ++b) {
          const uint2 q0 = qbf[4 * h + 2 * cc][b][lane], q1 = qbf[4 * h + 2 * cc + 1][b][lane];
          mma_bf16(c[b][j], a0, q0.x, q0.y);
          mma_bf16(c[b][j], a1, q1.x, q1.y);
        }
      }
}

// V rows that no row of the tile sees (seen) read as zero, so what stands in
// masked columns never reaches the sums.
template <int kNB>
__device__ __forceinline__ void tail_values(const uint8_t* vb, const uint32_t (&pk)[kNB][2][2],
                                            uint32_t seen, int g, int t, State<kNB>& s) {
  const int pg = perm(g);
  const uint8_t* vsub = vb + (pg >> 2) * (kTile / 2);
#pragma unroll
  for (int kk = 0; kk < 2; ++kk)
#pragma unroll
    for (int cc = 0; cc < 2; ++cc) {
      uint32_t w[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 16 * kk + 4 * i + t;
        uint4 v = lds128(vsub + r * 128 + (((2 * (pg & 3) + cc) ^ (r & 7)) << 4));
        if (!((seen >> r) & 1u)) v = make_uint4(0u, 0u, 0u, 0u);
        w[i][0] = v.x;
        w[i][1] = v.y;
        w[i][2] = v.z;
        w[i][3] = v.w;
      }
#pragma unroll
      for (int d = 0; d < 4; ++d) {  // dims 8 cc + 2 d, + 1
        const uint32_t a[4] = {__byte_perm(w[0][d], w[1][d], 0x5410),
                               __byte_perm(w[0][d], w[1][d], 0x7632),
                               __byte_perm(w[2][d], w[3][d], 0x5410),
                               __byte_perm(w[2][d], w[3][d], 0x7632)};
#pragma unroll
        for (int b = 0; b < kNB; ++b) mma_bf16(s.o[b][4 * cc + d], a, pk[b][kk][0], pk[b][kk][1]);
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
        l > 0.f ? (m - kPShift + __log2f(l)) * 0.69314718055994530942f : -INFINITY;
}

// Q rows of the tile in MMA fragment order: MMA 4 h + w covers dims
// 64 h + 16 t + 4 w..+3 of lane group t; lane 4 g + t has row g of the block.
// Thread: 8 dims of a row.
__device__ __forceinline__ uint4 load_q(const Params& p, int kvh, int row0, int n_rows) {
  const int r = threadIdx.x >> 4, c = threadIdx.x & 15;
  if (r >= n_rows) return make_uint4(0u, 0u, 0u, 0u);
  const int i = row0 + r, q = i / p.group;
  return *reinterpret_cast<const uint4*>(p.q + int64_t(q) * p.q_row_stride +
                                         int64_t(kvh * p.group + i - q * p.group) *
                                             p.q_head_stride + 8 * c);
}

template <int kNB>
__device__ __forceinline__ void stage_q(Smem& sm, uint4 v) {
  const int tid = threadIdx.x;
  if (tid >= 8 * kNB * 16) return;
  const int r = tid >> 4, c = tid & 15;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = __vmaxu2(top, w[i] & 0x7FFF7FFFu);
  top = max(top & 0xFFFFu, top >> 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  // the power of two at or below the row's largest |q|, as a float's exponent
  const uint32_t e = min(max((top & 0x7F80u) << 16, 27u << 23), 227u << 23);
  const float inv = __uint_as_float((254u << 23) - e);
  if (c == 0) sm.unit[r] = __uint_as_float(e);
  const int h = c >> 3, t = (c & 7) >> 1, k0 = 4 * h + 2 * (c & 1);
  const int lane = (r & 7) * 4 + t, block = r >> 3;
#pragma unroll
  for (int i = 0; i < 2; ++i) {  // dims 8 c + 4 i..+3: MMA k0 + i
    uint32_t f[2];
#pragma unroll
    for (int k = 0; k < 2; ++k)
      f[k] = pack_f16x2(__uint_as_float(w[2 * i + k] << 16) * inv,
                        __uint_as_float(w[2 * i + k] & 0xFFFF0000u) * inv);
    sm.q16[k0 + i][block][lane] = make_uint2(f[0], f[1]);
    sm.qbf[k0 + i][block][lane] = make_uint2(w[2 * i], w[2 * i + 1]);
  }
}

__device__ __forceinline__ uint32_t cluster_addr(const void* p, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void st_cluster_v4(uint32_t a, float4 v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(a), "f"(v.x), "f"(v.y),
               "f"(v.z), "f"(v.w)
               : "memory");
}
__device__ __forceinline__ void st_cluster_v2(uint32_t a, float x, float y) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(a), "f"(x), "f"(y) : "memory");
}
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

// CTA (split, KV head, tile of 8 kNB packed rows); sealed steps of 16 NT columns
template <int kNB, int NT>
__global__ void __launch_bounds__(kThreads, 1)
    rows_kernel(const __grid_constant__ CUtensorMap tm_k8,
                const __grid_constant__ CUtensorMap tm_v8,
                const __grid_constant__ CUtensorMap tm_kt,
                const __grid_constant__ CUtensorMap tm_vt, const Params p, const Split sp) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  // (offset from the array, so that the compiler knows these are shared loads)
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw + ((0u - smem_u32(smem_raw)) & 1023u));
  const int warp = warp_id(), lane = lane_id();
  const int g = lane >> 2, t = lane & 3, pg = perm(g);
  if (threadIdx.x == 0) sm.abort = 0;
  if (lane < kBuf) mbar_init(&sm.full[warp][lane], 1);
  fence_barrier_init();
  __syncwarp();
  const bool cluster = sp.splits > 1 && !sp.partials;
  if (cluster) cluster_arrive();  // waited for before anything is written to another CTA
  pdl_wait_then_release();  // launched with launch_pdl: nothing global is read before
  volatile int* abort = &sm.abort;
  const int kvh = blockIdx.y;
  constexpr int kRows = 8 * kNB;
  const int row0 = int(blockIdx.z) * kRows;  // first packed row
  const int n_rows = min(kRows, p.q_len * p.group - row0);
  // a tile's rows lie in one query tile: 128 group is a multiple of 16
  const int qt = (row0 / p.group) >> 7;
  const uint4 q_dims = load_q(p, kvh, row0, n_rows);
  Walk walk;
  walk.list = p.blk_list + size_t(qt) * p.n_kv128;
  walk.n_units = (NT == 4 ? 2 : 4) * p.blk_count[qt];
  walk.room = p.n_kv128;
  walk.stride = sp.splits * kWarps;
  walk.u = int(blockIdx.x) * kWarps + warp;
  walk.ahead = list_entry<NT>(walk, walk.u);
  uint8_t* ring = sm.ring[warp];
  // operand tile i (K of step n: 2 n, V: 2 n + 1) into buffer i % kBuf
  int issued = 0;
  int fill = 0;  // issued % kBuf
  auto issue = [&](const Step& c, bool is_v) {
    if (lane == 0) {
      uint64_t* bar = &sm.full[warp][fill];
      uint8_t* dst = ring + fill * kTile;
      mbar_arrive_expect_tx(bar, c.tail ? kTile : 16 * NT * HD);
      if (c.tail) {
        for (int h = 0; h < 2; ++h)
          tma_load_3d(dst + h * (kTile / 2), is_v ? &tm_vt : &tm_kt, bar, 64 * h,
                      c.col - p.tail_row0, kvh);
      } else {
        tma_load_3d(dst, is_v ? &tm_v8 : &tm_k8, bar, 0, c.col, kvh);
      }
    }
    ++issued;
    fill = fill + 1 == kBuf ? 0 : fill + 1;
  };
  Step none;
  none.col = -1;
  none.tail = none.second = none.partial = false;
  Step cur = next_step<NT>(p, walk, none);
  if (cur.col >= 0) {
    issue(cur, false);
    issue(cur, true);
  }
  int mrow[2 * kNB];  // the lane's rows in the query tile, -1: no such row
#pragma unroll
  for (int r = 0; r < 2 * kNB; ++r) {
    const int i = 8 * (r >> 1) + 2 * t + (r & 1);
    mrow[r] = i < n_rows ? ((row0 + i) / p.group) & 127 : -1;
  }
  Aside<kNB> a;  // of the current step
  if (cur.col >= 0) load_aside<kNB>(p, cur, kvh, qt, mrow, a);
  stage_q<kNB>(sm, q_dims);
  Step nxt = none;
  if (cur.col >= 0) nxt = next_step<NT>(p, walk, cur);
  if (nxt.col >= 0) issue(nxt, false);
  __syncthreads();  // Q fragments and the abort word

  State<kNB> s;
  s.unit = s.unit_max = 0.f;
  float q_unit[2 * kNB];  // the rows' score factors
#pragma unroll
  for (int r = 0; r < 2 * kNB; ++r) {
    s.m[r] = -INFINITY;
    s.l[r] = 0.f;
    q_unit[r] = p.scale_log2 * sm.unit[8 * (r >> 1) + 2 * t + (r & 1)];
  }
#pragma unroll
  for (int b = 0; b < kNB; ++b)
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) s.o[b][i][k] = 0.f;

  int used = 0;  // tiles used
  int at = 0;    // used % kBuf
  uint32_t parity = 0;
  bool ok = true;
  auto wait_tile = [&](int32_t where) {
    ok = __all_sync(0xffffffffu, mbar_wait(&sm.full[warp][at], parity, abort, p.status, where));
    return ok;
  };
  auto done_tile = [&]() {  // every lane has read the tile
    __syncwarp();
    ++used;
    if (++at == kBuf) {
      at = 0;
      parity ^= 1u;
    }
  };
  while (cur.col >= 0) {
    Step after = none;  // the step after next
    if (nxt.col >= 0) after = next_step<NT>(p, walk, nxt);
    uint64_t all = ~0ull, some = 0ull;
#pragma unroll
    for (int r = 0; r < 2 * kNB; ++r) {
      all &= a.bits[r];
      if (mrow[r] >= 0) some |= a.bits[r];
    }
    if (NT == 2 || cur.tail) all |= 0xffffffff00000000ull;
    const bool masked = __any_sync(0xffffffffu, all != ~0ull);
    const bool any = !masked || __any_sync(0xffffffffu, some != 0ull);
    if (!wait_tile(0x800)) break;
    // one step of 64 sealed or 32 bf16 columns
    if (cur.tail) {
      float c[kNB][2][4];
      tail_scores<kNB>(ring + at * kTile, sm.qbf, g, t, c);
      done_tile();
      if (nxt.col >= 0) issue(nxt, true);
      uint32_t pk[kNB][2][2];
      float sc[2 * kNB];
#pragma unroll
      for (int r = 0; r < 2 * kNB; ++r) sc[r] = p.scale_log2;
      if (any) softmax_step<kNB, 2, false>(c, a.bits, masked, sc, 1.f, pg, s, pk);
      // columns that some row sees
      const uint32_t seen = __reduce_or_sync(0xffffffffu, uint32_t(some));
      if (nxt.col >= 0) load_aside<kNB>(p, nxt, kvh, qt, mrow, a);
      if (!wait_tile(0x801)) break;
      if (any) tail_values<kNB>(ring + at * kTile, pk, seen, g, t, s);
    } else {
      float c[kNB][NT][4];
      sealed_scores<kNB, NT>(ring + at * kTile, sm.q16, g, t, c);
      done_tile();
      if (nxt.col >= 0) issue(nxt, true);
      uint32_t pk[kNB][NT][2];
      float sc[2 * kNB];
#pragma unroll
      for (int r = 0; r < 2 * kNB; ++r) sc[r] = score_factor(a.ks * q_unit[r]);
      if (any) softmax_step<kNB, NT, true>(c, a.bits, masked, sc, a.vs, pg, s, pk);
      if (nxt.col >= 0) load_aside<kNB>(p, nxt, kvh, qt, mrow, a);
      if (!wait_tile(0x802)) break;
      if (any) sealed_values<kNB, NT>(ring + at * kTile, pk, g, t, s);
    }
    done_tile();
    if (after.col >= 0) issue(after, false);
    cur = nxt;
    nxt = after;
  }
  if (!ok)  // copies in flight must land before the CTA's memory goes
    for (; used < issued; ++used)
      mbar_wait(&sm.full[warp][used % kBuf], uint32_t(used / kBuf) & 1u, abort, p.status, 0x803,
                false);

  // ---- join the CTA's warps
#pragma unroll
  for (int r = 0; r < 2 * kNB; ++r) {
    const int b = r >> 1, e = r & 1, row = 8 * b + 2 * t + e;
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) s.l[r] += __shfl_xor_sync(0xffffffffu, s.l[r], o);
    if (g == 0) sm.ml[warp][row] = make_float2(s.m[r], s.l[r]);
    float* dst = reinterpret_cast<float*>(ring) + row * (HD + 4) + 16 * pg;
#pragma unroll
    for (int i = 0; i < 8; i += 2)
      *reinterpret_cast<float4*>(dst + 2 * i) =
          make_float4(s.o[b][i][e] * s.unit, s.o[b][i][2 + e] * s.unit,
                      s.o[b][i + 1][e] * s.unit, s.o[b][i + 1][2 + e] * s.unit);
  }
  __syncthreads();
  const size_t tile = size_t(kvh) * gridDim.z + blockIdx.z;
  float* rec = sp.partials ? sp.partials + (tile * sp.splits + blockIdx.x) * kRecord : nullptr;
  const int per_cta = (kRows + sp.splits - 1) / sp.splits;
  if (cluster) cluster_wait();
  for (int idx = threadIdx.x; idx < n_rows * 32; idx += kThreads) {
    const int r = idx >> 5, d4 = idx & 31;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, sm.ml[w][r].x);
    const float nm = m == -INFINITY ? 0.f : -m;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float2 x = sm.ml[w][r];
      const float f = ex2_approx(x.x + nm);
      const float4 v = *reinterpret_cast<const float4*>(
          reinterpret_cast<const float*>(sm.ring[w]) + r * (HD + 4) + 4 * d4);
      l += x.y * f;
      acc.x += v.x * f;
      acc.y += v.y * f;
      acc.z += v.z * f;
      acc.w += v.w * f;
    }
    if (rec) {
      *reinterpret_cast<float4*>(rec + r * HD + 4 * d4) = acc;
      if (d4 == 0) reinterpret_cast<float2*>(rec + kMaxRows * HD)[r] = make_float2(m, l);
    } else if (cluster) {
      const int to = r % sp.splits, at_row = int(blockIdx.x) * per_cta + r / sp.splits;
      st_cluster_v4(cluster_addr(&sm.in_rows[at_row][d4], uint32_t(to)), acc);
      if (d4 == 0) st_cluster_v2(cluster_addr(&sm.in_ml[at_row], uint32_t(to)), m, l);
    } else {
      store_row(p, kvh, row0 + r, d4, acc, m, l);
    }
  }
  if (!cluster) return;
  // ---- join the cluster's CTAs: rows dealt out, each now in its CTA's memory
  cluster_arrive();
  cluster_wait();
  for (int i = warp; int(blockIdx.x) + sp.splits * i < n_rows; i += kWarps) {
    float2 x[kMaxCluster];
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < kMaxCluster; ++k) {
      x[k] = k < sp.splits ? sm.in_ml[k * per_cta + i] : make_float2(-INFINITY, 0.f);
      m = fmaxf(m, x[k].x);
    }
    const float nm = m == -INFINITY ? 0.f : -m;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
#pragma unroll
    for (int k = 0; k < kMaxCluster; ++k) {
      if (k >= sp.splits) break;
      const float4 v = sm.in_rows[k * per_cta + i][lane];
      const float f = ex2_approx(x[k].x + nm);
      l += x[k].y * f;
      acc.x += v.x * f;
      acc.y += v.y * f;
      acc.z += v.z * f;
      acc.w += v.w * f;
    }
    store_row(p, kvh, row0 + int(blockIdx.x) + sp.splits * i, lane, acc, m, l);
  }
}

// Join the splits: CTA (packed row, KV head), its warps the splits in turn, lane
// = 4 dims.  Latency: 4 us behind the rows kernel for 18 splits.
constexpr int kJoinWarps = 8;
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(const Params p, const Split sp) {
  pdl_wait_then_release();  // launched with launch_pdl
  __shared__ float4 acc_s[kJoinWarps][32];
  __shared__ float2 ml_s[kJoinWarps];
  const int row = blockIdx.x, kvh = blockIdx.y, warp = warp_id(), d4 = lane_id();
  const int r = row % sp.rows;
  const float* rec0 =
      sp.partials + (size_t(kvh) * sp.n_tiles + row / sp.rows) * sp.splits * kRecord;
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int kAt = 8;  // records in flight
  for (int i0 = warp; i0 < sp.splits; i0 += kJoinWarps * kAt) {
    float2 x[kAt];
    float4 v[kAt];
#pragma unroll
    for (int k = 0; k < kAt; ++k) {
      const int i = i0 + k * kJoinWarps;
      x[k] = make_float2(-INFINITY, 0.f);
      v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i < sp.splits) {
        const float* rec = rec0 + size_t(i) * kRecord;
        x[k] = __ldcg(reinterpret_cast<const float2*>(rec + kMaxRows * HD) + r);
        v[k] = __ldcg(reinterpret_cast<const float4*>(rec + r * HD) + d4);
      }
    }
    float m_new = m;
#pragma unroll
    for (int k = 0; k < kAt; ++k) m_new = fmaxf(m_new, x[k].x);
    const float nm = m_new == -INFINITY ? 0.f : -m_new;
    const float a = ex2_approx(m + nm);
    l *= a;
    acc.x *= a;
    acc.y *= a;
    acc.z *= a;
    acc.w *= a;
#pragma unroll
    for (int k = 0; k < kAt; ++k) {
      const float f = ex2_approx(x[k].x + nm);
      l += x[k].y * f;
      acc.x += v[k].x * f;
      acc.y += v[k].y * f;
      acc.z += v[k].z * f;
      acc.w += v[k].w * f;
    }
    m = m_new;
  }
  acc_s[warp][d4] = acc;
  if (d4 == 0) ml_s[warp] = make_float2(m, l);
  __syncthreads();
  if (warp > 0) return;
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) top = fmaxf(top, ml_s[w].x);
  const float nm = top == -INFINITY ? 0.f : -top;
  l = 0.f;
  acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) {
    const float2 x = ml_s[w];
    const float4 v = acc_s[w][d4];
    const float f = ex2_approx(x.x + nm);
    l += x.y * f;
    acc.x += v.x * f;
    acc.y += v.y * f;
    acc.z += v.z * f;
    acc.w += v.w * f;
  }
  store_row(p, kvh, row, d4, acc, top, l);
}

}  // namespace kv8r
}  // namespace hsd

namespace hsd_host {

using namespace hsd;

namespace {
constexpr int kMaxDevices = 64;
std::atomic<bool> g_attr_set[2][2][kMaxDevices];  // [16 rows][steps of 32][device]

auto rows_kernel_of(bool wide, bool fine) {
  if (fine) return wide ? kv8r::rows_kernel<2, 2> : kv8r::rows_kernel<1, 2>;
  return wide ? kv8r::rows_kernel<2, 4> : kv8r::rows_kernel<1, 4>;
}

int set_rows_attribute(bool wide, bool fine, int dev) {
  if (g_attr_set[wide][fine][dev].load(std::memory_order_acquire)) return HSD_OK;
  int rc = cuda_check(
      cudaFuncSetAttribute(rows_kernel_of(wide, fine), cudaFuncAttributeMaxDynamicSharedMemorySize,
                           int(kv8r::kSmem)),
      "cudaFuncSetAttribute(rows_kernel)");
  if (rc == HSD_OK)
    rc = cuda_check(cudaFuncSetAttribute(rows_kernel_of(wide, fine),
                                         cudaFuncAttributeNonPortableClusterSizeAllowed, 1),
                    "cudaFuncSetAttribute(rows_kernel)");
  if (rc == HSD_OK) g_attr_set[wide][fine][dev].store(true, std::memory_order_release);
  return rc;
}

// Packed rows of a tile: 8 when they are all, else 16.
int tile_rows(int q_len, int group) { return int64_t(q_len) * group <= 8 ? 8 : 16; }
int n_tiles(int q_len, int group) {
  const int r = tile_rows(q_len, group);
  return int((int64_t(q_len) * group + r - 1) / r);
}
// What the current device runs at once, looked up once per device.
struct Device {
  int sms = 148;
  int clusters[2][kv8r::kMaxCluster + 1];  // [16 rows][CTAs of a cluster]
};

// Clusters of s CTAs at once, 0 if none: SMs of a cluster lie in one group of the
// chip, so this is less than SMs / s.
int resident_clusters(bool wide, int s, int dev, int sms) {
  if (s == 1) return sms;
  if (set_rows_attribute(wide, false, dev) != HSD_OK) return 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(s * sms));
  cfg.blockDim = dim3(kv8r::kThreads);
  cfg.dynamicSmemBytes = kv8r::kSmem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(s);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  return cudaOccupancyMaxActiveClusters(&n, rows_kernel_of(wide, false), &cfg) == cudaSuccess ? n : 0;
}

const Device& current_device() {
  static Device table[kMaxDevices + 1];  // the last: no device
  static std::once_flag once[kMaxDevices + 1];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) {
    cudaGetLastError();
    dev = kMaxDevices;
  }
  std::call_once(once[dev], [dev] {
    Device& d = table[dev];
    int n = 0;
    if (dev < kMaxDevices &&
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && n > 0)
      d.sms = n;
    for (int wide = 0; wide < 2; ++wide)
      for (int s = 1; s <= kv8r::kMaxCluster; ++s)
        d.clusters[wide][s] =
            dev < kMaxDevices ? resident_clusters(wide, s, dev, d.sms) : 0;
    cudaGetLastError();
  });
  return table[dev];
}

// CTAs per tile, columns per step, and what the launch then takes.  A launch takes
// about 4.2 us (16 rows a tile: 5.2) and 2.7 us (3.4) for each step of a warp, 2 us (2.5)
// if sealed steps have 32 columns instead of 64: those pay where every warp then has
// one.  So the time goes by the waves of clusters and the steps; the join kernel (2 us)
// lets CTAs be dealt out without regard to clusters, or more than kMaxCluster of them
// to a tile.  Measured, 12/2 heads, one row: 1601 columns 5.6 us with steps of 32 (of
// 64: 6.4), 4097 columns 6.8 with a cluster of 9 and steps of 64 (of 32: 7.6; cluster of
// 8: 9.4), 8193 columns 7.0 with 33 CTAs, steps of 32 and the join (cluster of 16, steps
// of 64: 9.6).
Kv8RowsChoice choose(int q_len, int kv_len, int hq, int hkv) {
  const Device& dev = current_device();
  const int64_t tiles = int64_t(n_tiles(q_len, hq / hkv)) * hkv;
  const bool wide = tile_rows(q_len, hq / hkv) > 8;
  const float step_us[2][2] = {{2.7f, 2.f}, {3.4f, 2.5f}};  // [16 rows][steps of 32]
  Kv8RowsChoice best{1, false, false, 3.0e38f, dev.sms};
  for (int fine = 0; fine < 2; ++fine) {
    const int units = (kv_len + (fine ? 31 : 63)) / (fine ? 32 : 64);
    const int most = (units + kv8r::kWarps - 1) / kv8r::kWarps;
    auto consider = [&](int s, bool join, int64_t waves) {
      const int steps = (units + s * kv8r::kWarps - 1) / (s * kv8r::kWarps);
      const float us = float(waves) * ((wide ? 5.2f : 4.2f) + step_us[wide][fine] * float(steps)) +
                       (join ? 2.f : 0.f);
      if (us < best.us) best = {s, join, fine != 0, us, dev.sms};
    };
    consider(1, false, (tiles + dev.sms - 1) / dev.sms);
    for (int s = 2; s <= kv8r::kMaxCluster && s <= most; ++s)
      if (const int at_once = dev.clusters[wide][s])
        consider(s, false, (tiles + at_once - 1) / at_once);
    const int64_t s = std::min<int64_t>(dev.sms / tiles, most);
    if (s > 1) consider(int(s), true, 1);
  }
  return best;
}
}  // namespace

Kv8RowsChoice kv8_rows_choose(int q_len, int kv_len, int hq, int hkv) {
  return choose(q_len, kv_len, hq, hkv);
}

size_t kv8_rows_workspace_bytes(int q_len, int hq, int hkv, const Kv8RowsChoice& c) {
  if (!c.join) return 256;  // nothing, but a workspace all the same
  return size_t(n_tiles(q_len, hq / hkv)) * hkv * c.splits * kv8r::kRecord * sizeof(float);
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

int kv8_rows_launch(const Kv8AttnArgs& a, const Kv8RowsChoice& c) {
  const hsd::kv8a::Params& p = a.p;
  CUtensorMap k8, v8, kt, vt;
  const int64_t tail_rows = p.kv_len - p.tail_row0;
  const bool has8 = p.sealed > 0, has_tail = p.sealed < p.kv_len;
  const int box = c.fine ? 32 : 64;  // rows of a sealed step
  // a side without columns is never loaded; its map describes the other one
  int rc = HSD_OK;
  if (has8) {
    rc = kv8_map(&k8, a.k8, false, p.sealed, p.hkv, 128, a.k8_head_stride, box, "k8");
    if (!rc) rc = kv8_map(&v8, a.v8, false, p.sealed, p.hkv, 128, a.v8_head_stride, box, "v8");
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
  sp.rows = tile_rows(p.q_len, p.group);
  sp.splits = c.splits;
  sp.partials = c.join ? static_cast<float*>(a.workspace) : nullptr;
  if (sp.n_tiles > 65535 || p.hkv > 65535) {
    set_error("hsd_verify_attention_kv8: %d rows x %d heads exceed the launch's range", p.q_len,
              p.hq);
    return HSD_ERR_TOO_LARGE;
  }
  int dev = 0;
  rc = cuda_check(cudaGetDevice(&dev), "cudaGetDevice");
  if (rc) return rc;
  if (dev < 0 || dev >= kMaxDevices) {
    set_error("hsd_verify_attention_kv8: device ordinal %d >= %d", dev, kMaxDevices);
    return HSD_ERR_UNSUPPORTED;
  }
  const bool wide = sp.rows > 8;
  rc = set_rows_attribute(wide, c.fine, dev);
  if (rc) return rc;
  rc = launch_pdl(rows_kernel_of(wide, c.fine),
                  dim3(unsigned(sp.splits), unsigned(p.hkv), unsigned(sp.n_tiles)),
                  dim3(kv8r::kThreads), kv8r::kSmem, a.stream, "rows_kernel launch",
                  c.splits > 1 && !c.join ? unsigned(c.splits) : 0u, k8, v8, kt, vt, p, sp);
  if (rc || !sp.partials) return rc;
  return launch_pdl(kv8r::join_kernel,
                    dim3(unsigned(p.q_len * p.group), unsigned(p.hkv)),
                    dim3(kv8r::kJoinWarps * 32), 0, a.stream, "join_kernel launch", 0, p, sp);
}

}  // namespace hsd_host
