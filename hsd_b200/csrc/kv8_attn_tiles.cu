// Attention over the 8-bit cache for many query rows: tcgen05 tiles.
//
// One CTA = one 128-row query tile x two query heads of a KV group (slots),
// walking the tile's 128-column blocks; stream-K over one CTA per SM
// (attn_schedule.cuh).  Roles (24 warps):
//
//   warps 0-15  softmax: slot = warp / 8, column half = warp / 4 % 2, thread =
//               (row, 64 columns).  Two threads share a row, so every
//               scheduler has two warps of each slot to hide latency with;
//               they exchange the row's maximum through shared memory
//   warp 16     Q loader (TMA)
//   warps 17-18 MMA issuers, one thread per slot
//   warps 20-23 producers: 64-column halves that are sealed are loaded as int8
//               (16 bytes a lane, the next tile's loads in flight during this
//               tile's conversion), converted to bf16 exactly and written in
//               the MMA's 128-byte-swizzled layout; bf16 halves are copied
//
// TMEM (512 columns): slot s has S (fp32, 128 columns) at 256 s and O at
// 256 s + 128.  P (bf16, 64 columns) overwrites S and is the A operand of the
// PV MMA straight from tensor memory: shared-memory operand reads are what
// 128-column MMAs saturate (128 bytes per cycle), and the conversion's writes
// need room there.  One thread issues PV(j) then S(j+1), which run in that
// order, so S(j+1) complete implies PV(j) complete: a slot needs two barriers
// per block (S full, P full), its softmax runs under the other slot's MMAs,
// and O may be rescaled as soon as S is there.
//
// Scales: the half's K scale multiplies the scores; the V scale enters the
// exponent as its logarithm, so P carries it at no cost, and the half's row
// sum is divided by it again.  P is truncated to bf16 with the bias taken out
// of the exponent and the sum (truncation lowers a value by 0.282 % on
// average); sums and the running maximum are fp32.
//
// Items cut between CTAs: later pieces publish O / l in fp16 with a power of
// two per (row, half) -- 2^-12 of the row's largest value, where bf16 would
// add as much error as P's rounding -- and the owner of the first piece
// merges them.
#include <atomic>

#include "attn_schedule.cuh"
#include "kv8_attn.cuh"

#include <cuda_fp16.h>

namespace hsd {
namespace kv8t {

using kv8a::HD;

constexpr int BM = 128;
constexpr int BN = 128;
constexpr int NSLOT = 2;
constexpr int NSTAGE = 4;
constexpr int TILE_BYTES = BN * HD * 2;
constexpr int SUB_BYTES = 128 * 128;
constexpr int kSoftmaxThreads = 512;
constexpr int kThreads = 768;
constexpr int kMaxTiles = 1024;
constexpr float kRescaleLog2 = 8.0f;
constexpr float kPackBiasLog2 = 0.0040626743f;  // log2(1.00282)
constexpr float kPackBiasInv = 0.99718800f;     // 1 / 1.00282
// Partial record of one (CTA, slot): O / l in fp16 as [half][8 chunks][128
// rows] of 16 bytes, then (m, l, unit, 0) per (half, row).
constexpr int kRecData = 2 * 8 * 128 * 16;
constexpr int kRecBytes = kRecData + 2 * 128 * 16;

struct __align__(1024) Smem {
  uint8_t q[NSLOT][TILE_BYTES];
  uint8_t kv[NSTAGE][TILE_BYTES];
  float mx[NSLOT][2][128];  // block maxima of the two halves of a row
  float lx[NSLOT][2][128];  // their row sums, at the end of a piece
  uint64_t bar_q;
  uint64_t bar_q_free;
  uint64_t bar_full[NSTAGE];
  uint64_t bar_empty[NSTAGE];
  uint64_t bar_s_full[NSLOT];
  uint64_t bar_p_full[NSLOT];
  uint64_t bar_o_done[NSLOT];
  uint64_t bar_o_free[NSLOT];
  uint64_t bar_final[NSLOT];
  uint32_t tmem_base;
  int abort;
};
static_assert(sizeof(Smem) + 1024 <= 232448, "shared memory budget exceeded");

struct Params : kv8a::Params {
  const int32_t* tile_order;
  const int32_t* blk_prefix;
  const int8_t* k8;
  const int8_t* v8;
  int64_t k8_head_stride, v8_head_stride;
  const __nv_bfloat16* k_tail;
  const __nv_bfloat16* v_tail;
  int64_t kt_row_stride, kt_head_stride, vt_row_stride, vt_head_stride;
  uint8_t* partials;  // [G][NSLOT][kRecBytes]
  uint32_t* flags;    // [G][NSLOT][8]: rows of softmax warp w published (= generation + 1)
  uint32_t* sync;     // {generation, CTAs finished}
  int pairs, n_qtiles;
};

constexpr uint32_t kIdescS = idesc_bf16_f32(BM, BN, false, false);  // Q K^T
constexpr uint32_t kIdescO = idesc_bf16_f32(BM, HD, false, true);   // P V, V is MN-major

__device__ __forceinline__ void issue_s(uint32_t d_tmem, uint32_t q_smem, uint32_t k_smem) {
  const uint64_t a = sdesc_sw128(q_smem, 16, 1024);
  const uint64_t b = sdesc_sw128(k_smem, 16, 1024);
#pragma unroll
  for (int kk = 0; kk < HD / 16; ++kk) {
    const uint64_t off = uint64_t(((kk >> 2) * SUB_BYTES + (kk & 3) * 32) >> 4);
    umma_bf16_ss(d_tmem, a + off, b + off, kIdescS, kk > 0);
  }
}

// A from TMEM: 16 columns of K are 8 words.
__device__ __forceinline__ void issue_pv(uint32_t d_tmem, uint32_t p_tmem, uint32_t v_smem,
                                         bool acc) {
  const uint64_t b = sdesc_sw128(v_smem, SUB_BYTES, 1024);
#pragma unroll
  for (int kk = 0; kk < BN / 16; ++kk)
    umma_bf16_ts(d_tmem, p_tmem + kk * 8, b + uint64_t((kk * 2048) >> 4), kIdescO,
                 (acc || kk > 0) ? 1u : 0u);
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 unpack_f16x2(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ float log2_approx(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The producers' walk: K then V tile of every block of every piece.
struct Feed {
  int w, w1;
  attn::Piece pc;
  int j, kb;
  uint32_t entry;
  bool is_v;
};

__device__ __forceinline__ bool feed_next(const Params& p, Feed& f, bool first) {
  if (!first && !f.is_v) {
    f.is_v = true;
    return true;
  }
  if (first || f.j + 1 == f.pc.b1) {
    if (!attn::next_piece(p, f.w, f.w1, f.pc)) return false;
    f.j = f.pc.b0;
  } else {
    ++f.j;
  }
  f.is_v = false;
  f.entry = p.blk_list[size_t(f.pc.qt) * p.n_kv128 + f.j];
  f.kb = int(f.entry & 0xFFFFFFu);
  return true;
}

__device__ __forceinline__ bool half_sealed(const Params& p, const Feed& f, int hf) {
  return f.kb * BN + 64 * hf < p.sealed;
}

// int8 loads of half hf: lane (row, 16 dims), 32 rows x 64 dims a step.
__device__ __forceinline__ void load_half(const Params& p, const Feed& f, int hf, int ct,
                                          uint4 (&buf)[4]) {
  const int8_t* src = (f.is_v ? p.v8 + f.pc.kvh * p.v8_head_stride
                              : p.k8 + f.pc.kvh * p.k8_head_stride) +
                      int64_t(f.kb * BN + 64 * hf + (ct >> 2)) * HD + (ct & 3) * 16;
#pragma unroll
  for (int u = 0; u < 4; ++u)
    buf[u] = __ldg(reinterpret_cast<const uint4*>(src + (u >> 1) * (32 * HD) + (u & 1) * 64));
}

__device__ __forceinline__ void convert_half(uint32_t stage, int hf, int ct,
                                             const uint4 (&buf)[4]) {
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int row = 64 * hf + 32 * (u >> 1) + (ct >> 2);
    const uint32_t base = stage + uint32_t((u & 1) * SUB_BYTES + row * 128);
    const int c = 2 * (ct & 3);
    uint32_t o[8];
    kv8a::bytes_to_bf16(buf[u].x, o[0], o[1]);
    kv8a::bytes_to_bf16(buf[u].y, o[2], o[3]);
    kv8a::bytes_to_bf16(buf[u].z, o[4], o[5]);
    kv8a::bytes_to_bf16(buf[u].w, o[6], o[7]);
    st_shared_v4(base + (uint32_t(c ^ (row & 7)) << 4), o[0], o[1], o[2], o[3]);
    st_shared_v4(base + (uint32_t((c + 1) ^ (row & 7)) << 4), o[4], o[5], o[6], o[7]);
  }
}

// bf16 rows of half hf; columns past kv_len, and V rows of columns that no
// row of the query tile sees, are zero.
__device__ __forceinline__ void copy_half(const Params& p, const Feed& f, uint32_t stage, int hf,
                                          int ct) {
  const int col0 = f.kb * BN + 64 * hf;
  uint64_t seen = ~0ull;
  if (f.is_v) {
    if (!((f.entry >> (24 + 2 * hf)) & 1u)) {
      seen = 0ull;
    } else if ((f.entry >> (25 + 2 * hf)) & 1u) {
      const uint64_t* words = p.mask_words + (size_t(f.pc.qt) * p.n_kv64 + 2 * f.kb + hf) * 128;
      uint64_t w = 0ull;
#pragma unroll
      for (int k = 0; k < 4; ++k) w |= words[lane_id() + 32 * k];
      seen = uint64_t(__reduce_or_sync(0xffffffffu, uint32_t(w))) |
             (uint64_t(__reduce_or_sync(0xffffffffu, uint32_t(w >> 32))) << 32);
    }
  }
  const int64_t rs = f.is_v ? p.vt_row_stride : p.kt_row_stride;
  const __nv_bfloat16* src = (f.is_v ? p.v_tail + f.pc.kvh * p.vt_head_stride
                                     : p.k_tail + f.pc.kvh * p.kt_head_stride) +
                             int64_t(col0 - p.tail_row0) * rs + (ct & 15) * 8;
  const uint32_t base = stage + uint32_t(((ct >> 3) & 1) * SUB_BYTES);
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r = 8 * (4 * b + u) + (ct >> 4);
      v[u] = make_uint4(0u, 0u, 0u, 0u);
      if (col0 + r < p.kv_len && ((seen >> r) & 1ull))
        v[u] = __ldg(reinterpret_cast<const uint4*>(src + r * rs));
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int row = 64 * hf + 8 * (4 * b + u) + (ct >> 4);
      st_shared_v4(base + uint32_t(row * 128) + (uint32_t((ct & 7) ^ (row & 7)) << 4), v[u].x,
                   v[u].y, v[u].z, v[u].w);
    }
  }
}

__global__ void __launch_bounds__(kThreads, 1)
    tiles_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                      ~uintptr_t(1023));
  const int warp = warp_id(), lane = lane_id();
  const int per_tile = p.hkv * p.pairs;

  if (threadIdx.x == 0) {
    mbar_init(&sm.bar_q, 1);
    mbar_init(&sm.bar_q_free, NSLOT);
    for (int i = 0; i < NSTAGE; ++i) {
      mbar_init(&sm.bar_full[i], 128);
      mbar_init(&sm.bar_empty[i], NSLOT);
    }
    for (int i = 0; i < NSLOT; ++i) {
      mbar_init(&sm.bar_s_full[i], 1);
      mbar_init(&sm.bar_p_full[i], 256);
      mbar_init(&sm.bar_o_done[i], 1);
      mbar_init(&sm.bar_o_free[i], 256);
      mbar_init(&sm.bar_final[i], 1);
    }
    sm.abort = 0;
    fence_barrier_init();
  }
  if (warp == 0) {
    tmem_alloc(&sm.tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // launched with launch_pdl: nothing global is read before this point
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const uint32_t tmem = sm.tmem_base;
  volatile int* abort = &sm.abort;
  const int total = p.blk_prefix[p.n_qtiles] * per_tile;
  const int G = gridDim.x;
  const uint32_t gen = __ldcg(p.sync);
  const int w0 = attn::range_start(blockIdx.x, total, G);
  const int w1 = attn::range_start(blockIdx.x + 1, total, G);

  // Registers: launched with 80 x 768 = 61440; softmax 88 x 512 and the other
  // two warpgroups 64 x 256 are 61440 again.
  if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;\n" ::: "memory");
    if (warp >= 20) {
      // ---------------------------------------------------------- producers
      const int ct = int(threadIdx.x) - 640;
      Feed f;
      f.w = w0;
      f.w1 = w1;
      int stage = 0;
      uint32_t phase = 0;
      uint4 buf[2][4];
      bool have = feed_next(p, f, true);
      if (have) {
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
          if (half_sealed(p, f, hf)) load_half(p, f, hf, ct, buf[hf]);
      }
      while (have) {
        const bool ok = __all_sync(0xffffffffu, mbar_wait(&sm.bar_empty[stage], phase ^ 1u, abort,
                                                          p.status, 0x900));
        if (!ok) break;
        const uint32_t dst = smem_u32(sm.kv[stage]);
        Feed nx = f;
        const bool more = feed_next(p, nx, false);
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          if (half_sealed(p, f, hf))
            convert_half(dst, hf, ct, buf[hf]);
          else
            copy_half(p, f, dst, hf, ct);
          if (more && half_sealed(p, nx, hf)) load_half(p, nx, hf, ct, buf[hf]);
        }
        fence_async_shared();  // the tile's bytes -> visible to the MMAs (async proxy)
        mbar_arrive(&sm.bar_full[stage]);
        if (++stage == NSTAGE) {
          stage = 0;
          phase ^= 1u;
        }
        f = nx;
        have = more;
      }
    } else if (warp == 16 && lane == 0) {
      // ---------------------------------------------------------- Q loader
      tma_prefetch_desc(&tm_q);
      int pieces = 0;
      int w = w0;
      attn::Piece pc;
      while (attn::next_piece(p, w, w1, pc)) {
        if (pieces > 0 && !mbar_wait(&sm.bar_q_free, uint32_t(pieces - 1) & 1u, abort, p.status,
                                     0x910))
          break;
        mbar_arrive_expect_tx(&sm.bar_q, pc.nslot * TILE_BYTES);
        for (int s = 0; s < pc.nslot; ++s)
          for (int d = 0; d < 2; ++d)
            tma_load_3d(sm.q[s] + d * SUB_BYTES, &tm_q, &sm.bar_q, d * 64, pc.qt * BM, pc.h0 + s);
        ++pieces;
      }
      // every issued load must land before the CTA exits, also after an abort
      if (pieces > 0)
        mbar_wait(&sm.bar_q, uint32_t(pieces - 1) & 1u, abort, p.status, 0x911, false);
    } else if ((warp == 17 || warp == 18) && lane == 0) {
      // ---------------------------------------------------------- MMA issuers
      const int s = warp - 17;
      const uint32_t qa = smem_u32(sm.q[s]);
      const uint32_t kv0 = smem_u32(sm.kv[0]);
      const uint32_t t_s = tmem + s * 256;
      int stage = 0;
      uint32_t phase = 0;
      int np = 0;      // PV issued (p_full parity)
      int done = 0;    // pieces of this slot (o_free parity)
      int pieces = 0;  // all pieces (bar_q parity)
      bool issued_any = false;
      bool ok = true;
      auto advance = [&]() {
        if (++stage == NSTAGE) {
          stage = 0;
          phase ^= 1u;
        }
      };
      int w = w0;
      attn::Piece pc;
      while (ok && attn::next_piece(p, w, w1, pc)) {
        const int n = pc.b1 - pc.b0;
        if (s >= pc.nslot) {  // no head in slot 1: skip the piece's tiles
          for (int i = 0; i < 2 * n; ++i) advance();
          ++pieces;
          continue;
        }
        const int rel = pc.nslot == NSLOT ? 1 : NSLOT;  // releases owed per stage
        ok = mbar_wait(&sm.bar_q, uint32_t(pieces) & 1u, abort, p.status, 0x920 + s);
        if (!ok) break;
        for (int j = -1; j < n; ++j) {
          if (j >= 0) {  // PV(j): V tile and P
            ok = mbar_wait(&sm.bar_full[stage], phase, abort, p.status, 0x922 + s) &&
                 mbar_wait(&sm.bar_p_full[s], uint32_t(np) & 1u, abort, p.status, 0x924 + s) &&
                 // the softmax has read O of this slot's previous piece
                 (j > 0 || done == 0 ||
                  mbar_wait(&sm.bar_o_free[s], uint32_t(done - 1) & 1u, abort, p.status,
                            0x926 + s));
            if (!ok) break;
            tc_fence_after();
            issue_pv(t_s + 128, t_s, kv0 + stage * TILE_BYTES, j > 0);
            ++np;
            for (int k = 0; k < rel; ++k) umma_commit(&sm.bar_empty[stage]);
            advance();
            if (j + 1 == n) umma_commit(&sm.bar_o_done[s]);
          }
          if (j + 1 < n) {  // S(j + 1), behind PV(j) in the pipe: P's columns are free by then
            ok = mbar_wait(&sm.bar_full[stage], phase, abort, p.status, 0x928 + s);
            if (!ok) break;
            tc_fence_after();
            issue_s(t_s, qa, kv0 + stage * TILE_BYTES);
            issued_any = true;
            umma_commit(&sm.bar_s_full[s]);
            if (j + 2 == n)  // the piece's last S: Q is free once it completes
              for (int k = 0; k < rel; ++k) umma_commit(&sm.bar_q_free);
            for (int k = 0; k < rel; ++k) umma_commit(&sm.bar_empty[stage]);
            advance();
          }
        }
        ++done;
        ++pieces;
      }
      if (issued_any) {  // everything this thread issued has completed before TMEM is freed
        umma_commit(&sm.bar_final[s]);
        mbar_wait(&sm.bar_final[s], 0, abort, p.status, 0x92a + s, false);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 88;\n" ::: "memory");
    // ------------------------------------------------------------ softmax
    // No thread leaves the walk early: after an abort every wait returns at
    // once and the walk ends by itself, so the barrier of a row's two warps
    // always has both.
    const int s = warp >> 3;
    const int half = (warp >> 2) & 1;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t t_s = tmem + (uint32_t(quarter * 32) << 16) + s * 256;
    const uint32_t t_o = t_s + 128 + half * 64;
    const int pair_bar = 1 + s * 4 + quarter;  // the two warps of 32 rows
    float* my_mx = &sm.mx[s][half][r];
    const float* other_mx = &sm.mx[s][half ^ 1][r];
    int ns = 0;  // blocks (s_full parity)
    int no = 0;  // pieces (o_done parity)
    int w = w0;
    attn::Piece pc;
    while (attn::next_piece(p, w, w1, pc)) {
      if (s >= pc.nslot) continue;
      const int qt = pc.qt;
      const uint32_t* list = p.blk_list + size_t(qt) * p.n_kv128;
      const uint64_t* mrow = p.mask_words + size_t(qt) * p.n_kv64 * 128 + r;
      const float* ksc = p.k_scale + int64_t(pc.kvh) * p.scale_stride;
      const float* vsc = p.v_scale + int64_t(pc.kvh) * p.scale_stride;
      float m = -INFINITY, l = 0.f;
      // the next block's mask word and scales are fetched during this block
      uint64_t wd_next = 0;
      float ks_next = 1.f, vs_next = 1.f;
      auto prefetch = [&](uint32_t e) {
        const int t64 = 2 * int(e & 0xFFFFFFu) + half;
        wd_next = ((e >> (24 + 2 * half)) & 1u) ? ~0ull : 0ull;
        if ((e >> (25 + 2 * half)) & 1u) wd_next = mrow[size_t(t64) * 128];
        const bool sealed = t64 * 64 < p.sealed;
        ks_next = sealed ? __ldg(ksc + t64) : 1.f;
        vs_next = sealed ? __ldg(vsc + t64) : 1.f;
      };
      prefetch(list[pc.b0]);
      uint32_t e_next = pc.b0 + 1 < pc.b1 ? list[pc.b0 + 1] : 0u;
      for (int j = pc.b0; j < pc.b1; ++j) {
        const uint32_t mw[2] = {uint32_t(wd_next), uint32_t(wd_next >> 32)};
        const float sc = ks_next * p.scale_log2;
        const float vs = vs_next;
        mbar_wait(&sm.bar_s_full[s], uint32_t(ns) & 1u, abort, p.status, 0x930 + s);
        __syncwarp();
        ++ns;
        tc_fence_after();
        float x[64];
        {
          uint32_t u[2][32];
          tmem_ld32(t_s + half * 64, u[0]);
          tmem_ld32(t_s + half * 64 + 32, u[1]);
          tmem_wait_ld(u[0]);
          tmem_wait_ld(u[1]);
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i) x[c * 32 + i] = __uint_as_float(u[c][i]);
        }
        if ((mw[0] & mw[1]) != 0xffffffffu) {
#pragma unroll
          for (int i = 0; i < 64; ++i)
            x[i] = ((mw[i >> 5] >> (i & 31)) & 1u) ? x[i] : -INFINITY;
        }
        float mx4[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) mx4[k] = x[k];
#pragma unroll
        for (int i = 4; i + 8 <= 64; i += 8)
#pragma unroll
          for (int k = 0; k < 4; ++k) mx4[k] = fmax3(mx4[k], x[i + k], x[i + 4 + k]);
#pragma unroll
        for (int k = 0; k < 4; ++k) mx4[k] = fmaxf(mx4[k], x[60 + k]);
        const float mx = fmaxf(fmax3(mx4[0], mx4[1], mx4[2]), mx4[3]) * sc;
        *my_mx = mx;
        // both halves have read S (P overwrites it) and their maxima are written
        tc_fence_before();
        asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
        tc_fence_after();
        const float m_new = fmax3(m, mx, *other_mx);
        const bool need = m_new > m + kRescaleLog2;  // also from m = -inf
        const float alpha = need ? ex2_approx(m - m_new) : 1.f;
        if (need) m = m_new;
        // O holds the piece's earlier blocks: S(j) complete implies PV(j-1)
        if (j > pc.b0 && __any_sync(0xffffffffu, need)) {
          const uint64_t al2 = f2_pack(alpha, alpha);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t o[16];
            tmem_ld16(t_o + c * 16, o);
            tmem_wait_ld16(o);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              float lo, hi;
              f2_unpack(f2_mul(f2_pack(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1])),
                               al2),
                        lo, hi);
              o[2 * i] = __float_as_uint(lo);
              o[2 * i + 1] = __float_as_uint(hi);
            }
            tmem_st16(t_o + c * 16, o);
          }
        }
        const float nm = (m == -INFINITY ? 0.f : -m) + (kPackBiasLog2 + log2_approx(vs));
        const uint64_t sc2 = f2_pack(sc, sc);
        const uint64_t nm2 = f2_pack(nm, nm);
        uint64_t sum2[2] = {0ull, 0ull};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float xa, xb;
            f2_unpack(f2_fma(f2_pack(x[32 * c + 2 * i], x[32 * c + 2 * i + 1]), sc2, nm2), xa, xb);
            const float a = ex2_approx(xa);
            const float b = ex2_approx(xb);
            sum2[i & 1] = f2_add(sum2[i & 1], f2_pack(a, b));
            pk[i] = pack_bf16x2_trunc(a, b);
          }
          tmem_st16(t_s + half * 32 + c * 16, pk);
        }
        float s0, s1, s2, s3;
        f2_unpack(sum2[0], s0, s1);
        f2_unpack(sum2[1], s2, s3);
        l = l * alpha + ((s0 + s1) + (s2 + s3)) * __fdividef(kPackBiasInv, vs);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&sm.bar_p_full[s]);
        if (j + 1 < pc.b1) {
          prefetch(e_next);
          if (j + 2 < pc.b1) e_next = list[j + 2];
        }
      }
      // ---- end of the piece: O -> registers, then release O
      mbar_wait(&sm.bar_o_done[s], uint32_t(no) & 1u, abort, p.status, 0x932 + s);
      __syncwarp();
      ++no;
      tc_fence_after();
      float o[64];
      {
        uint32_t u[2][32];
        tmem_ld32(t_o, u[0]);
        tmem_ld32(t_o + 32, u[1]);
        tmem_wait_ld(u[0]);
        tmem_wait_ld(u[1]);
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i) o[c * 32 + i] = __uint_as_float(u[c][i]);
      }
      tc_fence_before();
      mbar_arrive(&sm.bar_o_free[s]);
      sm.lx[s][half][r] = l;
      asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
      l += sm.lx[s][half ^ 1][r];
      const bool whole = pc.b0 == 0 && pc.b1 == pc.nblk;
      const int flag = (s * 2 + half) * 4 + quarter;
      if (!whole && pc.start < w0) {
        // a later piece of an item begun by an earlier CTA: publish O / l
        uint8_t* rec = p.partials + (size_t(blockIdx.x) * NSLOT + s) * kRecBytes;
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 64; ++i) top = fmaxf(top, fabsf(o[i]));
        const float inv = l > 0.f ? 1.f / l : 0.f;
        // the power of two at or below the row's largest |O / l|
        const uint32_t e =
            min(max(__float_as_uint(top * inv) & 0x7f800000u, 27u << 23), 247u << 23);
        const float f = inv * __uint_as_float((254u << 23) - e);
        uint4* dst = reinterpret_cast<uint4*>(rec) + half * (8 * 128) + r;
#pragma unroll
        for (int c = 0; c < 8; ++c)
          dst[c * 128] = make_uint4(pack_f16x2(o[8 * c] * f, o[8 * c + 1] * f),
                                    pack_f16x2(o[8 * c + 2] * f, o[8 * c + 3] * f),
                                    pack_f16x2(o[8 * c + 4] * f, o[8 * c + 5] * f),
                                    pack_f16x2(o[8 * c + 6] * f, o[8 * c + 7] * f));
        reinterpret_cast<float4*>(rec + kRecData)[half * 128 + r] =
            make_float4(m, l, __uint_as_float(e), 0.f);
        __threadfence();
        __syncwarp();
        if (lane == 0) st_release_u32(p.flags + size_t(blockIdx.x) * 16 + flag, gen + 1u);
        continue;
      }
      if (!whole) {
        // this piece holds the item's first blocks: merge the later pieces,
        // the first pieces of the non-empty ranges blockIdx.x + 1 .. khi
        const int ib = pc.start + pc.nblk - 1;  // the item's last work unit
        for (int k = blockIdx.x + 1; k < G && attn::range_start(k, total, G) <= ib; ++k) {
          if (attn::range_start(k + 1, total, G) == attn::range_start(k, total, G)) continue;
          const uint8_t* rec = p.partials + (size_t(k) * NSLOT + s) * kRecBytes;
          const bool got = wait_flag(p.flags + size_t(k) * 16 + flag, gen + 1u, abort, p.status,
                                     0x934 + s, true);
          if (!__all_sync(0xffffffffu, got)) break;
          const float4 ml =
              __ldcg(reinterpret_cast<const float4*>(rec + kRecData) + half * 128 + r);
          const bool use = ml.y > 0.f;  // a piece that saw nothing of this row changes nothing
          const float nm = use ? fmaxf(m, ml.x) : m;
          const float a = use ? ex2_approx(m - nm) : 1.f;
          const float b = use ? ex2_approx(ml.x - nm) * ml.y : 0.f;
          const float bu = b * ml.z;
          const uint4* src = reinterpret_cast<const uint4*>(rec) + half * (8 * 128) + r;
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const uint4 v = __ldcg(src + c * 128);
            const uint32_t wv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 t = unpack_f16x2(wv[i]);
              o[8 * c + 2 * i] = o[8 * c + 2 * i] * a + t.x * bu;
              o[8 * c + 2 * i + 1] = o[8 * c + 2 * i + 1] * a + t.y * bu;
            }
          }
          l = l * a + b;
          m = nm;
        }
      }
      const int q = qt * BM + r;
      if (q < p.q_len) {
        const int h = pc.h0 + s;
        const float inv = l > 0.f ? 1.f / l : 0.f;
        uint4* dst =
            reinterpret_cast<uint4*>(p.out + (size_t(q) * p.hq + h) * HD + half * 64);
#pragma unroll
        for (int c = 0; c < 8; ++c)
          dst[c] = make_uint4(pack_bf16x2(o[8 * c] * inv, o[8 * c + 1] * inv),
                              pack_bf16x2(o[8 * c + 2] * inv, o[8 * c + 3] * inv),
                              pack_bf16x2(o[8 * c + 4] * inv, o[8 * c + 5] * inv),
                              pack_bf16x2(o[8 * c + 6] * inv, o[8 * c + 7] * inv));
        if (half == 0 && p.lse)
          p.lse[size_t(h) * p.q_len + q] =
              l > 0.f ? (m + __log2f(l)) * 0.69314718055994530942f : -INFINITY;
      }
    }
    // query tiles without any visible block: all their rows are fully masked
    for (int t = blockIdx.x; t < p.n_qtiles; t += G) {
      const int qt = p.tile_order[t];
      if (p.blk_count[qt] != 0) continue;
      const int rows = min(BM, p.q_len - qt * BM);
      uint4* dst = reinterpret_cast<uint4*>(p.out + size_t(qt) * BM * p.hq * HD);
      for (int i = threadIdx.x; i < rows * p.hq * (HD / 8); i += kSoftmaxThreads)
        dst[i] = make_uint4(0u, 0u, 0u, 0u);
      if (p.lse)
        for (int i = threadIdx.x; i < rows * p.hq; i += kSoftmaxThreads)
          p.lse[size_t(i / rows) * p.q_len + qt * BM + i % rows] = -INFINITY;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0) {
    // the last CTA to finish advances the generation for the next launch
    __threadfence();
    if (atomicAdd(p.sync + 1, 1u) == uint32_t(G) - 1u) {
      p.sync[1] = 0u;
      __threadfence();
      st_release_u32(p.sync, gen + 1u);
    }
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace kv8t
}  // namespace hsd

namespace hsd_host {

using namespace hsd;

namespace {
constexpr int kMaxDevices = 64;
std::atomic<bool> g_attr_set[kMaxDevices];
}  // namespace

size_t kv8_tiles_workspace_bytes() {
  return kKv8FlagBytes + size_t(kv8_sm_count()) * kv8t::NSLOT * kv8t::kRecBytes;
}

int kv8_tiles_launch(const Kv8AttnArgs& a, const hsd_plan_t& plan) {
  kv8t::Params p;
  static_cast<kv8a::Params&>(p) = a.p;
  if (plan.n_qtiles > kv8t::kMaxTiles) {
    set_error("hsd_verify_attention_kv8: q_len %d exceeds %d query tiles", p.q_len,
              kv8t::kMaxTiles);
    return HSD_ERR_TOO_LARGE;
  }
  CUtensorMap tq;
  int rc = kv8_map(&tq, p.q, true, p.q_len, p.hq, p.q_row_stride, p.q_head_stride, 128, "q");
  if (rc) return rc;
  const int grid = kv8_sm_count();
  if (256 + size_t(grid) * 64 > kKv8FlagBytes) {
    set_error("hsd_verify_attention_kv8: %d SMs exceed the workspace's flags", grid);
    return HSD_ERR_UNSUPPORTED;
  }
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  p.tile_order = plan.tile_order;
  p.blk_prefix = plan.blk_prefix;
  p.k8 = a.k8;
  p.v8 = a.v8;
  p.k8_head_stride = a.k8_head_stride;
  p.v8_head_stride = a.v8_head_stride;
  p.k_tail = static_cast<const __nv_bfloat16*>(a.k_tail);
  p.v_tail = static_cast<const __nv_bfloat16*>(a.v_tail);
  p.kt_row_stride = a.kt_row_stride;
  p.kt_head_stride = a.kt_head_stride;
  p.vt_row_stride = a.vt_row_stride;
  p.vt_head_stride = a.vt_head_stride;
  p.partials = ws + kKv8FlagBytes;
  p.flags = reinterpret_cast<uint32_t*>(ws + 256);
  p.sync = reinterpret_cast<uint32_t*>(ws);
  p.pairs = (p.group + 1) / 2;
  p.n_qtiles = plan.n_qtiles;
  const size_t smem = sizeof(kv8t::Smem) + 1024;
  int dev = 0;
  rc = cuda_check(cudaGetDevice(&dev), "cudaGetDevice");
  if (rc) return rc;
  if (dev < 0 || dev >= kMaxDevices) {
    set_error("hsd_verify_attention_kv8: device ordinal %d >= %d", dev, kMaxDevices);
    return HSD_ERR_UNSUPPORTED;
  }
  if (!g_attr_set[dev].load(std::memory_order_acquire)) {
    rc = cuda_check(cudaFuncSetAttribute(kv8t::tiles_kernel,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)),
                    "cudaFuncSetAttribute(tiles_kernel)");
    if (rc) return rc;
    g_attr_set[dev].store(true, std::memory_order_release);
  }
  return launch_pdl(kv8t::tiles_kernel, dim3(unsigned(grid)), dim3(kv8t::kThreads), smem,
                    a.stream, "tiles_kernel launch", 0, tq, p);
}

}  // namespace hsd_host
