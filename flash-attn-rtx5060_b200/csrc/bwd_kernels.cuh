// Kernels of the attention's backward pass.
//
//   P_ij  = exp(scale * q_i.k_j + bias_ij - lse_i)            (0 where key j is hidden from query i)
//   dS_ij = P_ij * (dO_i.v_j - delta_i),   delta_i = dO_i.O_i - dlse_i
//   dQ_i  = scale * sum_j dS_ij k_j,   dK_j = scale * sum_i dS_ij q_i,   dV_j = sum_i P_ij dO_i
//
// bwd_rows_kernel computes delta and the norms that the scaling of dS needs; bwd_kernel has a work item for every 128 rows
// of dQ and one for every 128 rows of dK and dV. Both kinds take the probabilities again (seven products a tile pair where
// one pass that also adds dQ up in global memory would have five), so that every sum stays in tensor memory, in one order:
// no atomics, no fp32 copy of dQ in HBM, the same bits every time.
//
// The operands of the second products are fp16, and P and dS of a long row are far below 1: P is kept as 2^14 P, and dS as
// 2^14 P * (dO.v - delta) / 2^e with 2^e above the head's bound max|dO_i| max|v_j| + max|delta_i|, so that neither overflows
// and a value is rounded to 11 bits down to 2^-28 of that bound (to 2^-25 of it in steps, below it is 0). The sums are fp32.
#pragma once
#include "fwd_params.h"
#include "ptx.cuh"

namespace fa {

struct BwdParams {
  const __half *o, *d_o, *v;  // bwd_rows_kernel
  const float* lse;           // [bh][seqlen]
  const float* d_lse;         // the same, or nullptr
  float* delta;               // [bh][seqlen]
  float* norms;               // [bh][tiles][3]: of 128 rows the largest |dO_i|, |v_i|, |delta_i|
  __half *dq, *dk, *dv;
  int seqlen, bh, heads, tiles;  // tiles: ceil(seqlen / 128)
  int head_group;                // heads whose work items are interleaved
  float scale, scale_log2;
  int causal, window_left, window_right;
  const float* alibi_slopes;
  int* status;
  int withhold;  // test build only: work item 0 leaves out a tile, so that a wait runs out
};

// 128 rows of a head a CTA, D / 8 lanes a row.
template <int D>
__global__ void __launch_bounds__(256) bwd_rows_kernel(const BwdParams p) {
  constexpr int kLanes = D / 8, kRows = 32 / kLanes;  // of a warp at a time
  __shared__ float s_max[8][3];
  griddep_wait();
  griddep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const size_t head = blockIdx.y;
  float top[3] = {0.f, 0.f, 0.f};
#pragma unroll 2
  for (int r = blockIdx.x * 128 + warp * 16 + lane / kLanes, i = 0; i < 16 / kRows; ++i, r += kRows) {
    float dot = 0.f, gg = 0.f, vv = 0.f;
    if (r < p.seqlen) {
      const size_t at = (head * p.seqlen + r) * D + (lane % kLanes) * 8;
      const uint4 a = *reinterpret_cast<const uint4*>(p.o + at), g = *reinterpret_cast<const uint4*>(p.d_o + at),
                  v = *reinterpret_cast<const uint4*>(p.v + at);
      const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, gw[4] = {g.x, g.y, g.z, g.w}, vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 x = __half22float2(*reinterpret_cast<const __half2*>(aw + k));
        const float2 y = __half22float2(*reinterpret_cast<const __half2*>(gw + k));
        const float2 z = __half22float2(*reinterpret_cast<const __half2*>(vw + k));
        dot = fmaf(x.x, y.x, fmaf(x.y, y.y, dot));
        gg = fmaf(y.x, y.x, fmaf(y.y, y.y, gg));
        vv = fmaf(z.x, z.x, fmaf(z.y, z.y, vv));
      }
    }
#pragma unroll
    for (int s = kLanes / 2; s > 0; s >>= 1) {
      dot += __shfl_xor_sync(0xffffffffu, dot, s);
      gg += __shfl_xor_sync(0xffffffffu, gg, s);
      vv += __shfl_xor_sync(0xffffffffu, vv, s);
    }
    if (r < p.seqlen) {
      if (p.d_lse) dot -= p.d_lse[head * p.seqlen + r];
      if (lane % kLanes == 0) p.delta[head * p.seqlen + r] = dot;
      top[0] = fmaxf(top[0], gg);
      top[1] = fmaxf(top[1], vv);
      top[2] = fmaxf(top[2], fabsf(dot));
    }
  }
#pragma unroll
  for (int k = 0; k < 3; ++k)
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], s));
  if (lane == 0)
    for (int k = 0; k < 3; ++k) s_max[warp][k] = top[k];
  __syncthreads();
  if (threadIdx.x < 3) {
    float m = 0.f;
    for (int w = 0; w < 8; ++w) m = fmaxf(m, s_max[w][threadIdx.x]);
    p.norms[(head * p.tiles + blockIdx.x) * 3 + threadIdx.x] = threadIdx.x < 2 ? sqrtf(m) : m;
  }
}

template <int D>
struct BwdCfg {
  static constexpr int kThreads = 384;
  static constexpr int kTileBytes = 128 * D * 2;
  static constexpr int kPanelBytes = 128 * 128;
  // Ring slots of the first and of the second column tensor. A first tile is held longest (for dQ from the scores of the
  // tile two ahead to its own product).
  static constexpr int kFirst = D == 128 ? 3 : 4, kSecond = D == 128 ? 2 : 4, kStats = 2;
  static constexpr int kOffFirst = 2 * kTileBytes;  // behind the item's own two tiles
  static constexpr int kOffSecond = kOffFirst + kFirst * kTileBytes;
  static constexpr int kOffStats = kOffSecond + kSecond * kTileBytes;  // per slot float[2][128]
  static constexpr int kOffBars = kOffStats + kStats * 1024;
  static constexpr int kNumBars = 1 + 2 * (kFirst + kSecond + kStats) + 6;
  static constexpr int kSmemBytes = kOffBars + kNumBars * 8 + 16;
  static constexpr uint32_t kTmemCols = 512;
  static constexpr int kRegSoftmax = 208, kRegOthers = 88;  // 256 * 208 + 128 * 88 = 384 * 168
};

// One work item: 128 rows of a head (queries for dQ, keys for dK and dV) against the columns (keys, queries) that they
// see, 128 at a time. With "first" and "second" for the column tensors (K and V; Q and dO) and the item's own two tiles A
// and B (Q and dO; K and V), both kinds compute
//   S = A first^T,  dP = B second^T,  dS,  acc1 += dS first      and for dK and dV also  acc0 += P second,
// every product with M = 128 rows in tensor-memory lanes.
struct BwdItem {
  int is_dq, bh, r0, begin, tiles;  // column tiles [begin, begin + tiles)
  int left, right;                  // row r sees columns [r - left, r + right], negative: unbounded
};

__device__ __forceinline__ BwdItem bwd_item(const BwdParams& p, int index) {
  const int per_group = 2 * p.tiles * p.head_group;
  const int first_head = index / per_group * p.head_group;
  const int heads = min(p.head_group, p.bh - first_head);
  const int in = index % per_group, rank = in / (2 * heads), rest = in % (2 * heads);
  BwdItem it;
  it.is_dq = rest >= heads;
  it.bh = first_head + rest % heads;
  const int wr = eff_window_right(p.causal, p.window_right);
  it.left = it.is_dq ? p.window_left : wr;
  it.right = it.is_dq ? wr : p.window_left;
  it.r0 = (it.is_dq ? p.tiles - 1 - rank : rank) * 128;  // under a causal mask the longest first
  it.begin = kv_tile_begin(it.r0, it.left);
  it.tiles = kv_tile_end(min(it.r0 + 127, p.seqlen - 1), it.right, p.seqlen) - it.begin;
  return it;
}

// 2^-e: see the top of this file. A bound that is zero, infinite or NaN leaves dS as it is. All lanes of a warp.
__device__ __forceinline__ float bwd_unit(const BwdParams& p, int bh, int lane) {
  float g = 0.f, v = 0.f, d = 0.f;
  for (int t = lane; t < p.tiles; t += 32) {
    const float* n = p.norms + (static_cast<size_t>(bh) * p.tiles + t) * 3;
    g = fmaxf(g, n[0]);
    v = fmaxf(v, n[1]);
    d = fmaxf(d, n[2]);
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) {
    g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, s));
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, s));
    d = fmaxf(d, __shfl_xor_sync(0xffffffffu, d, s));
  }
  const int exponent = static_cast<int>(__float_as_uint(fmaf(g, v, d)) >> 23 & 255u);  // of the bound, biased by 127
  if (exponent == 0 || exponent == 255) return 1.f;
  return __uint_as_float(static_cast<uint32_t>(min(max(127 - (exponent - 126), 27), 227)) << 23);
}

struct BwdBars {
  uint64_t *own_full, *first_full, *second_full, *stats_full, *first_empty, *second_empty, *stats_empty, *s_full, *dp_full,
      *p_ready, *ds_ready, *acc_full;
  volatile int* abort_flag;
};

// The eight softmax warps: a thread has one row and 64 columns of every tile (warps 0-3 the first 64, 4-7 the others).
// kDq: row statistics are the thread's own, P is not needed further; else they come by column through shared memory.
template <int D, bool kAlibi, bool kDq>
__device__ __forceinline__ bool bwd_softmax(const BwdParams& p, const BwdItem& it, const BwdBars& b, const uint8_t* smem,
                                            uint32_t tmem_base, int warp, int lane) {
  using Cfg = BwdCfg<D>;
  constexpr uint32_t kColDp = kDq ? 256 : 128;
  const int half = warp >> 2;
  const uint32_t lane_base = (warp & 3) * 32u;
  const int row = it.r0 + static_cast<int>(lane_base) + lane;
  const float unit = bwd_unit(p, it.bh, lane);
  const uint64_t scale2 = f2_pack(p.scale_log2, p.scale_log2), unit2 = f2_pack(unit, unit);
  float nl = -INFINITY, nd = 0.f;  // 14 - log2(e) * lse and -delta / 2^e of the row
  if (kDq && row < p.seqlen) {
    const size_t at = static_cast<size_t>(it.bh) * p.seqlen + row;
    nl = fmaf(p.lse[at], -1.4426950408889634f, 14.f);
    nd = -p.delta[at] * unit;
  }
  const float slope = kAlibi ? p.alibi_slopes[it.bh % p.heads] * 1.4426950408889634f : 0.f;
  const int r_last = min(it.r0 + 127, p.seqlen - 1);
  bool ok = true;
  for (int i = 0; i < it.tiles; ++i) {
    const int stage = i % Cfg::kStats;
    const uint32_t tS = tmem_addr(tmem_base, lane_base, (kDq ? (i & 1) * 128 : 0) + half * 64);
    const uint32_t tDp = tmem_addr(tmem_base, lane_base, kColDp + half * 64);
    const int c_tile = (it.begin + i) * 128, c0 = c_tile + half * 64;
    const bool cut = kv_tile_needs_mask(c_tile, it.r0, r_last, it.left, it.right, p.seqlen);
    const int c_lo = it.left >= 0 ? row - it.left - c0 : -1;
    const int c_hi = min(it.right >= 0 ? row + it.right : p.seqlen - 1, p.seqlen - 1) - c0;
    const float4* col_nl = reinterpret_cast<const float4*>(smem + Cfg::kOffStats + stage * 1024 + half * 256);
    const float4* col_nd = col_nl + 32;

    if (!kDq) ok = ok && mbar_wait_warp(b.stats_full + stage, (i / Cfg::kStats) & 1, b.abort_flag);
    ok = ok && (kDq ? mbar_wait_warp(b.s_full + (i & 1), (i >> 1) & 1, b.abort_flag)
                    : mbar_wait_warp(b.s_full, i & 1, b.abort_flag));
    if (!ok) return false;
    tc_fence_after();
    float e[64];
#pragma unroll
    for (int ch = 0; ch < 2; ++ch) {
      uint32_t r[32];
      tmem_ld32(tS + ch * 32, r);
      tmem_wait_ld();
      tmem_ld_fence(r);
#pragma unroll
      for (int c = 0; c < 32; c += 4) {
        float x[4];
        const float4 n = kDq ? make_float4(nl, nl, nl, nl) : col_nl[(ch * 32 + c) / 4];
        f2_unpack(f2_fma(f2_pack(__uint_as_float(r[c]), __uint_as_float(r[c + 1])), scale2, f2_pack(n.x, n.y)), x[0], x[1]);
        f2_unpack(f2_fma(f2_pack(__uint_as_float(r[c + 2]), __uint_as_float(r[c + 3])), scale2, f2_pack(n.z, n.w)), x[2],
                  x[3]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int col = ch * 32 + c + k;
          if (kAlibi) x[k] = fmaf(-slope, fabsf(static_cast<float>(row - c0 - col)), x[k]);
          if (cut && (col < c_lo || col > c_hi)) x[k] = -INFINITY;
          e[col] = ex2_approx(x[k]);
        }
      }
      if (!kDq) {
        uint32_t pk[16];
#pragma unroll
        for (int c = 0; c < 16; ++c) pk[c] = pack_f16x2(e[ch * 32 + 2 * c], e[ch * 32 + 2 * c + 1]);
        tmem_st16(tS + ch * 16, pk);
      }
    }
    if (!kDq) {
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      mbar_arrive_lane0(b.p_ready, lane);
    }
    ok = mbar_wait_warp(b.dp_full, i & 1, b.abort_flag);
    if (!ok) return false;
    tc_fence_after();
#pragma unroll
    for (int ch = 0; ch < 2; ++ch) {
      uint32_t r[32], pk[16];
      tmem_ld32(tDp + ch * 32, r);
      tmem_wait_ld();
      tmem_ld_fence(r);
#pragma unroll
      for (int c = 0; c < 32; c += 4) {
        const float4 n = kDq ? make_float4(nd, nd, nd, nd) : col_nd[(ch * 32 + c) / 4];
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
          float d0, d1;
          const uint64_t t = f2_fma(f2_pack(__uint_as_float(r[c + k]), __uint_as_float(r[c + k + 1])), unit2,
                                    k ? f2_pack(n.z, n.w) : f2_pack(n.x, n.y));
          f2_unpack(f2_mul(t, f2_pack(e[ch * 32 + c + k], e[ch * 32 + c + k + 1])), d0, d1);
          pk[(c + k) / 2] = pack_f16x2(d0, d1);
        }
      }
      tmem_st16((kDq ? tS : tDp) + ch * 16, pk);
    }
    tmem_wait_st();
    tc_fence_before();
    __syncwarp();
    mbar_arrive_lane0(b.ds_ready, lane);
    if (!kDq) mbar_arrive_lane0(b.stats_empty + stage, lane);
  }

  // ---- epilogue ----
  if (!mbar_wait_warp(b.acc_full, 0, b.abort_flag)) return false;
  tc_fence_after();
  const float ds_scale = p.scale * 0x1p-14f / unit;  // (a power of two but for p.scale)
  const float factor = kDq || half ? ds_scale : 0x1p-14f;
  const uint32_t acc = tmem_addr(tmem_base, lane_base, kDq ? 384 + half * (D / 2) : half ? 384 : 256);
  __half* out = (kDq ? p.dq + half * (D / 2) : half ? p.dk : p.dv) + (static_cast<size_t>(it.bh) * p.seqlen + row) * D;
#pragma unroll
  for (int ch = 0; ch < (kDq ? D / 64 : D / 32); ++ch) {
    uint32_t r[32];
    tmem_ld32(acc + ch * 32, r);
    tmem_wait_ld();
    tmem_ld_fence(r);
    if (row < p.seqlen) {
#pragma unroll
      for (int c = 0; c < 32; c += 8) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          w[k] = pack_f16x2(__uint_as_float(r[c + 2 * k]) * factor, __uint_as_float(r[c + 2 * k + 1]) * factor);
        *reinterpret_cast<uint4*>(out + ch * 32 + c) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
  return true;
}

// 12 warps: 0-7 softmax, 8 issues the products, 9 loads tiles, 10 loads the column statistics, 11 only donates registers.
// Tensor memory: for dK and dV S (P in its place) at column 0, dP (dS in its place) at 128, dV at 256, dK at 384; for dQ two
// S (dS in its place) at 0 and 128, dP at 256, dQ at 384. fp16 P and dS of columns 0-63 of a tile lie in the first 32 columns
// of their region, of columns 64-127 in columns 64-95, so that neither half of the warps writes where the other still reads.
template <int D, bool kAlibi>
__global__ void __launch_bounds__(384, 1)
bwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
           const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do,
           const __grid_constant__ BwdParams p) {
  using Cfg = BwdCfg<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kOffBars);
  BwdBars b;
  b.own_full = bars;
  b.first_full = bars + 1;
  b.first_empty = b.first_full + Cfg::kFirst;
  b.second_full = b.first_empty + Cfg::kFirst;
  b.second_empty = b.second_full + Cfg::kSecond;
  b.stats_full = b.second_empty + Cfg::kSecond;
  b.stats_empty = b.stats_full + Cfg::kStats;
  b.s_full = b.stats_empty + Cfg::kStats;  // two
  b.dp_full = b.s_full + 2;
  b.p_ready = b.s_full + 3;
  b.ds_ready = b.s_full + 4;
  b.acc_full = b.s_full + 5;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Cfg::kNumBars);
  b.abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == 8) {
    tmem_alloc(tmem_slot, Cfg::kTmemCols);
    tmem_relinquish();
  }
  if (threadIdx.x == 0) {
    mbar_init(b.own_full, 1);
    for (int i = 0; i < 2 * Cfg::kFirst; ++i) mbar_init(b.first_full + i, 1);    // and first_empty
    for (int i = 0; i < 2 * Cfg::kSecond; ++i) mbar_init(b.second_full + i, 1);  // and second_empty
    for (int i = 0; i < Cfg::kStats; ++i) {
      mbar_init(b.stats_full + i, 1);
      mbar_init(b.stats_empty + i, 8);
    }
    mbar_init(b.s_full, 1);
    mbar_init(b.s_full + 1, 1);
    mbar_init(b.dp_full, 1);
    mbar_init(b.p_ready, 8);
    mbar_init(b.ds_ready, 8);
    mbar_init(b.acc_full, 1);
    *b.abort_flag = 0;
    fence_mbar_init();
  }
  const BwdItem it = bwd_item(p, blockIdx.x);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  griddep_wait();
  griddep_launch();

  if (warp < 8) {
    reg_inc<Cfg::kRegSoftmax>();
    if (it.is_dq) bwd_softmax<D, kAlibi, true>(p, it, b, smem, tmem_base, warp, lane);
    else bwd_softmax<D, kAlibi, false>(p, it, b, smem, tmem_base, warp, lane);
  } else {
    reg_dec<Cfg::kRegOthers>();
    bool ok = true;
    if (warp == 8) {
      // ---- products ----
      constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);  // row stride, version, 128-byte swizzle
      constexpr uint32_t kKMajor = 1u << 16, kMnMajor = (Cfg::kPanelBytes >> 4) << 16;  // leading-dimension offsets
      constexpr uint32_t idesc_s = umma_idesc_f16(128, 128, 0, 0), idesc_acc = umma_idesc_f16(128, D, 0, 1);
      constexpr uint32_t kTile = Cfg::kTileBytes >> 4, kPanel16 = Cfg::kPanelBytes >> 4;
      auto low = [&](int offset) { return (smem_u32(smem + offset) >> 4) & 0x3fffu; };
      const uint32_t own = low(0), first = low(Cfg::kOffFirst), second = low(Cfg::kOffSecond);
      auto first_tile = [&](int i) { return first + i % Cfg::kFirst * kTile; };
      auto second_tile = [&](int i) { return second + i % Cfg::kSecond * kTile; };
      auto scores = [&](uint32_t col, uint32_t a, uint32_t tile) {
#pragma unroll
        for (int h = 0; h < D / 64; ++h)
          umma_qk64(tmem_base + col, (a + h * kPanel16) | kKMajor, (tile + h * kPanel16) | kKMajor, kDescHi, idesc_s, h);
      };
      // acc += X tile, fp16 X at column `x` as described above
      auto accumulate = [&](uint32_t col, uint32_t x, uint32_t tile, bool more) {
        umma_pv64(tmem_base + col, tmem_base + x, tile | kMnMajor, kDescHi, idesc_acc, more);
        umma_pv64(tmem_base + col, tmem_base + x + 64, (tile + 4 * (2048 >> 4)) | kMnMajor, kDescHi, idesc_acc, 1);
      };
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        ok = ok && mbar_wait_warp(bar, parity, b.abort_flag);
        tc_fence_after();
        return ok;
      };
      auto wait_first = [&](int i) { return wait(b.first_full + i % Cfg::kFirst, (i / Cfg::kFirst) & 1); };
      auto wait_second = [&](int i) { return wait(b.second_full + i % Cfg::kSecond, (i / Cfg::kSecond) & 1); };
      const int n = it.tiles;
      wait(b.own_full, 0);
      if (wait_first(0)) {
        scores(0, own, first_tile(0));
        umma_commit_warp(b.s_full);
      }
      if (it.is_dq) {
        if (n > 1 && wait_first(1)) {
          scores(128, own, first_tile(1));
          umma_commit_warp(b.s_full + 1);
        }
        if (wait_second(0)) {
          scores(256, own + kTile, second_tile(0));
          umma_commit_warp(b.dp_full);
          umma_commit_warp(b.second_empty);
        }
        for (int i = 0; i < n; ++i) {
          if (!wait(b.ds_ready, i & 1)) break;
          if (i + 1 < n) {  // the softmax of the next tile waits for this one first
            if (!wait_second(i + 1)) break;
            scores(256, own + kTile, second_tile(i + 1));
            umma_commit_warp(b.dp_full);
            umma_commit_warp(b.second_empty + (i + 1) % Cfg::kSecond);
          }
          accumulate(384, (i & 1) * 128, first_tile(i), i > 0);
          umma_commit_warp(b.first_empty + i % Cfg::kFirst);
          if (i + 2 < n) {
            if (!wait_first(i + 2)) break;
            scores((i & 1) * 128, own, first_tile(i + 2));
            umma_commit_warp(b.s_full + (i & 1));
          }
        }
      } else {
        if (wait_second(0)) {
          scores(128, own + kTile, second_tile(0));
          umma_commit_warp(b.dp_full);
        }
        for (int i = 0; i < n; ++i) {
          if (!wait(b.p_ready, i & 1)) break;
          accumulate(256, 0, second_tile(i), i > 0);
          umma_commit_warp(b.second_empty + i % Cfg::kSecond);
          if (i + 1 < n) {
            if (!wait_first(i + 1)) break;
            scores(0, own, first_tile(i + 1));
            umma_commit_warp(b.s_full);
          }
          if (!wait(b.ds_ready, i & 1)) break;
          accumulate(384, 128, first_tile(i), i > 0);
          umma_commit_warp(b.first_empty + i % Cfg::kFirst);
          if (i + 1 < n) {
            if (!wait_second(i + 1)) break;
            scores(128, own + kTile, second_tile(i + 1));
            umma_commit_warp(b.dp_full);
          }
        }
      }
      if (ok) umma_commit_warp(b.acc_full);
    } else if (warp == 9) {
      // ---- tiles ----
      if (elect_one()) {
        const CUtensorMap *own0 = it.is_dq ? &map_q : &map_k, *own1 = it.is_dq ? &map_do : &map_v;
        const CUtensorMap *first = it.is_dq ? &map_k : &map_q, *second = it.is_dq ? &map_v : &map_do;
        mbar_arrive_expect_tx(b.own_full, 2 * Cfg::kTileBytes);
        tma_load_4d(smem, own0, b.own_full, 0, it.r0, 0, it.bh);
        tma_load_4d(smem + Cfg::kTileBytes, own1, b.own_full, 0, it.r0, 0, it.bh);
        for (int i = 0; i < it.tiles; ++i) {
          const int c0 = (it.begin + i) * 128, f = i % Cfg::kFirst, s = i % Cfg::kSecond;
          ok = mbar_wait(b.first_empty + f, ((i / Cfg::kFirst) & 1) ^ 1, b.abort_flag);
          if (!ok) break;
          mbar_arrive_expect_tx(b.first_full + f, Cfg::kTileBytes);
          tma_load_4d(smem + Cfg::kOffFirst + f * Cfg::kTileBytes, first, b.first_full + f, 0, c0, 0, it.bh);
          ok = mbar_wait(b.second_empty + s, ((i / Cfg::kSecond) & 1) ^ 1, b.abort_flag);
          if (!ok) break;
          mbar_arrive_expect_tx(b.second_full + s, Cfg::kTileBytes);
#ifdef FA_TEST_WITHHOLD_LOAD
          if (p.withhold && blockIdx.x == 0 && i == it.tiles - 1) continue;
#endif
          tma_load_4d(smem + Cfg::kOffSecond + s * Cfg::kTileBytes, second, b.second_full + s, 0, c0, 0, it.bh);
        }
        // a give-up leaves loads in flight; let them land before the CTA retires
        if (!ok)
          for (int i = 0; i < 64; ++i) __nanosleep(2000);
      }
      __syncwarp();
    } else if (warp == 10 && !it.is_dq) {
      // ---- column statistics ----
      const float unit = bwd_unit(p, it.bh, lane);
      for (int i = 0; i < it.tiles; ++i) {
        const int stage = i % Cfg::kStats;
        float nl[4], nd[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int c = (it.begin + i) * 128 + k * 32 + lane;
          const size_t at = static_cast<size_t>(it.bh) * p.seqlen + c;
          nl[k] = c < p.seqlen ? fmaf(p.lse[at], -1.4426950408889634f, 14.f) : -INFINITY;
          nd[k] = c < p.seqlen ? -p.delta[at] * unit : 0.f;
        }
        if (!mbar_wait_warp(b.stats_empty + stage, ((i / Cfg::kStats) & 1) ^ 1, b.abort_flag)) break;
        float* to = reinterpret_cast<float*>(smem + Cfg::kOffStats + stage * 1024);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          to[k * 32 + lane] = nl[k];
          to[128 + k * 32 + lane] = nd[k];
        }
        __syncwarp();
        mbar_arrive_lane0(b.stats_full + stage, lane);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *b.abort_flag != 0) atomicExch(p.status, 1);
  if (warp == 8) tmem_dealloc(tmem_base, Cfg::kTmemCols);
}

}  // namespace fa
