// Kernels of the attention's backward pass.
//
//   P_ij  = exp(scale * q_i.k_j + bias_ij - lse_i)            (0 where key j is hidden from query i)
//   dS_ij = P_ij * (dO_i.v_j - delta_i),   delta_i = dO_i.O_i - dlse_i
//   dQ_i  = scale * sum_j dS_ij k_j,   dK_j = scale * sum_i dS_ij q_i,   dV_j = sum_i P_ij dO_i
//
// bwd_rows_kernel computes delta and the norms that the scaling of dS needs; bwd_kernel has a work item for every 128 rows
// of dQ and one for every 128 rows of dK and dV (few short heads: one launch, bwd_own_rows). Both kinds take the
// probabilities again (seven products a tile pair where one pass that also adds dQ up in global memory would have five), so
// that every sum stays in tensor memory, in one order: no atomics, no fp32 copy of dQ in HBM, the same bits every time.
//
// The operands of the second products are fp16, and P and dS of a long row are far below 1: P is kept as 2^14 P, and dS as
// 2^14 P * (dO.v - delta) / 2^e with 2^e above a bound of what follows P, so that neither overflows and a value is rounded to 11
// bits down to 2^-28 of the bound (to 2^-39 of it in steps of 2^-38, below it is 0). For dQ the bound is a row's own, |dO_i| max|v_j| +
// |delta_i| over the keys that its 128 rows see; for dK, whose sums run over the queries, that of 128 keys, max|dO_i| max|v_j| +
// max|delta_i| over the queries that see them. (One bound a head cost the rows beside a large one their precision: error of dQ 1.6e-3
// instead of 3e-4 beside a row of dO 2^18 times as large, 4096 rows.) Rows whose norms are infinite or NaN are left out of the
// maxima. The sums are fp32.
#pragma once
#include "fwd_params.h"
#include "ptx.cuh"

namespace fa {

struct BwdParams {
  const __half *o, *d_o, *v;  // for delta and the norms
  const float* lse;           // [bh][seqlen]
  const float* d_lse;         // the same, or nullptr
  float* delta;               // [bh][seqlen]
  float* norms;               // [bh][tiles][3]: of 128 rows the largest |dO_i|, |v_i|, |delta_i|
  __half *dq, *dk, *dv;       // the place of 128 rows of dq holds, until they are written, their |dO_i|^2 as floats in a row
  int seqlen, bh, heads, tiles;  // tiles: ceil(seqlen / 128)
  int head_group;                // heads whose work items are interleaved
  int kinds_apart;               // in such a group all items of dK and dV come first, not those of one rank
  float scale, scale_log2;
  int causal, window_left, window_right;
  const float* alibi_slopes;
  int* status;
  int withhold;  // test build only: work item 0 leaves out a tile, so that a wait runs out
};

// delta of row r of a head, and |dO_r|^2 and |v_r|^2: D / 8 lanes a row, all of which get the sums. All lanes of a warp.
template <int D>
__device__ __forceinline__ void bwd_row(const BwdParams& p, size_t head, int r, int lane, float& delta, float& gg, float& vv) {
  constexpr int kLanes = D / 8;
  delta = gg = vv = 0.f;
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
      delta = fmaf(x.x, y.x, fmaf(x.y, y.y, delta));
      gg = fmaf(y.x, y.x, fmaf(y.y, y.y, gg));
      vv = fmaf(z.x, z.x, fmaf(z.y, z.y, vv));
    }
  }
#pragma unroll
  for (int s = kLanes / 2; s > 0; s >>= 1) {
    delta += __shfl_xor_sync(0xffffffffu, delta, s);
    gg += __shfl_xor_sync(0xffffffffu, gg, s);
    vv += __shfl_xor_sync(0xffffffffu, vv, s);
  }
  if (p.d_lse && r < p.seqlen) delta -= p.d_lse[head * p.seqlen + r];
}

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, s));
  return x;
}

// A norm for the maxima: one that is infinite or NaN is left out. Its own row has no finite result whatever the scaling, and the
// others' has to be that of their own sizes (an infinite bound once left dS of the whole head unscaled: it overflowed).
__device__ __forceinline__ float bwd_norm(float x) { return x < INFINITY ? x : 0.f; }

// 128 rows of a head a CTA. Reads O, dO and V once: bound by bytes where rows are many (B1 H16 N8192 d128: 101 MB in 24 us under
// ncu, caches flushed), else by one round of loads and two reductions.
template <int D>
__global__ void __launch_bounds__(1024) bwd_rows_kernel(const BwdParams p) {
  constexpr int kRows = 32 / (D / 8);  // of a warp at a time
  __shared__ float s_max[32][3];
  griddep_wait();
  griddep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const size_t head = blockIdx.y;
  float top[3] = {0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4 / kRows; ++i) {
    const int r = blockIdx.x * 128 + warp * 4 + i * kRows + lane / (D / 8);
    float delta, gg, vv;
    bwd_row<D>(p, head, r, lane, delta, gg, vv);
    if (r < p.seqlen && lane % (D / 8) == 0) {
      p.delta[head * p.seqlen + r] = delta;
      reinterpret_cast<float*>(p.dq + (head * p.seqlen + blockIdx.x * 128) * D)[r % 128] = gg;
    }
    top[0] = fmaxf(top[0], bwd_norm(gg));
    top[1] = fmaxf(top[1], bwd_norm(vv));
    top[2] = fmaxf(top[2], bwd_norm(fabsf(delta)));
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const float m = warp_max(top[k]);
    if (lane == 0) s_max[warp][k] = m;
  }
  __syncthreads();
  if (warp < 3) {  // warp k: the largest of norm k
    const float m = warp_max(s_max[lane][warp]);
    if (lane == 0) p.norms[(head * p.tiles + blockIdx.x) * 3 + warp] = warp < 2 ? sqrt_approx(m) : m;
  }
}

template <int D>
struct BwdCfg {
  static constexpr int kSoftmaxWarps = 16;
  static constexpr int kThreads = (kSoftmaxWarps + 4) * 32;
  static constexpr int kTileBytes = 128 * D * 2;
  static constexpr int kPanelBytes = 128 * 128;
  // Ring slots of the first and of the second column tensor. A first tile is held longest (for dQ from the scores of the
  // tile two ahead to its own product).
  static constexpr int kFirst = D == 128 ? 3 : 4, kSecond = D == 128 ? 2 : 4, kStats = 2;
  static constexpr int kOffFirst = 2 * kTileBytes;  // behind the item's own two tiles
  static constexpr int kOffSecond = kOffFirst + kFirst * kTileBytes;
  static constexpr int kOffStats = kOffSecond + kSecond * kTileBytes;  // per slot float[2][128]
  static constexpr int kOffUnits = kOffStats + kStats * 1024;  // per slot, for dQ, the exponents of 128 rows' units, a byte each
  static constexpr int kOffBars = kOffUnits + kStats * 128;
  static constexpr int kNumBars = 2 * (kFirst + kSecond + kStats) + 10;
  static constexpr int kSmemBytes = kOffBars + kNumBars * 8 + 24;
  // kOwnRows: delta and |dO_i|^2 of all rows, 16 warps' three norms and a barrier. At head_dim 128, where there is no other room,
  // they lie in the first ring's third slot, which the single tile of 128 rows does not reach.
  static constexpr int kMaxOwnRows = 16384 / D;
  static constexpr int kOffOwnRows = D == 128 ? kOffFirst + 2 * kTileBytes : (kSmemBytes + 15) / 16 * 16;
  static constexpr int kOwnRowsBytes = kMaxOwnRows * 8 + 16 * 3 * 4 + 8;
  static constexpr int kSmemBytesOwnRows = D == 128 ? kSmemBytes : kOffOwnRows + kOwnRowsBytes;
  static_assert(D == 64 || kFirst * 128 > kMaxOwnRows);
  static constexpr uint32_t kTmemCols = 512;
  // Tensor memory: score regions of 128 columns, in which the fp16 operands of the second products take the place of the
  // scores that they are made of (32 columns' operand in the first 16 of the 32), and the accumulators. S has two regions for
  // dQ and at head_dim 64, where there is room: the scores of a tile are then computed while the tile before is worked on.
  static constexpr uint32_t kColS = 0, kColDp = 128, kColOdd = 256, kColDv = D == 128 ? 256 : 384,
                            kColDk = D == 128 ? 384 : 448, kColDq = 384;
  // launched with 96 registers a thread: 512 * 104 + 128 * 64 <= 640 * 96
  static constexpr int kRegSoftmax = 104, kRegOthers = 64;
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
  const unsigned per_group = 2 * p.tiles * p.head_group, group = static_cast<unsigned>(index) / per_group;
  const int first_head = group * p.head_group;
  const unsigned heads = min(p.head_group, p.bh - first_head);
  unsigned in = index - group * per_group;  // kinds apart: [kind][rank][head], else [rank][kind][head]
  const unsigned of_kind = p.tiles * heads;
  const bool second_kind = p.kinds_apart && in >= of_kind;
  if (second_kind) in -= of_kind;
  int rank = in / heads;
  const int head = in - rank * heads;
  BwdItem it;
  it.is_dq = p.kinds_apart ? second_kind : rank & 1;
  if (!p.kinds_apart) rank >>= 1;
  it.bh = first_head + head;
  const int wr = eff_window_right(p.causal, p.window_right);
  it.left = it.is_dq ? p.window_left : wr;
  it.right = it.is_dq ? wr : p.window_left;
  it.r0 = (it.is_dq ? p.tiles - 1 - rank : rank) * 128;  // under a causal mask the longest first
  it.begin = kv_tile_begin(it.r0, it.left);
  it.tiles = kv_tile_end(min(it.r0 + 127, p.seqlen - 1), it.right, p.seqlen) - it.begin;
  return it;
}

// The k-th work item of a CTA, or an index past the last: every other round of CTAs is dealt backwards, so that the CTAs'
// sums are alike although the items of a group of heads get shorter under a causal mask.
__device__ __forceinline__ int bwd_index(int k) {
  return k * static_cast<int>(gridDim.x) + static_cast<int>(k & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
}

// The exponent field of 2^-e (see the top of this file) for a bound. A bound of zero leaves dS as it is; one beyond fp32 (norms are
// finite, their sum need not be) is the largest.
__device__ __forceinline__ uint32_t bwd_unit_exponent(float bound) {
  const int exponent = static_cast<int>(__float_as_uint(bound) >> 23 & 255u);  // biased by 127
  return exponent == 0 ? 127u : static_cast<uint32_t>(min(max(127 - (exponent - 126), 27), 227));
}

// A role's place in a ring of slots, or on a barrier that is used again and again (one slot).
template <int kSlots>
struct Turn {
  int slot = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void advance() {
    if (++slot == kSlots) slot = 0, parity ^= 1;
  }
};

struct BwdBars {
  uint64_t *first_full, *first_empty, *second_full, *second_empty, *stats_full, *own_full, *own_empty, *s_full, *dp_full,
      *acc_full;  // s_full: two
  // p_ready: two, for even and odd tiles where S has two regions: a warp may then have handed over P of a tile before another
  // has that of the tile before
  uint64_t *stats_empty, *p_ready, *ds_ready, *acc_empty;
  volatile int* abort_flag;
  volatile float *unit, *slope;  // of the items of even and odd turn (unit: of dK)
};

// dK and dV at head_dim 128 have one region for S.
template <int D>
__device__ __forceinline__ constexpr bool bwd_two_s(bool is_dq) {
  return D == 64 || is_dq;
}

// Of every kBwdPolyOf pairs of exponentials one is taken on the FMA pipe instead of the special-function unit.
constexpr int kBwdPolyOf = 4;

// State that a softmax warp carries from item to item.
template <int D>
struct SoftmaxTurns {
  Turn<BwdCfg<D>::kStats> stats;
  uint32_t s = 0, dp = 0, acc = 0;  // parities; s: bit 0, bit 1 of either s_full
};

// Stores 32 rows of kPieces * 16 bytes, `rows` of which exist, from lanes that hold a row each. Written as they lie, a store
// instruction touches 32 lines for 16 bytes each, 5300 clocks for the dK and dV of an item at head_dim 128 (2700 this way), in the
// load/store unit that all warps share: B1 H4 N512 d128 16.8 -> 13.9 us, window 1024 2373 -> 2253. So groups of kPieces lanes
// first exchange their pieces: lane l gets piece l % kPieces of each of the group's rows, and an instruction writes whole rows.
template <int kPieces>
__device__ __forceinline__ void bwd_store_rows(__half* to, int stride, int rows, uint4 (&piece)[kPieces], int lane) {
#pragma unroll
  for (int s = 1; s < kPieces; s *= 2) {
    const bool upper = lane & s;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if (i & s) continue;
      const uint4 give = upper ? piece[i] : piece[i | s];
      const uint4 got = make_uint4(__shfl_xor_sync(0xffffffffu, give.x, s), __shfl_xor_sync(0xffffffffu, give.y, s),
                                   __shfl_xor_sync(0xffffffffu, give.z, s), __shfl_xor_sync(0xffffffffu, give.w, s));
      if (upper) piece[i] = got;
      else piece[i | s] = got;
    }
  }
  const int first = lane / kPieces * kPieces;
  to += static_cast<size_t>(first) * stride + lane % kPieces * 8;
#pragma unroll
  for (int i = 0; i < kPieces; ++i)
    if (first + i < rows) *reinterpret_cast<uint4*>(to + static_cast<size_t>(i) * stride) = piece[i];
}

// The sixteen softmax warps: a thread has one row and 32 columns of every tile (warps 0-3 the first 32, and so on), so that four
// warps a sub-partition hide one another's latencies (eight warps with 64 columns each: 10-20 % slower, and two groups of eight
// that take tiles in turn 10-30 %). A tile is a chain: wait, load S, exponentials, P, wait, load dP, dS. At head_dim 64 that chain
// and the power cap set the pace (3680 clocks for the two tiles of a pair, of which 1540 are exponentials); at head_dim 128 the
// products do, at the power cap.
// kDq: the statistics (14 - log2(e) * lse, -delta / 2^e and e) are the row's, P is not needed further; else they are the
// columns' (but for e), and P goes to the tensor cores too. Returns false once a wait has run out.
template <int D, bool kAlibi, bool kDq>
__device__ __forceinline__ bool bwd_softmax(const BwdParams& p, const BwdItem& it, BwdItem& next, const BwdBars& b,
                                            const uint8_t* smem, uint32_t tmem_base, int warp, int lane, int turn,
                                            SoftmaxTurns<D>& at) {
  using Cfg = BwdCfg<D>;
  const int quarter = warp >> 2;
  const uint32_t lane_base = (warp & 3) * 32u;
  const int row = it.r0 + static_cast<int>(lane_base) + lane;
  const uint64_t scale2 = f2_pack(p.scale_log2, p.scale_log2);
  const int r_last = min(it.r0 + 127, p.seqlen - 1);
  constexpr bool kTwoS = bwd_two_s<D>(kDq);
  const uint32_t tS = tmem_addr(tmem_base, lane_base, Cfg::kColS + quarter * 32);
  const uint32_t tDp = tmem_addr(tmem_base, lane_base, Cfg::kColDp + quarter * 32);
  bool ok = true;  // (looked at once a tile: a vote behind each wait costs more than the wait)
  float unit = 1.f, slope = 0.f, nl = 0.f, nd = 0.f;
  if (kDq) {
    ok &= mbar_wait(b.stats_full + at.stats.slot, at.stats.parity, b.abort_flag);
    const float* stats = reinterpret_cast<const float*>(smem + Cfg::kOffStats + at.stats.slot * 1024);
    nl = stats[lane_base + lane];
    nd = stats[128 + lane_base + lane];
    unit = __uint_as_float(static_cast<uint32_t>(smem[Cfg::kOffUnits + at.stats.slot * 128 + lane_base + lane]) << 23);
    if (kAlibi) slope = b.slope[turn & 1];
    __syncwarp();
    mbar_arrive_lane0(b.stats_empty + at.stats.slot, lane);
    at.stats.advance();
  }
  for (int i = 0; i < it.tiles; ++i) {
    const uint32_t tS_i = tS + (kTwoS && (i & 1) ? Cfg::kColOdd - Cfg::kColS : 0u);
    const int c_tile = (it.begin + i) * 128, c0 = c_tile + quarter * 32;
    const float4* col_nl = reinterpret_cast<const float4*>(smem + Cfg::kOffStats + at.stats.slot * 1024 + quarter * 128);
    const float4* col_nd = col_nl + 32;
    const bool cut = kv_tile_needs_mask(c_tile, it.r0, r_last, it.left, it.right, p.seqlen);

    if (!kDq) {
      ok &= mbar_wait(b.stats_full + at.stats.slot, at.stats.parity, b.abort_flag);
      if (i == 0) {
        unit = b.unit[turn & 1];
        if (kAlibi) slope = b.slope[turn & 1];
      }
    }
    const int odd = kTwoS ? i & 1 : 0;
    ok &= mbar_wait(b.s_full + odd, at.s >> odd & 1u, b.abort_flag);
    at.s ^= 1u << odd;
    tc_fence_after();
    uint32_t r[32];
    tmem_ld32(tS_i, r);
    tmem_wait_ld();
    tmem_ld_fence(r);
    float e[32];
#pragma unroll
    for (int c = 0; c < 32; c += 4) {
      const float4 n = kDq ? make_float4(nl, nl, nl, nl) : col_nl[c / 4];
      f2_unpack(f2_fma(f2_pack(__uint_as_float(r[c]), __uint_as_float(r[c + 1])), scale2, f2_pack(n.x, n.y)), e[c], e[c + 1]);
      f2_unpack(f2_fma(f2_pack(__uint_as_float(r[c + 2]), __uint_as_float(r[c + 3])), scale2, f2_pack(n.z, n.w)), e[c + 2],
                e[c + 3]);
    }
    if (kAlibi) {
#pragma unroll
      for (int c = 0; c < 32; ++c) e[c] = fmaf(-slope, fabsf(static_cast<float>(row - c0 - c)), e[c]);
    }
    if (cut) {
      const int c_lo = it.left >= 0 ? row - it.left - c0 : -1;
      const int c_hi = min(it.right >= 0 ? row + it.right : p.seqlen - 1, p.seqlen - 1) - c0;
#pragma unroll
      for (int c = 0; c < 32; ++c)
        if (c < c_lo || c > c_hi) e[c] = -INFINITY;
    }
#pragma unroll
    for (int c = 0; c < 32; c += 2) {
      if (kBwdPolyOf > 0 && c / 2 % (kBwdPolyOf > 0 ? kBwdPolyOf : 1) == 1) {
        exp2_poly(e[c], e[c + 1], e[c], e[c + 1]);
      } else {
        e[c] = ex2_approx(e[c]);
        e[c + 1] = ex2_approx(e[c + 1]);
      }
    }
    uint32_t pk[16];
    if (!kDq) {
#pragma unroll
      for (int c = 0; c < 16; ++c) pk[c] = pack_f16x2(e[2 * c], e[2 * c + 1]);
      tmem_st16(tS_i, pk);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      mbar_arrive_lane0(b.p_ready + odd, lane);
    }
    ok &= mbar_wait(b.dp_full, at.dp, b.abort_flag);
    at.dp ^= 1;
    tc_fence_after();
    tmem_ld32(tDp, r);
    tmem_wait_ld();
    tmem_ld_fence(r);
    const uint64_t unit2 = f2_pack(unit, unit);
#pragma unroll
    for (int c = 0; c < 32; c += 4) {
      const float4 n = kDq ? make_float4(nd, nd, nd, nd) : col_nd[c / 4];
#pragma unroll
      for (int k = 0; k < 4; k += 2) {
        float d0, d1;
        const uint64_t t = f2_fma(f2_pack(__uint_as_float(r[c + k]), __uint_as_float(r[c + k + 1])), unit2,
                                  k ? f2_pack(n.z, n.w) : f2_pack(n.x, n.y));
        f2_unpack(f2_mul(t, f2_pack(e[c + k], e[c + k + 1])), d0, d1);
        pk[(c + k) / 2] = pack_f16x2(d0, d1);
      }
    }
    tmem_st16(kDq ? tS_i : tDp, pk);
    tmem_wait_st();
    tc_fence_before();
    __syncwarp();
    mbar_arrive_lane0(b.ds_ready, lane);
    if (!kDq) {
      mbar_arrive_lane0(b.stats_empty + at.stats.slot, lane);
      at.stats.advance();
    }
    if (!__all_sync(0xffffffffu, ok)) return false;
  }

  // ---- epilogue: dQ a quarter of the columns a warp; dV the first eight warps, dK the others, half of the columns each ----
  // (the next item's place is worked out while the last product runs: after the epilogue it cost 1000 clocks)
  if (bwd_index(turn + 1) < 2 * p.tiles * p.bh) next = bwd_item(p, bwd_index(turn + 1));
  ok &= mbar_wait(b.acc_full, at.acc, b.abort_flag);
  at.acc ^= 1;
  tc_fence_after();
  constexpr int kCols = kDq ? D / 4 : D / 2;
  const int col = kDq ? quarter * kCols : (quarter & 1) * kCols;
  const float factor = kDq || quarter >= 2 ? p.scale * 0x1p-14f / unit : 0x1p-14f;
  const uint32_t acc =
      tmem_addr(tmem_base, lane_base, (kDq ? Cfg::kColDq : quarter >= 2 ? Cfg::kColDk : Cfg::kColDv) + col);
  __half* out = (kDq ? p.dq : quarter >= 2 ? p.dk : p.dv) +
                (static_cast<size_t>(it.bh) * p.seqlen + it.r0 + lane_base) * D + col;
  uint4 piece[kCols / 8];  // 16 bytes each
#pragma unroll
  for (int ch = 0; ch < kCols / 16; ++ch) {
    uint32_t r[16];
    tmem_ld16(acc + ch * 16, r);
    tmem_wait_ld();
    tmem_ld_fence16(r);
    uint32_t w[8];
#pragma unroll
    for (int c = 0; c < 8; ++c)
      w[c] = pack_f16x2(__uint_as_float(r[2 * c]) * factor, __uint_as_float(r[2 * c + 1]) * factor);
    piece[2 * ch] = make_uint4(w[0], w[1], w[2], w[3]);
    piece[2 * ch + 1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
  bwd_store_rows<kCols / 8>(out, D, p.seqlen - (it.r0 + static_cast<int>(lane_base)), piece, lane);
  tc_fence_before();
  __syncwarp();
  mbar_arrive_lane0(b.acc_empty, lane);
  return __all_sync(0xffffffffu, ok);
}

// The warp that issues the products of all items.
template <int D>
__device__ __forceinline__ bool bwd_issue(const BwdParams& p, const BwdBars& b, uint8_t* smem, uint32_t tmem_base) {
  using Cfg = BwdCfg<D>;
  constexpr uint32_t idesc_s = umma_idesc_f16(128, 128, 0, 0), idesc_acc = umma_idesc_f16(128, D, 0, 1);
  // descriptors of shared-memory operands: a constant high word (row stride, version, 128-byte swizzle), and low words that
  // differ by the start address
  constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
  constexpr uint32_t kKMajor = 1u << 16, kMnMajor = static_cast<uint32_t>(Cfg::kPanelBytes >> 4) << 16, kTile = Cfg::kTileBytes >> 4;
  const uint32_t own = smem_u32(smem) >> 4, first = smem_u32(smem + Cfg::kOffFirst) >> 4,
                 second = smem_u32(smem + Cfg::kOffSecond) >> 4;
  // scores: 128 x 128, over head_dim
  auto scores = [&](uint32_t col, uint32_t a, uint32_t tile) {
#pragma unroll
    for (int h = 0; h < D / 64; ++h)
      umma_qk64(tmem_base + col, (a + h * (Cfg::kPanelBytes >> 4)) | kKMajor, (tile + h * (Cfg::kPanelBytes >> 4)) | kKMajor,
                kDescHi, idesc_s, h);
  };
  // acc += X tile over 128 columns, fp16 X in the place of scores at column `x`
  auto accumulate = [&](uint32_t col, uint32_t x, uint32_t tile, bool more) {
    umma_x64(tmem_base + col, tmem_base + x, tile | kMnMajor, kDescHi, idesc_acc, more);
    umma_x64(tmem_base + col, tmem_base + x + 64, (tile + 4 * (2048 >> 4)) | kMnMajor, kDescHi, idesc_acc, 1);
  };
  bool ok = true;
  // (a wait that has run out is noticed at the end of the tile: a vote behind each costs more than the wait)
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    ok &= mbar_wait(bar, parity, b.abort_flag);
    tc_fence_after();
  };
  Turn<Cfg::kFirst> f_scores, f_acc;  // first tiles: whose scores come next, whose product comes next
  Turn<Cfg::kSecond> s_scores, s_acc;
  uint32_t p_at = 0, ds_at = 0, own_at = 0, acc_at = 1;  // parities, p_at of either p_ready (the accumulators are free at the start)
  BwdItem it, next = bwd_item(p, bwd_index(0));
  for (int k = 0; bwd_index(k) < 2 * p.tiles * p.bh && ok; ++k) {
    it = next;
    const int n = it.tiles;
    const bool two_s = bwd_two_s<D>(it.is_dq);
    auto s_col = [&](int i) { return two_s && (i & 1) ? Cfg::kColOdd : Cfg::kColS; };
    auto scores_first = [&](int i) {
      wait(b.first_full + f_scores.slot, f_scores.parity);
      scores(s_col(i), own, first + f_scores.slot * kTile);
      umma_commit_warp(b.s_full + (two_s ? i & 1 : 0));
      f_scores.advance();
    };
    auto scores_second = [&](int i) {
      wait(b.second_full + s_scores.slot, s_scores.parity);
      scores(Cfg::kColDp, own + kTile, second + s_scores.slot * kTile);
      umma_commit_warp(b.dp_full);
      umma_commit_warp(b.second_empty + s_scores.slot, it.is_dq);
      umma_commit_warp(b.own_empty, i + 1 == n);
      s_scores.advance();
    };
    auto product_first = [&](int i) {
      accumulate(it.is_dq ? Cfg::kColDq : Cfg::kColDk, it.is_dq ? s_col(i) : Cfg::kColDp, first + f_acc.slot * kTile, i > 0);
      umma_commit_warp(b.first_empty + f_acc.slot);
      f_acc.advance();
    };
    // S and dP of the item before have been used: its products stand in front of what follows here
    wait(b.own_full, own_at);
    own_at ^= 1;
    scores_first(0);
    scores_second(0);
    wait(b.acc_empty, acc_at);  // (before the odd S, which may lie where an accumulator of the item before is)
    acc_at ^= 1;
    if (two_s && n > 1) scores_first(1);
    if (bwd_index(k + 1) < 2 * p.tiles * p.bh) next = bwd_item(p, bwd_index(k + 1));
    if (it.is_dq) {
      for (int i = 0; i < n && ok; ++i) {
        wait(b.ds_ready, ds_at);
        ds_at ^= 1;
        if (i + 1 < n) scores_second(i + 1);  // the softmax of the next tile waits for this one first
        product_first(i);
        if (i + 2 < n) scores_first(i + 2);
        s_acc.advance();
        ok = __all_sync(0xffffffffu, ok);
      }
    } else {
      for (int i = 0; i < n && ok; ++i) {
        const int odd = two_s ? i & 1 : 0;
        wait(b.p_ready + odd, p_at >> odd & 1u);
        p_at ^= 1u << odd;
        accumulate(Cfg::kColDv, s_col(i), second + s_acc.slot * kTile, i > 0);
        umma_commit_warp(b.second_empty + s_acc.slot);
        s_acc.advance();
        if (i + 1 + two_s < n) scores_first(i + 1 + two_s);
        wait(b.ds_ready, ds_at);
        ds_at ^= 1;
        product_first(i);
        if (i + 1 < n) scores_second(i + 1);
        ok = __all_sync(0xffffffffu, ok);
      }
    }
    umma_commit_warp(b.acc_full);
  }
  return ok;
}

// The thread that loads the tiles of all items.
template <int D>
__device__ __forceinline__ bool bwd_load(const CUtensorMap& map_q, const CUtensorMap& map_k, const CUtensorMap& map_v,
                                         const CUtensorMap& map_do, const BwdParams& p, const BwdBars& b, uint8_t* smem) {
  using Cfg = BwdCfg<D>;
  Turn<Cfg::kFirst> f;
  Turn<Cfg::kSecond> s;
  Turn<1> own;
  own.parity = f.parity = s.parity = 1;  // (everything is free at the start)
  for (int k = 0, index; (index = bwd_index(k)) < 2 * p.tiles * p.bh; ++k) {
    const BwdItem it = bwd_item(p, index);
    const CUtensorMap *own0 = it.is_dq ? &map_q : &map_k, *own1 = it.is_dq ? &map_do : &map_v;
    const CUtensorMap *first = it.is_dq ? &map_k : &map_q, *second = it.is_dq ? &map_v : &map_do;
    for (int i = 0; i < it.tiles; ++i) {
      const int c0 = (it.begin + i) * 128;
      if (!mbar_wait(b.first_empty + f.slot, f.parity, b.abort_flag)) return false;
      mbar_arrive_expect_tx(b.first_full + f.slot, Cfg::kTileBytes);
      tma_load_4d(smem + Cfg::kOffFirst + f.slot * Cfg::kTileBytes, first, b.first_full + f.slot, 0, c0, 0, it.bh);
      f.advance();
      if (i == 0) {
        if (!mbar_wait(b.own_empty, own.parity, b.abort_flag)) return false;
        own.advance();
        mbar_arrive_expect_tx(b.own_full, 2 * Cfg::kTileBytes);
        tma_load_4d(smem, own0, b.own_full, 0, it.r0, 0, it.bh);
        tma_load_4d(smem + Cfg::kTileBytes, own1, b.own_full, 0, it.r0, 0, it.bh);
      }
      if (!mbar_wait(b.second_empty + s.slot, s.parity, b.abort_flag)) return false;
      mbar_arrive_expect_tx(b.second_full + s.slot, Cfg::kTileBytes);
#ifdef FA_TEST_WITHHOLD_LOAD
      if (!(p.withhold && index == 0 && i == it.tiles - 1))
#endif
        tma_load_4d(smem + Cfg::kOffSecond + s.slot * Cfg::kTileBytes, second, b.second_full + s.slot, 0, c0, 0, it.bh);
      s.advance();
    }
  }
  return true;
}

// What bwd_rows_kernel computes, by the softmax warps of a CTA for all rows of its one item's head; the norms of the rows that bound
// the item's dS.
template <int D>
__device__ __forceinline__ void bwd_own_rows(const BwdParams& p, const BwdItem& it, uint8_t* smem, int warp, int lane) {
  using Cfg = BwdCfg<D>;
  constexpr int kRows = 32 / (D / 8);  // of a warp at a time
  float* delta_of = reinterpret_cast<float*>(smem + Cfg::kOffOwnRows);
  float* norm_of = delta_of + Cfg::kMaxOwnRows;  // |dO_i|^2
  float* norms = norm_of + Cfg::kMaxOwnRows;
  float top[3] = {0.f, 0.f, 0.f};
#pragma unroll 4
  for (int r0 = warp * kRows; r0 < p.seqlen; r0 += 16 * kRows) {
    const int r = r0 + lane / (D / 8);
    float delta, gg, vv;
    bwd_row<D>(p, it.bh, r, lane, delta, gg, vv);
    if (r < p.seqlen && lane % (D / 8) == 0) {
      delta_of[r] = delta;
      norm_of[r] = gg;
    }
    const bool own = r / 128 == it.r0 / 128, column = r / 128 >= it.begin && r / 128 < it.begin + it.tiles;
    if (it.is_dq ? own : column) {
      top[0] = fmaxf(top[0], bwd_norm(gg));
      top[2] = fmaxf(top[2], bwd_norm(fabsf(delta)));
    }
    if (it.is_dq ? column : own) top[1] = fmaxf(top[1], bwd_norm(vv));
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const float m = warp_max(top[k]);
    if (lane == 0) norms[warp * 3 + k] = k < 2 ? sqrt_approx(m) : m;
  }
  __syncwarp();
  mbar_arrive_lane0(reinterpret_cast<uint64_t*>(norms + 48), lane);
}

// The warp that brings the statistics: for dK and dV those of every column tile, for dQ those of the item's own rows, each with its
// unit.
template <int D, bool kAlibi, bool kOwnRows>
__device__ __forceinline__ void bwd_stats(const BwdParams& p, const BwdBars& b, uint8_t* smem, int lane) {
  using Cfg = BwdCfg<D>;
  Turn<Cfg::kStats> at;
  at.parity = 1;
  griddep_wait();
  const float* delta_here = reinterpret_cast<const float*>(smem + Cfg::kOffOwnRows);
  const float* norm_here = delta_here + Cfg::kMaxOwnRows;
  const float* norms_here = norm_here + Cfg::kMaxOwnRows;
  for (int k = 0, index; (index = bwd_index(k)) < 2 * p.tiles * p.bh; ++k) {
    const BwdItem it = bwd_item(p, index);
    const int c0 = it.is_dq ? it.r0 : it.begin * 128;
    float nl[4], nd[4], g[4];
    auto load = [&](int i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = c0 + i * 128 + j * 32 + lane;
        const size_t from = static_cast<size_t>(it.bh) * p.seqlen + c;
        nl[j] = c < p.seqlen ? fmaf(p.lse[from], -1.4426950408889634f, 14.f) : -INFINITY;
        if (!kOwnRows) nd[j] = c < p.seqlen ? -p.delta[from] : 0.f;
      }
    };
    load(0);  // (on its way while the norms are read)
    if (!kOwnRows && it.is_dq) {  // (this CTA alone writes the rows, and not before it has these statistics)
      const float* norm_of = reinterpret_cast<const float*>(p.dq + (static_cast<size_t>(it.bh) * p.seqlen + it.r0) * D);
#pragma unroll
      for (int j = 0; j < 4; ++j) g[j] = it.r0 + j * 32 + lane < p.seqlen ? norm_of[j * 32 + lane] : 0.f;
    }
    const float slope = kAlibi ? p.alibi_slopes[it.bh % p.heads] * 1.4426950408889634f : 0.f;
    float norm[3] = {0.f, 0.f, 0.f};
    if (kOwnRows) {
      if (!mbar_wait_warp(reinterpret_cast<uint64_t*>(const_cast<float*>(norms_here + 48)), 0, b.abort_flag)) return;
      for (int j = 0; j < 3; ++j) norm[j] = lane < 16 ? norms_here[lane * 3 + j] : 0.f;
    } else {
      const float* norms = p.norms + static_cast<size_t>(it.bh) * p.tiles * 3;
      for (int t = it.begin + lane; t < it.begin + it.tiles; t += 32) {
        if (it.is_dq) {
          norm[1] = fmaxf(norm[1], norms[3 * t + 1]);
        } else {
          norm[0] = fmaxf(norm[0], norms[3 * t]);
          norm[2] = fmaxf(norm[2], norms[3 * t + 2]);
        }
      }
      if (!it.is_dq) norm[1] = norms[it.r0 / 128 * 3 + 1];
    }
    for (int j = 0; j < 3; ++j) norm[j] = warp_max(norm[j]);
    // of dK and dV; dQ has one a row
    const float unit = __uint_as_float(bwd_unit_exponent(fmaf(norm[0], norm[1], norm[2])) << 23);
    for (int i = 0; i < (it.is_dq ? 1 : it.tiles); ++i) {
      if (i > 0) load(i);
      if (kOwnRows) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int c = c0 + i * 128 + j * 32 + lane;
          nd[j] = c < p.seqlen ? -delta_here[c] : 0.f;
          g[j] = c < p.seqlen ? norm_here[c] : 0.f;
        }
      }
      if (!mbar_wait_warp(b.stats_empty + at.slot, at.parity, b.abort_flag)) return;
      float* to = reinterpret_cast<float*>(smem + Cfg::kOffStats + at.slot * 1024);
      if (it.is_dq) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t e = bwd_unit_exponent(fmaf(sqrt_approx(bwd_norm(g[j])), norm[1], bwd_norm(fabsf(nd[j]))));
          nd[j] *= __uint_as_float(e << 23);
          smem[Cfg::kOffUnits + at.slot * 128 + j * 32 + lane] = static_cast<uint8_t>(e);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) nd[j] *= unit;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        to[j * 32 + lane] = nl[j];
        to[128 + j * 32 + lane] = nd[j];
      }
      if (i == 0 && lane == 0) {
        b.unit[k & 1] = unit;
        if (kAlibi) b.slope[k & 1] = slope;
      }
      __syncwarp();
      mbar_arrive_lane0(b.stats_full + at.slot, lane);
      at.advance();
    }
  }
}

// One CTA a SM walks the work items bwd_index(0), bwd_index(1), ... (a CTA an item, started by the hardware, took 7 us an item
// for its start and end: window 1024 2576 -> 2153 us with all that came with it). Bound by the tensor pipe at head_dim 128: 4510
// clocks a pair of tiles for 3584 of products, 79 % busy at 1.3-1.5 GHz under the power cap; B2 H32 N8192 causal 3400-3560 us,
// 770-810 TFLOP/s of the five products that the gradient has; B2 H16 N4096 d64 causal 266-304 us. 20 warps: 0-15 softmax and
// epilogue, 16 issues the products, 17 loads tiles, 18 brings the statistics, 19 only donates registers.
// kOwnRows: short heads, an item a CTA, no bwd_rows_kernel: the softmax warps, idle until the first products, do its work for
// their CTA, each CTA for all rows of its head.
template <int D, bool kAlibi, bool kOwnRows>
__global__ void __launch_bounds__(640, 1)
bwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
           const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do,
           const __grid_constant__ BwdParams p) {
  using Cfg = BwdCfg<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kOffBars);
  BwdBars b;
  b.first_full = bars;
  b.first_empty = b.first_full + Cfg::kFirst;
  b.second_full = b.first_empty + Cfg::kFirst;
  b.second_empty = b.second_full + Cfg::kSecond;
  b.stats_full = b.second_empty + Cfg::kSecond;
  b.own_full = b.stats_full + Cfg::kStats;
  b.own_empty = b.own_full + 1;
  b.acc_full = b.own_full + 2;
  b.dp_full = b.own_full + 3;
  b.s_full = b.own_full + 4;
  b.stats_empty = b.own_full + 6;  // from here on it is the softmax warps that arrive
  b.p_ready = b.stats_empty + Cfg::kStats;
  b.ds_ready = b.p_ready + 2;
  b.acc_empty = b.p_ready + 3;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Cfg::kNumBars);
  b.abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  b.unit = reinterpret_cast<volatile float*>(tmem_slot + 2);
  b.slope = b.unit + 2;
  // The shuffles let the compiler see that the warp's number and the address in tensor memory are the same in all lanes: the
  // issuer's branch then is one that a warp takes as a whole, and the operands of its products are computed in uniform registers,
  // not moved there one by one. 17 -> 12 clocks for the instructions around a product, more where the softmax warps compete for
  // the issue slots: 8 heads x 2048 d64 41.4 -> 38.2 us, B8 H12 N1000 d64 128 -> 119, B2 H32 N8192 d128 causal 3790 -> 3400.
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (warp == 16) {
    tmem_alloc(tmem_slot, Cfg::kTmemCols);
    tmem_relinquish();
  }
  static_assert(Cfg::kNumBars <= 64);
  if (warp == 0) {  // (a thread for one barrier or two: one after the other they cost a short call 0.2 us)
    for (int i = lane; i < Cfg::kNumBars; i += 32) mbar_init(bars + i, bars + i >= b.stats_empty ? Cfg::kSoftmaxWarps : 1);
    if (lane == 0) {
      *b.abort_flag = 0;
      if (kOwnRows) mbar_init(reinterpret_cast<uint64_t*>(smem + Cfg::kOffOwnRows + Cfg::kOwnRowsBytes - 8), Cfg::kSoftmaxWarps);
    }
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  if (kOwnRows) griddep_wait();
  // bwd_rows_kernel lets this kernel in only behind its own griddep_wait(): whatever came before the two of them is complete,
  // and only the warp that reads what bwd_rows_kernel writes has to wait for it. (Every CTA has one, so whoever waits for this
  // kernel has waited for both.)
  griddep_launch();

  if (warp < Cfg::kSoftmaxWarps) {
    reg_inc<Cfg::kRegSoftmax>();
    BwdItem next = bwd_item(p, bwd_index(0));
    if (kOwnRows) bwd_own_rows<D>(p, next, smem, warp, lane);
    SoftmaxTurns<D> at;
    bool ok = true;
    for (int k = 0; bwd_index(k) < 2 * p.tiles * p.bh && ok; ++k) {
      const BwdItem it = next;
      ok = it.is_dq ? bwd_softmax<D, kAlibi, true>(p, it, next, b, smem, tmem_base, warp, lane, k, at)
                    : bwd_softmax<D, kAlibi, false>(p, it, next, b, smem, tmem_base, warp, lane, k, at);
    }
  } else {
    reg_dec<Cfg::kRegOthers>();
    if (warp == 16) {
      bwd_issue<D>(p, b, smem, tmem_base);
    } else if (warp == 17) {
      // (a give-up leaves loads in flight: they land before the CTA retires)
      if (elect_one() && !bwd_load<D>(map_q, map_k, map_v, map_do, p, b, smem))
        for (int i = 0; i < 64; ++i) __nanosleep(2000);
      __syncwarp();
    } else if (warp == 18) {
      bwd_stats<D, kAlibi, kOwnRows>(p, b, smem, lane);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *b.abort_flag != 0) atomicExch(p.status, 1);
  if (warp == 16) tmem_dealloc(tmem_base, Cfg::kTmemCols);
}

}  // namespace fa
