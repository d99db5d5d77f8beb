// The attention of new tokens over the paged cache for more than 16 rows (query heads of a key head times new tokens).
#pragma once
#include "paged_cache.cuh"

namespace fa {

template <int D>
struct WideCfg {
  static constexpr int kSoftmaxWarps = 8;
  static constexpr int kThreads = (kSoftmaxWarps + 4) * 32;
  static constexpr int kRows = 128;
  static constexpr int kKeys = kDecodeKeys<D>;
  static constexpr int kPanelBytes = kKeys * 128, kHalfBytes = kKeys * D * 2;  // 64 columns of a tile; K or V of a tile
  // Tiles whose scores have a place. At head_dim 64 a third is worth 10-13 % (16 x 8 tokens, 64 heads on 8, up to 32768: 160 ->
  // 138 us): the scores of a group's next tile are there before its P is done. At head_dim 128, where a tile's scores are half as
  // many and each tile held back is one less on its way, three or four cost such calls 2-4 %, and looking for what can be done next
  // costs more than it finds (2048 tokens over 8192 keys 404 -> 480).
  static constexpr int kRegions = D == 128 ? 2 : 3;
  static constexpr int kQBytes = kRows * D * 2;
  static constexpr int kStages = D == 128 ? 5 : 6;
  static constexpr int kOffRing = 2 * kQBytes;  // behind Q of this item and of the next
  static constexpr int kOffMl = kOffRing + kStages * 2 * kHalfBytes;
  static constexpr int kOffBars = kOffMl + 2 * kRows * 8;
  static constexpr int kNumBars = 2 * kStages + kRegions + 11;
  static constexpr int kSmemBytes = kOffBars + kNumBars * 8 + 16;
  // tensor memory: scores of either group of softmax warps, in which P takes their place, and its O
  static constexpr uint32_t kColO = kRegions * kKeys;
  static constexpr float kLazy = 8.f;
  static constexpr int kRoom = 7;  // in fp16: P is kept as 2^kRoom P
  static constexpr int kMaxCopies = kKeys / 32;
};

// A CTA's 128 rows are the M of tcgen05 products: S = Q K^T of a tile, then O += P V with P in tensor memory in the place of S
// (32 keys' operand in the first 16 of 32 columns). Two groups of four softmax warps take the tiles in turn, each with its S,
// its O and its statistics, so that a tile's chain (product, load, maximum, exponentials, P, product) has the time that two
// tiles of 32 KB take to arrive; they are joined at the end of the item, where both O lie in the same lanes. A thread has a row:
// no exchange for its maximum and sum. Where the rows fill half of the 128 or a quarter, M holds copies of them, of which each
// takes a part of a tile's keys (its P is 0 for the others), so that all warps share the exponentials; the copies are summed at
// the end of the item (32 rows d64 x up to 8192: 62 -> 46 us). The reference that a row's exponentials are taken against moves
// only when the maximum has grown by 2^8 over it, so that O is rarely rescaled, or along with another row of the warp that has to
// (the key that sets it has P = 1 exactly, one above it a P that is rounded); P is at most 2^8 and is rounded once to the cache's
// type, in fp16 as 2^7 P: half a step off down to 2^-21 of the row's maximum, and at most 2^-32 of that below. Warps whose rows are
// all padding only hand on. Everything is summed in an order that depends on the lengths alone.
// 12 warps: 0-7 softmax, 8 issues the products, 9 loads, 10 and 11 bring Q of the next item (with Q brought by the softmax warps
// themselves an item took 5000 clocks more).
// Bound by HBM where contexts are long: 16 x 8 tokens, 64 heads on 8 of 128, up to 32768 tokens 209 us (5.8 TB/s); by the chain
// where many tokens share the keys: 2048 tokens of 32 heads on 8 over 8192 keys, 241 GFLOP under the mask, in 404 us, an eighth
// of it for tiles that a row tile does not see (the line has a sequence's tiles for every row tile; of a prompt without a past it is
// half). An item's start and end take as long as six tiles.
template <typename T, int D>
__global__ void __launch_bounds__(WideCfg<D>::kThreads, 1)
decode_wide_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                   const __grid_constant__ DecodeParams p) {
  using Cfg = WideCfg<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Cfg::kOffBars);
  uint64_t* empty = full + Cfg::kStages;
  uint64_t* s_full = empty + Cfg::kStages;  // one a region
  uint64_t* o_full = s_full + Cfg::kRegions;
  uint64_t* o_done = o_full + 1;            // two, of either group: a product has been summed
  uint64_t* q_full = o_full + 3;            // two
  uint64_t* q_empty = o_full + 5;           // two
  uint64_t* p_ready = o_full + 7;           // of tile i the (i % 4)th: a warp may be a tile of its group ahead of another
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(full + Cfg::kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  // (shuffles: the compiler then sees that the issuing warp's operands are uniform)
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (warp == Cfg::kSoftmaxWarps) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < Cfg::kNumBars; ++i)
      mbar_init(full + i, full + i >= p_ready ? Cfg::kSoftmaxWarps / 2 : full + i >= q_empty ? Cfg::kSoftmaxWarps
                                                                       : full + i >= q_full ? 2 : 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  griddep_wait();
  DecodeWalk walk;
  walk.start(p, blockIdx.x, lane);
  griddep_launch();
  int kv_head, row_tile, t0, t1;
  bool ok = true;

  if (warp < Cfg::kSoftmaxWarps) {
    const int group = warp >> 2, in_tile = (warp & 3) * 32 + lane;
    const int rows = p.group * p.cache.tokens;
    // copies of the row tile among the 128 rows, and this warp's
    const int copies = rows <= Cfg::kRows / Cfg::kMaxCopies ? Cfg::kMaxCopies : rows <= Cfg::kRows / 2 ? 2 : 1;
    const int copy_rows = Cfg::kRows / copies, copy = in_tile / copy_rows;
    const int chunks = Cfg::kKeys / 32 / copies, first_chunk = copy * chunks;  // 32 keys of a tile each: this thread's
    const uint32_t t_o = tmem_addr(tmem, (warp & 3) * 32, Cfg::kColO);  // of group 0
    float2* ml = reinterpret_cast<float2*>(smem + Cfg::kOffMl);         // [group][row]
    uint32_t s_at = 0, done_at = 0, o_at = 0, q_at = 0;  // parities at the start of the item; s_at: a bit a region
    int loaded = 0;  // tiles of the items before
    constexpr int kRoom = std::is_same_v<T, __half> ? Cfg::kRoom : 0;
    while (walk.next(p, kv_head, row_tile, t0, t1)) {
      const int n = t1 - t0, r = row_tile * Cfg::kRows + in_tile % copy_rows;
      const int t = r / p.group, head = kv_head * p.group + r % p.group;
      const bool there = r < rows, real = there && t < walk.count;
      const bool idle = row_tile * Cfg::kRows + (warp & 3) * 32 % copy_rows >= rows;
      const int last_key = real ? walk.length - walk.count + t : -1, first_query = walk.length - walk.count;
      const int lo = p.window_left >= 0 ? first_query - p.window_left : 0;
      const float slope = real && p.alibi_slopes ? p.alibi_slopes[head] * 1.4426950408889634f : 0.f;
      float m = -INFINITY, l = 0.f;
      for (int i = group; i < n; i += 2) {
        const int key0 = (walk.first + t0 + i) * Cfg::kKeys;
        // does every row see every key of the tile?
        const bool cut = key0 + Cfg::kKeys > first_query + 1 ||
                         (p.window_left >= 0 && key0 < walk.length - 1 - p.window_left);
        const int region = i % Cfg::kRegions;
        const uint32_t t_s = tmem_addr(tmem, (warp & 3) * 32, region * Cfg::kKeys);
        ok &= mbar_wait(s_full + region, (s_at >> region ^ i / Cfg::kRegions) & 1, abort_flag);
        tc_fence_after();
        if (cut) {
          // what lies behind the last token, or in pages in front of the window, is not the sequence's: any bits at all, and
          // 0 * NaN is NaN
          const int stage = (loaded + i) % Cfg::kStages, key = key0 + in_tile % Cfg::kKeys;
          ok &= mbar_wait(full + stage, (loaded + i) / Cfg::kStages & 1, abort_flag);
          if (key >= walk.length || key < lo) {
            uint8_t* row = smem + Cfg::kOffRing + stage * 2 * Cfg::kHalfBytes + Cfg::kHalfBytes +
                           in_tile / Cfg::kKeys * Cfg::kPanelBytes + in_tile % Cfg::kKeys * 128;
#pragma unroll
            for (int c = 0; c < 8; ++c) reinterpret_cast<uint4*>(row)[c] = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (!idle) {
          auto values = [&](int chunk, float (&x)[32]) {  // scores in log2 units
            uint32_t s[32];
            tmem_ld32(t_s + chunk * 32, s);
            tmem_wait_ld();
            tmem_ld_fence(s);
#pragma unroll
            for (int c = 0; c < 32; ++c) x[c] = __uint_as_float(s[c]) * p.scale_log2;
            const int key = key0 + chunk * 32;
            if (p.alibi_slopes) {
#pragma unroll
              for (int c = 0; c < 32; ++c) x[c] = fmaf(-slope, fabsf(static_cast<float>(last_key - key - c)), x[c]);
            }
            if (cut) {
              const int from = p.window_left >= 0 ? last_key - p.window_left : 0;
#pragma unroll
              for (int c = 0; c < 32; ++c)
                if (key + c > last_key || key + c < from) x[c] = -INFINITY;
            }
          };
          // (the scores of kKept chunks stay in registers; where a thread has more, they are read again for the exponentials)
          constexpr int kKept = Cfg::kMaxCopies == 2 ? 2 : 1;
          float x[kKept][32], top = -INFINITY;
#pragma unroll 1
          for (int chunk = 0; chunk < chunks; chunk += kKept) {
#pragma unroll
            for (int k = 0; k < kKept; ++k) {
              if (chunk + k >= chunks) break;
              values(first_chunk + chunk + k, x[k]);
              float a = x[k][0], b = x[k][1];
#pragma unroll
              for (int c = 2; c < 32; c += 2) {
                a = fmaxf(a, x[k][c]);
                b = fmaxf(b, x[k][c + 1]);
              }
              top = fmaxf(top, fmaxf(a, b));
            }
          }
          if (__any_sync(0xffffffffu, top - m > Cfg::kLazy)) {  // (the difference is exact where a sum would be rounded)
            const float alpha = top > m ? ex2_approx(reference_of<kRoom>(m) - reference_of<kRoom>(top)) : 1.f;
            m = fmaxf(m, top);
            l *= alpha;
            if (i >= 2) {
              if (Cfg::kRegions > 2) {  // the group's last product has to be summed (else S came behind it)
                ok &= mbar_wait(o_done + group, (done_at ^ i / 2 ^ 1) & 1, abort_flag);
                tc_fence_after();
              }
#pragma unroll 1
              for (int c = 0; c < D; c += 32) {
                uint32_t o[32];
                tmem_ld32(t_o + group * D + c, o);
                tmem_wait_ld();
                tmem_ld_fence(o);
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
                tmem_st32(t_o + group * D + c, o);
              }
            }
          }
          const float off = m == -INFINITY ? 0.f : reference_of<kRoom>(m);
#pragma unroll 1
          for (int chunk = 0; chunk < chunks; chunk += kKept) {
#pragma unroll
            for (int k = 0; k < kKept; ++k) {
              if (chunk + k >= chunks) break;
              if (kKept == 1 && chunks > 1) values(first_chunk + chunk, x[k]);
              uint32_t w[16];
              float a = 0.f, b = 0.f;
#pragma unroll
              for (int c = 0; c < 32; c += 2) {
                const float e0 = ex2_approx(x[k][c] - off), e1 = ex2_approx(x[k][c + 1] - off);
                a += e0;
                b += e1;
                w[c / 2] = from_floats<T>(e0, e1);
              }
              l += a + b;
              tmem_st16(t_s + (first_chunk + chunk + k) * 32, w);
            }
          }
          // the other copies' keys
          const uint32_t zero[16] = {};
#pragma unroll
          for (int chunk = 0; chunk < Cfg::kKeys / 32; ++chunk)
            if (chunk < first_chunk || chunk >= first_chunk + chunks) tmem_st16(t_s + chunk * 32, zero);
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        mbar_arrive_lane0(p_ready + i % 4, lane);
      }
      loaded += n;
#pragma unroll
      for (int r = 0; r < Cfg::kRegions; ++r) s_at ^= ((n + Cfg::kRegions - 1 - r) / Cfg::kRegions & 1) << r;
      done_at ^= (n + 1 - group) / 2 & 1;

      const bool whole = t0 == 0 && t1 == walk.tiles;
      const long long out_row = (static_cast<long long>(walk.b) * p.q_heads + head) * p.cache.tokens + t;
      const long long part = (2ll * blockIdx.x + (t0 == 0 ? 1 : 0)) * p.part_rows + in_tile % copy_rows;
      // ---- the parts of both groups and of all copies joined ----
      ml[group * Cfg::kRows + in_tile] = make_float2(reference_of<kRoom>(m), l);  // what the sum and O were taken against
      if (n > 0) {
        ok &= mbar_wait(o_full, o_at, abort_flag);
        o_at ^= 1;
        tc_fence_after();
      }
      compute_sync<Cfg::kSoftmaxWarps * 32>();
      float top = -INFINITY, sum = 0.f;
      for (int c = 0; c < copies; ++c)
        for (int g = 0; g < 2; ++g) top = fmaxf(top, ml[g * Cfg::kRows + c * copy_rows + in_tile % copy_rows].x);
      const float off = top == -INFINITY ? 0.f : top;
      for (int c = 0; c < copies; ++c)
        for (int g = 0; g < 2; ++g) {
          const float2 other = ml[g * Cfg::kRows + c * copy_rows + in_tile % copy_rows];
          sum = fmaf(other.y, ex2_approx(other.x - off), sum);
        }
      const float s0 = ex2_approx(ml[in_tile].x - off), s1 = ex2_approx(ml[Cfg::kRows + in_tile].x - off);
      const float inv = sum != 0.f ? 1.f / sum : 0.f;
      auto joined = [&](int c, float (&o)[16]) {  // sixteen columns of both groups' O
        uint32_t v[16];
        if (n > 0) {
          tmem_ld16(t_o + c, v);
          tmem_wait_ld();
          tmem_ld_fence16(v);
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) o[k] = n > 0 ? __uint_as_float(v[k]) * s0 : 0.f;
        if (n > 1) {
          tmem_ld16(t_o + D + c, v);
          tmem_wait_ld();
          tmem_ld_fence16(v);
#pragma unroll
          for (int k = 0; k < 16; ++k) o[k] = fmaf(__uint_as_float(v[k]), s1, o[k]);
        }
      };
      auto write = [&](int c, const float4& x) {  // four columns
        if (whole)
          *reinterpret_cast<uint2*>(static_cast<T*>(p.o) + out_row * D + c) =
              real ? make_uint2(from_floats<T>(x.x * inv, x.y * inv), from_floats<T>(x.z * inv, x.w * inv)) : make_uint2(0, 0);
        else
          *reinterpret_cast<float4*>(p.part_o + part * D + c) = x;
      };
      if (copies == 1) {
        if (!idle)
#pragma unroll 1
          for (int c = group * (D / 2); c < (group + 1) * (D / 2); c += 16) {
            float o[16];
            joined(c, o);
            if (there)
#pragma unroll
              for (int k = 0; k < 16; k += 4) write(c + k, make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]));
          }
      } else {
        // Summed through the memory of Q in the copies' order, half of the columns at a time, of which either group has its own:
        // [row][D / 2 columns], 16-byte pieces shuffled by the row.
        auto at = [&](int row, int piece) {
          return reinterpret_cast<float4*>(smem + q_at * Cfg::kQBytes + row * (D * 2) + ((piece ^ (row & 7)) << 4));
        };
        const int first_piece = group * (D / 16), own = D / 16 / copies;
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          if (!idle)
#pragma unroll 1
            for (int step = 0; step < D / 64; ++step) {
              float o[16];
              joined(half * (D / 2) + group * (D / 4) + step * 16, o);
#pragma unroll
              for (int k = 0; k < 4; ++k)
                *at(in_tile, first_piece + step * 4 + k) = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
            }
          compute_sync<Cfg::kSoftmaxWarps * 32>();
          if (there)
            for (int k = copy * own; k < (copy + 1) * own; ++k) {
              float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
              for (int c = 0; c < copies; ++c) {
                const float4 y = *at(c * copy_rows + in_tile % copy_rows, first_piece + k);
                x = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
              }
              write(half * (D / 2) + group * (D / 4) + k * 4, x);
            }
          compute_sync<Cfg::kSoftmaxWarps * 32>();  // before the place is written again
        }
      }
      // (O may be written again, and with p_ready of the next item it will be, once both groups have read it)
      tc_fence_before();
      if (copies == 1) compute_sync<Cfg::kSoftmaxWarps * 32>();
      if (n > 0) {
        mbar_arrive_lane0(q_empty + q_at, lane);
        q_at ^= 1;
      }
      if (there && group == 0 && copy == 0) {
        if (!whole) *reinterpret_cast<float2*>(p.part_ml + part * 2) = make_float2(top, sum);
        else if (p.lse) p.lse[out_row] = real ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
      }
    }
  } else if (warp == Cfg::kSoftmaxWarps) {
    // ---- products ----
    constexpr uint32_t kType = std::is_same_v<T, __half> ? 0u : 1u << 7 | 1u << 10;
    constexpr uint32_t idesc_s = umma_idesc_f16(128, Cfg::kKeys, 0, 0) | kType, idesc_o = umma_idesc_f16(128, D, 0, 1) | kType;
    constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29), kKMajor = 1u << 16,
                       kMnMajor = static_cast<uint32_t>(Cfg::kPanelBytes >> 4) << 16;
    const uint32_t q_first = smem_u32(smem) >> 4, ring = smem_u32(smem + Cfg::kOffRing) >> 4;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      ok &= mbar_wait(bar, parity, abort_flag);
      tc_fence_after();
    };
    int s_stage = 0, o_stage = 0, q_buffer = 0;
    uint32_t s_phase = 0, q_phase = 0, p_at = 0, q = q_first;
    auto scores = [&](int region) {  // of the next tile, which is there
      const uint32_t k = ring + s_stage * (2 * Cfg::kHalfBytes >> 4);
#pragma unroll
      for (int h = 0; h < D / 64; ++h)
        umma_qk64(tmem + region * Cfg::kKeys, (q + h * (Cfg::kRows * 128 >> 4)) | kKMajor,
                  (k + h * (Cfg::kPanelBytes >> 4)) | kKMajor, kDescHi, idesc_s, h);
      umma_commit_warp(s_full + region);
      if (++s_stage == Cfg::kStages) s_stage = 0, s_phase ^= 1;
    };
    auto product = [&](int i, int region) {
      const int group = i & 1;
      const uint32_t v = ring + (o_stage * 2 * Cfg::kHalfBytes + Cfg::kHalfBytes >> 4);
#pragma unroll
      for (int c = 0; c < Cfg::kKeys / 64; ++c)
        umma_x64(tmem + Cfg::kColO + group * D, tmem + region * Cfg::kKeys + 64 * c, (v + c * (64 * 128 >> 4)) | kMnMajor, kDescHi,
                 idesc_o, i >= 2 || c > 0);
      umma_commit_warp(empty + o_stage);
      if (Cfg::kRegions > 2) umma_commit_warp(o_done + group);
      if (++o_stage == Cfg::kStages) o_stage = 0;
    };
    while (ok && walk.next(p, kv_head, row_tile, t0, t1)) {
      const int n = t1 - t0;
      if (n <= 0) continue;
      wait(q_full + q_buffer, q_phase);
      q = q_first + q_buffer * (Cfg::kQBytes >> 4);
      if (q_buffer ^= 1; q_buffer == 0) q_phase ^= 1;
      // (S goes where the P of a product in front of it was)
      if constexpr (Cfg::kRegions == 2) {
        for (int i = 0; i < 2 && i < n; ++i) {
          wait(full + s_stage, s_phase);
          scores(i);
        }
        for (int i = 0; i < n && ok; ++i) {
          wait(p_ready + i % 4, p_at >> i % 4 & 1u);
          p_at ^= 1u << i % 4;
          product(i, i & 1);
          if (i + 2 < n) {
            wait(full + s_stage, s_phase);
            scores(i & 1);
          }
          ok = __all_sync(0xffffffffu, ok);
        }
      } else {
        // S of as many tiles ahead as there are regions, each once its tile is there; O in the tiles' order, each once its P is
        // there; whichever can be done next
        int s_next = 0, polls = 0;
        for (int i = 0; i < n && ok;) {
          const int p_bar = i % 4;
          const bool ahead = s_next < min(n, i + Cfg::kRegions);
          if (ahead && __all_sync(0xffffffffu, mbar_test(full + s_stage, s_phase))) {
            tc_fence_after();
            scores(s_next % Cfg::kRegions);
            ++s_next;
            polls = 0;
          } else if (i < s_next && __all_sync(0xffffffffu, mbar_test(p_ready + p_bar, p_at >> p_bar & 1u))) {
            tc_fence_after();
            p_at ^= 1u << p_bar;
            product(i, i % Cfg::kRegions);
            ++i;
            polls = 0;
          } else if (!ahead) {  // only P can come
            ok = mbar_wait_warp(p_ready + p_bar, p_at >> p_bar & 1u, abort_flag);
          } else {
            __nanosleep(40);  // (the softmax warps beside this one need the issue slots)
            if ((++polls & 63) == 0) {
              if (polls >= 16 * FA_WAIT_LIMIT_POLLS) *abort_flag = 1;  // 0.4 s
              ok = __all_sync(0xffffffffu, *abort_flag == 0);
            }
          }
        }
      }
      umma_commit_warp(o_full);
    }
  } else if (warp == Cfg::kSoftmaxWarps + 1) {
    // ---- loads: a lane looks up the page of a box of a tile, for as many tiles at a time as there are lanes and the next ones
    // ahead (one tile at a time the table's latency was most of what a tile took), and brings its keys and values, 64 columns
    // at a time ----
    const int boxes = Cfg::kKeys / p.box_rows, at_once = 32 / boxes, of_tile = lane / boxes, box = lane % boxes;
    const uint32_t box_bytes = p.box_rows * 128;
    int stage = 0;
    uint32_t phase = 0;
    while (ok && walk.next(p, kv_head, row_tile, t0, t1)) {
      const int lo = p.window_left >= 0 && walk.length - walk.count > p.window_left
                         ? walk.length - walk.count - p.window_left : 0;
      const int* table = p.cache.page_table + walk.b * p.cache.table_stride;
      auto page_of = [&](int first_tile) {  // -1: the box holds nothing that is seen
        const int tile = first_tile + of_tile, key = (walk.first + tile) * Cfg::kKeys + box * p.box_rows;
        if (tile >= t1 || key >= walk.length || key + p.box_rows <= lo) return -1;
        const int page = table[key / p.cache.page_size];
        if (page >= 0 && page < p.cache.num_pages) return page;
        atomicExch(p.cache.bad_index, 1);
        return -1;
      };
      int next_page = page_of(t0);
      for (int t = t0; ok && t < t1; t += at_once) {
        const int page = next_page;
        next_page = page_of(t + at_once);
        for (int j = 0; j < at_once && t + j < t1; ++j) {
          ok = mbar_wait_warp(empty + stage, phase ^ 1, abort_flag);
          if (!ok) break;
          bool mine = of_tile == j && page >= 0;
          const unsigned here = __ballot_sync(0xffffffffu, mine);
          if (lane == 0) mbar_arrive_expect_tx(full + stage, 2 * (D / 64) * box_bytes * __popc(here));
          __syncwarp();
#ifdef FA_TEST_WITHHOLD_LOAD
          if (p.withhold && walk.b == 0 && t + j == walk.tiles - 1) mine = false;
#endif
          if (mine) {
            uint8_t* dst = smem + Cfg::kOffRing + stage * 2 * Cfg::kHalfBytes + box * box_bytes;
            const int row = ((walk.first + t + j) * Cfg::kKeys + box * p.box_rows) % p.cache.page_size;
#pragma unroll
            for (int h = 0; h < D / 64; ++h) {
              tma_load_5d(dst + h * Cfg::kPanelBytes, &map_k, full + stage, 0, row, h, kv_head, page);
              tma_load_5d(dst + Cfg::kHalfBytes + h * Cfg::kPanelBytes, &map_v, full + stage, 0, row, h, kv_head, page);
            }
          }
          if (++stage == Cfg::kStages) stage = 0, phase ^= 1;
        }
      }
    }
  } else {
    // ---- Q of the next item: two warps, neighbouring lanes neighbouring pieces of a row ----
    const int rows = p.group * p.cache.tokens;
    const int copy_rows = rows <= Cfg::kRows / Cfg::kMaxCopies ? Cfg::kRows / Cfg::kMaxCopies
                          : rows <= Cfg::kRows / 2             ? Cfg::kRows / 2 : Cfg::kRows;
    int buffer = 0;
    uint32_t phase = 0;
    while (ok && walk.next(p, kv_head, row_tile, t0, t1)) {
      if (t1 <= t0) continue;
      ok = mbar_wait_warp(q_empty + buffer, phase ^ 1, abort_flag);
      if (!ok) break;
      constexpr int kPieces = D / 8, kAtOnce = 8;
      for (int i0 = (warp & 1) * 32 + lane; i0 < Cfg::kRows * kPieces; i0 += 64 * kAtOnce) {
        uint4 piece[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
          const int i = i0 + 64 * k, c = i % kPieces, r = row_tile * Cfg::kRows + i / kPieces % copy_rows, t = r / p.group;
          const T* q = static_cast<const T*>(p.q.data) + walk.b * p.q.batch_stride +
                       (kv_head * p.group + r - t * p.group) * p.q.head_stride + t * p.q.token_stride + c * 8;
          piece[k] = r < rows && t < walk.count ? *reinterpret_cast<const uint4*>(q) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
          const int i = i0 + 64 * k, c = i % kPieces, row = i / kPieces;
          *reinterpret_cast<uint4*>(smem + buffer * Cfg::kQBytes + c / 8 * (Cfg::kRows * 128) + row * 128 +
                                    ((c % 8 ^ (row & 7)) << 4)) = piece[k];
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      mbar_arrive_lane0(q_full + buffer, lane);
      if (buffer ^= 1; buffer == 0) phase ^= 1;
    }
  }
  if (!ok && lane == 0) atomicExch(p.status, 1);
  tc_fence_before();
  __syncthreads();
  if (warp == Cfg::kSoftmaxWarps) tmem_dealloc(tmem, 512);
  if (*abort_flag)
    for (int i = 0; i < 64; ++i) __nanosleep(2000);  // loads in flight land before the CTA retires
}

}  // namespace fa
