// Kernels of the paged key-value cache: new keys and values enter it (cache_append_kernel), and the newest tokens of every
// sequence attend to what it holds (decode_kernel here, decode_wide_kernel where there are many rows, and decode_join_kernel for
// the sequences that several CTAs shared).
//
// The keys and values of a sequence lie in pages of `page_size` tokens that its row of the page table names in order:
// token j is row j % page_size of page table[j / page_size]. Nothing of a page behind the sequence's last token, and no
// entry of the table behind its last page, is read.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "ptx.cuh"

namespace fa {

struct CacheView {
  long long page_stride, head_stride, token_stride;  // elements
  int num_pages, page_size, kv_heads;
  const int* page_table;  // [batch][table_stride], max_pages entries a row
  long long table_stride;
  int max_pages;
  const int* lengths;  // tokens of every sequence, the new ones included
  const int* counts;   // new tokens of every sequence, or nullptr: `tokens` each
  int batch, tokens;
  int* bad_index;  // device word, set to 1 where an index in device memory is out of range
};

struct StridedRows {  // [batch][head][token] rows of head_dim contiguous elements
  const void* data;
  long long batch_stride, head_stride, token_stride;  // elements
};

// Length and number of new tokens of sequence b, within what the table and the call can hold: 0 <= count <= tokens,
// count <= length <= max_pages * page_size. Anything else is reported and cut to that.
__device__ __forceinline__ void sequence_of(const CacheView& c, int b, int& length, int& count) {
  const int len = c.lengths[b];
  const int cnt = c.counts ? c.counts[b] : c.tokens;
  const long long room = static_cast<long long>(c.max_pages) * c.page_size;
  length = len < 0 ? 0 : len > room ? static_cast<int>(room) : len;
  count = cnt < 0 ? 0 : cnt > c.tokens ? c.tokens : cnt;
  // (a sequence of length 0 is one that is not there: it needs no count of its own)
  if (length != len || (len > 0 && (count != cnt || count > length))) atomicExch(c.bad_index, 1);
  if (count > length) count = length;
}

template <typename T>
__device__ __forceinline__ float2 to_float2(uint32_t v) {
  if constexpr (std::is_same_v<T, __half>) return __half22float2(*reinterpret_cast<__half2*>(&v));
  else return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v));
}
template <typename T>
__device__ __forceinline__ uint32_t from_floats(float lo, float hi) {
  if constexpr (std::is_same_v<T, __half>) {
    return pack_f16x2(lo, hi);
  } else {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------------------------------------------------
struct AppendParams {
  CacheView cache;
  void *k_pages, *v_pages;
  StridedRows k, v, q;  // q.data may be nullptr
  void* q_out;          // [batch][q_heads][tokens][head_dim]
  int q_heads;
  const float* rotary;  // [positions][rotary_dim]: rotary_dim / 2 cosines, then as many sines; nullptr: nothing is rotated
  int rotary_dim, positions, interleaved;
  int row_units;  // (2 * kv_heads + q_heads) * (head_dim / 16)
};

// Rotates the four pairs of neighbours of an 16-byte piece.
template <typename T>
__device__ __forceinline__ uint4 turn_pairs(const uint4& x, const float* cosines, const float* sines) {
  const float4 cs = *reinterpret_cast<const float4*>(cosines), sn = *reinterpret_cast<const float4*>(sines);
  auto one = [](uint32_t v, float c, float s) {
    const float2 z = to_float2<T>(v);
    return from_floats<T>(z.x * c - z.y * s, z.x * s + z.y * c);
  };
  return make_uint4(one(x.x, cs.x, sn.x), one(x.y, cs.y, sn.y), one(x.z, cs.z, sn.z), one(x.w, cs.w, sn.w));
}

// One thread moves two 16-byte pieces of one row, half of the rotated part (or of the rest of the row) apart, so that both
// elements of every pair of a rotation by halves are in one thread and neighbouring threads move neighbouring pieces. Keys and
// queries are turned in fp32 by the cosine and sine of their position and rounded once; values, and what lies behind
// rotary_dim, are copied as bits. Bound by the bytes moved (rows of padding are not read); a step of generation by the launch
// and three dependent reads (length, page, row). A grid of blocks per token: its divisions cost a block's threads little,
// where one thread per piece of a long line of pieces spent its time on 64-bit remainders, and waited for rows of padding:
// 8 x 2048 tokens, half of them padding, 48 heads: 66.2 -> 43.6 us.
template <typename T, int D>
__global__ void __launch_bounds__(128) cache_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int kUnits = D / 16;
  const int unit = blockIdx.y * 128 + threadIdx.x;
  const int t = blockIdx.x % p.cache.tokens, b = blockIdx.x / p.cache.tokens;
  griddep_wait();
  int length, count;
  sequence_of(p.cache, b, length, count);
  if (unit >= p.row_units) return;
  const int h = unit / kUnits, c = unit % kUnits;
  const bool is_q = h >= 2 * p.cache.kv_heads, is_v = !is_q && h >= p.cache.kv_heads;
  const int head = is_q ? h - 2 * p.cache.kv_heads : is_v ? h - p.cache.kv_heads : h;
  const bool real = t < count;
  if (!real && !is_q) return;

  const int turned = is_v ? 0 : p.rotary_dim;
  const bool turn = c < turned / 16;
  const int part = turn ? turned / 2 : (D - turned) / 2;  // what the two pieces are apart
  const int at0 = turn ? c * 8 : turned + (c - turned / 16) * 8, at1 = at0 + part;
  const int position = length - count + t;
  uint4 x0 = make_uint4(0, 0, 0, 0), x1 = x0;
  if (real) {
    const StridedRows& src = is_q ? p.q : is_v ? p.v : p.k;
    const T* from = static_cast<const T*>(src.data) + b * src.batch_stride + head * src.head_stride + t * src.token_stride;
    x0 = *reinterpret_cast<const uint4*>(from + at0);
    x1 = *reinterpret_cast<const uint4*>(from + at1);
  }
  T* to;
  if (is_q) {
    to = static_cast<T*>(p.q_out) + ((static_cast<long long>(b) * p.q_heads + head) * p.cache.tokens + t) * D;
  } else {
    const int page = p.cache.page_table[b * p.cache.table_stride + position / p.cache.page_size];
    if (page < 0 || page >= p.cache.num_pages) {
      atomicExch(p.cache.bad_index, 1);
      return;
    }
    to = static_cast<T*>(is_v ? p.v_pages : p.k_pages) + page * p.cache.page_stride + head * p.cache.head_stride +
         (position % p.cache.page_size) * p.cache.token_stride;
  }
  if (real && turned > 0 && position >= p.positions) {  // no angles: nothing of the row is written
    atomicExch(p.cache.bad_index, 1);
    return;
  }
  if (real && turn) {
    const float* cosines = p.rotary + static_cast<long long>(position) * p.rotary_dim;
    const float* sines = cosines + p.rotary_dim / 2;
    if (p.interleaved) {
      x0 = turn_pairs<T>(x0, cosines + at0 / 2, sines + at0 / 2);
      x1 = turn_pairs<T>(x1, cosines + at1 / 2, sines + at1 / 2);
    } else {
      uint32_t a[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
      float cs[8], sn[8];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        *reinterpret_cast<float4*>(cs + 4 * i) = *reinterpret_cast<const float4*>(cosines + at0 + 4 * i);
        *reinterpret_cast<float4*>(sn + 4 * i) = *reinterpret_cast<const float4*>(sines + at0 + 4 * i);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 lo = to_float2<T>(a[i]), hi = to_float2<T>(a[4 + i]);
        a[i] = from_floats<T>(lo.x * cs[2 * i] - hi.x * sn[2 * i], lo.y * cs[2 * i + 1] - hi.y * sn[2 * i + 1]);
        a[4 + i] = from_floats<T>(lo.x * sn[2 * i] + hi.x * cs[2 * i], lo.y * sn[2 * i + 1] + hi.y * cs[2 * i + 1]);
      }
      x0 = make_uint4(a[0], a[1], a[2], a[3]);
      x1 = make_uint4(a[4], a[5], a[6], a[7]);
    }
  }
  *reinterpret_cast<uint4*>(to + at0) = x0;
  *reinterpret_cast<uint4*>(to + at1) = x1;
}

// ---------------------------------------------------------------------------------------------------------------------
// attention of the newest tokens
// ---------------------------------------------------------------------------------------------------------------------
// Keys of a tile: 32 KB of keys and values.
template <int D>
constexpr int kDecodeKeys = D == 128 ? 64 : 128;

struct DecodeParams {
  CacheView cache;
  StridedRows q;
  void* o;     // [batch][q_heads][tokens][head_dim]
  float* lse;  // [batch][q_heads][tokens], or nullptr
  int q_heads, group;  // group: query heads of a key head
  float scale_log2;
  int window_left;  // < 0: unbounded
  const float* alibi_slopes;
  int tile_shift;  // a tile has 2^tile_shift keys
  int box_rows;   // rows of a page that one TMA box brings: the largest power of two that divides page_size, a tile at most
  int row_tiles;  // of the group * tokens rows of a key head
  int ctas;
  int cluster;     // CTAs of a cluster that share an item and join it themselves (1: a CTA an item), or 0: the line below
  float* part_o;   // [ctas][2][part_rows][head_dim]
  float* part_ml;  // [ctas][2][part_rows][2]: what the exponentials were taken against (log2 units) and their sum
  int part_rows;   // rows of a row tile
  int item_units;  // tiles of keys that an item's beginning and end take as long as
  int* status;
  int withhold;    // test build only: sequence 0 never gets its last tile
};

// The work is one line of tiles of 32 KB: sequence by sequence, in each key head by key head (and row tile by row tile), the
// tiles that the new tokens see. Every CTA takes an equal stretch of the line, to within a tile. A (sequence, key head, row
// tile) that lies within one stretch is finished there; one that is cut has its parts written as (maximum, sum, unnormalised
// output) and joined by decode_join_kernel in the order of the line, so the results depend on the lengths alone. Where few
// items are short, or many are very short, an item has a cluster of CTAs, or one CTA, to itself instead, and no second launch.
struct DecodeLine {
  __device__ static void tiles_of(const DecodeParams& p, int b, int& first, int& tiles, int& length, int& count) {
    sequence_of(p.cache, b, length, count);
    const int lo = p.window_left >= 0 && length - count > p.window_left ? length - count - p.window_left : 0;
    first = lo >> p.tile_shift;
    tiles = count > 0 ? ((length - 1) >> p.tile_shift) + 1 - first : 0;
  }
  // What an item takes up on the line: p.item_units for its beginning and end (Q, the join of the warps and the output take a CTA
  // about as long as so many tiles), then its tiles.
  __device__ static int units_of(const DecodeParams& p, int tiles) { return tiles > 0 ? tiles + p.item_units : 0; }
  // Sums the units of an item of every sequence, and of those in front of `upto`. All lanes of a warp call it.
  __device__ static void sum(const DecodeParams& p, int upto, int& all, int& before, int lane) {
    all = before = 0;
    for (int b = lane; b < p.cache.batch; b += 32) {
      int first, tiles, length, count;
      tiles_of(p, b, first, tiles, length, count);
      all += units_of(p, tiles);
      if (b < upto) before += units_of(p, tiles);
    }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) {
      all += __shfl_xor_sync(0xffffffffu, all, s);
      before += __shfl_xor_sync(0xffffffffu, before, s);
    }
  }

  // CTA c has the units [start(c), start(c + 1)).
  int base, more;  // units of a CTA; CTAs that have one more
  __device__ DecodeLine(const DecodeParams& p, int all) {
    const int total = all * p.cache.kv_heads * p.row_tiles;
    base = total / p.ctas;
    more = total - base * p.ctas;
  }
  __device__ int start(int c) const { return c * base + min(c, more); }
  __device__ int cta_of(int unit) const {
    const int in_more = more * (base + 1);
    return unit < in_more ? unit / (base + 1) : more + (unit - in_more) / base;
  }
};

// A stretch of the line, walked item by item; every role of a CTA walks it for itself.
struct DecodeWalk {
  int at, end;  // of the line
  int b_start;  // where sequence b starts
  int b, first, tiles, length, count;

  __device__ void start(const DecodeParams& p, int cta, int lane) {
    if (p.cluster > 0) {  // one item: `at` and `end` count items
      b = cta / (p.cluster * p.cache.kv_heads * p.row_tiles);
      DecodeLine::tiles_of(p, b, first, tiles, length, count);
      at = 0;
      end = 1;
      return;
    }
    const int per = p.cache.kv_heads * p.row_tiles;
    b = b_start = at = end = 0;
    // the sequence that holds the start, 32 at a time
    for (int b0 = 0; b0 < p.cache.batch; b0 += 32) {
      int f = 0, n = 0, len = 0, cnt = 0;
      if (b0 + lane < p.cache.batch) DecodeLine::tiles_of(p, b0 + lane, f, n, len, cnt);
      int upto = DecodeLine::units_of(p, n);
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, s);
        if (lane >= s) upto += v;
      }
      if (b0 == 0) {
        int all = __shfl_sync(0xffffffffu, upto, 31), before;
        if (p.cache.batch > 32) DecodeLine::sum(p, 0, all, before, lane);
        const DecodeLine line(p, all);
        at = line.start(cta);
        end = line.start(cta + 1);
      }
      upto = b_start + upto * per;
      const unsigned found = __ballot_sync(0xffffffffu, upto > at);
      if (found) {
        const int src = __ffs(found) - 1;
        b = b0 + src;
        first = __shfl_sync(0xffffffffu, f, src);
        tiles = __shfl_sync(0xffffffffu, n, src);
        length = __shfl_sync(0xffffffffu, len, src);
        count = __shfl_sync(0xffffffffu, cnt, src);
        b_start = __shfl_sync(0xffffffffu, upto, src) - DecodeLine::units_of(p, tiles) * per;
        return;
      }
      b_start = __shfl_sync(0xffffffffu, upto, 31);
    }
    at = end;  // (nothing is left for this CTA)
  }
  // The next item of which the stretch holds tiles: key head, row tile, and its tiles [t0, t1) of [0, tiles).
  __device__ bool next(const DecodeParams& p, int& kv_head, int& row_tile, int& t0, int& t1) {
    if (p.cluster > 0) {
      if (at >= end) return false;
      const int item = blockIdx.x / p.cluster % (p.cache.kv_heads * p.row_tiles);
      kv_head = item / p.row_tiles;
      row_tile = item % p.row_tiles;
      const int share = (tiles + p.cluster - 1) / p.cluster, rank = blockIdx.x % p.cluster;
      t0 = min(rank * share, tiles);
      t1 = min(t0 + share, tiles);
      at = end;
      return true;
    }
    const int per = p.cache.kv_heads * p.row_tiles;
    while (at < end) {
      while (at >= b_start + DecodeLine::units_of(p, tiles) * per) {
        b_start += DecodeLine::units_of(p, tiles) * per;
        ++b;
        DecodeLine::tiles_of(p, b, first, tiles, length, count);
      }
      const int units = DecodeLine::units_of(p, tiles), item = (at - b_start) / units, from = at - b_start - item * units;
      const int to = min(from + end - at, units);
      at += to - from;
      t0 = max(from - p.item_units, 0);
      t1 = to - p.item_units;
      kv_head = item / p.row_tiles;
      row_tile = item % p.row_tiles;
      if (t1 > t0) return true;
    }
    return false;
  }
};

// 16 rows: four warps that compute and two CTAs a SM. More rows: eight warps and one CTA a SM, whose threads have the registers
// for 32 keys' scores at a time (a warp's work on a tile is one chain of latencies: 16 keys or 32 take it about as long).
template <int D, int kRowWarps>
struct DecodeCfg {
  static constexpr int kWarps = kRowWarps == 1 ? 4 : 8;
  static constexpr int kThreads = kWarps * 32 + 32;  // and one that loads
  static constexpr int kCtasPerSm = kRowWarps == 1 ? 2 : 1;
  static constexpr int kRows = 16 * kRowWarps;
  static constexpr int kKeys = kDecodeKeys<D>;
  static constexpr int kKeyWarps = kWarps / kRowWarps;
  static constexpr int kWarpKeys = kKeys / kKeyWarps;  // of a tile, a warp's
  static constexpr int kChunk = kWarpKeys < 32 ? kWarpKeys : 32;  // of them at a time
  static constexpr int kHalfBytes = kKeys * D * 2;  // K or V of a tile
  static constexpr int kStages = 6 / kCtasPerSm;
  static constexpr int kOffJoin = kStages * 2 * kHalfBytes;
  static constexpr int kJoinBytes = (kKeyWarps / 2) * kRows * D * 4;  // O of half of the key warps
  static constexpr int kOffMl = kOffJoin + kJoinBytes;  // maxima and sums of all warps' rows
  static constexpr int kOffBars = kOffMl + kWarps * 16 * 8;
  static constexpr int kSmemBytes = kOffBars + kStages * 16 + 16;
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void tma_load_5d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2,
                                            int c3, int c4) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
      :
      : "r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2),
        "r"(c3), "r"(c4)
      : "memory");
}
// Two floats from the shared memory of CTA `rank` of the cluster, at the place of `here` in this CTA's.
__device__ __forceinline__ float2 dsmem_ld2(const void* here, uint32_t rank) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
               : "=f"(v.x), "=f"(v.y)
               : "r"(mapa_u32(smem_u32(here), rank))
               : "memory");
  return v;
}
// What exponentials are taken against for a maximum of m, so that the largest is 2^kRoom. Rounded up: scores so large that fp32 has
// steps of 4 and more there would else be taken against something further below, up to 2^16, which fp16 does not hold.
template <int kRoom>
__device__ __forceinline__ float reference_of(float m) {
  return kRoom > 0 ? __fadd_ru(m, -static_cast<float>(kRoom)) : m;
}
// barrier of the warps that compute
template <int kThreads>
__device__ __forceinline__ void compute_sync() {
  asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
}

// A CTA's warps take 16 * kRowWarps rows (a row: one query head of the key head's group and one new token) and share a tile's
// keys. The products run as m16n8k16 matrix instructions: a step of generation reads every key for a handful of rows, so HBM is
// what bounds it (at 16 rows a tile of 32 KB is 128 such instructions of an SM), and rows that are padding cost nothing that
// matters: 64 sequences of up to 32768 tokens, 32 heads on 8 of 128, 4.8 GB in 704-741 us; one of 131072 in 89 us (6.0 TB/s, 5 of
// them start and join). More than 16 rows leave the warps latency-bound (16 x 8 tokens, 64 heads on 8, up to 32768 tokens: 352 us
// for 1.2 GB), so there decode_wide_kernel takes all but short work. Scores, maxima, sums and O are fp32; P is rounded to the
// cache's type for the second product, as the operand has to be, and its sum is taken unrounded. In fp16 it is kept as 2^14 P, so
// that it is half a step off down to 2^-28 of the row's maximum. (Kept as P, what lies 17 nats below the maximum was off by up to
// all of itself: the tail of 131071 keys behind one that dominates them, 4e-3 of the weight, came out a quarter too large.)
template <typename T, int D, int kRowWarps>
__global__ void __launch_bounds__(DecodeCfg<D, kRowWarps>::kThreads, DecodeCfg<D, kRowWarps>::kCtasPerSm)
decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
              const __grid_constant__ DecodeParams p) {
  using Cfg = DecodeCfg<D, kRowWarps>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Cfg::kOffBars);
  uint64_t* empty = full + Cfg::kStages;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + Cfg::kStages);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < Cfg::kStages; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, Cfg::kWarps);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  griddep_wait();
  DecodeWalk walk;
  walk.start(p, blockIdx.x, lane);
  griddep_launch();
  int kv_head, row_tile, t0, t1, stage = 0;
  uint32_t phase = 0;

  if (warp == Cfg::kWarps) {
    // ---- loads: lane i brings box i of the tile's keys and of its values ----
    const int boxes = Cfg::kKeys / p.box_rows;
    const uint32_t box_bytes = p.box_rows * D * 2;
    bool ok = true;
    while (ok && walk.next(p, kv_head, row_tile, t0, t1)) {
      const int lo = p.window_left >= 0 && walk.length - walk.count > p.window_left
                         ? walk.length - walk.count - p.window_left : 0;
      const int* table = p.cache.page_table + walk.b * p.cache.table_stride;
      auto page_of = [&](int tile) {  // -1: the box holds nothing that is seen
        const int key = (walk.first + tile) * Cfg::kKeys + lane * p.box_rows;
        if (lane >= boxes || tile >= t1 || key >= walk.length || key + p.box_rows <= lo) return -1;
        const int page = table[key / p.cache.page_size];
        if (page >= 0 && page < p.cache.num_pages) return page;
        atomicExch(p.cache.bad_index, 1);
        return -1;
      };
      int page = page_of(t0);
      for (int t = t0; t < t1; ++t) {
        const int next_page = page_of(t + 1);
        ok = mbar_wait_warp(empty + stage, phase ^ 1, abort_flag);
        if (!ok) break;
        const unsigned here = __ballot_sync(0xffffffffu, page >= 0);
        if (lane == 0) mbar_arrive_expect_tx(full + stage, 2 * box_bytes * __popc(here));
        __syncwarp();
#ifdef FA_TEST_WITHHOLD_LOAD
        if (p.withhold && walk.b == 0 && t == walk.tiles - 1) page = -1;
#endif
        if (page >= 0) {
          uint8_t* dst = smem + stage * 2 * Cfg::kHalfBytes + lane * box_bytes;
          const int row = ((walk.first + t) * Cfg::kKeys + lane * p.box_rows) % p.cache.page_size;
          tma_load_5d(dst, &map_k, full + stage, 0, row, 0, kv_head, page);
          tma_load_5d(dst + Cfg::kHalfBytes, &map_v, full + stage, 0, row, 0, kv_head, page);
        }
        page = next_page;
        if (++stage == Cfg::kStages) stage = 0, phase ^= 1;
      }
    }
    if (!ok && lane == 0) {
      atomicExch(p.status, 1);
      for (int i = 0; i < 64; ++i) __nanosleep(2000);  // loads in flight land before the CTA retires
    }
    if (p.cluster > 1) {  // the barriers of the join below
      __syncwarp();
      cluster_sync_all();
      cluster_sync_all();
    }
    return;
  }

  // ---- compute ----
  const int row_warp = warp % kRowWarps, key_warp = warp / kRowWarps;
  const int quad = lane >> 2, in_quad = lane & 3;  // fragments: rows quad and quad + 8, columns 2 * in_quad and the next
  const int rows = p.group * p.cache.tokens;
  // where this lane's rows of the operands of ldmatrix start: K as [key][d], V (transposed on the way) as [key][d]
  const int k_row = key_warp * Cfg::kWarpKeys + (lane >> 4) * 8 + (lane & 7), k_chunk = (lane >> 3) & 1;
  const int v_row = key_warp * Cfg::kWarpKeys + (lane & 15), v_chunk = lane >> 4;
  const int box_shift = __ffs(p.box_rows) - 1;
  auto row_base = [&](int row) {  // of a row of the tile, first 128 bytes; its other panel is box_rows * 128 further
    return (row >> box_shift) * (p.box_rows * D * 2) + (row & (p.box_rows - 1)) * 128;
  };
  const uint32_t panel = p.box_rows * 128;
  constexpr int kRoom = std::is_same_v<T, __half> ? 14 : 0;  // P is kept as 2^kRoom P
  bool ok = true;  // once a wait has run out, the warp goes on with whatever is there: the others may wait for it

  while (walk.next(p, kv_head, row_tile, t0, t1)) {
    // this thread's two rows
    uint32_t qf[D / 16][4];
    float slope[2];
    int last_key[2], out_row[2];  // the last key that the row sees; its place in the outputs, -1: there is none
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = row_tile * Cfg::kRows + row_warp * 16 + quad + 8 * i;
      const int t = r / p.group, head = kv_head * p.group + r % p.group;
      const bool there = r < rows, real = there && t < walk.count;
      out_row[i] = there ? (walk.b * p.q_heads + head) * p.cache.tokens + t : -1;
      last_key[i] = real ? walk.length - walk.count + t : -1;
      slope[i] = real && p.alibi_slopes ? p.alibi_slopes[head] * 1.4426950408889634f : 0.f;
      const T* q = static_cast<const T*>(p.q.data) + walk.b * p.q.batch_stride + head * p.q.head_stride +
                   t * p.q.token_stride + 2 * in_quad;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        qf[k][i] = real ? *reinterpret_cast<const uint32_t*>(q + 16 * k) : 0u;
        qf[k][2 + i] = real ? *reinterpret_cast<const uint32_t*>(q + 16 * k + 8) : 0u;
      }
    }
    const int first_query = walk.length - walk.count;
    float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;

    for (int t = t0; t < t1; ++t) {
      ok &= mbar_wait(full + stage, phase, abort_flag);  // (looked at once an item: a vote costs more than the wait)
      {
        const int key0 = (walk.first + t) * Cfg::kKeys;
        const uint32_t k_smem = smem_u32(smem + stage * 2 * Cfg::kHalfBytes), v_smem = k_smem + Cfg::kHalfBytes;
        // does every row see every key of the tile?
        const bool cut = key0 + Cfg::kKeys > first_query + 1 ||
                         (p.window_left >= 0 && key0 < walk.length - 1 - p.window_left);
#pragma unroll 1
        for (int chunk = 0; chunk < Cfg::kWarpKeys; chunk += Cfg::kChunk) {
        float s[Cfg::kChunk / 8][4];
#pragma unroll
        for (int n = 0; n < Cfg::kChunk / 16; ++n) {
          const uint32_t base = k_smem + row_base(k_row + chunk + 16 * n);
          // (two partial sums each where a warp has 16 keys only: four chains of products instead of two)
          constexpr int kSplit = Cfg::kChunk == 16 ? 2 : 1;
          float part[kSplit][2][4] = {};
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            uint32_t b[4];
            ldsm4(base + (k / 4) * panel + ((((k % 4) * 2 + k_chunk) ^ (k_row & 7)) << 4), b);
            mma16816<T>(part[k % kSplit][0], qf[k], b[0], b[1]);
            mma16816<T>(part[k % kSplit][1], qf[k], b[2], b[3]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) s[2 * n + h][i] = kSplit == 2 ? part[0][h][i] + part[kSplit - 1][h][i] : part[0][h][i];
        }
        const int warp_key = key0 + key_warp * Cfg::kWarpKeys + chunk + 2 * in_quad;
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < Cfg::kChunk / 8; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = warp_key + 8 * n + (i & 1), r = i >> 1;
            float x = s[n][i] * p.scale_log2;
            if (p.alibi_slopes) x = fmaf(-slope[r], fabsf(static_cast<float>(last_key[r] - key)), x);
            if (cut && (key > last_key[r] || (p.window_left >= 0 && key < last_key[r] - p.window_left))) x = -INFINITY;
            s[n][i] = x;
            top[r] = fmaxf(top[r], x);
          }
        float scale[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
          top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
          top[r] = fmaxf(top[r], m[r]);
        }
        if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            scale[r] = top[r] == -INFINITY ? 1.f : ex2_approx(reference_of<kRoom>(m[r]) - reference_of<kRoom>(top[r]));
            m[r] = top[r];
            l[r] *= scale[r];
          }
#pragma unroll
          for (int n = 0; n < D / 8; ++n) {
            o[n][0] *= scale[0];
            o[n][1] *= scale[0];
            o[n][2] *= scale[1];
            o[n][3] *= scale[1];
          }
        }
        const float off[2] = {m[0] == -INFINITY ? 0.f : reference_of<kRoom>(m[0]),
                              m[1] == -INFINITY ? 0.f : reference_of<kRoom>(m[1])};
#pragma unroll
        for (int n = 0; n < Cfg::kChunk / 16; ++n) {
          uint32_t pf[4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float* x = s[2 * n + h];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = ex2_approx(x[i] - off[i >> 1]);
            l[0] += x[0] + x[1];
            l[1] += x[2] + x[3];
            pf[2 * h] = from_floats<T>(x[0], x[1]);
            pf[2 * h + 1] = from_floats<T>(x[2], x[3]);
          }
          const uint32_t base = v_smem + row_base(v_row + chunk + 16 * n);
          if (cut) {
            // what lies behind the last token, or in pages in front of the window, is not the sequence's: any bits at all,
            // and 0 * NaN is NaN
            uint32_t keep[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int key = warp_key + 16 * n + 8 * h;
              const int lo = p.window_left >= 0 ? first_query - p.window_left : 0;
              keep[h] = (key < walk.length && key >= lo ? 0xffffu : 0u) |
                        (key + 1 < walk.length && key + 1 >= lo ? 0xffff0000u : 0u);
            }
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
              uint32_t b[4];
              ldsm4_trans(base + (d / 4) * panel + ((((d % 4) * 2 + v_chunk) ^ (v_row & 7)) << 4), b);
              mma16816<T>(o[2 * d], pf, b[0] & keep[0], b[1] & keep[1]);
              mma16816<T>(o[2 * d + 1], pf, b[2] & keep[0], b[3] & keep[1]);
            }
          } else {
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
              uint32_t b[4];
              ldsm4_trans(base + (d / 4) * panel + ((((d % 4) * 2 + v_chunk) ^ (v_row & 7)) << 4), b);
              mma16816<T>(o[2 * d], pf, b[0], b[1]);
              mma16816<T>(o[2 * d + 1], pf, b[2], b[3]);
            }
          }
        }
        }
      }
      __syncwarp();
      mbar_arrive_lane0(empty + stage, lane);
      if (++stage == Cfg::kStages) stage = 0, phase ^= 1;
    }

    ok = __all_sync(0xffffffffu, ok);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      m[r] = reference_of<kRoom>(m[r]);  // from here on what the sum and O were taken against
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
    if constexpr (Cfg::kKeyWarps > 1) {
      // join the key warps: a common maximum, then the outputs pairwise through shared memory
      float2* ml = reinterpret_cast<float2*>(smem + Cfg::kOffMl);
      if (in_quad == 0) {
        ml[warp * 16 + quad] = make_float2(m[0], l[0]);
        ml[warp * 16 + quad + 8] = make_float2(m[1], l[1]);
      }
      compute_sync<Cfg::kWarps * 32>();
      float scale[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < Cfg::kKeyWarps; ++w) top = fmaxf(top, ml[(w * kRowWarps + row_warp) * 16 + quad + 8 * r].x);
        const float off = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < Cfg::kKeyWarps; ++w) {
          const float2 other = ml[(w * kRowWarps + row_warp) * 16 + quad + 8 * r];
          sum += other.y * ex2_approx(other.x - off);
        }
        scale[r] = ex2_approx(m[r] - off);
        m[r] = top;
        l[r] = sum;
      }
#pragma unroll
      for (int step = Cfg::kKeyWarps / 2; step > 0; step /= 2) {
        float2* buf = reinterpret_cast<float2*>(smem + Cfg::kOffJoin) +
                      ((key_warp % step) * kRowWarps + row_warp) * (16 * D / 2) + lane;
        if (key_warp >= step && key_warp < 2 * step) {
#pragma unroll
          for (int n = 0; n < D / 8; ++n) {
            const float c0 = step == Cfg::kKeyWarps / 2 ? scale[0] : 1.f, c1 = step == Cfg::kKeyWarps / 2 ? scale[1] : 1.f;
            buf[(2 * n) * 32] = make_float2(o[n][0] * c0, o[n][1] * c0);
            buf[(2 * n + 1) * 32] = make_float2(o[n][2] * c1, o[n][3] * c1);
          }
        }
        compute_sync<Cfg::kWarps * 32>();
        if (key_warp < step) {
#pragma unroll
          for (int n = 0; n < D / 8; ++n) {
            const float c0 = step == Cfg::kKeyWarps / 2 ? scale[0] : 1.f, c1 = step == Cfg::kKeyWarps / 2 ? scale[1] : 1.f;
            const float2 a = buf[(2 * n) * 32], c = buf[(2 * n + 1) * 32];
            o[n][0] = fmaf(o[n][0], c0, a.x);
            o[n][1] = fmaf(o[n][1], c0, a.y);
            o[n][2] = fmaf(o[n][2], c1, c.x);
            o[n][3] = fmaf(o[n][3], c1, c.y);
          }
        }
        compute_sync<Cfg::kWarps * 32>();
      }
    }
    if (p.cluster > 1) {
      // this CTA's part of every row, for the CTA of the cluster that finishes it
      if (key_warp == 0) {
        float* part_o = reinterpret_cast<float*>(smem + Cfg::kOffJoin) + (row_warp * 16 + quad) * D + 2 * in_quad;
        float2* part_ml = reinterpret_cast<float2*>(smem + Cfg::kOffMl) + row_warp * 16 + quad;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
#pragma unroll
          for (int n = 0; n < D / 8; ++n)
            *reinterpret_cast<float2*>(part_o + 8 * r * D + 8 * n) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
          if (in_quad == 0) part_ml[8 * r] = make_float2(m[r], l[r]);
        }
      }
      break;  // a cluster has one item
    }
    if (key_warp == 0) {
      const bool whole = t0 == 0 && t1 == walk.tiles;
      const long long part =
          (2ll * blockIdx.x + (t0 == 0 ? 1 : 0)) * Cfg::kRows + row_warp * 16 + quad;  // of the first part, or a later one
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        if (out_row[r] < 0) continue;
        const bool real = last_key[r] >= 0;
        if (whole) {
          const float inv = real && l[r] != 0.f ? 1.f / l[r] : 0.f;
          T* to = static_cast<T*>(p.o) + static_cast<long long>(out_row[r]) * D + 2 * in_quad;
#pragma unroll
          for (int n = 0; n < D / 8; ++n)
            *reinterpret_cast<uint32_t*>(to + 8 * n) =
                real ? from_floats<T>(o[n][2 * r] * inv, o[n][2 * r + 1] * inv) : 0u;
          if (p.lse && in_quad == 0) p.lse[out_row[r]] = real ? (m[r] + log2f(l[r])) * 0.6931471805599453f : -INFINITY;
        } else {
          float* to = p.part_o + (part + 8 * r) * D + 2 * in_quad;
#pragma unroll
          for (int n = 0; n < D / 8; ++n) *reinterpret_cast<float2*>(to + 8 * n) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
          if (in_quad == 0)
            *reinterpret_cast<float2*>(p.part_ml + (part + 8 * r) * 2) = make_float2(m[r], l[r]);
        }
      }
    }
  }
  if (p.cluster > 1) {
    // CTA `rank` finishes the rows rank, rank + cluster, ...: a warp a row, the parts in the order of their keys
    cluster_sync_all();
    constexpr int kOwn = D / 32;  // elements of a lane
    const int rank = blockIdx.x % p.cluster;
    for (int tile_row = rank + p.cluster * warp; tile_row < Cfg::kRows; tile_row += p.cluster * Cfg::kWarps) {
      const int r = row_tile * Cfg::kRows + tile_row;
      if (r >= rows) break;
      const int t = r / p.group, head = kv_head * p.group + r % p.group;
      const bool real = t < walk.count;
      float2 ml = make_float2(-INFINITY, 0.f);
      if (lane < p.cluster) ml = dsmem_ld2(smem + Cfg::kOffMl + tile_row * 8, lane);
      float top = ml.x;
#pragma unroll
      for (int i = 4; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
      const float off = top == -INFINITY ? 0.f : top, scale = ex2_approx(ml.x - off);
      float sum = 0.f, out[kOwn];
#pragma unroll
      for (int i = 0; i < kOwn; ++i) out[i] = 0.f;
#pragma unroll 8
      for (int c = 0; c < p.cluster; ++c) {
        const float s = __shfl_sync(0xffffffffu, scale, c);
        sum = fmaf(__shfl_sync(0xffffffffu, ml.y, c), s, sum);
#pragma unroll
        for (int i = 0; i < kOwn; i += 2) {
          const float2 x = dsmem_ld2(smem + Cfg::kOffJoin + (tile_row * D + lane * kOwn + i) * 4, c);
          out[i] = fmaf(x.x, s, out[i]);
          out[i + 1] = fmaf(x.y, s, out[i + 1]);
        }
      }
      top = __shfl_sync(0xffffffffu, top, 0);  // (lanes from the eighth on have seen no part)
      const long long row = (static_cast<long long>(walk.b) * p.q_heads + head) * p.cache.tokens + t;
      const float inv = real && sum != 0.f ? 1.f / sum : 0.f;
      T* to = static_cast<T*>(p.o) + row * D + lane * kOwn;
#pragma unroll
      for (int i = 0; i < kOwn; i += 2)
        *reinterpret_cast<uint32_t*>(to + i) = real ? from_floats<T>(out[i] * inv, out[i + 1] * inv) : 0u;
      if (p.lse && lane == 0) p.lse[row] = real ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
    }
    cluster_sync_all();  // the others may still read here
  }
  if (!ok && lane == 0) atomicExch(p.status, 1);
}

// kWarps warps a row: nothing to do where one CTA had the whole item; else the parts are joined, every warp those of its turn
// in the order of the line, then the warps in their order. Rows of sequences without keys, and rows of padding, are set to
// O = 0 and a log-sum-exp of -infinity.
template <typename T, int D, int kWarps>
__global__ void __launch_bounds__(128, 6) decode_join_kernel(const __grid_constant__ DecodeParams p) {
  constexpr int kOwn = D / 32;  // elements of a lane
  __shared__ float s_o[kWarps][D];
  __shared__ float2 s_ml[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, turn = warp % kWarps;
  const long long row = kWarps == 4 ? blockIdx.x : blockIdx.x * 4ll + warp;
  if (row >= static_cast<long long>(p.cache.batch) * p.q_heads * p.cache.tokens) return;
  const int t = static_cast<int>(row % p.cache.tokens);
  const int bh = static_cast<int>(row / p.cache.tokens), head = bh % p.q_heads, b = bh / p.q_heads;
  // decode_kernel lets this kernel in only behind its own griddep_wait(), so the lengths are there already
  int first, tiles, length, count;
  DecodeLine::tiles_of(p, b, first, tiles, length, count);
  const bool real = tiles > 0 && t < count;
  int c0 = 0, c1 = -1;  // the CTAs of the row's item
  const int r = t * p.group + head % p.group;
  if (real) {
    int all, before;
    DecodeLine::sum(p, b, all, before, lane);
    const int item = head / p.group * p.row_tiles + r / p.part_rows;
    const DecodeLine line(p, all);
    const int from = before * p.cache.kv_heads * p.row_tiles + item * DecodeLine::units_of(p, tiles) + p.item_units;
    c0 = line.cta_of(from);
    c1 = line.cta_of(from + tiles - 1);
  }
  griddep_wait();
  if (real && c0 == c1) return;
  auto part = [&](int c) { return (2ll * c + (c == c0 ? 1 : 0)) * p.part_rows + r % p.part_rows; };
  float o[kOwn], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < kOwn; ++i) o[i] = 0.f;
  for (int base = c0 + turn; base <= c1; base += 32 * kWarps) {  // 32 parts at a time, one a lane
    const int mine = base + lane * kWarps;
    const float2 ml = mine <= c1 ? *reinterpret_cast<const float2*>(p.part_ml + 2 * part(mine)) : make_float2(-INFINITY, 0.f);
    float top = ml.x;
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
    top = fmaxf(top, m);
    const float off = top == -INFINITY ? 0.f : top;
    const float old = ex2_approx(m - off), scale = ex2_approx(ml.x - off);
    m = top;
    l *= old;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) o[i] *= old;
    const int n = min((c1 - base) / kWarps + 1, 32);
#pragma unroll 4
    for (int k = 0; k < n; ++k) {
      const float s = __shfl_sync(0xffffffffu, scale, k);
      const float* from = p.part_o + part(base + k * kWarps) * D + lane * kOwn;
      l = fmaf(__shfl_sync(0xffffffffu, ml.y, k), s, l);
#pragma unroll
      for (int i = 0; i < kOwn; i += 2) {
        const float2 x = *reinterpret_cast<const float2*>(from + i);
        o[i] = fmaf(x.x, s, o[i]);
        o[i + 1] = fmaf(x.y, s, o[i + 1]);
      }
    }
  }
  if constexpr (kWarps > 1) {
#pragma unroll
    for (int i = 0; i < kOwn; ++i) s_o[turn][lane * kOwn + i] = o[i];
    if (lane == 0) s_ml[turn] = make_float2(m, l);
    __syncthreads();
    if (turn > 0) return;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, s_ml[w].x);
    const float off = m == -INFINITY ? 0.f : m;
    l = 0.f;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) o[i] = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float s = ex2_approx(s_ml[w].x - off);
      l = fmaf(s_ml[w].y, s, l);
#pragma unroll
      for (int i = 0; i < kOwn; ++i) o[i] = fmaf(s_o[w][lane * kOwn + i], s, o[i]);
    }
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;
  T* to = static_cast<T*>(p.o) + row * D + lane * kOwn;
#pragma unroll
  for (int i = 0; i < kOwn; i += 2) *reinterpret_cast<uint32_t*>(to + i) = from_floats<T>(o[i] * inv, o[i + 1] * inv);
  if (p.lse && lane == 0) p.lse[row] = (m + log2f(l)) * 0.6931471805599453f;
}

}  // namespace fa
