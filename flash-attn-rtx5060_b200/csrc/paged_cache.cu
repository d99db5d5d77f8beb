// Host side of the paged key-value cache: argument checks, tensor maps and launches of flash_cache_append and flash_decode.
#include <cmath>
#include <cstring>

#include "decode_plan.h"
#include "host.h"
#include "paged_cache.cuh"
#include "paged_cache_wide.cuh"

using namespace fa_host;

namespace {

constexpr long long kJoinBlocks = 148 * 6;

int check_cache(const fa_paged_cache* c, int batch, int tokens, int q_heads) {
  if (!c) return fail(FA_INVALID_ARG, "cache is null");
  if (!c->k || !c->v || !c->page_table || !c->lengths) return fail(FA_INVALID_ARG, "null pointer in the cache");
  if (c->dtype != FA_FP16 && c->dtype != FA_BF16) return fail(FA_UNSUPPORTED, "dtype must be FA_FP16 or FA_BF16");
  if (c->head_dim != 64 && c->head_dim != 128) return fail(FA_UNSUPPORTED, "head_dim must be 64 or 128");
  if (batch <= 0 || tokens <= 0) return fail(FA_INVALID_ARG, "batch and tokens must be positive");
  if (c->kv_heads <= 0 || c->num_pages <= 0 || c->max_pages <= 0)
    return fail(FA_INVALID_ARG, "kv_heads, num_pages and max_pages must be positive");
  if (c->page_size <= 0 || c->page_size % 8 != 0) return fail(FA_UNSUPPORTED, "page_size must be a multiple of 8");
  if (static_cast<long long>(c->max_pages) * c->page_size > 0x7fffffffLL - 65536)
    return fail(FA_INVALID_ARG, "max_pages * page_size does not fit 31 bits");
  if (c->table_stride < c->max_pages && batch > 1)
    return fail(FA_INVALID_ARG, "table_stride is smaller than max_pages");
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15)
    return fail(FA_INVALID_ARG, "pages must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(c->page_table) | reinterpret_cast<uintptr_t>(c->lengths) |
       reinterpret_cast<uintptr_t>(c->counts)) & 3)
    return fail(FA_INVALID_ARG, "page_table, lengths and counts must be 4-byte aligned");
  const long long strides[3] = {c->page_stride, c->head_stride, c->token_stride};
  const int extents[3] = {c->num_pages, c->kv_heads, c->page_size};
  for (int i = 0; i < 3; ++i)
    if (extents[i] > 1 && (strides[i] < c->head_dim || strides[i] % 8 != 0 || strides[i] >= 1ll << 38))
      return fail(FA_INVALID_ARG, "strides of the pages must be multiples of 8 elements, of head_dim or more");
  if (q_heads < 0 || q_heads % c->kv_heads != 0)
    return fail(FA_INVALID_ARG, "the query heads must be a multiple of kv_heads");
  return FA_OK;
}

int check_rows(const fa_rows* r, int batch, int heads, int tokens) {
  if (!r || !r->data) return fail(FA_INVALID_ARG, "null rows");
  if (reinterpret_cast<uintptr_t>(r->data) & 15) return fail(FA_INVALID_ARG, "rows must be 16-byte aligned");
  const long long strides[3] = {r->batch_stride, r->head_stride, r->token_stride};
  const int extents[3] = {batch, heads, tokens};
  for (int i = 0; i < 3; ++i)
    if (extents[i] > 1 && (strides[i] < 0 || strides[i] % 8 != 0))
      return fail(FA_INVALID_ARG, "strides of the rows must be multiples of 8 elements and not negative");
  return FA_OK;
}

// (a stride along an extent of 1 may be anything: it is not used)
fa::StridedRows rows_of(const fa_rows* r) {
  return fa::StridedRows{r->data, r->batch_stride, r->head_stride, r->token_stride};
}

fa::CacheView view_of(const fa_paged_cache* c, int batch, int tokens, DeviceState* s) {
  return fa::CacheView{c->page_stride, c->head_stride, c->token_stride, c->num_pages, c->page_size, c->kv_heads,
                       c->page_table, c->table_stride, c->max_pages, c->lengths, c->counts, batch, tokens,
                       s->status + 1};
}

// 5-D map over the pages of K or V: {64 contiguous elements, token of the page, 64-wide panel, head, page}. One box is
// `box_rows` tokens and `box_panels` panels of a head, [panel][token][64] in shared memory with the 128-byte swizzle.
int make_page_map(CUtensorMap* map, const fa_paged_cache* c, void* base, int box_rows, int box_panels) {
  EncodeTiledFn enc = encode_tiled_fn();
  if (!enc) return fail(FA_CUDA_ERROR, "cuTensorMapEncodeTiled entry point not available");
  const cuuint64_t row = 2ull * c->head_dim;
  cuuint64_t dims[5] = {64, (cuuint64_t)c->page_size, (cuuint64_t)(c->head_dim / 64), (cuuint64_t)c->kv_heads,
                        (cuuint64_t)c->num_pages};
  cuuint64_t strides[4] = {2ull * c->token_stride, 128, c->kv_heads > 1 ? 2ull * c->head_stride : row,
                           c->num_pages > 1 ? 2ull * c->page_stride : row};
  cuuint32_t box[5] = {64, (cuuint32_t)box_rows, (cuuint32_t)box_panels, 1, 1};
  cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  CUresult r = enc(map, c->dtype == FA_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, base,
                   dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(FA_CUDA_ERROR, "cuTensorMapEncodeTiled refused the map of the pages");
  return FA_OK;
}

template <typename T, int D>
int launch_join(const fa::DecodeParams& p, cudaStream_t st, bool early) {
  const long long rows = static_cast<long long>(p.cache.batch) * p.q_heads * p.cache.tokens;
  // a row by the four warps of a block while that is one wave of blocks
  cudaError_t e =
      rows <= kJoinBlocks
          ? launch_early(fa::decode_join_kernel<T, D, 4>, dim3(static_cast<unsigned>(rows)), 128, 0, st, early, p)
          : launch_early(fa::decode_join_kernel<T, D, 1>, dim3(static_cast<unsigned>((rows + 3) / 4)), 128, 0, st, early, p);
  if (e != cudaSuccess) return fail_cuda("launch decode_join_kernel", e);
  return FA_OK;
}

using DecodeKernel = void (*)(CUtensorMap, CUtensorMap, fa::DecodeParams);
template <typename T, int D>
int launch_decode(DecodeKernel kernel, int threads, int smem, const fa_paged_cache* c, int box_panels, const fa::DecodeParams& p,
                  cudaStream_t st, bool early) {
  CUtensorMap mk, mv;
  int rc = make_page_map(&mk, c, c->k, p.box_rows, box_panels);
  if (rc != FA_OK || (rc = make_page_map(&mv, c, c->v, p.box_rows, box_panels)) != FA_OK) return rc;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return fail_cuda("cudaFuncSetAttribute(MaxDynamicSharedMemorySize)", e);
  const unsigned grid =
      p.cluster > 0 ? static_cast<unsigned>(p.cluster) * p.cache.batch * p.cache.kv_heads * p.row_tiles : p.ctas;
  e = launch_early_in_clusters(kernel, p.cluster > 0 ? p.cluster : 1, dim3(grid), threads, smem, st, early, mk, mv, p);
  if (e != cudaSuccess) return fail_cuda("launch of the decoding kernel", e);
  return p.cluster > 0 ? FA_OK : launch_join<T, D>(p, st, early);
}

template <typename T, int D, int kRowWarps>
int launch_narrow(const fa_paged_cache* c, const fa::DecodeParams& p, cudaStream_t st, bool early) {
  using Cfg = fa::DecodeCfg<D, kRowWarps>;
  return launch_decode<T, D>(fa::decode_kernel<T, D, kRowWarps>, Cfg::kThreads, Cfg::kSmemBytes, c, D / 64, p, st, early);
}

template <typename T, int D>
int launch_rows(const fa::DecodePlan& plan, const fa_paged_cache* c, const fa::DecodeParams& p, cudaStream_t st, bool early) {
  using Cfg = fa::WideCfg<D>;
  if (plan.wide) return launch_decode<T, D>(fa::decode_wide_kernel<T, D>, Cfg::kThreads, Cfg::kSmemBytes, c, 1, p, st, early);
  return plan.part_rows == 16   ? launch_narrow<T, D, 1>(c, p, st, early)
         : plan.part_rows == 32 ? launch_narrow<T, D, 2>(c, p, st, early)
                                : launch_narrow<T, D, 4>(c, p, st, early);
}

int decode(const fa_paged_cache* cache, const fa_rows* q, void* o, float* lse, int batch, int tokens, int q_heads,
           float softmax_scale, int window_left, const float* alibi_slopes, void* workspace, size_t workspace_bytes, void* stream,
           int withhold) {
  int rc = check_cache(cache, batch, tokens, q_heads);
  if (rc != FA_OK) return rc;
  if (q_heads <= 0) return fail(FA_INVALID_ARG, "q_heads must be positive");
  if ((rc = check_rows(q, batch, q_heads, tokens)) != FA_OK) return rc;
  if (!o || (reinterpret_cast<uintptr_t>(o) & 15)) return fail(FA_INVALID_ARG, "o must be there and 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(lse) | reinterpret_cast<uintptr_t>(alibi_slopes)) & 3)
    return fail(FA_INVALID_ARG, "lse and alibi_slopes must be 4-byte aligned");
  if ((rc = check_scale(softmax_scale)) != FA_OK) return rc;
  if (static_cast<double>(batch) * q_heads * tokens > 0x7fffffff - 256)  // (so are a key head's rows, filled up to row tiles)
    return fail(FA_INVALID_ARG, "too many rows");
  if (!workspace || workspace_bytes < flash_decode_workspace_bytes(tokens, q_heads, cache->kv_heads, cache->head_dim))
    return fail(FA_INVALID_ARG, "workspace is null or smaller than flash_decode_workspace_bytes()");
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return fail(FA_INVALID_ARG, "workspace must be 16-byte aligned");

  DeviceState* s = nullptr;
  bool captured = false;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if ((rc = device_state_for(st, &s, &captured)) != FA_OK) return rc;
  if (!s->is_sm100) return fail(FA_UNSUPPORTED, "this library runs on compute capability 10.x (B200) only");
  if (softmax_scale <= 0.f) softmax_scale = 1.0f / sqrtf(static_cast<float>(cache->head_dim));

  fa::DecodeParams p;
  memset(&p, 0, sizeof(p));
  p.cache = view_of(cache, batch, tokens, s);
  p.q = rows_of(q);
  p.o = o;
  p.lse = lse;
  p.q_heads = q_heads;
  p.group = q_heads / cache->kv_heads;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.window_left = window_left;
  p.alibi_slopes = alibi_slopes;
  p.box_rows = cache->page_size & -cache->page_size;
  const int tile_keys = cache->head_dim == 128 ? fa::kDecodeKeys<128> : fa::kDecodeKeys<64>;
  if (p.box_rows > tile_keys) p.box_rows = tile_keys;
  p.tile_shift = cache->head_dim == 128 ? 6 : 7;
  const fa::DecodePlan plan = fa::decode_plan(batch, tokens, p.group, cache->kv_heads,
                                              static_cast<long long>(cache->max_pages) * cache->page_size, window_left, tile_keys);
  if (static_cast<double>(plan.items) * (plan.tiles + 8) > 0x7fffffff - 512)
    return fail(FA_INVALID_ARG, "more tiles of keys than 31 bits count");
  p.ctas = plan.ctas;
  p.part_rows = plan.part_rows;
  p.row_tiles = static_cast<int>(plan.row_tiles);
  p.cluster = plan.cluster;
  p.item_units = plan.wide ? 6 : 1;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = p.part_o + static_cast<size_t>(2) * p.ctas * p.part_rows * cache->head_dim;
  p.status = s->status;
  p.withhold = withhold;
  if (cache->dtype == FA_FP16)
    return cache->head_dim == 64 ? launch_rows<__half, 64>(plan, cache, p, st, !captured)
                                 : launch_rows<__half, 128>(plan, cache, p, st, !captured);
  return cache->head_dim == 64 ? launch_rows<__nv_bfloat16, 64>(plan, cache, p, st, !captured)
                               : launch_rows<__nv_bfloat16, 128>(plan, cache, p, st, !captured);
}

}  // namespace

extern "C" {

int flash_cache_append(const fa_paged_cache* cache, const fa_rows* k, const fa_rows* v, const fa_rows* q, void* q_out,
                       int batch, int tokens, int q_heads, const float* rotary, int rotary_dim, int rotary_positions,
                       int interleaved, void* stream) {
  int rc = check_cache(cache, batch, tokens, q_heads);
  if (rc != FA_OK) return rc;
  if ((rc = check_rows(k, batch, cache->kv_heads, tokens)) != FA_OK) return rc;
  if ((rc = check_rows(v, batch, cache->kv_heads, tokens)) != FA_OK) return rc;
  const bool has_q = q != nullptr;
  if (has_q != (q_out != nullptr) || has_q != (q_heads > 0))
    return fail(FA_INVALID_ARG, "q, q_out and q_heads come together or not at all");
  if (has_q && (rc = check_rows(q, batch, q_heads, tokens)) != FA_OK) return rc;
  if (reinterpret_cast<uintptr_t>(q_out) & 15) return fail(FA_INVALID_ARG, "q_out must be 16-byte aligned");
  if (has_q && !rotary) return fail(FA_INVALID_ARG, "queries are taken only to be rotated");
  if (rotary) {
    if (rotary_dim <= 0 || rotary_dim > cache->head_dim || rotary_dim % 16 != 0)
      return fail(FA_UNSUPPORTED, "rotary_dim must be a multiple of 16, up to head_dim");
    if (rotary_positions <= 0) return fail(FA_INVALID_ARG, "rotary_positions must be positive");
    if (reinterpret_cast<uintptr_t>(rotary) & 15) return fail(FA_INVALID_ARG, "rotary must be 16-byte aligned");
  }
  const long long row_units = (2ll * cache->kv_heads + q_heads) * (cache->head_dim / 16);  // of a token
  if (static_cast<long long>(batch) * tokens > 0x7fffffffLL || row_units > 65535ll * 128)
    return fail(FA_INVALID_ARG, "too many rows");

  DeviceState* s = nullptr;
  bool captured = false;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if ((rc = device_state_for(st, &s, &captured)) != FA_OK) return rc;
  if (!s->is_sm100) return fail(FA_UNSUPPORTED, "this library runs on compute capability 10.x (B200) only");
  fa::AppendParams p;
  memset(&p, 0, sizeof(p));
  p.cache = view_of(cache, batch, tokens, s);
  p.k_pages = cache->k;
  p.v_pages = cache->v;
  p.k = rows_of(k);
  p.v = rows_of(v);
  if (has_q) p.q = rows_of(q);
  p.q_out = q_out;
  p.q_heads = q_heads;
  p.rotary = rotary;
  p.rotary_dim = rotary ? rotary_dim : 0;
  p.positions = rotary_positions;
  p.interleaved = interleaved ? 1 : 0;
  p.row_units = static_cast<int>(row_units);
  const bool half = cache->dtype == FA_FP16, d64 = cache->head_dim == 64;
  const auto kernel = half ? (d64 ? fa::cache_append_kernel<__half, 64> : fa::cache_append_kernel<__half, 128>)
                           : (d64 ? fa::cache_append_kernel<__nv_bfloat16, 64> : fa::cache_append_kernel<__nv_bfloat16, 128>);
  const dim3 grid(static_cast<unsigned>(batch) * tokens, static_cast<unsigned>((row_units + 127) / 128));
  cudaError_t e = launch_early(kernel, grid, 128, 0, st, !captured, p);
  if (e != cudaSuccess) return fail_cuda("launch cache_append_kernel", e);
  return FA_OK;
}

size_t flash_decode_workspace_bytes(int tokens, int q_heads, int kv_heads, int head_dim) {
  if (tokens <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0 || head_dim <= 0) return 0;
  const long long rows = static_cast<long long>(q_heads / kv_heads) * tokens;
  return static_cast<size_t>(2) * fa::decode_ctas(rows) * fa::decode_part_rows(rows, true) * (head_dim + 2) * sizeof(float);
}

int flash_decode(const fa_paged_cache* cache, const fa_rows* q, void* o, float* lse, int batch, int tokens, int q_heads,
                 float softmax_scale, int window_left, const float* alibi_slopes, void* workspace, size_t workspace_bytes,
                 void* stream) {
  return decode(cache, q, o, lse, batch, tokens, q_heads, softmax_scale, window_left, alibi_slopes, workspace, workspace_bytes,
                stream, 0);
}

#ifdef FA_TEST_WITHHOLD_LOAD
// Test build only: sequence 0 never gets its last tile.
int flash_decode_test_withhold(const fa_paged_cache* cache, const fa_rows* q, void* o, float* lse, int batch, int tokens,
                               int q_heads, float softmax_scale, int window_left, const float* alibi_slopes, void* workspace,
                               size_t workspace_bytes, void* stream) {
  return decode(cache, q, o, lse, batch, tokens, q_heads, softmax_scale, window_left, alibi_slopes, workspace, workspace_bytes,
                stream, 1);
}
#endif

}  // extern "C"
