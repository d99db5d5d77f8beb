// Host side of flash_backward: argument checks, workspace, tensor maps and launches.
#include <cmath>
#include <cstring>

#include "bwd_kernels.cuh"
#include "host.h"

using namespace fa_host;

namespace {

size_t align256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

struct Range {
  const void* at;  // nullptr: nothing
  size_t bytes;
};
bool overlap(const Range& a, const Range& b) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
  return a.at && b.at && (x < y ? y - x < a.bytes : x - y < b.bytes);
}

template <int D, bool kAlibi, bool kOwnRows>
int launch_main(const CUtensorMap (&maps)[4], const fa::BwdParams& p, int ctas, cudaStream_t st, bool early) {
  using Cfg = fa::BwdCfg<D>;
  constexpr int smem = kOwnRows ? Cfg::kSmemBytesOwnRows : Cfg::kSmemBytes;
  constexpr auto kernel = fa::bwd_kernel<D, kAlibi, kOwnRows>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return fail_cuda("cudaFuncSetAttribute(MaxDynamicSharedMemorySize)", e);
  e = launch_early(kernel, dim3(ctas), Cfg::kThreads, smem, st, early, maps[0], maps[1], maps[2], maps[3], p);
  if (e != cudaSuccess) return fail_cuda("launch bwd_kernel", e);
  return FA_OK;
}

template <int D, bool kAlibi>
int launch(const CUtensorMap (&maps)[4], const fa::BwdParams& p, int num_sms, cudaStream_t st, bool early) {
  const int items = 2 * p.tiles * p.bh;
  // Short heads that are one wave of items: every CTA finds its head's delta and norms itself. us on the GPU, two launches ->
  // one: B1 H4 N128 d64 7.3 -> 6.0, B4 H18 N128 d128 causal 11.8 -> 10.5, B1 H4 N256 d64 8.5 -> 8.3; with more rows every CTA
  // reads too much: N384 d64 9.7 -> 10.4, N256 d128 10.6 -> 11.6. The call takes the host 5.8 instead of 7.9.
  if (p.seqlen <= fa::BwdCfg<D>::kMaxOwnRows && items <= num_sms)
    return launch_main<D, kAlibi, true>(maps, p, items, st, early);
  cudaError_t e = launch_early(fa::bwd_rows_kernel<D>, dim3(p.tiles, p.bh), 1024, 0, st, early, p);
  if (e != cudaSuccess) return fail_cuda("launch bwd_rows_kernel", e);
  return launch_main<D, kAlibi, false>(maps, p, items < num_sms ? items : num_sms, st, early);
}

int backward(const void* q, const void* k, const void* v, const void* o, const void* d_o, const float* lse,
             const float* d_lse, void* dq, void* dk, void* dv, int batch, int heads, int seqlen, int head_dim,
             float softmax_scale, int is_causal, int window_left, int window_right, const float* alibi_slopes,
             void* workspace, size_t workspace_bytes, void* stream, int withhold) {
  if (!q || !k || !v || !o || !d_o || !lse || !dq || !dk || !dv) return fail(FA_INVALID_ARG, "null tensor pointer");
  if (batch <= 0 || heads <= 0 || seqlen <= 0) return fail(FA_INVALID_ARG, "batch, heads and seqlen must be positive");
  if (head_dim != 64 && head_dim != 128) return fail(FA_UNSUPPORTED, "head_dim must be 64 or 128");
  uintptr_t any = 0;
  for (const void* t : {q, k, v, o, d_o, static_cast<const void*>(dq), static_cast<const void*>(dk),
                        static_cast<const void*>(dv)})
    any |= reinterpret_cast<uintptr_t>(t);
  if (any & 15) return fail(FA_INVALID_ARG, "tensor pointers must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(lse) | reinterpret_cast<uintptr_t>(d_lse) | reinterpret_cast<uintptr_t>(alibi_slopes)) & 3)
    return fail(FA_INVALID_ARG, "lse, d_lse and alibi_slopes must be 4-byte aligned");
  int rc = check_scale(softmax_scale);
  if (rc != FA_OK) return rc;
  const long long bh = static_cast<long long>(batch) * heads;
  const long long tiles = (static_cast<long long>(seqlen) + 127) / 128;
  if (bh > 65535) return fail(FA_UNSUPPORTED, "batch*heads must not exceed 65535");
  if (2 * bh * tiles > 0x7fffffffLL) return fail(FA_INVALID_ARG, "too many work items");
  if (!workspace || workspace_bytes < flash_backward_workspace_bytes(batch, heads, seqlen))
    return fail(FA_INVALID_ARG, "workspace is null or smaller than flash_backward_workspace_bytes()");
  if (reinterpret_cast<uintptr_t>(workspace) & 255) return fail(FA_INVALID_ARG, "workspace must be 256-byte aligned");

  DeviceState* s = nullptr;
  bool captured = false;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if ((rc = device_state_for(st, &s, &captured)) != FA_OK) return rc;
  if (!s->is_sm100) return fail(FA_UNSUPPORTED, "this library runs on compute capability 10.x (B200) only");
  // (results are written while other items still read the inputs, and dq holds norms before)
  const size_t rows = static_cast<size_t>(bh) * seqlen, whole = rows * head_dim * 2;
  const Range written[4] = {{dq, whole}, {dk, whole}, {dv, whole}, {workspace, flash_backward_workspace_bytes(batch, heads, seqlen)}};
  const Range read[8] = {{q, whole}, {k, whole}, {v, whole}, {o, whole}, {d_o, whole}, {lse, rows * 4}, {d_lse, rows * 4},
                         {alibi_slopes, static_cast<size_t>(heads) * 4}};
  for (int i = 0; i < 4; ++i) {
    for (const Range& r : read)
      if (overlap(written[i], r)) return fail(FA_INVALID_ARG, "dq, dk, dv and the workspace must not overlap the inputs");
    for (int j = 0; j < i; ++j)
      if (overlap(written[i], written[j])) return fail(FA_INVALID_ARG, "dq, dk, dv and the workspace must not overlap one another");
  }
  if (softmax_scale <= 0.f) softmax_scale = 1.0f / sqrtf(static_cast<float>(head_dim));

  fa::BwdParams p;
  memset(&p, 0, sizeof(p));
  p.o = static_cast<const __half*>(o);
  p.d_o = static_cast<const __half*>(d_o);
  p.v = static_cast<const __half*>(v);
  p.lse = lse;
  p.d_lse = d_lse;
  p.delta = static_cast<float*>(workspace);
  p.norms = p.delta + align256(sizeof(float) * bh * seqlen) / sizeof(float);
  p.dq = static_cast<__half*>(dq);
  p.dk = static_cast<__half*>(dk);
  p.dv = static_cast<__half*>(dv);
  p.seqlen = seqlen;
  p.bh = static_cast<int>(bh);
  p.heads = heads;
  p.tiles = static_cast<int>(tiles);
  p.scale = softmax_scale;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.causal = is_causal ? 1 : 0;
  p.window_left = norm_window(window_left, seqlen);
  p.window_right = norm_window(window_right, seqlen);
  p.alibi_slopes = alibi_slopes;
  p.status = s->status;
  p.withhold = withhold;
  // heads whose Q, K, V and dO (of which every one is read by as many CTAs as it has tiles) stay within 64 MB of L2
  const long long group = (64ll << 20) / (4ll * seqlen * head_dim * 2);
  p.head_group = static_cast<int>(group < 1 ? 1 : group > bh ? bh : group);

  // Items come in falling order of their time. A mask that bounds one side only makes them unequal, so there the order is by
  // rank; else they differ by their kind: dK and dV take a fifth longer than dQ. us, by rank -> kinds apart: 8 heads x 2048 d64,
  // 256 items on 148 CTAs 46.9 -> 41.4, 37 x 4096 d128 866 -> 835; but causal 8 x 2048 d128 35.8 -> 41.9.
  const bool left = p.window_left >= 0, right = p.causal || p.window_right >= 0;
  p.kinds_apart = left == right;

  CUtensorMap maps[4];
  const void* tensors[4] = {q, k, v, d_o};
  for (int i = 0; i < 4; ++i)
    if ((rc = make_map(&maps[i], tensors[i], p.bh, seqlen, head_dim, 128)) != FA_OK) return rc;
  if (head_dim == 64)
    return alibi_slopes ? launch<64, true>(maps, p, s->num_sms, st, !captured) : launch<64, false>(maps, p, s->num_sms, st, !captured);
  return alibi_slopes ? launch<128, true>(maps, p, s->num_sms, st, !captured) : launch<128, false>(maps, p, s->num_sms, st, !captured);
}

}  // namespace

extern "C" {

size_t flash_backward_workspace_bytes(int batch, int heads, int seqlen) {
  if (batch <= 0 || heads <= 0 || seqlen <= 0) return 0;
  const size_t bh = static_cast<size_t>(batch) * heads, n = seqlen;
  return align256(sizeof(float) * bh * n) + align256(sizeof(float) * 3 * bh * ((n + 127) / 128));
}

int flash_backward(const void* q, const void* k, const void* v, const void* o, const void* d_o, const float* lse,
                   const float* d_lse, void* dq, void* dk, void* dv, int batch, int heads, int seqlen, int head_dim,
                   float softmax_scale, int is_causal, int window_left, int window_right, const float* alibi_slopes,
                   void* workspace, size_t workspace_bytes, void* stream) {
  return backward(q, k, v, o, d_o, lse, d_lse, dq, dk, dv, batch, heads, seqlen, head_dim, softmax_scale, is_causal,
                  window_left, window_right, alibi_slopes, workspace, workspace_bytes, stream, 0);
}

#ifdef FA_TEST_WITHHOLD_LOAD
// Test build only: work item 0 never gets its last tile.
int flash_backward_test_withhold(const void* q, const void* k, const void* v, const void* o, const void* d_o,
                                 const float* lse, void* dq, void* dk, void* dv, int batch, int heads, int seqlen,
                                 int head_dim, void* workspace, size_t workspace_bytes, void* stream) {
  return backward(q, k, v, o, d_o, lse, nullptr, dq, dk, dv, batch, heads, seqlen, head_dim, 0.f, 0, -1, -1, nullptr,
                  workspace, workspace_bytes, stream, 1);
}
#endif

}  // extern "C"
