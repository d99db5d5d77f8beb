// What the host sides of the library's entry points share: error texts, the record of a device, tensor maps.
// Defined in flash_forward.cu.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <mutex>

#include "../../include/flash_forward_b200.h"

namespace fa_host {

// Sets the calling thread's error text and returns `code`.
int fail(int code, const char* fmt, const char* a = "", const char* b = "");
int fail_cuda(const char* what, cudaError_t e);

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver entry point is looked up at run time so that the library links against the CUDA
// runtime only and can be loaded (for symbol checks) on a machine without a driver.
EncodeTiledFn encode_tiled_fn();

constexpr int kMaxDevices = 64;
// Launches in flight at the same time must not share a pair of scheduler words (the kernel leaves its pair at zero).
// The first kOwnedSlots streams that are used on a device each own a pair: launches on one stream run one after the
// other, so nothing more is needed. Streams are told apart by their id, which is never used again after a stream is
// destroyed (nothing tells this library that one was, so its pair stays taken until flash_forward_shutdown()). Launches
// on any further stream take the 64 remaining pairs in turn, and one that reuses a pair last used on ANOTHER stream
// first makes its stream wait for that earlier launch (an event per pair). (With an event behind every launch a call
// cost 1 us more on the host, and the kernel behind it could not start early. 256 owners: eight times one of
// PyTorch's stream pools; finding the last of them takes 0.1 us.)
constexpr int kOwnedSlots = 256;
constexpr int kSchedSlots = kOwnedSlots + 64;
constexpr size_t kDeviceWords = 4 + 2 * kSchedSlots;
struct DeviceState {
  std::mutex mu;
  bool probed = false;
  bool is_sm100 = false;
  int num_sms = 0;
  // device words: [0] status (a wait that ran out), [1] an index in device memory that was out of range, then, from the
  // fifth on, kSchedSlots pairs of scheduler words
  int* status = nullptr;
  int num_owned = 0;                           // pairs 0 .. num_owned-1 belong to the streams owner[]
  unsigned long long owner[kOwnedSlots] = {};  // stream ids
  unsigned next_sched = 0;
  cudaEvent_t slot_done[kSchedSlots] = {};     // recorded behind the last launch that used the pair
  unsigned long long slot_stream[kSchedSlots] = {};  // the id of that launch's stream
  bool slot_used[kSchedSlots] = {};
  unsigned long long acquired_by = 0;  // the stream id of the launch between sched_acquire and sched_release
  bool attr_set[29] = {};
};

// The record of the current device; the first call on a device allocates its words.
int device_state(DeviceState** out);

// The same for an entry point that may be captured into a CUDA graph: the first call on a device, which allocates, is
// refused with FA_UNSUPPORTED on a stream that is being captured. *captured says whether `st` is.
int device_state_for(cudaStream_t st, DeviceState** out, bool* captured);

// 4-D map over one [bh][seqlen][head_dim] fp16 tensor: {64 contiguous elements, row, 64-wide
// panel, head}. One box = 128 rows x all panels of one head, landing in shared memory as
// [panel][row][64] with the 128-byte swizzle a UMMA descriptor expects. Out-of-range rows of
// a ragged last tile read as zero.
int make_map(CUtensorMap* map, const void* base, int bh, int seqlen, int head_dim, int box_rows, int box_panels = 0);

// A window that reaches past either end of the sequence for every row is no window. Mapping it to
// "unbounded" (-1) here keeps the tile arithmetic (row - window_left, row + window_right) inside int
// for every legal argument, INT_MAX included.
inline int norm_window(int w, int seqlen) { return (w < 0 || w >= seqlen) ? -1 : w; }

// FA_OK, or FA_INVALID_ARG for a softmax scale that the kernels cannot take.
int check_scale(float softmax_scale);

// Launches `kernel` with programmatic stream serialization if `early`: its prologue may run while the kernel in front of
// it in the stream ends, and it has to wait (griddepcontrol.wait) before it touches global memory. Not in a captured
// graph: two such launches in a row would leave a programmatic edge there, and cudaGraphGetEdges and the like, which
// report plain edges only, would answer cudaErrorLossyQuery for the caller's whole graph.
template <typename... Params, typename... Args>
cudaError_t launch_early_in_clusters(void (*kernel)(Params...), int cluster, dim3 grid, int threads, int smem, cudaStream_t st,
                                     bool early, Args&&... args) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = early ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}
template <typename... Params, typename... Args>
cudaError_t launch_early(void (*kernel)(Params...), dim3 grid, int threads, int smem, cudaStream_t st, bool early,
                         Args&&... args) {
  return launch_early_in_clusters(kernel, 1, grid, threads, smem, st, early, args...);
}

}  // namespace fa_host
