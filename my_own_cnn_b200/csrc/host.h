// Host services of the library shared by its translation units (defined in b200q.cu): error
// messages, per-device state, stream workspaces.  Internal: hidden from the library's users.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <array>
#include <cstddef>
#include <cstdint>
#include <mutex>

#include "../../include/b200q.h"

namespace b200q {

#define B200Q_HIDDEN __attribute__((visibility("hidden")))

// Sets the calling thread's message and returns `code`.
B200Q_HIDDEN int host_fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
B200Q_HIDDEN int host_cuda_fail(cudaError_t e, const char* what);
// cudaGetLastError() after a launch as a status.
B200Q_HIDDEN int host_check_launch(const char* what);
// SM count of the current device, the device address of its error word and (index) its number.
constexpr int kMaxDevices = 64;
B200Q_HIDDEN int host_device(int* sms, int** err, int* index = nullptr);
// Scratch of a stream: kScratchBytes, and kSplitCounters arrival counters that are zero before and after every kernel that uses
// them.  Made by the first call on the stream and never moved.  While the stream is captured it is the graph's own (refused
// where the stream has none yet), so that a graph may be replayed beside other graphs and calls; it is used again when the
// graph is destroyed.
constexpr size_t kScratchBytes = 8u << 20;
constexpr int kSplitCounters = 1 << 16;
// While it lives no other thread's call gets the same scratch: a call's launches lie together in the stream.
struct ScratchHold {
  std::unique_lock<std::mutex> lock;
  void* bytes = nullptr;
  unsigned* counters = nullptr;
  cudaStream_t stream = nullptr;
  cudaEvent_t* after = nullptr;
  B200Q_HIDDEN void launched() const;  // the call's last kernel is in the stream
};
B200Q_HIDDEN int host_scratch(cudaStream_t stream, ScratchHold* hold);
B200Q_HIDDEN void host_set_path(int path);
// Bound of a wait on an mbarrier, in SM clocks.
B200Q_HIDDEN long long host_wait_limit();
// A rank-3 tensor map with the 128-byte swizzle and zeros outside: sizes and box in elements, strides of the outer two in bytes.
B200Q_HIDDEN int host_tensor_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, std::array<uint64_t, 3> size,
                                 uint64_t stride1, uint64_t stride2, std::array<uint32_t, 3> box);

// Launches a kernel that begins with wait_for_previous(): its blocks may take their places while the stream's previous kernel
// drains, and wait there until that one has ended and its writes can be seen.  `cluster` blocks make a cluster.
template <typename... P, typename... A>
int host_launch(const char* what, void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t stream,
                int cluster, const A&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {static_cast<unsigned>(cluster), 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, P(args)...);
  return e == cudaSuccess ? host_check_launch(what) : host_cuda_fail(e, what);
}

// Codes of g_dev_err for bad values that only the device sees; 0x1xx are timeouts (common.cuh).
constexpr int kDevErrBadPosition = 0x201;
constexpr int kDevErrBadSlot = 0x202;
constexpr int kDevErrBadPage = 0x203;
constexpr int kDevErrBadLength = 0x204;
constexpr int kDevErrBadStarts = 0x205;

}  // namespace b200q
