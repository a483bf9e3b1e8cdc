// bb200_internal.h — helpers shared by the translation units of libbb200.so (host side).
#pragma once
#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdint.h>

#include <atomic>

#include "../../include/bb200.h"

namespace bb200 {

// Record a formatted message as this thread's last error and return `status`.
int fail(int status, const char* fmt, ...);

// Map a cudaError_t of the runtime layer to a status (0 stays 0) and record its string.
int check_runtime(cudaError_t err, const char* what);

// After a kernel launch: pick up launch-configuration errors without synchronising.
inline int check_launch(const char* what) { return check_runtime(cudaGetLastError(), what); }

// The configuration of a launch with programmatic stream serialisation: the kernel's CTAs may be placed while the kernel
// before it on `stream` drains.  ONLY for kernels that run `dependent_launch_prologue()` (below) before their first
// global-memory access.  A capturing stream takes the ordinary launch.  `cluster`: CTAs of a cluster along x.
struct DependentLaunch {
  cudaLaunchConfig_t config = {};
  cudaLaunchAttribute attributes[2] = {};
  DependentLaunch(dim3 grid, dim3 block, unsigned cluster, size_t dynamic_smem, cudaStream_t stream) {
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    const bool capturing = cudaStreamIsCapturing(stream, &capture) != cudaSuccess || capture != cudaStreamCaptureStatusNone;
    config.gridDim = grid;
    config.blockDim = block;
    config.dynamicSmemBytes = dynamic_smem;
    config.stream = stream;
    config.attrs = attributes;
    if (!capturing) {
      attributes[config.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attributes[config.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
      attributes[config.numAttrs].id = cudaLaunchAttributeClusterDimension;
      attributes[config.numAttrs].val.clusterDim.x = cluster;
      attributes[config.numAttrs].val.clusterDim.y = 1;
      attributes[config.numAttrs++].val.clusterDim.z = 1;
    }
  }
  DependentLaunch(const DependentLaunch&) = delete;  // config points to attributes
  DependentLaunch& operator=(const DependentLaunch&) = delete;
};

template <typename... Params, typename... Args>
inline void launch_dependent_cluster(void (*kernel)(Params...), dim3 grid, dim3 block, unsigned cluster, size_t dynamic_smem,
                                     cudaStream_t stream, const Args&... args) {
  DependentLaunch launch(grid, block, cluster, dynamic_smem, stream);
  cudaLaunchKernelEx(&launch.config, kernel, static_cast<Params>(args)...);  // the caller reads the status with check_launch()
}

template <typename... Params, typename... Args>
inline void launch_dependent(void (*kernel)(Params...), dim3 grid, dim3 block, size_t dynamic_smem, cudaStream_t stream, const Args&... args) {
  launch_dependent_cluster(kernel, grid, block, 1, dynamic_smem, stream, args...);
}

#ifdef __CUDACC__
// First statement of a kernel launched with launch_dependent(): lets the kernel behind this one be placed early in its
// turn, then waits until the kernel before this one has completed and its writes are visible.  Without the launch
// attribute both instructions do nothing.
__device__ __forceinline__ void dependent_launch_prologue() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
#endif

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

inline bool aligned32(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31u) == 0; }

inline size_t dtype_bytes(bb200_dtype t) {
  switch (t) {
    case BB200_F32: case BB200_I32: return 4;
    case BB200_BF16: case BB200_F16: return 2;
    case BB200_I64: return 8;
    case BB200_I8: case BB200_I1: return 1;
  }
  return 0;
}

// Device status word for bounded waits (0 = clean).  Defined in abi_driver.cu.
int* device_status_word();

// TMA descriptor encoding through the lazily loaded driver (abi_driver.cu).
int encode_tensormap_2d(void* map_out, bb200_dtype dtype, const void* base, uint64_t rows, uint64_t cols,
                        uint64_t row_stride_bytes, uint32_t box_rows, uint32_t box_cols, int swizzle);

// 3-D variant: extents (dim0 innermost), byte strides of dim1 and dim2, box extents.
int encode_tensormap_3d(void* map_out, bb200_dtype dtype, const void* base, uint64_t dim0, uint64_t dim1, uint64_t dim2,
                        uint64_t stride1_bytes, uint64_t stride2_bytes, uint32_t box0, uint32_t box1, uint32_t box2,
                        int swizzle);

// ---- stream-ordered workspaces (workspace.cu) ------------------------------------------------------------------------
// Devices that per-device tables of this library cover.
constexpr int kMaxWorkspaceDevices = 64;

// The pool that workspaces of `device` come from (nullptr: it could not be created).  A pool of this library's own that
// keeps what is freed (release threshold = everything): the device's default pool hands memory back at every
// synchronisation, and a caller that synchronises between two calls would then pay a fresh allocation (about 130 us)
// for every call.
cudaMemPool_t workspace_pool(int device);

// Streaming multiprocessors of the current device.
int multiprocessor_count();

// Memory for one call: taken in stream order from the current device's pool, given back in stream order by release()
// (or the destructor).  Two calls, on one stream or on several, never share it; recorded into a launch graph it becomes
// an allocation of that graph's own.
class Workspace {
 public:
  explicit Workspace(cudaStream_t stream) : stream_(stream) {}
  ~Workspace() { release(nullptr); }
  Workspace(const Workspace&) = delete;
  Workspace& operator=(const Workspace&) = delete;
  int take(size_t bytes, const char* what);  // a status; data() is 256-byte aligned afterwards
  int release(const char* what);             // a status; `what` names the caller in the error text
  char* data() const { return data_; }

 private:
  cudaStream_t stream_;
  char* data_ = nullptr;
};

// Whether the current device can hold a cluster of 16 CTAs of KERNEL (with `threads` threads and `shared_bytes` of dynamic
// shared memory, the same in every call): beyond the portable eight, it depends on the multiprocessors that are there.
// Asked once per kernel and device.
template <auto KERNEL> bool sixteen_fit(int threads, size_t shared_bytes) {
  static std::atomic<int> answers[kMaxWorkspaceDevices];  // 0: not asked yet, 1: no, 2: yes
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= kMaxWorkspaceDevices) return false;
  int answer = answers[device].load(std::memory_order_relaxed);
  if (!answer) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(16);
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = shared_bytes;
    cudaLaunchAttribute attribute = {};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = 16;
    attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    int clusters = 0;
    answer = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
                     cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared_bytes) == cudaSuccess &&
                     cudaOccupancyMaxActiveClusters(&clusters, KERNEL, &config) == cudaSuccess && clusters > 0
                 ? 2
                 : 1;
    cudaGetLastError();  // a "no" is no error of the call
    answers[device].store(answer, std::memory_order_relaxed);
  }
  return answer == 2;
}

// Raise KERNEL's limit of dynamic shared memory to `bytes` on the current device, once per kernel and device (`bytes` is the
// same in every call; two threads doing it at once is harmless).
template <auto KERNEL> int allow_shared_memory(int bytes, const char* what) {
  static std::atomic<bool> done[kMaxWorkspaceDevices];
  int device = 0;
  if (int status = check_runtime(cudaGetDevice(&device), what)) return status;
  const bool known = device >= 0 && device < kMaxWorkspaceDevices;
  if (known && done[device].load(std::memory_order_relaxed)) return BB200_OK;
  if (int status = check_runtime(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), what)) return status;
  if (known) done[device].store(true, std::memory_order_relaxed);
  return BB200_OK;
}

// Whether [a, a + a_bytes) and [b, b + b_bytes) share memory (null pointers share none).
inline bool overlap(const void* a, size_t a_bytes, const void* b, size_t b_bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x && y && x < y + b_bytes && y < x + a_bytes;
}

}  // namespace bb200
