// workspace.cu — stream-ordered workspaces of the operators that need device memory for the length of one call.
#include <atomic>
#include <mutex>

#include "bb200_internal.h"

namespace bb200 {

cudaMemPool_t workspace_pool(int device) {
  static std::mutex guard;
  static cudaMemPool_t pools[kMaxWorkspaceDevices] = {};
  if (device < 0 || device >= kMaxWorkspaceDevices) return nullptr;
  std::lock_guard<std::mutex> lock(guard);
  if (!pools[device]) {
    cudaMemPoolProps props = {};
    props.allocType = cudaMemAllocationTypePinned;
    props.handleTypes = cudaMemHandleTypeNone;
    props.location.type = cudaMemLocationTypeDevice;
    props.location.id = device;
    cudaMemPool_t created = nullptr;
    if (cudaMemPoolCreate(&created, &props) != cudaSuccess) {
      cudaGetLastError();
      return nullptr;
    }
    unsigned long long keep_everything = ~0ull;
    cudaMemPoolSetAttribute(created, cudaMemPoolAttrReleaseThreshold, &keep_everything);
    pools[device] = created;
  }
  return pools[device];
}

int multiprocessor_count() {
  static std::atomic<int> counts[kMaxWorkspaceDevices];
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= kMaxWorkspaceDevices) return 148;
  int count = counts[device];
  if (!count) {
    if (cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || count < 1) count = 148;
    counts[device] = count;
  }
  return count;
}

int Workspace::take(size_t bytes, const char* what) {
  int device = 0;
  if (int status = check_runtime(cudaGetDevice(&device), what)) return status;
  cudaMemPool_t pool = workspace_pool(device);
  if (!pool) return fail(BB200_E_NO_DRIVER, "%s: could not create the workspace pool", what);
  void* taken = nullptr;
  if (int status = check_runtime(cudaMallocFromPoolAsync(&taken, bytes, pool, stream_), what)) return status;
  data_ = static_cast<char*>(taken);
  return BB200_OK;
}

int Workspace::release(const char* what) {
  if (!data_) return BB200_OK;
  const cudaError_t err = cudaFreeAsync(data_, stream_);
  data_ = nullptr;
  return what ? check_runtime(err, what) : BB200_OK;
}

}  // namespace bb200
