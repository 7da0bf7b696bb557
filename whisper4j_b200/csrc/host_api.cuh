// host_api.cuh — error reporting shared by the files that define C entry points.
#pragma once
#include <cuda_runtime.h>

#include <atomic>

#include "../../include/whisper4j_cuda.h"

namespace w4j {

// Sets the calling thread's w4j_last_error() message and returns `code` (runtime.cu).
int set_err(int code, const char *fmt, ...);

// Makes `device` current on the calling thread and puts the caller's device back at the end of the call.
class DeviceGuard {
  public:
    explicit DeviceGuard(int device) {
        static std::atomic<int> count{0};  // devices do not come and go
        int n = count.load(std::memory_order_relaxed);
        if (n == 0 && (cudaGetDeviceCount(&n) != cudaSuccess || n == 0)) {
            cudaGetLastError();
            rc_ = set_err(W4J_ERR_CUDA, "no CUDA device available");
            return;
        }
        count.store(n, std::memory_order_relaxed);
        if (device < 0 || device >= n) {
            rc_ = set_err(W4J_ERR_ARG, "device %d out of range (%d devices)", device, n);
        } else if (cudaGetDevice(&before_) != cudaSuccess ||
                   (before_ != device && cudaSetDevice(device) != cudaSuccess)) {
            cudaGetLastError();
            before_ = -1;
            rc_ = set_err(W4J_ERR_CUDA, "device %d cannot be made current", device);
        } else if (before_ == device) {
            before_ = -1;  // nothing to put back
        }
    }
    ~DeviceGuard() {
        if (before_ >= 0) cudaSetDevice(before_);
    }
    DeviceGuard(const DeviceGuard &) = delete;
    DeviceGuard &operator=(const DeviceGuard &) = delete;
    int rc() const { return rc_; }

  private:
    int before_ = -1, rc_ = W4J_OK;
};

// Once for each device: lets a kernel use all of the opt-in shared memory beside its static arrays.
template <auto Kern>
inline cudaError_t prepare() {
    static std::atomic<uint64_t> done{0};
    int dev = 0, optin = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (dev < 64 && (done.load(std::memory_order_acquire) & bit)) return cudaSuccess;
    cudaFuncAttributes fa;
    if ((e = cudaDeviceGetAttribute(&optin, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev)) != cudaSuccess) return e;
    if ((e = cudaFuncGetAttributes(&fa, Kern)) != cudaSuccess) return e;
    e = cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, optin - (int)fa.sharedSizeBytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
    return e;
}

// Launch with programmatic dependent launch: the kernel may be scheduled while its predecessor in the
// stream still runs, so every one of its threads executes griddepcontrol.wait before it touches global
// memory that the predecessor may write or still read.
template <auto Kern, typename... Args>
inline cudaError_t launch_after(dim3 grid, dim3 block, size_t smem, cudaStream_t s, int cluster, Args... args) {
    const cudaError_t e = prepare<Kern>();
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute at[2];
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = at;
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
    if (cluster > 1) {
        at[1].id = cudaLaunchAttributeClusterDimension;
        at[1].val.clusterDim.x = cluster;
        at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
        cfg.numAttrs = 2;
    }
    return cudaLaunchKernelEx(&cfg, Kern, args...);
}

}  // namespace w4j

// A failed call leaves its error as the thread's last CUDA error (cudaGetLastError); it is consumed
// here, so a later launch check does not report an earlier, already handled failure (a refused
// allocation, for instance).
#define CUDA_TRY(expr)                                                                             \
    do {                                                                                           \
        cudaError_t e_ = (expr);                                                                   \
        if (e_ != cudaSuccess) {                                                                   \
            cudaGetLastError();                                                                    \
            return w4j::set_err(e_ == cudaErrorMemoryAllocation ? W4J_ERR_OOM : W4J_ERR_CUDA, "%s: %s (%s:%d)", \
                                #expr, cudaGetErrorString(e_), __FILE__, __LINE__);                \
        }                                                                                          \
    } while (0)

#define TRY(expr)            \
    do {                     \
        int r_ = (expr);     \
        if (r_ < 0) return r_; \
    } while (0)
