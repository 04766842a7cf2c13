// What the entry points ask of the current device (included by every source file of the library).
#include <atomic>
#include <cstdint>
#include <mutex>

static int device_ready()
{
    static std::atomic<bool> found{false};       // (a device that was there stays)
    if (found.load(std::memory_order_relaxed)) return LMZ_GPU_OK;
    int n = 0;
    if (cudaGetDeviceCount(&n) != cudaSuccess || n < 1) {
        cudaGetLastError();
        return fail_msg(LMZ_GPU_ENODEV, "no CUDA device");
    }
    found = true;
    return LMZ_GPU_OK;
}

// Kernels ask for more dynamic shared memory than the default 48 KiB; the
// opt-in is per device and is made once.
template <class K>
static int opt_in_smem(K kernel, uint32_t bytes, bool *done /* [64] by device */)
{
    int dev = 0;
    CK("cudaGetDevice", cudaGetDevice(&dev));
    static std::mutex mu;
    std::lock_guard<std::mutex> lock(mu);
    if (dev >= 0 && dev < 64 && done[dev]) return LMZ_GPU_OK;
    CK("cudaFuncSetAttribute",
       cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    if (dev >= 0 && dev < 64) done[dev] = true;
    return LMZ_GPU_OK;
}

static int sm_count(int *out)
{
    static int cached[64];
    int dev = 0;
    CK("cudaGetDevice", cudaGetDevice(&dev));
    if (dev >= 0 && dev < 64 && cached[dev]) { *out = cached[dev]; return LMZ_GPU_OK; }
    int n = 0;
    CK("cudaDeviceGetAttribute", cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
    if (dev >= 0 && dev < 64) cached[dev] = n;
    *out = n;
    return LMZ_GPU_OK;
}
