// The dynamic shared-memory limit of a kernel, raised as its launches need it.
// Host code only, without device helpers, so that it also compiles as plain C++.
#pragma once

#include <cuda_runtime_api.h>

#include <atomic>
#include <mutex>

namespace bee_b200 {

int fail(int code, const char* fmt, ...);
int api_fail(cudaError_t e, const char* fmt, ...);

// cudaFuncSetAttribute applies to the current device, so the limit is kept per
// device.  Launches of one kernel may need different sizes, from several host
// threads at once: the limit only ever grows, and whoever raises it does so
// under the lock, so that no smaller size is set after a larger one and `raised`
// never says more than the kernel has.  Keep one instance per kernel as a
// function-local static.
constexpr int kMaxDevices = 64;
struct SmemLimit {
    std::atomic<int> raised[kMaxDevices]{};
    std::mutex raising;
    template <typename Kernel>
    int ensure(Kernel kernel, int bytes, const char* what) {
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices)
            return fail(cudaErrorInvalidDevice, "%s: no usable current device", what);
        if (raised[dev].load(std::memory_order_acquire) >= bytes) return 0;
        const std::lock_guard<std::mutex> lock(raising);
        if (raised[dev].load(std::memory_order_relaxed) >= bytes) return 0;
        cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e != cudaSuccess) return api_fail(e, "%s: shared memory attribute: %s", what, cudaGetErrorString(e));
        raised[dev].store(bytes, std::memory_order_release);
        return 0;
    }
};

}  // namespace bee_b200
