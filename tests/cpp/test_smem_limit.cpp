// SmemLimit against a fake CUDA runtime: two host threads make the first calls
// for one kernel, one with a large and one with a small size, and the fake lets
// each call to cudaFuncSetAttribute wait (a bounded time) for the other one:
// the large size is set, then the small one, and the small call returns first.
#include "smem_limit.cuh"

#include <chrono>
#include <cstdio>
#include <thread>

namespace {

constexpr int kBig = 209920, kSmall = 105472;
std::atomic<int> limit{49152}, calls{0};
std::atomic<bool> big_set{false}, small_done{false};

void await(const std::atomic<bool>& flag, int ms) {
    for (int i = 0; i < ms && !flag; ++i) std::this_thread::sleep_for(std::chrono::milliseconds(1));
}

void kernel() {}

}  // namespace

extern "C" cudaError_t CUDARTAPI cudaGetDevice(int* device) {
    *device = 0;
    return cudaSuccess;
}
extern "C" const char* CUDARTAPI cudaGetErrorString(cudaError_t) { return "fake"; }
extern "C" cudaError_t CUDARTAPI cudaFuncSetAttribute(const void*, cudaFuncAttribute, int value) {
    ++calls;
    if (value == kBig) {
        limit = value;
        big_set = true;
        await(small_done, 200);
    } else {
        await(big_set, 200);
        limit = value;
    }
    return cudaSuccess;
}

namespace bee_b200 {
int fail(int code, const char*, ...) { return code; }
int api_fail(cudaError_t e, const char*, ...) { return static_cast<int>(e); }
}  // namespace bee_b200

int main() {
    static bee_b200::SmemLimit smem;
    int rc_big = -1, rc_small = -1;
    std::thread a([&] { rc_big = smem.ensure(kernel, kBig, "big"); });
    std::thread b([&] {
        rc_small = smem.ensure(kernel, kSmall, "small");
        small_done = true;
    });
    a.join();
    b.join();
    bool ok = rc_big == 0 && rc_small == 0 && limit == kBig && smem.raised[0] == kBig;
    const int before = calls;
    ok = ok && smem.ensure(kernel, kSmall, "again") == 0 && smem.ensure(kernel, kBig, "again") == 0 && calls == before;
    std::printf("limit %d, recorded %d, calls %d: %s\n", limit.load(), smem.raised[0].load(), calls.load(), ok ? "ok" : "WRONG");
    return ok ? 0 : 1;
}
