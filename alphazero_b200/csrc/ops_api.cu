// Errors and device status of the training operators (include/minigo_ops.h).
#include "ops_common.cuh"

#include <atomic>

namespace mgb {
namespace ops {
namespace {

__device__ int g_op_status;
constexpr int kMaxDevices = 64;

}  // namespace

std::string& last_op_error() {
    thread_local std::string message;
    return message;
}

int* op_status_word() {
    static std::atomic<int*> known[kMaxDevices];
    int device = 0;
    check(cudaGetDevice(&device), "cudaGetDevice");
    need(device >= 0 && device < kMaxDevices, "device index out of range");
    int* p = known[device].load(std::memory_order_acquire);
    if (p == nullptr) {
        void* q = nullptr;
        check(cudaGetSymbolAddress(&q, g_op_status), "cudaGetSymbolAddress(status)");
        p = static_cast<int*>(q);
        known[device].store(p, std::memory_order_release);
    }
    return p;
}

}  // namespace ops
}  // namespace mgb

using namespace mgb::ops;

extern "C" const char* mg_op_error(void) { return last_op_error().c_str(); }

extern "C" int mg_op_synchronize(int device, void* stream) {
    return guarded([&] {
        OnDevice on(device);
        auto s = static_cast<cudaStream_t>(stream);
        int status = 0;
        int* word = op_status_word();
        check(cudaMemcpyAsync(&status, word, sizeof status, cudaMemcpyDeviceToHost, s), "cudaMemcpyAsync");
        check(cudaStreamSynchronize(s), "cudaStreamSynchronize");
        if (status == 0) return;
        check(cudaMemsetAsync(word, 0, sizeof status, s), "cudaMemsetAsync");
        check(cudaStreamSynchronize(s), "cudaStreamSynchronize");
        fail(MG_E_DEVICE, "a kernel gave up a bounded wait (device status " + std::to_string(status) + ")");
    });
}
