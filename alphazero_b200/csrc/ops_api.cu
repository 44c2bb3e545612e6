// Errors and device status of the training operators (include/minigo_ops.h).
#include "ops_common.cuh"

#include <atomic>

namespace mgb {
namespace ops {
namespace {

__device__ int g_op_status;
constexpr int kMaxDevices = 64;

// 32 columns per block; 32 threads share a column's rows.
template <int DT>
__global__ void __launch_bounds__(1024) add_rows_kernel(const float* sums, int64_t rows, int64_t cols, float alpha,
                                                        const int* count, typename Elem<DT>::T* out) {
    __shared__ float part[32][33];
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
    griddep_launch_dependents();
    griddep_wait();
    float s = 0.0f;
    if (c < cols)
#pragma unroll 8
        for (int64_t r = slice; r < rows; r += 32) s += sums[r * cols + c];
    part[slice][lane] = s;
    __syncthreads();
    if (slice > 0 || c >= cols) return;
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += part[i][lane];
    out[c] = Elem<DT>::put(s * (count ? alpha / (float)max(*count, 1) : alpha));
}

}  // namespace

std::string& last_op_error() {
    thread_local std::string message;
    return message;
}

void add_rows(int dtype, const float* sums, int64_t rows, int64_t cols, float alpha, const int* count,
              void* out, Queue& q) {
    const dim3 grid((unsigned)((cols + 31) / 32));
    if (dtype == MG_PREC_BF16)
        q.launch("add_rows_kernel", add_rows_kernel<MG_PREC_BF16>, grid, 1024, 0, sums, rows, cols, alpha, count,
                 static_cast<__nv_bfloat16*>(out));
    else
        q.launch("add_rows_kernel", add_rows_kernel<MG_PREC_FP16>, grid, 1024, 0, sums, rows, cols, alpha, count,
                 static_cast<__half*>(out));
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
