// Matrix products of the training operators: C[i][j] = sum_k A[i][k] B[j][k]
// with a fused epilogue.
#pragma once

#include "ops_common.cuh"

namespace mgb {
namespace ops {

// Element (i, k) is at data[i * row + k * col].
struct GemmOperand {
    const void* data;
    int64_t row, col;
};

// out = act(alpha * acc + bias) + res_scale * res; z = alpha * acc + bias.
struct GemmEpilogue {
    const void* bias = nullptr;      // [n]
    const void* res = nullptr;       // [m][n]
    int64_t r_row = 0, r_col = 0;
    void* out = nullptr;             // [m][n], row stride ld
    void* z = nullptr;               // [m][n], row stride ld
    float* out32 = nullptr;          // [m][n] fp32 instead of out
    int64_t ld = 0;
    float res_scale = 0.0f;
    int act = MG_ACT_NONE;
    float alpha = 1.0f;
    const int* count = nullptr;      // alpha is divided by max(*count, 1)
};

void launch_gemm(int dtype, const GemmOperand& a, const GemmOperand& b, int64_t m, int64_t n,
                 int64_t k, const GemmEpilogue& e, cudaStream_t stream);

__device__ __forceinline__ float activate(float z, int act) {
    switch (act) {
        case MG_ACT_RELU: return z < 0.0f ? 0.0f : z;  // NaN stays
        case MG_ACT_SILU: return z / (1.0f + expf(-z));
        case MG_ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
        default: return z;
    }
}

}  // namespace ops
}  // namespace mgb
