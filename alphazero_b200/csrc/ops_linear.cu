// Linear layer with bias, activation and residual, and its gradients
// (include/minigo_ops.h).
#include "ops_gemm.cuh"

#include <algorithm>

namespace mgb {
namespace ops {
namespace {

__device__ __forceinline__ float slope(float z, int act) {
    switch (act) {
        case MG_ACT_RELU: return z > 0.0f ? 1.0f : 0.0f;
        case MG_ACT_SILU: {
            const float p = 1.0f / (1.0f + expf(-z));
            return p * (1.0f + z * (1.0f - p));
        }
        case MG_ACT_GELU:
            return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) +
                   z * expf(-0.5f * z * z) * 0.39894228040143268f;
        default: return 1.0f;
    }
}

// g = grad * act'(z) and db = sum of g over rows; one thread per column.
template <int DT>
__global__ void __launch_bounds__(256) slope_kernel(mg_linear_backward_args a, void* g) {
    using E = Elem<DT>;
    using T = typename E::T;
    const int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (j >= a.n) return;
    float sum = 0.0f;
    for (int64_t i = 0; i < a.m; ++i) {
        float v = E::get(static_cast<const T*>(a.grad)[i * a.g_row + j * a.g_col]);
        if (a.activation != MG_ACT_NONE)
            v *= slope(E::get(static_cast<const T*>(a.z)[i * a.z_row + j * a.z_col]), a.activation);
        if (g) static_cast<T*>(g)[i * a.n + j] = E::put(v);
        sum += v;
    }
    if (a.db) static_cast<T*>(a.db)[j] = E::put(sum);
}

void check_sizes(int64_t m, int64_t n, int64_t k) {
    const int64_t top = int64_t(1) << 31;
    need(m >= 0 && n >= 1 && k >= 1, "sizes: m >= 0, n >= 1, k >= 1");
    need(m < top && n < top && k < top, "m, n and k must be below 2^31");
}

void check(const mg_linear_args& a) {
    check_sizes(a.m, a.n, a.k);
    need(a.dtype == MG_PREC_BF16 || a.dtype == MG_PREC_FP16, "dtype must be MG_PREC_BF16 or MG_PREC_FP16");
    need(a.activation >= MG_ACT_NONE && a.activation <= MG_ACT_GELU, "activation is not an MG_ACT_* value");
    need(a.m == 0 || (a.x && a.weight && a.y), "x, weight or y is null");
    need(a.x_row >= 0 && a.x_col >= 0 && a.w_row >= 0 && a.w_col >= 0 && a.r_row >= 0 && a.r_col >= 0,
         "a stride is negative");
}

void check(const mg_linear_backward_args& a) {
    check_sizes(a.m, a.n, a.k);
    need(a.dtype == MG_PREC_BF16 || a.dtype == MG_PREC_FP16, "dtype must be MG_PREC_BF16 or MG_PREC_FP16");
    need(a.activation >= MG_ACT_NONE && a.activation <= MG_ACT_GELU, "activation is not an MG_ACT_* value");
    need(a.m == 0 || a.grad, "grad is null");
    need(a.m == 0 || !a.dx || a.weight, "dx needs the weight");
    need(a.m == 0 || !a.dw || a.x, "dw needs x");
    need(a.m == 0 || a.activation == MG_ACT_NONE || a.z, "an activation's backward pass needs z");
    need(a.g_row >= 0 && a.g_col >= 0 && a.x_row >= 0 && a.x_col >= 0 && a.w_row >= 0 &&
             a.w_col >= 0 && a.z_row >= 0 && a.z_col >= 0,
         "a stride is negative");
}

void linear(const mg_linear_args& a, Workspace& w, bool go, cudaStream_t s) {
    if (!go || a.m == 0) return;
    w.require();
    GemmEpilogue e;
    e.bias = a.bias;
    e.res = a.residual;
    e.r_row = a.r_row;
    e.r_col = a.r_col;
    e.out = a.y;
    e.z = a.z;
    e.ld = a.n;
    e.res_scale = a.residual_scale;
    e.act = a.activation;
    launch_gemm(a.dtype, {a.x, a.x_row, a.x_col}, {a.weight, a.w_row, a.w_col}, a.m, a.n, a.k, e, s);
}

void linear_backward(const mg_linear_backward_args& a, Workspace& w, bool go, cudaStream_t s) {
    const bool has_g = a.activation != MG_ACT_NONE && a.m > 0;
    void* g = has_g ? w.take((size_t)a.m * a.n * 2) : nullptr;
    if (!go) return;
    w.require();
    if (a.db || has_g) {
        const unsigned blocks = (unsigned)((a.n + 255) / 256);
        if (a.dtype == MG_PREC_BF16) slope_kernel<MG_PREC_BF16><<<blocks, 256, 0, s>>>(a, g);
        else slope_kernel<MG_PREC_FP16><<<blocks, 256, 0, s>>>(a, g);
        launched("slope_kernel");
    }
    const GemmOperand gr = has_g ? GemmOperand{g, a.n, 1} : GemmOperand{a.grad, a.g_row, a.g_col};
    GemmEpilogue e;
    e.ld = a.k;
    if (a.dx && a.m > 0) {
        e.out = a.dx;
        launch_gemm(a.dtype, gr, {a.weight, a.w_col, a.w_row}, a.m, a.k, a.n, e, s);
    }
    if (a.dw) {
        e.out = a.dw;
        launch_gemm(a.dtype, {gr.data, gr.col, gr.row}, {a.x, a.x_col, a.x_row}, a.n, a.k, a.m, e, s);
    }
}

}  // namespace
}  // namespace ops
}  // namespace mgb

using namespace mgb::ops;

extern "C" int mg_linear_workspace(const mg_linear_args* args, size_t* bytes) {
    return guarded([&] {
        need(args != nullptr && bytes != nullptr, "args or bytes is null");
        check(*args);
        Workspace w;
        linear(*args, w, false, nullptr);
        *bytes = w.used();
    });
}

extern "C" int mg_linear(const mg_linear_args* args, void* workspace, size_t workspace_bytes,
                         void* stream) {
    return guarded([&] {
        need(args != nullptr, "args is null");
        check(*args);
        OnDevice on(args->device);
        Workspace w(workspace, workspace_bytes);
        linear(*args, w, true, static_cast<cudaStream_t>(stream));
    });
}

extern "C" int mg_linear_backward_workspace(const mg_linear_backward_args* args, size_t* bytes) {
    return guarded([&] {
        need(args != nullptr && bytes != nullptr, "args or bytes is null");
        check(*args);
        Workspace w;
        linear_backward(*args, w, false, nullptr);
        *bytes = w.used();
    });
}

extern "C" int mg_linear_backward(const mg_linear_backward_args* args, void* workspace,
                                  size_t workspace_bytes, void* stream) {
    return guarded([&] {
        need(args != nullptr, "args is null");
        check(*args);
        OnDevice on(args->device);
        Workspace w(workspace, workspace_bytes);
        linear_backward(*args, w, true, static_cast<cudaStream_t>(stream));
    });
}
