// Linear layer with bias, activation and residual, and its gradients
// (include/minigo_ops.h).
#include "ops_gemm.cuh"

#include <algorithm>

namespace mgb {
namespace ops {
namespace {

// act'(z) of the smooth ones.
__device__ __forceinline__ float slope(float z, int act) {
    switch (act) {
        case MG_ACT_SILU: {
            const float p = logistic(z);
            return p * (1.0f + z * (1.0f - p));
        }
        case MG_ACT_GELU: {
            float bell;
            const float phi = normal_cdf(z, &bell);
            return phi + z * bell * 0.39894228040143268f;
        }
        default: return 1.0f;
    }
}

// A ReLU that is shut lets nothing through, an infinity or NaN neither.
__device__ __forceinline__ float times_slope(float v, float z, int act) {
    if (act == MG_ACT_RELU) return z > 0.0f ? v : 0.0f;
    return v * slope(z, act);
}

// g = grad * act'(z) (if g is set) and, per block of rows, the column sums of
// grad * act'(z) before their rounding.  One pass; a thread has V adjacent
// columns (V = 8: 16-byte accesses) of every eighth row of its block, the
// eight sums of a column meet in shared memory.  Blocks past across * down
// copy operands.  Bound by memory, for GELU by its instructions as well: 8192
// x 8192 bf16 take 80 us, 5 TB/s of the two matrices read and one written.
template <int DT, int V>
__global__ void __launch_bounds__(256)
    slope_kernel(mg_linear_backward_args a, uint16_t* g, int64_t ldg, int rows_per_block, float* sums, int64_t across,
                 int64_t down, Packs packs) {
    using E = Elem<DT>;
    using T = typename E::T;
    __shared__ float part[8][32 * V];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    griddep_launch_dependents();
    griddep_wait();
    if (blockIdx.x >= across * down) return pack_block(packs, (int)(blockIdx.x - across * down));
    const int64_t bx = blockIdx.x % across, by = blockIdx.x / across;
    const int64_t c = bx * (32 * V) + lane * V;
    const int64_t r0 = by * rows_per_block, r1 = min(a.m, r0 + rows_per_block);
    const T* dy = static_cast<const T*>(a.grad);
    const T* z = static_cast<const T*>(a.z);
    float sum[V] = {};
    if (c < a.n)
#pragma unroll 2
        for (int64_t r = r0 + warp; r < r1; r += 8) {
            alignas(16) T dv[V], zv[V];
            if constexpr (V == 8) {
                *reinterpret_cast<uint4*>(dv) = __ldg(reinterpret_cast<const uint4*>(dy + r * a.g_row + c));
                if (g) *reinterpret_cast<uint4*>(zv) = __ldg(reinterpret_cast<const uint4*>(z + r * a.z_row + c));
            } else {
                dv[0] = dy[r * a.g_row + c * a.g_col];
                if (g) zv[0] = z[r * a.z_row + c * a.z_col];
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float v = E::get(dv[i]);
                if (g) {
                    v = times_slope(v, E::get(zv[i]), a.activation);
                    dv[i] = E::put(v);
                }
                sum[i] += v;
            }
            if (g) {
                if constexpr (V == 8) *reinterpret_cast<uint4*>(g + r * ldg + c) = *reinterpret_cast<uint4*>(dv);
                else reinterpret_cast<T*>(g)[r * ldg + c] = dv[0];
            }
        }
    if (sums == nullptr) return;
#pragma unroll
    for (int i = 0; i < V; ++i) part[warp][lane * V + i] = sum[i];
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * V; i += 256) {
        const int64_t col = bx * (32 * V) + i;
        if (col >= a.n) continue;
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) s += part[w][i];
        sums[by * a.n + col] = s;
    }
}

void check_sizes(int64_t m, int64_t n, int64_t k) {
    const int64_t top = (int64_t(1) << 31) - 1024;  // whole tiles still count in 32 bits
    need(m >= 0 && n >= 1 && k >= 1, "sizes: m >= 0, n >= 1, k >= 1");
    need(m < top && n < top && k < top, "m, n and k must be below 2^31 - 1024");
}

void check(const mg_linear_args& a) {
    check_sizes(a.m, a.n, a.k);
    need(a.dtype == MG_PREC_BF16 || a.dtype == MG_PREC_FP16, "dtype must be MG_PREC_BF16 or MG_PREC_FP16");
    need(a.activation >= MG_ACT_NONE && a.activation <= MG_ACT_GELU, "activation is not an MG_ACT_* value");
    need(a.m == 0 || (a.x && a.weight && a.y), "x, weight or y is null");
    need(a.x_row >= 0 && a.x_col >= 0 && a.w_row >= 0 && a.w_col >= 0 && a.r_row >= 0 && a.r_col >= 0,
         "a stride is negative");
    need_aligned(a.x, 2, "x");
    need_aligned(a.weight, 2, "weight");
    need_aligned(a.bias, 2, "bias");
    need_aligned(a.residual, 2, "residual");
    need_aligned(a.y, 2, "y");
    need_aligned(a.z, 2, "z");
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
    need_aligned(a.grad, 2, "grad");
    need_aligned(a.x, 2, "x");
    need_aligned(a.weight, 2, "weight");
    need_aligned(a.z, 2, "z");
    need_aligned(a.dx, 2, "dx");
    need_aligned(a.dw, 2, "dw");
    need_aligned(a.db, 2, "db");
}

void linear(const mg_linear_args& a, Workspace& w, bool go, Queue& q) {
    if (a.m == 0) return;
    Packs packs;
    GemmJob job;
    job.a = stage_operand(w, packs, {a.x, a.x_row, a.x_col}, a.m, a.k);
    job.b = stage_operand(w, packs, {a.weight, a.w_row, a.w_col}, a.n, a.k);
    job.m = a.m;
    job.n = a.n;
    job.k = a.k;
    job.e.bias = a.bias;
    job.e.res = a.residual;
    job.e.r_row = a.r_row;
    job.e.r_col = a.r_col;
    job.e.out = a.y;
    job.e.z = a.z;
    job.e.ld = a.n;
    job.e.res_scale = a.residual_scale;
    job.e.act = a.activation;
    Post post;
    if (go) {
        w.require();
        packs.launch(q);
    }
    gemm(w, go, a.dtype, &job, 1, post, q);
    if (go) post.launch(a.dtype, q);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

void linear_backward(const mg_linear_backward_args& a, Workspace& w, bool go, Queue& q) {
    if (!a.dx && !a.dw && !a.db) return;
    if (a.m == 0) {
        if (!go) return;
        if (a.dw) q.clear(a.dw, (size_t)a.n * a.k * 2);
        if (a.db) q.clear(a.db, (size_t)a.n * 2);
        return;
    }
    Packs packs;
    Post post;
    GemmJob jobs[2];
    int count = 0;
    const bool has_g = a.activation != MG_ACT_NONE;
    const int64_t ldg = (a.n + 7) / 8 * 8;
    uint16_t* g = has_g ? w.take<uint16_t>((size_t)a.m * ldg * 2) : nullptr;
    StagedOperand gs;
    gs.data = g;
    gs.ld = ldg;
    if (!has_g && (a.dx || a.dw)) gs = stage_operand(w, packs, {a.grad, a.g_row, a.g_col}, a.m, a.n);
    if (a.dx) {
        GemmJob& j = jobs[count++];
        j.a = gs;
        j.b = stage_operand(w, packs, {a.weight, a.w_col, a.w_row}, a.k, a.n);
        j.m = a.m;
        j.n = a.k;
        j.k = a.n;
        j.e.out = a.dx;
        j.e.ld = a.k;
    }
    if (a.dw) {
        GemmJob& j = jobs[count++];
        j.a = transposed(gs);
        j.b = stage_operand(w, packs, {a.x, a.x_col, a.x_row}, a.k, a.m);
        j.m = a.n;
        j.n = a.k;
        j.k = a.m;
        j.e.out = a.dw;
        j.e.ld = a.k;
    }
    if (a.db || has_g) {
        const bool vec = a.n % 8 == 0 && aligned16(a.grad) && a.g_col == 1 && a.g_row % 8 == 0 &&
                         (!has_g || (aligned16(a.z) && a.z_col == 1 && a.z_row % 8 == 0));
        const int64_t across = (a.n + (vec ? 255 : 31)) / (vec ? 256 : 32);
        // about four blocks per SM, at least 32 rows each
        const int64_t want = std::max<int64_t>(1, 148 * 4 / across);
        const int rows = (int)std::max<int64_t>(32, (a.m + want - 1) / want);
        const int64_t down = (a.m + rows - 1) / rows;
        float* sums = a.db ? w.take<float>((size_t)down * a.n * 4) : nullptr;
        if (go) {
            w.require();
            const int64_t blocks = across * down + packs.blocks();
            need(blocks < (int64_t(1) << 31), "too many blocks");
            const bool bf = a.dtype == MG_PREC_BF16;
            const auto kernel = vec ? (bf ? slope_kernel<MG_PREC_BF16, 8> : slope_kernel<MG_PREC_FP16, 8>)
                                    : (bf ? slope_kernel<MG_PREC_BF16, 1> : slope_kernel<MG_PREC_FP16, 1>);
            q.launch("slope_kernel", kernel, dim3((unsigned)blocks), 256, 0, a, g, ldg, rows, sums, across, down,
                     packs);
            if (a.db) post.add = AddRowsTask{sums, down, a.n, 1.0f, Count{}, a.db, nullptr, nullptr};
        }
    } else if (go) {
        w.require();
        packs.launch(q);
    }
    if (count > 0) gemm(w, go, a.dtype, jobs, count, post, q);
    if (go) post.launch(a.dtype, q);
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
        Queue q(nullptr);
        linear(*args, w, false, q);
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
        Queue q(stream);
        linear(*args, w, true, q);
    });
}

extern "C" int mg_linear_backward_workspace(const mg_linear_backward_args* args, size_t* bytes) {
    return guarded([&] {
        need(args != nullptr && bytes != nullptr, "args or bytes is null");
        check(*args);
        Workspace w;
        Queue q(nullptr);
        linear_backward(*args, w, false, q);
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
        Queue q(stream);
        linear_backward(*args, w, true, q);
    });
}
