// Linear softmax cross entropy without the logits, with its gradients
// (include/minigo_ops.h).
//
// Rows are taken in pieces: a piece's logits are written to the workspace,
// turned into the row losses and (with gradients) into d, and used up by the
// two products before the next piece overwrites them.
#include "ops_gemm.cuh"

#include <algorithm>
#include <cfloat>
#include <cmath>

namespace mgb {
namespace ops {
namespace {

constexpr size_t kPieceBytes = size_t(512) << 20;  // of logits at a time

__global__ void __launch_bounds__(1024) count_kernel(mg_cross_entropy_args a, int* count) {
    __shared__ int part[32];
    int c = 0;
    for (int64_t i = threadIdx.x; i < a.n; i += 1024)
        c += index_at(a.targets, a.target_bytes, i * a.target_stride, a.vocab) >= 0;
    c = __reduce_add_sync(~0u, c);
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = c;
    __syncthreads();
    if (threadIdx.x < 32) {
        c = __reduce_add_sync(~0u, part[threadIdx.x]);
        if (threadIdx.x == 0) *count = c;
    }
}

// d is kept times 2^14 in fp16, so that small probabilities keep their bits.
template <int DT>
constexpr float kDScale = DT == MG_PREC_FP16 ? 16384.0f : 1.0f;

// One block per row: its loss, and its d.
template <int DT>
__global__ void __launch_bounds__(256)
    row_kernel(mg_cross_entropy_args a, int64_t row0, const float* logits, void* d) {
    using E = Elem<DT>;
    using T = typename E::T;
    __shared__ float sm[256], ss[256];
    const int64_t i = row0 + blockIdx.x;
    const float* l = logits + (int64_t)blockIdx.x * a.vocab;
    T* out = static_cast<T*>(d) + (int64_t)blockIdx.x * a.vocab;
    const int64_t t = index_at(a.targets, a.target_bytes, i * a.target_stride, a.vocab);
    if (t < 0) {
        if (threadIdx.x == 0) a.row_loss[i] = 0.0f;
        if (d)
            for (int64_t v = threadIdx.x; v < a.vocab; v += 256) out[v] = E::put(0.0f);
        return;
    }
    float m = -INFINITY, s = 0.0f;
    for (int64_t v = threadIdx.x; v < a.vocab; v += 256) m = fmaxf(m, l[v]);
    sm[threadIdx.x] = m;
    __syncthreads();
    for (int w = 128; w > 0; w /= 2) {
        if (threadIdx.x < w) sm[threadIdx.x] = fmaxf(sm[threadIdx.x], sm[threadIdx.x + w]);
        __syncthreads();
    }
    m = sm[0];
    const float ref = m == -INFINITY ? 0.0f : m;
    for (int64_t v = threadIdx.x; v < a.vocab; v += 256) s += expf(l[v] - ref);
    ss[threadIdx.x] = s;
    __syncthreads();
    for (int w = 128; w > 0; w /= 2) {
        if (threadIdx.x < w) ss[threadIdx.x] += ss[threadIdx.x + w];
        __syncthreads();
    }
    s = ss[0];
    const float lse = ref + logf(s);
    if (threadIdx.x == 0) a.row_loss[i] = l[t] == -INFINITY ? INFINITY : lse - l[t];
    if (d)
        for (int64_t v = threadIdx.x; v < a.vocab; v += 256) {
            const float p = s == 0.0f ? 0.0f : expf(l[v] - lse);
            out[v] = E::put((p - (v == t ? 1.0f : 0.0f)) * kDScale<DT>);
        }
}

__global__ void __launch_bounds__(1024) loss_kernel(mg_cross_entropy_args a, const int* count) {
    __shared__ float part[1024];
    float s = 0.0f;
    for (int64_t i = threadIdx.x; i < a.n; i += 1024) s += a.row_loss[i];
    part[threadIdx.x] = s;
    __syncthreads();
    for (int w = 512; w > 0; w /= 2) {
        if (threadIdx.x < w) part[threadIdx.x] += part[threadIdx.x + w];
        __syncthreads();
    }
    if (threadIdx.x == 0) *a.loss = part[0] / (float)max(*count, 1);
}

// db = sum of d over the piece's rows, added to what earlier pieces gave.
template <int DT>
__global__ void __launch_bounds__(256)
    column_kernel(int64_t vocab, int64_t rows, const void* d, float* sums, bool first, void* db,
                  float alpha, const int* count) {
    using E = Elem<DT>;
    using T = typename E::T;
    const int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (v >= vocab) return;
    float s = first ? 0.0f : sums[v];
    for (int64_t i = 0; i < rows; ++i) s += E::get(static_cast<const T*>(d)[i * vocab + v]);
    sums[v] = s;
    if (db) static_cast<T*>(db)[v] = E::put(s * alpha / (float)max(*count, 1));
}

// dw = alpha / count * (sums of the pieces).
template <int DT>
__global__ void __launch_bounds__(256)
    weight_kernel(int64_t total, float* sums, const float* piece, bool first, void* dw, float alpha,
                  const int* count) {
    using E = Elem<DT>;
    using T = typename E::T;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const float s = (first ? 0.0f : sums[i]) + piece[i];
    sums[i] = s;
    if (dw) static_cast<T*>(dw)[i] = E::put(s * alpha / (float)max(*count, 1));
}

template <int DT>
void run(const mg_cross_entropy_args& a, Workspace& w, bool go, cudaStream_t s) {
    using T = typename Elem<DT>::T;
    const bool grads = a.dw != nullptr;  // an empty dx may be null
    const int64_t piece = std::min<int64_t>(std::max<int64_t>(a.n, 1),
                                            std::max<int64_t>(1, kPieceBytes / 4 / a.vocab));
    int* count = w.take<int>(4);
    float* logits = w.take<float>((size_t)piece * a.vocab * 4);
    T* d = grads ? w.take<T>((size_t)piece * a.vocab * 2) : nullptr;
    float* sums = grads ? w.take<float>((size_t)a.vocab * 4) : nullptr;
    float* part = grads ? w.take<float>((size_t)a.vocab * a.dim * 4) : nullptr;
    float* total = grads ? w.take<float>((size_t)a.vocab * a.dim * 4) : nullptr;
    if (!go) return;
    w.require();
    count_kernel<<<1, 1024, 0, s>>>(a, count);
    launched("count_kernel");
    const GemmOperand weight{a.weight, a.w_row, a.w_col};
    const float alpha = a.grad_scale / kDScale<DT>;
    if (grads && a.n == 0) {
        check(cudaMemsetAsync(a.dw, 0, (size_t)a.vocab * a.dim * 2, s), "cudaMemsetAsync");
        if (a.db) check(cudaMemsetAsync(a.db, 0, (size_t)a.vocab * 2, s), "cudaMemsetAsync");
    }
    for (int64_t row0 = 0; row0 < a.n; row0 += piece) {
        const int64_t rows = std::min(piece, a.n - row0);
        const bool last = row0 + rows == a.n;
        const T* x = static_cast<const T*>(a.x) + row0 * a.x_row;
        GemmEpilogue e;
        e.bias = a.bias;
        e.out32 = logits;
        e.ld = a.vocab;
        launch_gemm(DT, {x, a.x_row, a.x_col}, weight, rows, a.vocab, a.dim, e, s);
        row_kernel<DT><<<(unsigned)rows, 256, 0, s>>>(a, row0, logits, d);
        launched("row_kernel");
        if (!grads) continue;
        GemmEpilogue ex;
        ex.out = static_cast<T*>(a.dx) + row0 * a.dim;
        ex.ld = a.dim;
        ex.alpha = alpha;
        ex.count = count;
        launch_gemm(DT, {d, a.vocab, 1}, {a.weight, a.w_col, a.w_row}, rows, a.dim, a.vocab, ex, s);
        GemmEpilogue ew;
        ew.out32 = part;
        ew.ld = a.dim;
        launch_gemm(DT, {d, 1, a.vocab}, {x, a.x_col, a.x_row}, a.vocab, a.dim, rows, ew, s);
        weight_kernel<DT><<<(unsigned)((a.vocab * a.dim + 255) / 256), 256, 0, s>>>(
            a.vocab * a.dim, total, part, row0 == 0, last ? a.dw : nullptr, alpha, count);
        launched("weight_kernel");
        column_kernel<DT><<<(unsigned)((a.vocab + 255) / 256), 256, 0, s>>>(
            a.vocab, rows, d, sums, row0 == 0, last ? a.db : nullptr, alpha, count);
        launched("column_kernel");
    }
    loss_kernel<<<1, 1024, 0, s>>>(a, count);
    launched("loss_kernel");
}

void check(const mg_cross_entropy_args& a) {
    const int64_t top = int64_t(1) << 31;
    need(a.n >= 0 && a.vocab >= 1 && a.dim >= 1, "sizes: n >= 0, vocab >= 1, dim >= 1");
    need(a.n < top && a.vocab < top && a.dim < top, "n, vocab and dim must be below 2^31");
    need(a.dtype == MG_PREC_BF16 || a.dtype == MG_PREC_FP16, "dtype must be MG_PREC_BF16 or MG_PREC_FP16");
    need(a.target_bytes == 8 || a.target_bytes == 4, "targets are int64 or int32 (target_bytes 8 or 4)");
    need(a.target_stride >= 0 && a.x_row >= 0 && a.x_col >= 0 && a.w_row >= 0 && a.w_col >= 0,
         "a stride is negative");
    need(a.weight && a.loss, "weight or loss is null");
    need(a.n == 0 || (a.x && a.targets && a.row_loss), "x, targets or row_loss is null");
    const bool grads = a.dx || a.dw || a.db;
    need(!grads || (a.dw && (a.n == 0 || a.dx)), "gradients: give both dx and dw, or neither (and no db)");
    need(!grads || (a.db != nullptr) == (a.bias != nullptr), "db goes with a bias");
}

void cross_entropy(const mg_cross_entropy_args& a, Workspace& w, bool go, cudaStream_t s) {
    if (a.dtype == MG_PREC_BF16) run<MG_PREC_BF16>(a, w, go, s);
    else run<MG_PREC_FP16>(a, w, go, s);
}

}  // namespace
}  // namespace ops
}  // namespace mgb

using namespace mgb::ops;

extern "C" int mg_cross_entropy_workspace(const mg_cross_entropy_args* args, size_t* bytes) {
    return guarded([&] {
        need(args != nullptr && bytes != nullptr, "args or bytes is null");
        check(*args);
        Workspace w;
        cross_entropy(*args, w, false, nullptr);
        *bytes = w.used();
    });
}

extern "C" int mg_cross_entropy(const mg_cross_entropy_args* args, void* workspace,
                                size_t workspace_bytes, void* stream) {
    return guarded([&] {
        need(args != nullptr, "args is null");
        check(*args);
        OnDevice on(args->device);
        Workspace w(workspace, workspace_bytes);
        cross_entropy(*args, w, true, static_cast<cudaStream_t>(stream));
    });
}
