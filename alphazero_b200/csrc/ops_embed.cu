// Embedding lookup with scaling and its gradient (include/minigo_ops.h).
#include "ops_common.cuh"

#include <algorithm>

namespace mgb {
namespace ops {
namespace {

template <int DT>
__global__ void __launch_bounds__(256) embed_kernel(mg_embed_args a) {
    using E = Elem<DT>;
    using T = typename E::T;
    for (int64_t i = blockIdx.x; i < a.n; i += gridDim.x) {
        const int64_t t = index_at(a.tokens, a.token_bytes, i * a.token_stride, a.vocab);
        const T* row = static_cast<const T*>(a.table) + t * a.table_row;
        T* out = static_cast<T*>(a.out) + i * a.dim;
        for (int64_t c = threadIdx.x; c < a.dim; c += 256)
            out[c] = E::put(t < 0 ? 0.0f : E::get(row[c]) * a.scale);
    }
}

// One block per vocabulary entry, which looks for its tokens.
template <int DT>
__global__ void __launch_bounds__(256) embed_backward_kernel(mg_embed_backward_args a) {
    using E = Elem<DT>;
    using T = typename E::T;
    __shared__ int hits[256];
    for (int64_t v = blockIdx.x; v < a.vocab; v += gridDim.x)
        for (int64_t c0 = 0; c0 < a.dim; c0 += 256) {
            const int64_t c = c0 + threadIdx.x;
            float sum = 0.0f;
            for (int64_t i0 = 0; i0 < a.n; i0 += 256) {
                const int64_t i = i0 + threadIdx.x;
                hits[threadIdx.x] =
                    i < a.n && index_at(a.tokens, a.token_bytes, i * a.token_stride, a.vocab) == v;
                if (__syncthreads_or(hits[threadIdx.x]))
                    for (int j = 0; j < 256; ++j)
                        if (hits[j] && c < a.dim)
                            sum += E::get(static_cast<const T*>(a.grad)[(i0 + j) * a.grad_row + c]);
                __syncthreads();
            }
            if (c < a.dim) static_cast<T*>(a.d_table)[v * a.dim + c] = E::put(sum * a.scale);
        }
}

void check_tokens(const void* p, int bytes, int64_t stride, int64_t n) {
    need(bytes == 8 || bytes == 4, "tokens are int64 or int32 (token_bytes 8 or 4)");
    need(n == 0 || p != nullptr, "tokens is null");
    need(stride >= 0, "token_stride is negative");
}

void check(const mg_embed_args& a) {
    need(a.n >= 0 && a.vocab >= 1 && a.dim >= 1, "sizes: n >= 0, vocab >= 1, dim >= 1");
    need(a.vocab < (int64_t(1) << 31), "vocab must be below 2^31");
    need(a.dtype >= MG_PREC_BF16 && a.dtype <= MG_PREC_FP32, "dtype is not an MG_PREC_* value");
    check_tokens(a.tokens, a.token_bytes, a.token_stride, a.n);
    need(a.table_row >= 0, "table_row is negative");
    need(a.n == 0 || (a.table != nullptr && a.out != nullptr), "table or out is null");
}

void check(const mg_embed_backward_args& a) {
    need(a.n >= 0 && a.vocab >= 1 && a.dim >= 1, "sizes: n >= 0, vocab >= 1, dim >= 1");
    need(a.n < (int64_t(1) << 31) && a.vocab < (int64_t(1) << 31), "n and vocab must be below 2^31");
    need(a.dtype >= MG_PREC_BF16 && a.dtype <= MG_PREC_FP32, "dtype is not an MG_PREC_* value");
    check_tokens(a.tokens, a.token_bytes, a.token_stride, a.n);
    need(a.grad_row >= 0, "grad_row is negative");
    need(a.d_table != nullptr && (a.n == 0 || a.grad != nullptr), "grad or d_table is null");
}

template <int DT>
void embed(const mg_embed_args& a, cudaStream_t s) {
    embed_kernel<DT><<<(unsigned)std::min<int64_t>(a.n, 1 << 20), 256, 0, s>>>(a);
    launched("embed_kernel");
}

template <int DT>
void embed_backward(const mg_embed_backward_args& a, cudaStream_t s) {
    embed_backward_kernel<DT><<<(unsigned)std::min<int64_t>(a.vocab, 1 << 20), 256, 0, s>>>(a);
    launched("embed_backward_kernel");
}

}  // namespace
}  // namespace ops
}  // namespace mgb

using namespace mgb::ops;

extern "C" int mg_embed(const mg_embed_args* args, void* stream) {
    return guarded([&] {
        need(args != nullptr, "args is null");
        check(*args);
        if (args->n == 0) return;
        OnDevice on(args->device);
        auto s = static_cast<cudaStream_t>(stream);
        if (args->dtype == MG_PREC_BF16) embed<MG_PREC_BF16>(*args, s);
        else if (args->dtype == MG_PREC_FP16) embed<MG_PREC_FP16>(*args, s);
        else embed<MG_PREC_FP32>(*args, s);
    });
}

extern "C" int mg_embed_backward_workspace(const mg_embed_backward_args* args, size_t* bytes) {
    return guarded([&] {
        need(args != nullptr && bytes != nullptr, "args or bytes is null");
        check(*args);
        *bytes = 0;
    });
}

extern "C" int mg_embed_backward(const mg_embed_backward_args* args, void* workspace,
                                 size_t workspace_bytes, void* stream) {
    return guarded([&] {
        need(args != nullptr, "args is null");
        check(*args);
        OnDevice on(args->device);
        auto s = static_cast<cudaStream_t>(stream);
        if (args->dtype == MG_PREC_BF16) embed_backward<MG_PREC_BF16>(*args, s);
        else if (args->dtype == MG_PREC_FP16) embed_backward<MG_PREC_FP16>(*args, s);
        else embed_backward<MG_PREC_FP32>(*args, s);
    });
}
