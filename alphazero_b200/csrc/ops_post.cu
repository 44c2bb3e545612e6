// The small launches around the products: copies of operands before them,
// sums after them (ops_gemm.cuh).  What remains after a call's products is one
// launch, since each costs a few us whatever it does (4 for a loss alone, 9
// with 16 splits of a 362 x 256 product and 148 rows of column sums, of which
// most is the latency of its loads).
#include "ops_gemm.cuh"

#include <algorithm>

namespace mgb {
namespace ops {
namespace {

__global__ void __launch_bounds__(256) pack_kernel(Packs packs) {
    griddep_launch_dependents();
    griddep_wait();
    pack_block(packs, blockIdx.x);
}

constexpr int kPostThreads = 1024;
constexpr int kManySplits = 8;  // from here on warps share the splits of a row

// 128 columns of 32 rows, a warp per row and four columns per lane; with
// many splits, of four rows, whose splits eight warps share.
template <int DT>
__device__ __forceinline__ void finish_block(const FinishTask& t, int64_t block, float4* shared) {
    using E = Elem<DT>;
    using T = typename E::T;
    const GemmEpilogue& e = t.e;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int slices = t.splits >= kManySplits ? 8 : 1, rows = 32 / slices;
    const int64_t across = (t.n + 127) / 128;
    const int64_t i = block / across * rows + warp / slices, c = block % across * 128 + lane * 4;
    const int slice = warp % slices;
    const float alpha = scaled_alpha(e.alpha, e.count, lane);
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const bool in = i < t.m && c < t.n;
    if (in)
#pragma unroll 4
        for (int s = slice; s < t.splits; s += slices) {
            const float4 p = *reinterpret_cast<const float4*>(t.part + (s * t.m_pad + i) * t.ld32 + c);
            v.x += p.x, v.y += p.y, v.z += p.z, v.w += p.w;
        }
    if (slices > 1) {
        shared[threadIdx.x] = v;
        __syncthreads();
        if (slice > 0) return;
        for (int s = 1; s < slices; ++s) {
            const float4 p = shared[threadIdx.x + 32 * s];
            v.x += p.x, v.y += p.y, v.z += p.z, v.w += p.w;
        }
    }
    if (!in) return;
    float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        if (c + q >= t.n) break;
        if (e.acc32) x[q] += e.acc32[i * e.ld32 + c + q];
        if (e.out32) {
            e.out32[i * e.ld32 + c + q] = x[q];
            continue;
        }
        float y = x[q] * alpha;
        if (e.bias) y += E::get(static_cast<const T*>(e.bias)[c + q]);
        if (e.z) static_cast<T*>(e.z)[i * e.ld + c + q] = E::put(y);
        y = activate(y, e.act);
        if (e.res) y += e.res_scale * E::get(static_cast<const T*>(e.res)[i * e.r_row + (c + q) * e.r_col]);
        static_cast<T*>(e.out)[i * e.ld + c + q] = E::put(y);
    }
}

// `slices` threads share a column: one where there are few rows, up to 32.
__host__ __device__ inline int add_rows_slices(int64_t rows) { return rows <= 16 ? 1 : rows <= 256 ? 8 : 32; }

template <int DT>
__device__ __forceinline__ void add_rows_block(const AddRowsTask& t, int64_t block, float* shared) {
    const int slices = add_rows_slices(t.rows), columns = kPostThreads / slices;
    const int slice = threadIdx.x / columns, lane = threadIdx.x % columns;
    const int64_t c = block * columns + lane;
    const float alpha = scaled_alpha(t.alpha, t.count, threadIdx.x & 31);
    float s = 0.0f;
    if (c < t.cols)
#pragma unroll 8
        for (int64_t r = slice; r < t.rows; r += slices) s += t.sums[r * t.cols + c];
    if (slices > 1) {
        shared[threadIdx.x] = s;
        __syncthreads();
        s = 0.0f;
        if (slice == 0)
            for (int i = 0; i < slices; ++i) s += shared[i * columns + lane];
    }
    if (slice > 0 || c >= t.cols) return;
    if (t.acc != nullptr) s += t.acc[c];
    if (t.acc_out != nullptr) t.acc_out[c] = s;
    else static_cast<typename Elem<DT>::T*>(t.out)[c] = Elem<DT>::put(s * alpha);
}

__device__ __forceinline__ void loss_block(const LossTask& t, float2* shared) {
    float s = 0.0f;
    int c = 0;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < t.n; i += kPostThreads) s += t.part[i];
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < t.counts_n; i += kPostThreads) c += t.counts[i];
    shared[threadIdx.x] = make_float2(s, __int_as_float(c));
    __syncthreads();
    for (int w = kPostThreads / 2; w > 0; w /= 2) {
        if (threadIdx.x < w) {
            const float2 x = shared[threadIdx.x], y = shared[threadIdx.x + w];
            shared[threadIdx.x] =
                make_float2(x.x + y.x, __int_as_float(__float_as_int(x.y) + __float_as_int(y.y)));
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) *t.loss = shared[0].x / (float)max(__float_as_int(shared[0].y), 1);
}

template <int DT>
__global__ void __launch_bounds__(kPostThreads) post_kernel(Post p) {
    __shared__ float4 shared[kPostThreads];
    griddep_launch_dependents();
    griddep_wait();
    int64_t block = blockIdx.x;
    for (int i = 0; i < 2; ++i) {
        if (i >= p.finishes) break;
        if (block < p.finish[i].blocks) return finish_block<DT>(p.finish[i], block, shared);
        block -= p.finish[i].blocks;
    }
    if (p.loss.loss != nullptr) {
        if (block == 0) return loss_block(p.loss, reinterpret_cast<float2*>(shared));
        --block;
    }
    if (p.add.sums != nullptr) add_rows_block<DT>(p.add, block, reinterpret_cast<float*>(shared));
}

}  // namespace

void Packs::launch(Queue& q) const {
    if (count > 0) q.launch("pack_kernel", pack_kernel, dim3(blocks()), 256, 0, *this);
}

void Post::launch(int dtype, Queue& q) {
    int64_t blocks = 0;
    for (int i = 0; i < finishes; ++i) {
        FinishTask& t = finish[i];
        const int rows = t.splits >= kManySplits ? 4 : 32;
        t.blocks = (t.m + rows - 1) / rows * ((t.n + 127) / 128);
        blocks += t.blocks;
    }
    if (loss.loss != nullptr) ++blocks;
    if (add.sums != nullptr) {
        const int columns = kPostThreads / add_rows_slices(add.rows);
        blocks += (add.cols + columns - 1) / columns;
    }
    if (blocks > 0) {
        need(blocks < (int64_t(1) << 31), "too many blocks");
        q.launch("post_kernel", dtype == MG_PREC_BF16 ? post_kernel<MG_PREC_BF16> : post_kernel<MG_PREC_FP16>,
                 dim3((unsigned)blocks), kPostThreads, 0, *this);
    }
    *this = Post{};
}

}  // namespace ops
}  // namespace mgb
