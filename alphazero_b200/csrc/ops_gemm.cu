// 64 x 64 tiles, 4 x 4 outputs per thread, operands of any strides.
#include "ops_gemm.cuh"

namespace mgb {
namespace ops {
namespace {

constexpr int kTile = 64, kStep = 16;

template <int DT>
__global__ void __launch_bounds__(256)
    gemm_kernel(GemmOperand a, GemmOperand b, int64_t m, int64_t n, int64_t k, GemmEpilogue e) {
    using E = Elem<DT>;
    using T = typename E::T;
    __shared__ float sa[kStep][kTile + 1], sb[kStep][kTile + 1];
    const int64_t i0 = (int64_t)blockIdx.x * kTile, j0 = (int64_t)blockIdx.y * kTile;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const T* pa = static_cast<const T*>(a.data);
    const T* pb = static_cast<const T*>(b.data);
    float acc[4][4] = {};
    for (int64_t k0 = 0; k0 < k; k0 += kStep) {
        for (int t = threadIdx.x; t < kTile * kStep; t += 256) {
            const int r = t / kStep, c = t % kStep;
            const int64_t i = i0 + r, j = j0 + r, kk = k0 + c;
            sa[c][r] = i < m && kk < k ? E::get(pa[i * a.row + kk * a.col]) : 0.0f;
            sb[c][r] = j < n && kk < k ? E::get(pb[j * b.row + kk * b.col]) : 0.0f;
        }
        __syncthreads();
        for (int c = 0; c < kStep; ++c)
            for (int r = 0; r < 4; ++r)
                for (int s = 0; s < 4; ++s) acc[r][s] += sa[c][ty * 4 + r] * sb[c][tx * 4 + s];
        __syncthreads();
    }
    const float alpha = e.count ? e.alpha / (float)max(*e.count, 1) : e.alpha;
    for (int r = 0; r < 4; ++r)
        for (int s = 0; s < 4; ++s) {
            const int64_t i = i0 + ty * 4 + r, j = j0 + tx * 4 + s;
            if (i >= m || j >= n) continue;
            float v = acc[r][s] * alpha;
            if (e.bias) v += E::get(static_cast<const T*>(e.bias)[j]);
            if (e.out32) {
                e.out32[i * e.ld + j] = v;
                continue;
            }
            if (e.z) static_cast<T*>(e.z)[i * e.ld + j] = E::put(v);
            v = activate(v, e.act);
            if (e.res)
                v += e.res_scale * E::get(static_cast<const T*>(e.res)[i * e.r_row + j * e.r_col]);
            static_cast<T*>(e.out)[i * e.ld + j] = E::put(v);
        }
}

}  // namespace

void launch_gemm(int dtype, const GemmOperand& a, const GemmOperand& b, int64_t m, int64_t n,
                 int64_t k, const GemmEpilogue& e, cudaStream_t stream) {
    const dim3 grid((unsigned)((m + kTile - 1) / kTile), (unsigned)((n + kTile - 1) / kTile));
    if (dtype == MG_PREC_BF16)
        gemm_kernel<MG_PREC_BF16><<<grid, 256, 0, stream>>>(a, b, m, n, k, e);
    else
        gemm_kernel<MG_PREC_FP16><<<grid, 256, 0, stream>>>(a, b, m, n, k, e);
    launched("gemm_kernel");
}

}  // namespace ops
}  // namespace mgb
