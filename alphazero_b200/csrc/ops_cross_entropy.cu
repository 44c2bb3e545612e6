// Linear softmax cross entropy without the logits, with its gradients
// (include/minigo_ops.h).
//
// Forward: the product's epilogue turns each tile of logits into a maximum
// and a sum per row and block of columns; the logits leave the chip in
// no form.  combine_kernel joins the blocks of a row.  Where there are few
// columns (kRowsColumns) the product's launch has whole rows, and leaves their
// losses and d itself.
//
// With gradients each tile also leaves exp(l - its block's maximum) in 16
// bits (Prob16, ops_gemm.cuh), for a piece of the rows at a time.  Once a
// row's logsumexp is known, d_kernel turns the piece into d in place, and
// two products use it up: dx = d W and dw += d^T x.  So the product x W^T is
// computed once (6 n V D operations in all), where making d from the inputs
// again after the forward pass would compute it twice (8 n V D).
#include "ops_gemm.cuh"

#include <algorithm>
#include <cmath>

namespace mgb {
namespace ops {
namespace {

// Of a piece of the rows' probabilities, or without gradients of its statistics,
// at a time.  Each further piece costs the fp32 sums of dw a trip through memory.
constexpr size_t kPieceBytes = size_t(1) << 30;

// The number of counted rows, per block: only where there are several pieces
// (else combine_kernel counts).
constexpr int kCountBlocks = 148;

__global__ void __launch_bounds__(1024) count_kernel(Indices target, int64_t n, int* counts) {
    griddep_launch_dependents();
    griddep_wait();
    int c = 0;
    for (int64_t i = (int64_t)blockIdx.x * 1024 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 1024)
        c += target.at(i) >= 0;
    c = __reduce_add_sync(~0u, c);
    __shared__ int part[32];
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = c;
    __syncthreads();
    if (threadIdx.x >= 32) return;
    c = __reduce_add_sync(~0u, part[threadIdx.x]);
    if (threadIdx.x == 0) counts[blockIdx.x] = c;
}

// (m, s) of a sum s exp(m) joined with another's.
__device__ __forceinline__ void join(float& m, float& s, float2 p) {
    const float top = fmaxf(m, p.x), ref = top == -INFINITY ? 0.0f : top;
    s = s * exp2f((m - ref) * 1.4426950408889634f) + p.y * exp2f((p.x - ref) * 1.4426950408889634f);
    m = top;
}

// The same of the warp's lanes.
__device__ __forceinline__ void join_lanes(float& m, float& s) {
    float top = m;
#pragma unroll
    for (int d = 16; d > 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
    s *= exp2f((m - (top == -INFINITY ? 0.0f : top)) * 1.4426950408889634f);
#pragma unroll
    for (int d = 16; d > 0; d /= 2) s += __shfl_xor_sync(~0u, s, d);
    m = top;
}

// A row's loss, given that it is counted: log(s exp(m)) - at, the difference of
// large numbers first, so that what is left of it when the target is the
// maximum, log(s), keeps its bits.
__device__ __forceinline__ float loss_of(float m, float s, float at) {
    return at == -INFINITY ? INFINITY : (m - at) + logf(s);
}

// A few rows without gradients: their losses and the mean in one launch, by a
// cluster whose CTAs have two rows each and leave their losses with the first.
// Bound by latency: 7 us for 13 rows of 2364 blocks of columns (65536 classes); a
// block per row and another launch for the mean took longer.
constexpr int kFewRows = 16;

__global__ void __cluster_dims__(kFewRows / 2, 1, 1) __launch_bounds__(1024)
    few_rows_kernel(int rows, int blocks, const float2* part, int64_t part_ld, Indices target, const float* logit,
                    float* row_loss, float* loss) {
    __shared__ float2 sums[32];
    __shared__ float2 losses[kFewRows];  // the first CTA's: a row's loss and 1, or zeros
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, half = warp >> 4;
    const int rank = (int)cluster_rank(), row = rank + half * (kFewRows / 2);
    griddep_launch_dependents();
    cluster_sync();  // all CTAs have begun: their shared memory can be written
    griddep_wait();
    float m = -INFINITY, s = 0.0f;
    if (row < rows)
#pragma unroll 8
        for (int b = threadIdx.x & 511; b < blocks; b += 512) join(m, s, part[(int64_t)b * part_ld + row]);
    join_lanes(m, s);
    if (lane == 0) sums[warp] = make_float2(m, s);
    __syncthreads();
    if ((warp & 15) == 0) {
        const float2 p = lane < 16 ? sums[half * 16 + lane] : make_float2(-INFINITY, 0.0f);
        m = p.x;
        s = p.y;
        join_lanes(m, s);
        if (lane == 0) {
            const bool counted = row < rows && target.at(row) >= 0;
            const float l = counted ? loss_of(m, s, logit[row]) : 0.0f;
            if (row < rows) row_loss[row] = l;
            asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(map_to_rank(smem_u32(&losses[row]), 0)), "f"(l),
                         "f"(counted ? 1.0f : 0.0f)
                         : "memory");
        }
    }
    __syncwarp();
    cluster_sync();
    if (rank > 0 || threadIdx.x > 0) return;
    float all = 0.0f, count = 0.0f;
    for (int r = 0; r < rows; ++r) {
        all += losses[r].x;
        count += losses[r].y;
    }
    *loss = all / fmaxf(count, 1.0f);
}

// Bound by latency: 13 us for 4096 rows of 513 blocks of columns.
// Maximum m and log2 of the sum s of exp(l - m) and the loss per row, and the
// loss summed per block: a thread per row where a row has few blocks of
// columns; with many, 32 threads per row, or where there are few rows too, a
// block per row.  A row of -inf has log2 s = -inf.  counts, if set: the counted rows per block.
enum Combine : int { kThreadPerRow, kWarpPerRow, kBlockPerRow };
constexpr int kFewBlocks = 16;

template <Combine HOW>
__global__ void __launch_bounds__(HOW == kThreadPerRow ? 128 : 1024)
    combine_kernel(int64_t rows, int blocks, const float2* part, int64_t part_ld, Indices target,
                   const float* logit, float2* stat, float* row_loss, float* loss_part, int* counts) {
    constexpr bool FEW = HOW == kThreadPerRow;
    __shared__ float2 tile[FEW ? 1 : 32][33];
    __shared__ float losses[FEW ? 128 : 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    griddep_launch_dependents();
    griddep_wait();
    constexpr int kRows = FEW ? 128 : HOW == kBlockPerRow ? 1 : 32;
    const int64_t row0 = (int64_t)blockIdx.x * kRows;
    const int64_t row = row0 + (FEW ? threadIdx.x : HOW == kBlockPerRow ? 0 : warp);
    float m = -INFINITY, s = 0.0f;
    if constexpr (FEW) {
        if (row < rows)
#pragma unroll 4
            for (int b = 0; b < blocks; ++b) join(m, s, part[(int64_t)b * part_ld + row]);
    } else if constexpr (HOW == kBlockPerRow) {
#pragma unroll 4
        for (int b = threadIdx.x; b < blocks; b += 1024) join(m, s, part[(int64_t)b * part_ld + row]);
        join_lanes(m, s);
        tile[0][warp] = make_float2(m, s);
        __syncthreads();
        m = tile[0][lane].x;
        s = tile[0][lane].y;
        join_lanes(m, s);
    } else {
        // read along the rows, a warp per block of columns in turn; then turned round
        if (row0 + lane < rows)
#pragma unroll 8
            for (int b = warp; b < blocks; b += 32) join(m, s, part[(int64_t)b * part_ld + row0 + lane]);
        tile[warp][lane] = make_float2(m, s);
        __syncthreads();
        m = tile[lane][warp].x;
        s = tile[lane][warp].y;
        join_lanes(m, s);
    }
    float loss = 0.0f;
    bool counted = false;
    if (row < rows) {
        counted = target.at(row) >= 0;
        if (counted) loss = loss_of(m, s, logit[row]);
        if (FEW || lane == 0) {  // (a block per row: every warp has the row, and writes the same)
            stat[row] = make_float2(m, log2f(s));
            row_loss[row] = loss;
        }
    }
    if constexpr (HOW == kBlockPerRow) {
        if (threadIdx.x == 0) {
            loss_part[blockIdx.x] = loss;
            if (counts) counts[blockIdx.x] = counted;
        }
        return;
    }
    losses[FEW ? threadIdx.x : warp] = loss;
    const int all = __syncthreads_count(counted) / (FEW ? 1 : 32);
    if (warp > 0) return;
    loss = 0.0f;
    for (int i = lane; i < kRows; i += 32) loss += losses[i];
#pragma unroll
    for (int d = 16; d > 0; d /= 2) loss += __shfl_xor_sync(~0u, loss, d);
    if (lane == 0) {
        loss_part[blockIdx.x] = loss;
        if (counts) counts[blockIdx.x] = all;
    }
}

// probs (Prob16, per block of `block` columns) -> d = (softmax - onehot) in
// place, and its column sums before rounding per block of rows.  A thread
// has 8 adjacent columns; `wide` of the block's eight warps lie side by side
// (up to 4 KB of a row at once; with one, 512 bytes, the same work took a
// half longer), the others take further rows.  The factor from the
// block's maximum to the row's softmax, exp(m_block - m) / s, is one exp per
// thread and row; near the row's maximum it is exact to the last bits, which
// the difference to one where a target has nearly everything needs.
// Bound by memory: 4096 x 65544 take 213 us, 5 TB/s read and written.
// Block 0 also adds up counts, if set, to count; each step of rows has a block
// that looks for rows whose x would reach dw through d = 0 (CleanRows).
template <int DT>
__global__ void __launch_bounds__(256)
    d_kernel(int rows, int64_t vocab, int block, uint16_t* probs, int64_t ld, const float2* part, int64_t part_ld,
             const float2* stat, Indices target, int wide, int rows_per_block, float* sums, const int* counts,
             int64_t counts_n, int* count, CleanRows clean) {
    using E = Elem<DT>;
    using T = typename E::T;
    __shared__ float acc[8][256];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int deep = 8 / wide, down = warp / wide;
    const int64_t c = ((int64_t)blockIdx.x * wide + warp % wide) * 256 + lane * 8;
    const int r0 = blockIdx.y * rows_per_block, r1 = min(rows, r0 + rows_per_block);
    float sum[8] = {};
    griddep_launch_dependents();
    griddep_wait();
    if (counts != nullptr && blockIdx.x == 0 && blockIdx.y == 0 && warp == 0) {
        int n = 0;
        for (int64_t i = lane; i < counts_n; i += 32) n += counts[i];
        n = __reduce_add_sync(~0u, n);
        if (lane == 0) *count = n;
    }
    const int steps = (rows + kStepRows - 1) / kStepRows, step0 = blockIdx.y * gridDim.x + blockIdx.x;
    const auto is_bad = [&](int g) {
        const int row = g * kStepRows + threadIdx.x;
        return threadIdx.x < kStepRows && row < rows && !isfinite(stat[row].y) && target.at(row) < 0;
    };
    const bool bad = step0 < steps && is_bad(step0);  // its loads are ahead of the others
    if (c < vocab) {
        const float2* mine = part + c / block * part_ld;
        const int64_t step = deep * ld;
        uint16_t* p = probs + (int64_t)(r0 + down) * ld + c;
        const int column = (int)c;
        // four rows at a time, their loads before the first store (which, for
        // all that is known, might be to what they read)
        constexpr int kRows = 4;
        for (int r = r0 + down; r < r1; r += deep * kRows, p += kRows * step) {
            uint4 u[kRows];
            int t[kRows];
            float2 f[kRows];
            float m[kRows];
#pragma unroll
            for (int q = 0; q < kRows; ++q) {
                const int row = r + deep * q;
                if (row >= r1) continue;
                u[q] = *reinterpret_cast<const uint4*>(p + q * step);
                t[q] = target.at(row);
                f[q] = stat[row];
                m[q] = mine[row].x;
            }
#pragma unroll
            for (int q = 0; q < kRows; ++q) {
                if (r + deep * q >= r1) break;
                const uint32_t w[4] = {u[q].x, u[q].y, u[q].z, u[q].w};
                // a row that is not counted (whatever it holds) and one of -inf have no probabilities
                float scale = exp2_flush((m[q] - f[q].x) * 1.4426950408889634f - f[q].y) * 0x1p112f;  // Prob16's
                if (f[q].y == -INFINITY || t[q] < 0) scale = 0.0f;
                float v[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[2 * i] = __uint_as_float((w[i] << 11) & 0x07fff800u) * scale;
                    v[2 * i + 1] = __uint_as_float((w[i] >> 5) & 0x07fff800u) * scale;
                }
                const uint32_t hot = (uint32_t)(t[q] - column);
                if (hot < 8 && t[q] >= 0)
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (hot == i) v[i] -= 1.0f;
                if (sums != nullptr)
#pragma unroll
                    for (int i = 0; i < 8; ++i) sum[i] += v[i];
                alignas(16) T d[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] = E::put(v[i] * kDScale<DT>);
                *reinterpret_cast<uint4*>(p + q * step) = *reinterpret_cast<uint4*>(d);
            }
        }
    }
    for (int g = step0; g < steps; g += gridDim.x * gridDim.y) {
        const bool any = __syncthreads_or(g == step0 ? bad : is_bad(g));
        if (threadIdx.x == 0) clean.use[g] = any;
        if (any) clean_step(clean, g, rows, target, threadIdx.x, 256);
    }
    if (sums == nullptr) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[warp][lane * 8 + i] = sum[i];
    __syncthreads();
    for (int i = threadIdx.x; i < wide * 256; i += 256) {
        const int64_t col = (int64_t)blockIdx.x * wide * 256 + i;
        if (col >= vocab) break;
        float s = 0.0f;
        for (int w = i / 256; w < 8; w += wide) s += acc[w][i % 256];
        sums[(int64_t)blockIdx.y * vocab + col] = s;
    }
}

template <int DT>
void run(const mg_cross_entropy_args& a, Workspace& w, bool go, Queue& q) {
    using T = typename Elem<DT>::T;
    const bool grads = a.dw != nullptr;  // an empty dx may be null
    if (a.n == 0) {
        if (!go) return;
        q.clear(a.loss, 4);
        if (grads) q.clear(a.dw, (size_t)a.vocab * a.dim * 2);
        if (a.db) q.clear(a.db, (size_t)a.vocab * 2);
        return;
    }
    const int64_t ld = (a.vocab + 7) / 8 * 8;
    // pieces of equal length, whole tiles; a block of columns has at least 64 (few rows are one piece)
    const int64_t per = grads ? 2 * ld : 8 * ((a.vocab + 63) / 64);
    const int64_t most = std::max<int64_t>(256, (int64_t)kPieceBytes / per / 256 * 256);
    const int64_t count_pieces = (a.n + most - 1) / most;
    const int64_t piece = std::min(a.n, ((a.n + count_pieces - 1) / count_pieces + 255) / 256 * 256);
    Packs packs;
    StagedOperand x = stage_operand(w, packs, {a.x, a.x_row, a.x_col}, a.n, a.dim);
    const StagedOperand weight = stage_operand(w, packs, {a.weight, a.w_row, a.w_col}, a.vocab, a.dim);
    SoftmaxJob shape;
    shape.a = x;
    shape.b = weight;
    shape.m = piece;
    shape.n = a.vocab;
    shape.k = a.dim;
    const bool rows_whole = gemm_rows_pays(shape, grads);
    const bool few = !grads && !rows_whole && a.n <= kFewRows;
    const SoftmaxBlocks cut = gemm_softmax_blocks(shape, grads);
    const int block = cut.columns, blocks = cut.count;

    Indices target;
    target.data = a.targets;
    target.bytes = a.target_bytes;
    target.stride = a.target_stride;
    target.limit = a.vocab;
    const size_t per_row = rows_whole ? 0 : (size_t)piece * 4;
    float* logit = w.take<float>(per_row);
    float2* stat = w.take<float2>(2 * per_row);
    float2* part = w.take<float2>(blocks * 2 * per_row);
    uint16_t* probs = grads ? w.take<uint16_t>((size_t)piece * ld * 2) : nullptr;
    // a copy of x as x lies, of which few steps are ever written
    StagedOperand other = x;
    other.ld = ((x.mn ? piece : a.dim) + 7) / 8 * 8;
    CleanRows clean;
    if (grads) {
        clean.clean = w.take<uint16_t>((size_t)(x.mn ? a.dim : piece) * other.ld * 2);
        clean.use = w.take<uint16_t>((size_t)(piece + 255) / 256 * (256 / kStepRows) * 2);
    }
    other.data = clean.clean;
    clean.row = x.mn ? 1 : x.ld;
    clean.col = x.mn ? x.ld : 1;
    clean.clean_row = x.mn ? 1 : other.ld;
    clean.clean_col = x.mn ? other.ld : 1;
    clean.dim = a.dim;
    int wide = 1;
    while (wide < 8 && wide * 256 < a.vocab) wide *= 2;
    const int64_t across = (a.vocab + 256 * wide - 1) / (256 * wide);
    // up to eight blocks per SM, at least sixteen rows per warp and block
    const int64_t want = std::max<int64_t>(1, 148 * 8 / across);
    const int down_rows = (int)std::max<int64_t>(128 / wide, (piece + want - 1) / want);
    const int ctas = gemm_rows_ctas(piece);
    const int64_t down = rows_whole ? ctas : (piece + down_rows - 1) / down_rows;  // of a whole piece
    float* sums = a.db ? w.take<float>((size_t)down * a.vocab * 4) : nullptr;
    float* db32 = a.db && count_pieces > 1 ? w.take<float>((size_t)a.vocab * 4) : nullptr;  // of earlier pieces
    const int64_t ld32 = (a.dim + 7) / 8 * 8;
    float* dw32 = grads && count_pieces > 1 ? w.take<float>((size_t)((a.vocab + 255) / 256 * 256) * ld32 * 4) : nullptr;

    const Combine how = blocks <= kFewBlocks ? kThreadPerRow : piece <= 2 * 148 ? kBlockPerRow : kWarpPerRow;
    const int64_t combine_rows = how == kThreadPerRow ? 128 : how == kBlockPerRow ? 1 : 32;
    const int64_t parts = rows_whole ? ctas : (piece + combine_rows - 1) / combine_rows;  // of a piece's loss
    float* loss_part = w.take<float>((size_t)(parts * count_pieces) * 4);
    const bool apart = count_pieces > 1;  // rows counted by a kernel of their own
    const int counts_n = (int)(apart ? std::min<int64_t>(kCountBlocks, (a.n + 1023) / 1024) : parts);
    int* counts = w.take<int>((size_t)counts_n * 4);
    int* total = w.take<int>(4);
    const Count count = rows_whole ? Count{counts, counts_n} : Count{total, 1};
    if (go) {
        w.require();
        packs.launch(q);
        if (apart) q.launch("count_kernel", count_kernel, dim3((unsigned)counts_n), 1024, 0, target, a.n, counts);
    }
    const float alpha = a.grad_scale / kDScale<DT>;
    int64_t losses = 0;
    size_t piece_scratch = 0;
    Post post;
    for (int64_t row0 = 0; row0 < a.n; row0 += piece) {
        const int64_t rows = std::min(piece, a.n - row0);
        const bool first = row0 == 0, last = row0 + rows == a.n;
        StagedOperand xp = x;  // row0 is a multiple of 256: still aligned
        xp.data = static_cast<const uint16_t*>(x.data) + row0 * (x.mn ? 1 : x.ld);
        clean.x = static_cast<const uint16_t*>(xp.data);
        if (go && rows_whole) {
            RowsJob f;
            f.a = xp;
            f.b = weight;
            f.m = rows;
            f.n = a.vocab;
            f.k = a.dim;
            f.e.bias = a.bias;
            f.e.target = target.from(row0);
            f.e.row_loss = a.row_loss + row0;
            f.e.loss = loss_part + losses;
            f.e.counts = apart ? nullptr : counts;
            f.e.d = probs;
            f.e.ld = ld;
            f.e.sums = sums;
            f.e.clean = clean;
            gemm_rows(DT, f, q);
            losses += gemm_rows_ctas(rows);
        } else if (go) {
            SoftmaxJob f;
            f.a = xp;
            f.b = weight;
            f.m = rows;
            f.n = a.vocab;
            f.k = a.dim;
            f.e.bias = a.bias;
            f.e.target = target.from(row0);
            f.e.logit = logit;
            f.e.part = part;
            f.e.part_ld = piece;
            f.e.probs = probs;
            f.e.probs_ld = ld;
            gemm_softmax(DT, f, block, q);
            if (few) {
                q.launch("few_rows_kernel", few_rows_kernel, dim3(kFewRows / 2), 1024, 0, (int)rows, blocks, part, piece, target,
                         logit, a.row_loss, a.loss);
                return;
            }
            const int64_t combine_blocks = (rows + combine_rows - 1) / combine_rows;
            const auto kernel = how == kThreadPerRow  ? combine_kernel<kThreadPerRow>
                                : how == kBlockPerRow ? combine_kernel<kBlockPerRow>
                                                      : combine_kernel<kWarpPerRow>;
            q.launch("combine_kernel", kernel, dim3((unsigned)combine_blocks), how == kThreadPerRow ? 128 : 1024, 0, rows,
                     blocks, part, piece, target.from(row0), logit, stat, a.row_loss + row0, loss_part + losses,
                     apart ? nullptr : counts);
            losses += combine_blocks;
        }
        if (!grads) continue;
        const int64_t these = rows_whole ? gemm_rows_ctas(rows) : (rows + down_rows - 1) / down_rows;
        if (go && !rows_whole) {
            q.launch("d_kernel", d_kernel<DT>, dim3((unsigned)across, (unsigned)these), 256, 0, (int)rows, a.vocab, block,
                     probs, ld, part, piece, stat, target.from(row0), wide, down_rows,
                     sums, first ? counts : nullptr, (int64_t)counts_n, total, clean);
        }
        StagedOperand d;
        d.data = probs;
        d.ld = ld;
        GemmJob jobs[2];
        GemmJob& jx = jobs[0];
        jx.a = d;
        jx.b = transposed(weight);
        jx.m = rows;
        jx.n = a.dim;
        jx.k = a.vocab;
        jx.e.out = static_cast<T*>(a.dx) + row0 * a.dim;
        jx.e.ld = a.dim;
        jx.e.alpha = alpha;
        jx.e.count = count;
        GemmJob& jw = jobs[1];
        jw.a = transposed(d);
        jw.b = transposed(xp);
        jw.use_other = clean.use;
        jw.b_other = transposed(other);
        jw.m = a.vocab;
        jw.n = a.dim;
        jw.k = rows;
        jw.e.ld32 = ld32;
        jw.e.acc32 = first ? nullptr : dw32;
        jw.e.out32 = last ? nullptr : dw32;
        jw.e.out = a.dw;
        jw.e.ld = a.dim;
        jw.e.alpha = alpha;
        jw.e.count = count;
        Workspace again = w;  // every piece's scratch is the same
        gemm(again, go, DT, jobs, 2, post, q);
        if (go) {
            if (sums)
                post.add = AddRowsTask{sums,  these, a.vocab, alpha * kDScale<DT>, count, a.db, first ? nullptr : db32,
                                       last ? nullptr : db32};
            if (!last) post.launch(DT, q);
            continue;
        }
        piece_scratch = std::max(piece_scratch, again.used() - w.used());
    }
    if (!go) {
        w.take(piece_scratch);
        return;
    }
    post.loss = LossTask{loss_part, losses, counts, counts_n, a.loss};
    post.launch(DT, q);
}

void check(const mg_cross_entropy_args& a) {
    const int64_t top = (int64_t(1) << 31) - 1024;  // whole tiles still count in 32 bits
    need(a.n >= 0 && a.vocab >= 1 && a.dim >= 1, "sizes: n >= 0, vocab >= 1, dim >= 1");
    need(a.n < top && a.vocab < top && a.dim < top, "n, vocab and dim must be below 2^31 - 1024");
    need(a.dtype == MG_PREC_BF16 || a.dtype == MG_PREC_FP16, "dtype must be MG_PREC_BF16 or MG_PREC_FP16");
    need(a.target_bytes == 8 || a.target_bytes == 4, "targets are int64 or int32 (target_bytes 8 or 4)");
    need(a.target_stride >= 0 && a.x_row >= 0 && a.x_col >= 0 && a.w_row >= 0 && a.w_col >= 0,
         "a stride is negative");
    need(a.weight && a.loss, "weight or loss is null");
    need(a.n == 0 || (a.x && a.targets && a.row_loss), "x, targets or row_loss is null");
    const bool grads = a.dx || a.dw || a.db;
    need(!grads || (a.dw && (a.n == 0 || a.dx)), "gradients: give both dx and dw, or neither (and no db)");
    need(!grads || (a.db != nullptr) == (a.bias != nullptr), "db goes with a bias");
    need_aligned(a.x, 2, "x");
    need_aligned(a.weight, 2, "weight");
    need_aligned(a.bias, 2, "bias");
    need_aligned(a.targets, a.target_bytes, "targets");
    need_aligned(a.loss, 4, "loss");
    need_aligned(a.row_loss, 4, "row_loss");
    need_aligned(a.dx, 2, "dx");
    need_aligned(a.dw, 2, "dw");
    need_aligned(a.db, 2, "db");
}

void cross_entropy(const mg_cross_entropy_args& a, Workspace& w, bool go, Queue& q) {
    if (a.dtype == MG_PREC_BF16) run<MG_PREC_BF16>(a, w, go, q);
    else run<MG_PREC_FP16>(a, w, go, q);
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
        Queue q(nullptr);
        cross_entropy(*args, w, false, q);
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
        Queue q(stream);
        cross_entropy(*args, w, true, q);
    });
}
