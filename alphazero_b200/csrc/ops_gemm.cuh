// Matrix products of the training operators: C[i][j] = sum_k A[i][k] B[j][k]
// in bf16 or fp16 with 32-bit sums, with a fused epilogue.
#pragma once

#include "ops_common.cuh"

namespace mgb {
namespace ops {

// Element (i, k) is at data[i * row + k * col].
struct GemmOperand {
    const void* data;
    int64_t row, col;
};

// An operand a TMA map can describe: 16-byte aligned, one unit stride, the
// other (ld) a multiple of 8.  mn: the unit stride runs along i, not k.
struct StagedOperand {
    const void* data = nullptr;
    int64_t ld = 0;
    bool mn = false;
};

// A number that earlier kernels left in n parts.
struct Count {
    const int* parts = nullptr;
    int n = 0;
};
// Its sum, to every lane of the calling warp.
__device__ __forceinline__ int count_total(const Count& c, int lane) {
    int s = 0;
#pragma unroll 4
    for (int i = lane; i < c.n; i += 32) s += c.parts[i];
    return __reduce_add_sync(~0u, s);
}

// z = alpha * acc + bias; out = act(z) + res_scale * res, both 16-bit.
struct GemmEpilogue {
    const void* bias = nullptr;      // [n]
    const void* res = nullptr;       // [m][n]
    int64_t r_row = 0, r_col = 0;
    void* out = nullptr;             // [m][n], row stride ld
    void* z = nullptr;               // [m][n], row stride ld
    // acc + acc32 in fp32, row stride ld32 (a multiple of 8), and nothing
    // else; room for m rounded up to 256 rows
    float* out32 = nullptr;
    const float* acc32 = nullptr;    // fp32 sums of earlier pieces, added to acc
    int64_t ld = 0, ld32 = 0;
    float res_scale = 0.0f;
    int act = MG_ACT_NONE;
    float alpha = 1.0f;
    Count count;                     // if set, alpha is divided by max(count, 1)
};
// To be called by whole warps.
__device__ __forceinline__ float scaled_alpha(float alpha, const Count& count, int lane) {
    return count.parts != nullptr ? alpha / (float)max(count_total(count, lane), 1) : alpha;
}

// Steps of 64 elements of the contraction, in which a product may take an
// operand from somewhere else.
constexpr int kStepRows = 64;

struct GemmJob {
    StagedOperand a, b;
    int64_t m = 0, n = 0, k = 0;
    GemmEpilogue e;
    // If set, per step of k: whether it is to be read from b_other, a matrix
    // like b, instead.
    const uint16_t* use_other = nullptr;
    StagedOperand b_other;
};

// Rows of x that are not counted have d = 0, which leaves them out of
// dw = d^T x unless they hold an infinity or NaN.  The kernel that knows
// the rows' softmax sees such a row by its logits (one that is not finite
// makes every logit an infinity or NaN, so the row's sum of exponentials is
// NaN or zero) and copies its step of rows with zeros in place of the rows
// that are not counted; dw's product reads that step from the copy.
struct CleanRows {
    const uint16_t* x = nullptr;
    int64_t row = 0, col = 0;
    uint16_t* clean = nullptr;
    int64_t clean_row = 0, clean_col = 0;
    uint16_t* use = nullptr;  // [steps], or as bytes per 32 rows: not zero where the copy is to be read
    int64_t dim = 0;
};

// One step's copy, by `count` threads (whole warps): a warp per row, 16 bytes
// per lane where rows lie along x (a StagedOperand's are 16-byte aligned).
// Small code, since kernels carry it that hardly ever run it: 32768 rows of 256,
// 362 classes take 99 us instead of 54 where 3% of the rows are NaN and not counted.
__device__ __forceinline__ void clean_step(const CleanRows& c, int step, int rows, const Indices& target, int thread,
                                           int count) {
    const int lane = thread & 31, first = step * kStepRows, end = min(first + kStepRows, rows);
    const bool along = c.col == 1;
#pragma unroll 1
    for (int i = first + thread / 32; i < end; i += count / 32) {
        const bool keep = target.at(i) >= 0;
        const uint16_t* const in = c.x + i * c.row;
        uint16_t* const out = c.clean + i * c.clean_row;
        int64_t j = lane;
        if (along) {
#pragma unroll 1
            for (j = lane * 8; j + 8 <= c.dim; j += 256) {
                const uint4 v = __ldg(reinterpret_cast<const uint4*>(in + j));
                *reinterpret_cast<uint4*>(out + j) = keep ? v : make_uint4(0, 0, 0, 0);
            }
            j = c.dim / 8 * 8 + lane;
        }
#pragma unroll 1
        for (; j < c.dim; j += 32) out[j * c.clean_col] = keep ? in[j * c.col] : 0;
    }
}

// Products of up to this many rows, both operands K-major, are bound by
// reading B once: they take a kernel of their own (ops_skinny.cu).
constexpr int kSkinnyRows = 16;

// Softmax statistics of l = acc + bias instead of a product (the forward
// half of the cross entropy).  A row's columns are taken in blocks
// (gemm_softmax_blocks()); per block and row
//   part[block * part_ld + row] = (max, sum of exp(l - max)),
// (-inf, 0) for a block of -inf; logit[row] = l at the row's target; and, if
// probs is set, probs[row * probs_ld + col] = exp(l - max) as a Prob16.
struct SoftmaxEpilogue {
    const void* bias = nullptr;       // [n]
    Indices target;                   // [m]
    float* logit = nullptr;           // [m]
    float2* part = nullptr;
    int64_t part_ld = 0;
    uint16_t* probs = nullptr;
    int64_t probs_ld = 0;             // a multiple of 8, at least n
};
struct SoftmaxJob {
    StagedOperand a, b;
    int64_t m = 0, n = 0, k = 0;
    SoftmaxEpilogue e;
};
// d is kept times 2^14 in fp16, so that small probabilities keep their bits.
template <int DT>
constexpr float kDScale = DT == MG_PREC_FP16 ? 16384.0f : 1.0f;

struct SoftmaxBlocks {
    int columns;  // of each, or 0: some number (not to be used with probs)
    int count;
};
// The blocks of the largest job that shares part's layout; even: all have
// the same number of columns.
SoftmaxBlocks gemm_softmax_blocks(const SoftmaxJob& job, bool even);
// `columns` of those.
void gemm_softmax(int dtype, const SoftmaxJob& job, int columns, Queue& q);

// The same, whole rows at a time, where n is small: the sums of 256 rows and
// up to kRowsColumns columns stay in TMEM until the rows' softmax is known,
// which then leaves the chip as d = (softmax - onehot) * kDScale.  Each of
// the gemm_rows_ctas(m) CTAs also leaves its rows' summed loss, how many of
// them are counted and the column sums of d / kDScale before its rounding.
constexpr int kRowsColumns = 512;
struct RowsEpilogue {
    const void* bias = nullptr;    // [n]
    Indices target;                // [m]
    float* row_loss = nullptr;     // [m]
    float* loss = nullptr;         // [ctas]
    int* counts = nullptr;         // [ctas], or null
    uint16_t* d = nullptr;         // [m][n], row stride ld; null: no gradient
    int64_t ld = 0;                // a multiple of 8
    float* sums = nullptr;         // [ctas][n], or null
    CleanRows clean;               // with d
};
struct RowsJob {
    StagedOperand a, b;
    int64_t m = 0, n = 0, k = 0;
    RowsEpilogue e;
};
bool gemm_rows_pays(const SoftmaxJob& job, bool grads);
int gemm_rows_ctas(int64_t m);
void gemm_rows(int dtype, const RowsJob& job, Queue& q);

void skinny(int dtype, const GemmJob& job, Queue& q);
SoftmaxBlocks skinny_blocks(int64_t m, int64_t n, int64_t k, bool even);
void skinny_softmax(int dtype, const SoftmaxJob& job, int block, Queue& q);

// The tensor map of an operand of rows x k, in boxes of tile_rows (at most 64
// where it lies along its rows) x 64.
void encode_operand(CUtensorMap* map, int dtype, const StagedOperand& s, int64_t rows, int64_t k, int tile_rows);

// A number in [0, 1] in 16 bits: 4 bits of exponent and 12 of fraction, no
// sign (relative error 2^-14 from 2^-14 up, absolute 2^-28 below).  A block's
// largest is 1, so the range is where the block's probabilities are, and the
// rounding is far below the one to bf16 or fp16 that follows, down to 2^-19 of the
// block's largest; what is below 2^-29 of it is lost.  It is an fp32 value scaled
// by 2^-112, whose exponent then has four bits, cut to its top 16 bits below the
// exponent's fourth: bits << 11, times 2^112.
__device__ __forceinline__ uint32_t prob16(float v) {
    return (__float_as_uint(v * 0x1p-112f) + 0x400u) >> 11;
}
// Two of them in one word.  (The byte permutation is written out: as shifts
// and an or, nvcc 12.9 -O3 drops the high half.)
__device__ __forceinline__ uint32_t prob16x2(float low, float high) {
    return __byte_perm(prob16(low), prob16(high), 0x5410);
}

// Copies of operands that do not lie right, made by blocks of the kernel that
// comes first in a call (a launch of their own would cost as much as the
// copy).  Lines of `len` elements (strides line, step) become lines of ld.
struct PackTask {
    const uint16_t* in;
    uint16_t* out;
    int64_t line, step, lines, len, ld;
    int blocks;
};
struct Packs {
    PackTask task[3];
    int count = 0;
    int blocks() const {
        int n = 0;
        for (int i = 0; i < count; ++i) n += task[i].blocks;
        return n;
    }
    void launch(Queue& q) const;  // on their own, if there are any
};

// The share of block `block` (0 .. blocks() - 1): a warp per line and 512
// columns, 16 bytes per lane and store.
__device__ __forceinline__ void pack_block(const Packs& packs, int block) {
    int i = 0;
    while (block >= packs.task[i].blocks) block -= packs.task[i++].blocks;
    const PackTask& t = packs.task[i];
    const int warps = blockDim.x >> 5;
    const int64_t across = (t.len + 511) / 512, tasks = t.lines * across;
    const int64_t line = t.line, len = t.len, step = t.step, ld = t.ld, span = (t.lines - 1) * line + len;
    const uint16_t* const in = t.in;
    uint16_t* const out = t.out;
    for (int64_t at = (int64_t)block * warps + (threadIdx.x >> 5); at < tasks; at += (int64_t)t.blocks * warps) {
        const int64_t r = at / across, c = at % across * 512 + (threadIdx.x & 31) * 8;
        uint4 v[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int64_t col = c + 256 * k;
            if (col >= len) continue;
            if (step == 1) {
                v[k] = load8_unaligned(in + r * line + col, r * line + col, span);
            } else {
                uint32_t h[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) h[e] = col + e < len ? in[r * line + (col + e) * step] : 0;
                v[k] = make_uint4(__byte_perm(h[0], h[1], 0x5410), __byte_perm(h[2], h[3], 0x5410),
                                  __byte_perm(h[4], h[5], 0x5410), __byte_perm(h[6], h[7], 0x5410));
            }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (c + 256 * k < len) *reinterpret_cast<uint4*>(out + r * ld + c + 256 * k) = v[k];
    }
}

// What is left to do after the products of a call, in one launch: products
// whose K was split are summed and given their epilogue, partial column sums
// are added up, and the cross entropy's loss is.
struct FinishTask {
    const float* part;
    int splits;
    int64_t m_pad, m, n, ld32;
    GemmEpilogue e;
    int64_t blocks;
};
// s[c] = acc[c] (if set) + the sum of `rows` rows of sums, in a fixed order:
// out[c] = alpha / max(count, 1) * s[c], or instead acc_out[c] = s[c].
struct AddRowsTask {
    const float* sums;
    int64_t rows, cols;
    float alpha;
    Count count;
    void* out;
    const float* acc;
    float* acc_out;
};
struct LossTask {  // loss = sum of part[0 .. n) / max(sum of counts[0 .. counts_n), 1)
    const float* part;
    int64_t n;
    const int* counts;
    int64_t counts_n;
    float* loss;
};
struct Post {
    FinishTask finish[2];
    int finishes = 0;
    AddRowsTask add{};   // sums set: to do
    LossTask loss{};     // loss set: to do
    void launch(int dtype, Queue& q);  // if there is anything, which is then done
};

// Gives an operand of `rows` x k in a form the products read: itself where
// it lies right, else a copy in the workspace, to be made by `packs`.
StagedOperand stage_operand(Workspace& w, Packs& packs, const GemmOperand& op, int64_t rows, int64_t k);
// The same matrix with i and k exchanged.
inline StagedOperand transposed(StagedOperand s) {
    s.mn = !s.mn;
    return s;
}

// One or two products in one launch (the one with more k first); `post` gets
// what then remains to be done.
void gemm(Workspace& w, bool go, int dtype, GemmJob* jobs, int count, Post& post, Queue& q);

// 2^x; below 2^-126, 0.
__device__ __forceinline__ float exp2_flush(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 1 / x to a unit or two in the last place, for 1 <= x (0 at infinity).
__device__ __forceinline__ float reciprocal(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Phi(z), the normal distribution function, and exp(-z^2 / 2): formula
// 7.1.26 of Abramowitz and Stegun for erf(|z| / sqrt 2), which is within
// 1.5e-7 and needs one exponential that GELU's slope shares.
__device__ __forceinline__ float normal_cdf(float z, float* bell) {
    const float t = reciprocal(fmaf(0.3275911f * 0.70710678118654752f, fabsf(z), 1.0f));
    float p = fmaf(0.5f * 1.061405429f, t, 0.5f * -1.453152027f);
    p = fmaf(p, t, 0.5f * 1.421413741f);
    p = fmaf(p, t, 0.5f * -0.284496736f);
    p = fmaf(p, t, 0.5f * 0.254829592f);
    *bell = exp2_flush(z * -0.72134752044448170f * z);
    const float tail = p * t * *bell;
    return z < 0.0f ? tail : 1.0f - tail;
}
// 1 / (1 + exp(-z)).
__device__ __forceinline__ float logistic(float z) { return reciprocal(1.0f + exp2_flush(z * -1.4426950408889634f)); }

__device__ __forceinline__ float activate(float z, int act) {
    float bell;
    switch (act) {
        case MG_ACT_RELU: asm("max.NaN.f32 %0, %0, 0f00000000;" : "+f"(z)); return z;  // NaN stays
        case MG_ACT_SILU: return z * logistic(z);
        case MG_ACT_GELU: return z * normal_cdf(z, &bell);
        default: return z;
    }
}

}  // namespace ops
}  // namespace mgb
