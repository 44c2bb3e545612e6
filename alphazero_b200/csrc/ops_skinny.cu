// Products of up to 16 rows: y = x W^T with few tokens, where the time is the
// one read of W.
//
// W's rows are the M side of mma.sync.m16n8k16 and the tokens its N side, so
// no work is padded beyond 8 tokens; the products are far from the limit of
// even these instructions.  A contraction may run in any order as long as
// both operands agree, so a lane takes 8 consecutive elements of a row in one
// 16-byte load and lets them stand for the element pairs that the fragment
// layout wants from two steps: W goes from memory to the tensor cores through
// registers alone, kAhead steps at a time, past L1, where x stays.  65536 rows
// of 2048: 41 us for one token, 43 for 8 (95% of the copy rate), 53 for 13,
// where x's loads are as many as W's and warps wait for both.  (For 13 tokens
// a queue through shared memory by cp.async, with blocks that go on to further
// rows without draining it, took 73 us; steps loaded one by one as others are
// used up, 72; 32 rows per warp, which halve x's loads, 54, but 64 instead of
// 56 for 16384 rows of 8192.)
//
// A warp has 16 rows of W; up to eight warps share 16 rows, each with a part
// of K, and add up in shared memory in a fixed order: short blocks, so that
// the card is full from the first wave to the last.  (On CTA pairs, tiles of
// 256 x BN with 13 rows in use take 75 us: the tensor work is 16 times as
// much.)
#include "ops_gemm.cuh"

#include <algorithm>
#include <cmath>

namespace mgb {
namespace ops {
namespace {

struct SkinnyArgs {
    const uint16_t* x;  // [m][k], row stride ldx
    const uint16_t* w;  // [n][k], row stride ldw
    int64_t ldx, ldw;
    int m, n, k;
    int share;   // warps per 16 rows
    int k_part;  // of K per warp, a multiple of 32
    GemmEpilogue e;
    SoftmaxEpilogue s;
};

// 8 elements of a row from k on, zeros past its end.
__device__ __forceinline__ uint4 load8(const uint16_t* row, int k, int end) {
    if (k >= end) return make_uint4(0, 0, 0, 0);
    if (k + 8 <= end) return __ldg(reinterpret_cast<const uint4*>(row + k));
    uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (k + i < end) v[i / 2] |= (uint32_t)row[k + i] << (i & 1 ? 16 : 0);
    return make_uint4(v[0], v[1], v[2], v[3]);
}

// Of W, which is read once: no place in L1, where x stays.
__device__ __forceinline__ uint4 load_once(const uint16_t* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}

template <int DT>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    if constexpr (DT == MG_PREC_BF16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The epilogue of W's rows [n0, n0 + rows), whose parts are in `sums`.
template <int DT, int TOKENS, bool SOFTMAX>
__device__ __forceinline__ void finish(const SkinnyArgs& a, const float (&sums)[128][TOKENS + 1], int n0, int rows,
                                       int group) {
    using E = Elem<DT>;
    using T = typename E::T;
    const auto total = [&](int r, int token) {  // of row r of the block
        float v = 0.0f;
        for (int p = 0; p < a.share; ++p) v += sums[(r / 16 * a.share + p) * 16 + r % 16][token];
        return v;
    };
    if constexpr (SOFTMAX) {
        const SoftmaxEpilogue& e = a.s;
        // 256 / TOKENS lanes per token, each with every so many-th column
        constexpr int kLanes = 256 / TOKENS, kEach = 128 / kLanes;
        const int token = threadIdx.x / kLanes, first = threadIdx.x % kLanes;
        const int target = token < a.m ? e.target.at(token) : -1;
        float l[kEach], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int r = first + kLanes * i, col = n0 + r;
            l[i] = -INFINITY;
            if (r < rows && col < a.n) {
                l[i] = total(r, token) + (e.bias ? E::get(static_cast<const T*>(e.bias)[col]) : 0.0f);
                if (col == target) e.logit[token] = l[i];
            }
            top = fmaxf(top, l[i]);
        }
#pragma unroll
        for (int d = kLanes / 2; d > 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
        const float ref = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int r = first + kLanes * i;
            if (r >= rows) break;
            l[i] = exp2f((l[i] - ref) * 1.4426950408889634f);
            sum += l[i];
            if (e.probs != nullptr && token < a.m && n0 + r < a.n)
                e.probs[token * e.probs_ld + n0 + r] = (uint16_t)prob16(l[i]);
        }
#pragma unroll
        for (int d = kLanes / 2; d > 0; d /= 2) sum += __shfl_xor_sync(~0u, sum, d);
        if (first == 0 && token < a.m) e.part[(int64_t)group * e.part_ld + token] = make_float2(top, sum);
    } else {
        const GemmEpilogue& e = a.e;
        const float alpha = e.alpha;
        for (int i = threadIdx.x; i < rows * a.m; i += 256) {
            const int r = i % rows, token = i / rows;
            const int64_t col = n0 + r;
            if (col >= a.n) continue;
            float v = total(r, token) * alpha;
            if (e.bias) v += E::get(static_cast<const T*>(e.bias)[col]);
            if (e.z) static_cast<T*>(e.z)[token * e.ld + col] = E::put(v);
            v = activate(v, e.act);
            if (e.res) v += e.res_scale * E::get(static_cast<const T*>(e.res)[token * e.r_row + col * e.r_col]);
            static_cast<T*>(e.out)[token * e.ld + col] = E::put(v);
        }
    }
}

// TILES: tokens in eights.  SOFTMAX: statistics of the block's columns, else
// the linear layer's epilogue.
template <int DT, int TILES, bool SOFTMAX>
__global__ void __launch_bounds__(256, 3) skinny_kernel(SkinnyArgs a) {
    constexpr int kTokens = 8 * TILES;
    constexpr int kAhead = 4;  // steps of 32 elements of K whose W is in flight per warp
    __shared__ float sums[128][kTokens + 1];  // [warp * 16 + row][token]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int part = warp % a.share, rows = 128 / a.share;
    const int n0 = blockIdx.x * rows;
    griddep_launch_dependents();
    griddep_wait();
    const int row = n0 + warp / a.share * 16 + g;
    const int begin = part * a.k_part, end = min(a.k, begin + a.k_part);
    const uint16_t* w0 = a.w + (int64_t)min(row, a.n - 1) * a.ldw;
    const uint16_t* w1 = a.w + (int64_t)min(row + 8, a.n - 1) * a.ldw;
    const uint16_t* x[TILES];
#pragma unroll
    for (int i = 0; i < TILES; ++i) x[i] = a.x + (int64_t)min(8 * i + g, a.m - 1) * a.ldx;
    float c[TILES][4] = {};
    const auto multiply = [&](int i, uint4 u0, uint4 u1, uint4 v) {
        mma16816<DT>(c[i], u0.x, u1.x, u0.y, u1.y, v.x, v.y);
        mma16816<DT>(c[i], u0.z, u1.z, u0.w, u1.w, v.z, v.w);
    };
    int k = begin + 8 * t;
    for (; k - 8 * t + 32 * kAhead <= end; k += 32 * kAhead) {
        uint4 u0[kAhead], u1[kAhead];
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
            u0[q] = load_once(w0 + k + 32 * q);
            u1[q] = load_once(w1 + k + 32 * q);
        }
#pragma unroll
        for (int q = 0; q < kAhead; ++q)
#pragma unroll
            for (int i = 0; i < TILES; ++i)
                multiply(i, u0[q], u1[q], __ldg(reinterpret_cast<const uint4*>(x[i] + k + 32 * q)));
    }
    for (; k - 8 * t < end; k += 32) {
        const uint4 u0 = load8(w0, k, end), u1 = load8(w1, k, end);
#pragma unroll
        for (int i = 0; i < TILES; ++i) multiply(i, u0, u1, load8(x[i], k, end));
    }
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
        sums[warp * 16 + g][8 * i + 2 * t] = c[i][0];
        sums[warp * 16 + g][8 * i + 2 * t + 1] = c[i][1];
        sums[warp * 16 + g + 8][8 * i + 2 * t] = c[i][2];
        sums[warp * 16 + g + 8][8 * i + 2 * t + 1] = c[i][3];
    }
    __syncthreads();
    finish<DT, kTokens, SOFTMAX>(a, sums, n0, rows, blockIdx.x);
}

template <class Job>
SkinnyArgs lay_out(const Job& j) {
    SkinnyArgs a{};
    a.x = static_cast<const uint16_t*>(j.a.data);
    a.w = static_cast<const uint16_t*>(j.b.data);
    a.ldx = j.a.ld;
    a.ldw = j.b.ld;
    a.m = (int)j.m;
    a.n = (int)j.n;
    a.k = (int)j.k;
    return a;
}

// Warps per 16 rows: as many as have at least four steps of K each.
int share_of(int64_t k) {
    int share = 1;
    while (share < 8 && k > share * 128) share *= 2;
    return share;
}

template <bool SOFTMAX>
void launch(int dtype, SkinnyArgs& a, Queue& q) {
    a.k_part = ((a.k + a.share - 1) / a.share + 31) / 32 * 32;
    const int rows = 128 / a.share;
    const dim3 grid((unsigned)((a.n + rows - 1) / rows));
    const bool bf = dtype == MG_PREC_BF16;
    const auto kernel = a.m <= 8 ? (bf ? skinny_kernel<MG_PREC_BF16, 1, SOFTMAX> : skinny_kernel<MG_PREC_FP16, 1, SOFTMAX>)
                                 : (bf ? skinny_kernel<MG_PREC_BF16, 2, SOFTMAX> : skinny_kernel<MG_PREC_FP16, 2, SOFTMAX>);
    q.launch("skinny_kernel", kernel, grid, 256, 0, a);
}

// ---- nine to sixteen tokens, many rows of W ----
//
// W's rows are the M side of tcgen05.mma (128 per tile) and the tokens its N
// side; both come to shared memory by TMA, so that neither L1 nor the issue of
// loads limits the one read of W: up to kStages steps of it are on their way
// per SM.  A thread of the four epilogue warps has a row of W and all tokens;
// tiles alternate between two halves of the TMEM.  Tiles have as many
// rows as give every SM the same number of them (an SM reads about 65 GB/s
// alone, so a last round on some is no faster than one on all); what the
// other rows of the products hold is not used.  CTAs begin at different steps
// of k, so that they do not all ask for the same piece of x.  65536 rows of
// 2048 and 13 tokens: 46 us, 90% of the rate of a plain copy.

constexpr int kTileRows = 128, kTileTokens = 16, kStepK = 64, kChunks = 2, kStages = 5;  // a stage has kChunks of kStepK
constexpr uint32_t kWBytes = kTileRows * kStepK * 2, kXBytes = kTileTokens * kStepK * 2, kStageBytes = kChunks * (kWBytes + kXBytes);
// A stage's eight products each add to sums of their own: the tensor cores cut
// their running sums, so long chains come out too small (ops_gemm.cu).
constexpr int kSums = kChunks * kStepK / 16;
constexpr int kStreamThreads = 32 * 6;
constexpr int kStreamSmem = kStages * kStageBytes + (2 * kStages + 5) * 8 + 16;

struct alignas(64) StreamArgs {
    CUtensorMap tw, tx;
    int m, n, steps, tiles;
    int rows;    // of W per tile, up to kTileRows
    int groups;  // of 32 columns or fewer, SOFTMAX
    GemmEpilogue e;
    SoftmaxEpilogue s;
    int* err;
};

// The lane's row of W is column `col`, past the warp's part if it is not
// below `end`; v: its sums, per token.
template <int DT, bool SOFTMAX>
__device__ __forceinline__ void stream_epilogue(const StreamArgs& a, float (&v)[kTileTokens], int col, int end,
                                                int group, int target, int lane) {
    using E = Elem<DT>;
    using T = typename E::T;
    if constexpr (SOFTMAX) {
        const SoftmaxEpilogue& e = a.s;
        const float bias = e.bias != nullptr && col < end ? E::get(static_cast<const T*>(e.bias)[col]) : 0.0f;
        float2 mine = make_float2(-INFINITY, 0.0f);  // lane i: token i's
#pragma unroll
        for (int t = 0; t < kTileTokens; ++t) {
            if (t >= a.m) break;
            const float l = col < end ? v[t] + bias : -INFINITY;
            if (col == __shfl_sync(~0u, target, t) && col < end) e.logit[t] = l;
            float top = l;
#pragma unroll
            for (int d = 16; d > 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
            const float p = exp2f((l - (top == -INFINITY ? 0.0f : top)) * 1.4426950408889634f);
            if (e.probs != nullptr && col < end) e.probs[t * e.probs_ld + col] = (uint16_t)prob16(p);
            float sum = p;
#pragma unroll
            for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(~0u, sum, d);
            if (lane == t) mine = make_float2(top, sum);
        }
        if (lane < a.m && group < a.groups) e.part[(int64_t)group * e.part_ld + lane] = mine;
    } else {
        const GemmEpilogue& e = a.e;
        if (col >= end) return;
        const float bias = e.bias != nullptr ? E::get(static_cast<const T*>(e.bias)[col]) : 0.0f;
#pragma unroll
        for (int t = 0; t < kTileTokens; ++t) {
            if (t >= a.m) break;
            float y = v[t] * e.alpha + bias;
            if (e.z) static_cast<T*>(e.z)[t * e.ld + col] = E::put(y);
            y = activate(y, e.act);
            if (e.res) y += e.res_scale * E::get(static_cast<const T*>(e.res)[t * e.r_row + col * e.r_col]);
            static_cast<T*>(e.out)[t * e.ld + col] = E::put(y);
        }
    }
}

template <int DT, bool SOFTMAX>
__global__ void __launch_bounds__(kStreamThreads, 1) stream_kernel(const __grid_constant__ StreamArgs a) {
    extern __shared__ __align__(1024) uint8_t ring[];
    uint64_t* full = reinterpret_cast<uint64_t*>(ring + kStages * kStageBytes);  // a stage has landed
    uint64_t* empty = full + kStages;                                            // its products are complete
    uint64_t* tfull = empty + kStages;                                           // [2] a tile's sums are complete
    uint64_t* tempty = tfull + 2;                                                // [2] they have been read
    uint64_t* done = tempty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(smem_u32(&full[s]), 1);
            mbar_init(smem_u32(&empty[s]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&tfull[i]), 1);
            mbar_init(smem_u32(&tempty[i]), 4);
        }
        mbar_init(smem_u32(done), 1);
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_slot), 2 * kSums * kTileTokens);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    griddep_launch_dependents();
    griddep_wait();

    if (warp == 0) {
        int s = 0, round = 0;
        int64_t used = 0;
        bool ok = true;
        for (int tile = blockIdx.x; ok && tile < a.tiles; tile += gridDim.x)
            for (int k = 0; k < a.steps; ++k) {
                if (!mbar_wait_warp(smem_u32(&empty[s]), (round & 1) ^ 1, a.err, kErrWaitProducer)) {
                    ok = false;
                    break;
                }
                const uint32_t at = smem_u32(ring + s * kStageBytes), bar = smem_u32(&full[s]);
                const int from = (k + (int)blockIdx.x) % a.steps * kChunks;
                if (elect_one()) {
                    mbar_arrive_expect_tx(bar, kChunks * (a.rows * kStepK * 2 + kXBytes));
#pragma unroll
                    for (int i = 0; i < kChunks; ++i) {
                        tma_load_2d(at + i * kWBytes, &a.tw, bar, (from + i) * kStepK, tile * a.rows);
                        tma_load_2d(at + kChunks * kWBytes + i * kXBytes, &a.tx, bar, (from + i) * kStepK, 0);
                    }
                }
                ++used;
                if (++s == kStages) {
                    s = 0;
                    ++round;
                }
            }
        // every load has landed before this CTA ends
        for (int i = 0; i < kStages && i < used; ++i) {
            if (--s < 0) {
                s = kStages - 1;
                --round;
            }
            mbar_wait_warp(smem_u32(&full[s]), round & 1, a.err, kErrWaitDrain);
        }
    } else if (warp == 1) {
        constexpr uint32_t idesc = idesc_f16(kTileRows, kTileTokens, DT == MG_PREC_BF16);
        const uint64_t w0 = smem_desc_sw128(smem_u32(ring)), x0 = smem_desc_sw128(smem_u32(ring) + kChunks * kWBytes);
        int s = 0, round = 0, count = 0;
        bool ok = true;
        for (int tile = blockIdx.x; ok && tile < a.tiles; tile += gridDim.x, ++count) {
            const int buf = count & 1;
            if (!mbar_wait_warp(smem_u32(&tempty[buf]), ((count >> 1) & 1) ^ 1, a.err, kErrWaitMma)) break;
            tc_fence_after();
            for (int k = 0; k < a.steps; ++k) {
                if (!mbar_wait_warp(smem_u32(&full[s]), round & 1, a.err, kErrWaitMma)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint64_t w = w0 + s * (kStageBytes >> 4), x = x0 + s * (kStageBytes >> 4);
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < kSums; ++kk)
                        mma_f16(tmem_base + (buf * kSums + kk) * kTileTokens, w + kk / 4 * (kWBytes >> 4) + kk % 4 * 2,
                                x + kk / 4 * (kXBytes >> 4) + kk % 4 * 2, idesc, k > 0);
                    mma_commit(smem_u32(&empty[s]));
                    if (k + 1 == a.steps) mma_commit(smem_u32(&tfull[buf]));
                }
                if (++s == kStages) {
                    s = 0;
                    ++round;
                }
            }
        }
        // products still in flight finish before TMEM is freed
        if (elect_one()) mma_commit(smem_u32(done));
        mbar_wait_warp(smem_u32(done), 0, a.err, kErrWaitDrain);
    } else {
        const int quarter = warp & 3, parts = (a.rows + 31) / 32;  // of a tile, a warp each
        const int target = SOFTMAX && lane < a.m ? a.s.target.at(lane) : -1;
        int count = 0;
        for (int tile = blockIdx.x; tile < a.tiles; tile += gridDim.x, ++count) {
            const int buf = count & 1;
            if (!mbar_wait_warp(smem_u32(&tfull[buf]), (count >> 1) & 1, a.err, kErrWaitEpilogue)) break;
            tc_fence_after();
            float v[kTileTokens] = {};
#pragma unroll
            for (int i = 0; i < kSums; ++i) {
                uint32_t r[kTileTokens];
                tmem_ld_16cols(tmem_base + (buf * kSums + i) * kTileTokens + ((uint32_t)quarter << 21), r);
                tmem_ld_wait(r);
#pragma unroll
                for (int t = 0; t < kTileTokens; ++t) v[t] += __uint_as_float(r[t]);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&tempty[buf]));
            const int first = tile * a.rows + quarter * 32, end = min(a.n, (tile + 1) * a.rows);
            if (quarter < parts) stream_epilogue<DT, SOFTMAX>(a, v, first + lane, end, tile * parts + quarter, target, lane);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem_base, 2 * kSums * kTileTokens);
}

// Rows of W per tile: as many as give each SM as many tiles.
int stream_rows(int64_t n) {
    const int64_t rounds = (n + 148 * kTileRows - 1) / (148 * kTileRows);
    return (int)((n + 148 * rounds - 1) / (148 * rounds));
}
// In us, this way and by the kernel above, 9 and 16 tokens, rows of W x k:
// 65536 x 2048 46 and 48, 54 and 56; 16384 x 8192 46 and 47, 57 and 58; 131072
// x 1000 50 and 51, 74 and 83; 19072 x 2048 17 and 18, 17 and 18; 8192 x 2048
// 10 and 11, 11 and 11; 16384 x 512 7 and 8, 8 and 8; 4096 x 4096 15 and 16, 10
// and 10 (tiles of few rows: a step's latency).
bool streams(int64_t m, int64_t n, int64_t k) { return m > 8 && n >= 148 * 64 && n * k >= int64_t(1) << 25; }

template <bool SOFTMAX, class Job>
void stream(int dtype, const Job& j, int rows, StreamArgs& a, Queue& q) {
    a.rows = rows;
    encode_operand(&a.tw, dtype, j.b, j.n, j.k, rows);
    encode_operand(&a.tx, dtype, j.a, j.m, j.k, kTileTokens);
    a.m = (int)j.m;
    a.n = (int)j.n;
    a.steps = (int)((j.k + kChunks * kStepK - 1) / (kChunks * kStepK));
    a.tiles = (int)((j.n + rows - 1) / rows);
    a.err = op_status_word();
    const auto kernel = dtype == MG_PREC_BF16 ? stream_kernel<MG_PREC_BF16, SOFTMAX> : stream_kernel<MG_PREC_FP16, SOFTMAX>;
    check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kStreamSmem),
          "cudaFuncSetAttribute(stream_kernel)");
    q.launch("stream_kernel", kernel, dim3((unsigned)std::min(a.tiles, 148)), kStreamThreads, kStreamSmem, a);
}

}  // namespace

SoftmaxBlocks skinny_blocks(int64_t m, int64_t n, int64_t k, bool even) {
    if (!streams(m, n, k)) return {128 / share_of(k), (int)((n * share_of(k) + 127) / 128)};
    if (even) return {32, (int)((n + 31) / 32)};
    const int rows = stream_rows(n);
    return {0, (int)((n + rows - 1) / rows) * ((rows + 31) / 32)};
}

void skinny(int dtype, const GemmJob& j, Queue& q) {
    if (streams(j.m, j.n, j.k)) {
        StreamArgs s{};
        s.e = j.e;
        return stream<false>(dtype, j, stream_rows(j.n), s, q);
    }
    SkinnyArgs a = lay_out(j);
    a.e = j.e;
    a.share = share_of(a.k);
    launch<false>(dtype, a, q);
}

void skinny_softmax(int dtype, const SoftmaxJob& j, int block, Queue& q) {
    if (streams(j.m, j.n, j.k)) {
        StreamArgs s{};
        s.s = j.e;
        s.groups = skinny_blocks(j.m, j.n, j.k, block > 0).count;
        return stream<true>(dtype, j, block > 0 ? kTileRows : stream_rows(j.n), s, q);
    }
    SkinnyArgs a = lay_out(j);
    a.s = j.e;
    a.share = share_of(a.k);
    launch<true>(dtype, a, q);
}

}  // namespace ops
}  // namespace mgb
