// Tensor-core products of the training operators on pairs of SMs.
//
// C = A B^T by tiles of 256 x BN (BN 256 or 128), a CTA pair
// (tcgen05, cta_group::2) per tile: each CTA holds 128 rows of A, half of
// the BN rows of B and 128 x BN fp32 sums in TMEM, so a K step of 64 moves
// 16 + BN / 16 KB per CTA for 128 x BN x 64 multiply-adds.  One CTA with a
// 128 x 256 tile of its own would move 48 KB for the same work: more than
// L2 gives 148 SMs at the tensor cores' rate.
//
// Either operand may lie along k (K-major) or along its own rows (MN-major):
// TMA writes both with the 128-byte swizzle, and the instruction and matrix
// descriptors say which, so the gradients' products read x, the weight and
// g where they are, with no transposing pass.
//
// Warps of each CTA (persistent over its tiles):
//   warp 0     TMA producer (one thread), a ring of kStages K steps
//   warp 1     TMEM; in the even CTA also the MMA issuer (one thread)
//   warps 2-9  epilogue: warp w reads TMEM lanes 32 (w % 4) .. + 31 (a thread
//              owns a row) and half of the columns, 64 at a time, through
//              swizzled blocks of shared memory that TMA stores (and, for the
//              residual, loads a chunk ahead, past the end of a tile).  Short
//              products are bound by these stores: the card writes 3.6 TB/s
//              (torch's zero_), 5100 cycles for an SM's 128 x 256 sums, and an
//              epilogue without a residual takes 5600; a lane's own 16-byte
//              stores to 32 rows at once took 14000
// The sums are double-buffered in TMEM: a tile's epilogue overlaps the next
// tile's products.  Every wait is bounded (ptx_sm100.cuh).
//
// Long products are bound by the tensor cores, and in a loop, as any such
// product, by the power cap: 8192 x 4096 x 4096 with GELU 210 us a call in a loop,
// 1.31 PFLOP/s (a profiled launch by itself 175, with the tensor pipe 86% active);
// 16384 x 4096 x 4096 with GELU, residual and z kept 500, 1.10 (one call after a
// pause 424, 1.30).  A product with 256 elements to a sum is bound by its
// epilogue: 184832 x 256 x 256 with a residual 66 us, 4.3 TB/s, without it 45.
#include "ops_gemm.cuh"

#include <algorithm>
#include <cmath>
#include <cudaTypedefs.h>

namespace mgb {
namespace ops {
namespace {

// Where sums end in 32 bits (the losses), K steps that the tensor cores add up
// on their own.  They cut off what does not fit a sum, so a chain of products
// comes out too small by about 1e-9 of itself for each of its elements; sums
// of such chains are rounded to nearest.  Losses of 2000 rows of 4096, 8000
// classes: off by 6e-7 of themselves as one chain, 1.5e-7 by 16 steps, 8e-8 by
// 8; 4096 rows of 2048, 65536 classes take 700, 702 and 723 us.
constexpr int kChain = 16;
constexpr int kRowsCta = 128;          // rows of a tile per CTA
constexpr int kRowsPair = 256;
constexpr int kBK = kStepRows;         // K elements per stage
constexpr int kPairs = 74;             // of SMs on a B200 (148)
constexpr int kGroup = 8;              // row tiles walked together (their B tiles stay in L2)
constexpr int kBlockBytes = 4096;      // 32 rows of 128 bytes: 64 columns of 16 bits or 32 of fp32
constexpr int kWarpBytes = 2 * kBlockBytes;  // per epilogue warp

enum Epi : int { kStore, kSoftmax, kRows };

template <int BN>
struct Config {
    static constexpr int kEpiWarps = 8;
    static constexpr int kStages = BN == 256 ? 5 : 6;
    static constexpr uint32_t kABytes = kRowsCta * kBK * 2;
    static constexpr uint32_t kBBytes = BN / 2 * kBK * 2;
    static constexpr uint32_t kStageBytes = kABytes + kBBytes;
    static constexpr int kCols = BN / 2;  // of a tile per epilogue warp
    static constexpr int kBarriers = 2 * kStages + 9 + 2 * kEpiWarps;
    // ring + per epilogue warp its blocks and 16-bit bias + barriers + TMEM address
    static constexpr int kSmem = kStages * kStageBytes + kEpiWarps * (kWarpBytes + kCols * 2) + kBarriers * 8 + 16;
    static_assert(kSmem <= 232448, "shared memory of an SM");
};

// kRows has 16 epilogue warps (its time is theirs: with eight, two per
// scheduler, it took 28 us instead of 25 for 32768 rows of 256 and 362
// columns), a stage less and more shared memory of their own: per warp two
// blocks of 32 x 32 16-bit elements and, in 32 bits, the bias, sums and counts
// of its columns (32 of every 128), per CTA the exchange of row statistics
// ([2][4][128] float2), the barriers for that and each warp's loss and count.
template <int EPI>
constexpr int kEpiWarps = EPI == kRows ? 16 : 8;
template <int EPI>
constexpr int kThreads = 32 * (2 + kEpiWarps<EPI>);
constexpr int kRowsColumnsWarp = kRowsColumns / 4;
constexpr int kRowsStages = Config<128>::kStages - 1;
constexpr int kRowsBlock = 2048;
constexpr int kRowsWarpBytes = 2 * kRowsBlock + kRowsColumnsWarp * 12;
constexpr int kRowsStats = 2 * 4 * kRowsCta * 8;
constexpr int kRowsSmem = kRowsStages * Config<128>::kStageBytes + kEpiWarps<kRows> * (kRowsWarpBytes + 16) + kRowsStats +
                          Config<128>::kBarriers * 8 + 16;
static_assert(kRowsSmem <= 232448, "shared memory of an SM");

struct JobArgs {
    int m, n, kblocks;
    int tiles_m, tiles_n, splits, kb_split;
    int a_mn, b_mn;
    int by_tma;  // outputs, z and residual go through their tensor maps
    int m_pad;   // rows of out32 per split
    int across;  // kRows: column tiles of a unit
    int chain;   // kSoftmax: K steps whose products add up in TMEM
    const uint16_t* use_other;  // GemmJob's
    GemmEpilogue e;
    SoftmaxEpilogue s;
    RowsEpilogue r;
};

struct alignas(64) KernelArgs {
    CUtensorMap ta[2], tb[2];
    CUtensorMap to[2];   // out, out32 or probs
    CUtensorMap tz, tr;  // z and residual of job 0
    CUtensorMap tb_other;  // of the job with use_other
    JobArgs job[2];
    int units[2];
    int head_start;  // units of job 1 that a pair does while others finish their last unit of job 0
    int* err;
};

// The units of a pair: job 0's round robin, then job 1's, handed out in the
// order in which the pairs come free (pairs with one unit of job 0 fewer
// start head_start units of job 1 earlier).  Index i of job 0 and of job 1,
// or -1 when the pair has no more of that job.
struct UnitWalk {
    int pairs, p, n0, n1, extra, ahead;
    __device__ UnitWalk(const KernelArgs& a, int pair, int total) : pairs(total), p(pair) {
        n0 = a.units[0];
        n1 = a.units[1];
        extra = n0 % pairs;
        ahead = extra ? a.head_start : 0;
    }
    __device__ __forceinline__ int unit(int job, int i) const {
        if (job == 0) {
            const int u = p + i * pairs;
            return u < n0 ? u : -1;
        }
        const int early = pairs - extra;
        int u = ahead * early + i * pairs + p;
        if (p >= extra) u = i < ahead ? i * early + (p - extra) : u - ahead * pairs;
        return u < n1 ? u : -1;
    }
};

// Where a job's units lie.  The job's sizes are read once into registers:
// a kernel parameter under a variable index is a load, and so are they
// after every asm statement that may touch memory.
struct Tiling {
    int tiles, tiles_m, per, full, splits, kb_split, kblocks;
    float inv_tiles, inv_per, inv_full, inv_last;
    __device__ explicit Tiling(const JobArgs& j) {
        tiles_m = j.tiles_m;
        tiles = j.tiles_m * j.tiles_n;
        per = kGroup * j.tiles_n;
        full = tiles_m / kGroup;  // groups of kGroup row tiles
        splits = j.splits;
        kb_split = j.kb_split;
        kblocks = j.kblocks;
        inv_tiles = 1.0f / tiles;
        inv_per = 1.0f / per;
        inv_full = 1.0f / kGroup;
        inv_last = 1.0f / max(1, tiles_m % kGroup);
    }
};

// n / d for 0 <= n < 2^24, with inv = 1 / d; the remainder stays in n.
__device__ __forceinline__ int divide(int& n, int d, float inv) {
    int q = (int)(__int2float_rn(n) * inv);
    n -= q * d;
    if (n < 0) {
        n += d;
        --q;
    }
    if (n >= d) {
        n -= d;
        ++q;
    }
    return q;
}

struct Tile {
    int m0, n0, kb0, kb1, split;
    __device__ __forceinline__ Tile(const Tiling& j, int unit, int bn) {
        split = j.splits > 1 ? divide(unit, j.tiles, j.inv_tiles) : 0;
        const int group = divide(unit, j.per, j.inv_per);
        const bool last = group >= j.full;
        const int column = divide(unit, last ? j.tiles_m - j.full * kGroup : kGroup, last ? j.inv_last : j.inv_full);
        m0 = (group * kGroup + unit) * kRowsPair;
        n0 = column * bn;
        kb0 = split * j.kb_split;
        kb1 = min(kb0 + j.kb_split, j.kblocks);
    }
};

template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (DT == MG_PREC_BF16) {
        __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<uint32_t*>(&h);
    } else {
        __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<uint32_t*>(&h);
    }
}
template <int DT>
__device__ __forceinline__ float2 unpack2(uint32_t u) {
    if constexpr (DT == MG_PREC_BF16) return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&u));
    else return __half22float2(*reinterpret_cast<__half2*>(&u));
}

// Byte offset of 16-byte piece q of row r in a block of 128-byte rows as TMA
// swizzles it.
__device__ __forceinline__ uint32_t swizzle128(int r, int q) { return r * 128 + ((q ^ (r & 7)) << 4); }

// An epilogue warp's two blocks of shared memory, used in turn.  A residual
// block lands where the result is then written: each lane replaces its own
// row.
struct WarpBlocks {
    uint8_t* blocks;   // [2][4096]
    uint64_t* landed;  // [2] a residual block has arrived
    int lane;
    int next = 0;        // block of the next chunk of columns
    uint32_t phase = 0;  // bit b: parity of landed[b]
    int flying = 0;      // residual blocks on their way

    __device__ __forceinline__ uint8_t* at(int b) const { return blocks + b * kBlockBytes; }
    // At most N of the warp's stores still read shared memory.
    template <int N>
    __device__ __forceinline__ void settle() {
        if (lane == 0) bulk_wait_read_n<N>();
        __syncwarp();
    }
    // Lane's 32 columns of 16 bits, the first (h = 0) or second half of block b.
    template <class Words>
    __device__ __forceinline__ void write16(int b, int h, Words word) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *reinterpret_cast<uint4*>(at(b) + swizzle128(lane, 4 * h + q)) =
                make_uint4(word(4 * q), word(4 * q + 1), word(4 * q + 2), word(4 * q + 3));
    }
    __device__ __forceinline__ void write32(int b, const float (&v)[32]) {
#pragma unroll
        for (int q = 0; q < 8; ++q)
            *reinterpret_cast<float4*>(at(b) + swizzle128(lane, q)) =
                make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
    }
    // Starts the store of block b.
    __device__ __forceinline__ void store(int b, const CUtensorMap* map, int col, int row) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
            tma_store_2d(map, smem_u32(at(b)), col, row);
            bulk_commit();
        }
    }
    // A chunk's residual into block b (settled), and the wait for it.
    __device__ __forceinline__ void start_res(int b, const CUtensorMap* map, int col, int row) {
        if (lane == 0) {
            const uint32_t bar = smem_u32(&landed[b]);
            mbar_arrive_expect_tx(bar, kBlockBytes);
            tma_load_2d(smem_u32(at(b)), map, bar, col, row);
        }
        ++flying;
    }
    __device__ __forceinline__ bool wait_res(int b, int* err, int code) {
        const bool ok = mbar_wait_warp(smem_u32(&landed[b]), phase >> b & 1, err, code);
        phase ^= 1u << b;
        --flying;
        return ok;
    }
};

// A block from or to a matrix that no tensor map describes (any strides and
// alignment): a row at a time, so that the warp's accesses are in order.
__device__ __forceinline__ void load_rows(uint8_t* block, const uint16_t* p, int64_t row, int64_t col, int rows,
                                          int cols, int lane) {
    __syncwarp();
#pragma unroll 8
    for (int r = 0; r < 32; ++r)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int c = lane + 32 * k;
            if (r < rows && c < cols)
                *reinterpret_cast<uint16_t*>(block + swizzle128(r, c >> 3) + (c & 7) * 2) = p[r * row + c * col];
        }
    __syncwarp();
}

// Two elements per lane; rows that begin off a 4-byte boundary are shifted by
// one element between the lanes, and their first and last go on their own.
__device__ __forceinline__ void store_row(uint16_t* q, uint32_t w, bool odd, int cols, int lane) {
    const int c = 2 * lane;
    if (!odd) {
        if (c + 1 < cols) *reinterpret_cast<uint32_t*>(q + c) = w;
        else if (c < cols) q[c] = (uint16_t)w;
        return;
    }
    const uint32_t up = __byte_perm(w, __shfl_down_sync(~0u, w, 1), 0x5432);  // elements c + 1, c + 2
    if (c + 2 < cols) *reinterpret_cast<uint32_t*>(q + c + 1) = up;
    // of an even number of columns the last one's place is its lane's second
    const bool last = c + 2 == cols;
    if (lane == 0 || last) q[last && lane > 0 ? c + 1 : 0] = (uint16_t)(last && lane > 0 ? w >> 16 : w);
    if (lane == 0 && last) q[1] = (uint16_t)(w >> 16);
}

__device__ __forceinline__ void store_rows(const uint8_t* block, uint16_t* p, int64_t row, int rows, int cols,
                                           int lane) {
    __syncwarp();
    const bool odd = (reinterpret_cast<uintptr_t>(p) & 2) != 0, turns = (row & 1) != 0;  // from row to row
    const uint32_t at = smem_u32(block) + (lane & 3) * 4;
    const auto word = [&](int r) {
        uint32_t w;
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(at + swizzle128(r, lane >> 2)));
        return w;
    };
    if (rows == 32 && cols == 64) {
#pragma unroll 4
        for (int r = 0; r < 32; r += 2, p += 2 * row) {
            const uint32_t w0 = word(r), w1 = word(r + 1);
            store_row(p, w0, odd, 64, lane);
            store_row(p + row, w1, odd != turns, 64, lane);
        }
        return;
    }
    for (int r = 0; r < rows; ++r, p += row) store_row(p, word(r), odd != (turns && (r & 1)), cols, lane);
}

__device__ __forceinline__ void activate_all(float (&v)[32], int act) {
    if (act == MG_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = activate(v[i], MG_ACT_RELU);
    } else if (act == MG_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = activate(v[i], MG_ACT_SILU);
    } else if (act == MG_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = activate(v[i], MG_ACT_GELU);
    }
}

// v = v * alpha + bias of 32 columns.
template <int DT>
__device__ __forceinline__ void add_bias(float (&v)[32], float alpha, const uint16_t* sbias) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const uint4 u = *reinterpret_cast<const uint4*>(sbias + q * 8);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 b = unpack2<DT>(w[i]);
            v[q * 8 + 2 * i] = fmaf(v[q * 8 + 2 * i], alpha, b.x);
            v[q * 8 + 2 * i + 1] = fmaf(v[q * 8 + 2 * i + 1], alpha, b.y);
        }
    }
}

// What a warp's epilogue needs of a job, in registers.
struct EpilogueJob {
    int m, n, m_pad, act;
    bool by_tma, has_z, has_res, has_acc32, has_out32;
    float alpha, res_scale;
    __device__ EpilogueJob(const JobArgs& j, int lane) {
        const GemmEpilogue& e = j.e;
        m = j.m;
        n = j.n;
        m_pad = j.m_pad;
        act = e.act;
        by_tma = j.by_tma != 0;
        has_z = e.z != nullptr;
        has_res = e.res != nullptr;
        has_acc32 = e.acc32 != nullptr;
        has_out32 = e.out32 != nullptr;
        alpha = scaled_alpha(e.alpha, e.count, lane);
        res_scale = e.res_scale;
    }
};

// Columns [n0 + c0, + kCols) of rows [m0, + 32) of a finished tile, whose
// sums are given back by `release` as soon as they are in registers.  False
// if a wait gave up.
// The residual's block after the tile's last starts at column after_col (-1:
// there is none) of row after_row.
template <int BN, int DT, class Release>
__device__ __forceinline__ bool epilogue(const KernelArgs& a, int job, const EpilogueJob& j, const Tile& t, int m0,
                                         int c0, uint32_t taddr, WarpBlocks& blocks, const uint16_t* sbias,
                                         int after_col, int after_row, Release release) {
    const GemmEpilogue& e = a.job[job].e;
    const int rows = min(32, j.m - m0), lane = blocks.lane;
    const int width = rows > 0 ? min(Config<BN>::kCols, j.n - t.n0 - c0) : 0;
    if (width <= 0) release();
#pragma unroll 1
    for (int c = 0; c < width; c += 32) {
        const int col = t.n0 + c0 + c, h = c >> 5 & 1;
        const bool ends = h == 1 || c + 32 >= width;  // of a chunk of 64 columns
        const int cols = min(64, width - c);
        if (!j.has_out32 && h == 0) {
            if (!j.by_tma) {
                blocks.settle<0>();
                if (j.has_res)
                    load_rows(blocks.at(blocks.next), static_cast<const uint16_t*>(e.res) + m0 * e.r_row + col * e.r_col,
                              e.r_row, e.r_col, rows, cols, lane);
            } else if (j.has_z) {
                blocks.settle<0>();
            } else if (j.has_res) {
                if (!blocks.wait_res(blocks.next, a.err, kErrWaitEpilogue)) return false;
                blocks.settle<0>();  // the chunk before's store, a chunk ago
                if (c + 64 < width) blocks.start_res(blocks.next ^ 1, &a.tr, col + 64, m0);
                else if (after_col >= 0) blocks.start_res(blocks.next ^ 1, &a.tr, after_col, after_row);
            } else {
                blocks.settle<1>();
            }
        }
        uint32_t r[32];
        tmem_ld_32cols(taddr + c, r);
        tmem_ld_wait();
        if (c + 32 >= width) release();
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
        if (j.has_acc32 && lane < rows) {
            const float* p = e.acc32 + (int64_t)(m0 + lane) * e.ld32 + col;
            uint32_t u[32];
#pragma unroll
            for (int q = 0; q < 4; ++q)  // ld32 is a multiple of 8
                if (c + q * 8 < width) ld_once_v8(p + q * 8, u + q * 8);
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (c + i / 8 * 8 < width) v[i] += __uint_as_float(u[i]);
        }
        if (j.has_out32) {
            blocks.settle<1>();
            blocks.write32(blocks.next, v);
            blocks.store(blocks.next, &a.to[job], col, t.split * j.m_pad + m0);
            blocks.next ^= 1;
            continue;
        }
        add_bias<DT>(v, j.alpha, sbias + c);
        const auto word = [&](int i) { return pack2<DT>(v[2 * i], v[2 * i + 1]); };
        const int col64 = col - 32 * h;
        if (j.has_z) blocks.write16(blocks.next ^ 1, h, word);
        activate_all(v, j.act);
        if (j.has_res) {
            uint4 u[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (!(j.has_z && j.by_tma))
                    u[q] = *reinterpret_cast<const uint4*>(blocks.at(blocks.next) + swizzle128(lane, 4 * h + q));
                else if (lane < rows && c + 8 * q < width)
                    u[q] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(e.res) +
                                                                (int64_t)(m0 + lane) * e.r_row + col + 8 * q));
                else
                    u[q] = make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint32_t w[4] = {u[q].x, u[q].y, u[q].z, u[q].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 f = unpack2<DT>(w[i]);
                    v[q * 8 + 2 * i] += j.res_scale * f.x;
                    v[q * 8 + 2 * i + 1] += j.res_scale * f.y;
                }
            }
        }
        blocks.write16(blocks.next, h, word);
        if (!ends) continue;
        if (j.by_tma) {
            if (j.has_z) blocks.store(blocks.next ^ 1, &a.tz, col64, m0);
            blocks.store(blocks.next, &a.to[job], col64, m0);
        } else {
            const int64_t at = (int64_t)m0 * e.ld + col64;
            const int stored = min(64, width - (c - 32 * h));
            if (j.has_z) store_rows(blocks.at(blocks.next ^ 1), static_cast<uint16_t*>(e.z) + at, e.ld, rows, stored, lane);
            store_rows(blocks.at(blocks.next), static_cast<uint16_t*>(e.out) + at, e.ld, rows, stored, lane);
        }
        blocks.next ^= 1;
    }
    return true;
}

// As tmem_ld_32cols into floats.
__device__ __forceinline__ void tmem_ld_32cols_to(uint32_t taddr, float* v) {
    uint32_t r[32];
    tmem_ld_32cols(taddr, r);
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
// No use of v moves above this point (it is loaded asynchronously until the
// wait before).
__device__ __forceinline__ void pin(float (&v)[32]) {
#pragma unroll
    for (int i = 0; i < 32; ++i) asm volatile("" : "+f"(v[i]));
}

// Softmax statistics of the same columns and rows.  A thread has its row's
// block to itself, in registers, so the maximum and the sum need no exchange.
// The tile's sums come in `parts`, which are added here.
template <int BN, int DT, class Wait, class Release, class Address>
__device__ __forceinline__ bool softmax_epilogue(const KernelArgs& a, const SoftmaxEpilogue& e, int m, int n,
                                                 const Tile& t, int m0, int c0, int target, WarpBlocks& blocks,
                                                 const uint16_t* sbias, int parts, Wait wait, Release release,
                                                 Address address) {
    const int row = m0 + blocks.lane;
    const int first = t.n0 + c0;
    constexpr int W = Config<BN>::kCols;
    const int width = m0 < m ? min(W, n - first) : 0;
    target -= first;
    float l[W];
    for (int p = 0; p < parts; ++p) {
        if (!wait(p)) return false;
        const uint32_t taddr = address(p);
        if (p == 0) {
#pragma unroll
            for (int c = 0; c < W; c += 32)
                if (c < width) tmem_ld_32cols_to(taddr + c, l + c);
            tmem_ld_wait();
#pragma unroll
            for (int c = 0; c < W; c += 32) pin(*reinterpret_cast<float(*)[32]>(l + c));
        } else {
#pragma unroll
            for (int c = 0; c < W; c += 16) {
                if (c >= width) break;
                uint32_t r[16];
                tmem_ld_16cols(taddr + c, r);
                tmem_ld_wait(r);
#pragma unroll
                for (int i = 0; i < 16; ++i) l[c + i] += __uint_as_float(r[i]);
            }
        }
        release(p);
    }
    if (width <= 0) return true;
    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, logit = 0.0f;
#pragma unroll
    for (int c = 0; c < W; c += 32) {
        if (c >= width) break;
        float(&v)[32] = *reinterpret_cast<float(*)[32]>(l + c);
        add_bias<DT>(v, 1.0f, sbias + c);  // -inf past the last column
#pragma unroll
        for (int i = 0; i < 32; ++i) top[i & 3] = fmaxf(top[i & 3], v[i]);
        if (__any_sync(~0u, target >= c && target < c + 32)) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (target == c + i) logit = v[i];
        }
    }
    const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
    const float ref = most == -INFINITY ? 0.0f : most;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < W; c += 32) {
        if (c >= width) break;
        float(&v)[32] = *reinterpret_cast<float(*)[32]>(l + c);
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            // the difference first: exact near the maximum, and in range for any finite logits
            v[i] = exp2_flush((v[i] - ref) * 1.4426950408889634f);
            sum[i & 3] += v[i];
        }
        if (e.probs != nullptr) {
            const int h = c >> 5 & 1;
            if (h == 0) blocks.settle<1>();
            blocks.write16(blocks.next, h, [&](int i) { return prob16x2(v[2 * i], v[2 * i + 1]); });
            if (h == 1 || c + 32 >= width) {
                blocks.store(blocks.next, &a.to[0], first + c - 32 * h, m0);
                blocks.next ^= 1;
            }
        }
    }
    if (row < m) {
        if (target >= 0 && target < width) e.logit[row] = logit;
        e.part[(int64_t)(first / W) * e.part_ld + row] =
            make_float2(most, (sum[0] + sum[1]) + (sum[2] + sum[3]));
    }
    return true;
}

// Two fp32 numbers side by side: sums and products of both are one instruction.
struct Two {
    uint64_t u;
    __device__ __forceinline__ explicit Two(uint64_t bits) : u(bits) {}
    __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(u) : "f"(a), "f"(b)); }
    __device__ __forceinline__ void get(float& a, float& b) const {
        asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(u));
    }
};
__device__ __forceinline__ Two operator+(Two a, Two b) {
    asm("add.rn.f32x2 %0, %0, %1;" : "+l"(a.u) : "l"(b.u));
    return a;
}
__device__ __forceinline__ Two operator*(Two a, Two b) {
    asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(a.u) : "l"(b.u));
    return a;
}
__device__ __forceinline__ Two mul_add(Two a, Two b, Two c) {
    asm("fma.rn.f32x2 %0, %0, %1, %2;" : "+l"(a.u) : "l"(b.u), "l"(c.u));
    return a;
}

// Sum over the warp's lanes of v[i], to lane i: each step halves the columns
// that a lane still has and doubles the rows in their sums.
__device__ __forceinline__ float sum_lanes(float (&v)[32], int lane) {
#pragma unroll
    for (int d = 16; d > 0; d /= 2) {
        const bool up = (lane & d) != 0;
#pragma unroll
        for (int i = 0; i < d; ++i) {
            const float keep = up ? v[i + d] : v[i], give = up ? v[i] : v[i + d];
            v[i] = keep + __shfl_xor_sync(~0u, give, d);
        }
    }
    return v[0];
}

// v[at], at in [0, 32), by halves.
__device__ __forceinline__ float pick(const float (&v)[32], uint32_t at) {
    float t[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) t[i] = at & 16 ? v[i + 16] : v[i];
#pragma unroll
    for (int d = 8; d > 0; d /= 2)
#pragma unroll
        for (int i = 0; i < d; ++i) t[i] = at & d ? t[i + d] : t[i];
    return t[0];
}

// What an epilogue warp of kRows keeps in shared memory for its columns
// (32 of every 128), and adds up over its units.
struct RowsWarp {
    uint8_t* blocks;  // [2][kRowsBlock]
    float* bias;      // [kRowsColumnsWarp] -inf past the last column
    float* columns;   // [kRowsColumnsWarp] sums of the probabilities of counted rows
    int* targets;     // [kRowsColumnsWarp] how many rows' target the column is
    int next = 0;     // block
    float loss = 0.0f;
    int counted = 0;
};

// A unit of kRows: 32 rows from m0 on, of which this warp has columns
// share * 32 .. + 31 of every 128; the others are three warps' with which it
// exchanges maximum and sum.  The sums of products are read from TMEM
// twice, since a row of them has no room in registers and an exponential
// costs no more than keeping one in fewer bits would.  The loops stay rolled:
// written out, each instruction would be fetched once or twice in all, and
// warps waited for that most (with eight warps, 34 us instead of 28).  wait(t) and release(t): column tile t's sums are complete, are
// no longer needed.
template <int DT, class Wait, class Release, class Exchange, class Address>
__device__ __forceinline__ bool rows_epilogue(const KernelArgs& a, const RowsEpilogue& e, int m, int n, int across,
                                              int m0, int share, int target, int lane, RowsWarp& own,
                                              Wait wait, Release release, Exchange exchange, Address address) {
    constexpr float kLog2e = 1.4426950408889634f;
    const int row = m0 + lane, first = share * 32;
    if (m0 >= m) {
        for (int t = 0; t < across; ++t) {
            if (!wait(t)) return false;
            release(t);
        }
        if (e.d != nullptr && share == 0 && lane == 0) reinterpret_cast<uint8_t*>(e.clean.use)[m0 / 32] = 0;
        return true;
    }
    // logits of 32 columns
    const auto load = [&](int t, float(&v)[32]) {
        tmem_ld_32cols_to(address(t), v);
        const float4* bias = reinterpret_cast<const float4*>(own.bias + t * 32);
        tmem_ld_wait();
        pin(v);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float4 b = bias[i];
            (Two(v[4 * i], v[4 * i + 1]) + Two(b.x, b.y)).get(v[4 * i], v[4 * i + 1]);
            (Two(v[4 * i + 2], v[4 * i + 3]) + Two(b.z, b.w)).get(v[4 * i + 2], v[4 * i + 3]);
        }
    };
    float top = -INFINITY, sum = 0.0f;
#pragma unroll 1
    for (int t = 0; t < across; ++t) {
        if (!wait(t)) return false;
        if (t * 128 + first >= n) continue;
        float v[32];
        load(t, v);
        float most[4] = {top, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 16; ++i)
            asm("max.f32 %0, %0, %1, %2;" : "+f"(most[i & 3]) : "f"(v[2 * i]), "f"(v[2 * i + 1]));
        const float next = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
        const float ref = next == -INFINITY ? 0.0f : next;
        Two part[2] = {Two(0.0f, 0.0f), Two(0.0f, 0.0f)};
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float x, y;
            ((Two(v[2 * i], v[2 * i + 1]) + Two(-ref, -ref)) * Two(kLog2e, kLog2e)).get(x, y);
            part[i & 1] = part[i & 1] + Two(exp2_flush(x), exp2_flush(y));
        }
        float x, y;
        (part[0] + part[1]).get(x, y);
        sum = sum * exp2_flush((top - ref) * kLog2e) + (x + y);
        top = next;
    }
    float2 all[4];
    if (!exchange(make_float2(top, sum), all)) return false;
    top = fmaxf(fmaxf(all[0].x, all[1].x), fmaxf(all[2].x, all[3].x));
    const float ref = top == -INFINITY ? 0.0f : top;
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += all[i].y * exp2_flush((all[i].x - ref) * kLog2e);
    const float shift = sum == 0.0f ? 0.0f : -log2f(sum);  // no sum: every logit is -inf
    const bool grads = e.d != nullptr, live = target >= 0, all_live = __all_sync(~0u, live);
    float logit = 0.0f;
#pragma unroll 1
    for (int t = 0; t < across; ++t) {
        const int col = t * 128 + first;
        const uint32_t hot = (uint32_t)(target - col);
        const bool any = __any_sync(~0u, hot < 32);
        if (col >= n || (!grads && !any)) {
            release(t);
            continue;
        }
        float v[32];
        load(t, v);
        release(t);
        if (any) {
            const float at = pick(v, hot);
            if (hot < 32) logit = at;
        }
        if (!grads) continue;
        // softmax as one exponential, whose argument is exact near the maximum
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float x, y;
            mul_add(Two(v[2 * i], v[2 * i + 1]) + Two(-ref, -ref), Two(kLog2e, kLog2e), Two(shift, shift)).get(x, y);
            v[2 * i] = exp2_flush(x);
            v[2 * i + 1] = exp2_flush(y);
        }
        if (!all_live)  // a row that is not counted, whatever it holds
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = live ? v[i] : 0.0f;
        // 64 bytes per row, as TMA swizzles them
        uint8_t* block = own.blocks + own.next * kRowsBlock + lane * 64;
        const auto place = [&](int q) { return block + ((q ^ (lane >> 1 & 3)) << 4); };
        if (lane == 0) bulk_wait_read_n<1>();
        __syncwarp();
        const auto word = [&](int i) { return pack2<DT>(v[2 * i] * kDScale<DT>, v[2 * i + 1] * kDScale<DT>); };
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *reinterpret_cast<uint4*>(place(q)) = make_uint4(word(4 * q), word(4 * q + 1), word(4 * q + 2), word(4 * q + 3));
        if (hot < 32) {
            using E = Elem<DT>;
            const float d = exp2_flush(fmaf(logit - ref, kLog2e, shift)) - 1.0f;
            reinterpret_cast<typename E::T*>(place(hot >> 3))[hot & 7] = E::put(d * kDScale<DT>);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
            tma_store_2d(&a.to[0], smem_u32(block), col, m0);
            bulk_commit();
        }
        own.next ^= 1;
        if (e.sums != nullptr) own.columns[t * 32 + lane] += sum_lanes(v, lane);
    }
    if (grads && share == 0) {
        const bool bad = row < m && !live && !(sum > 0.0f && sum < INFINITY);
        const bool any = __any_sync(~0u, bad);
        if (lane == 0) reinterpret_cast<uint8_t*>(e.clean.use)[m0 / 32] = any;
        // (two warps may copy a step, and then write the same)
        if (__builtin_expect(any, false)) clean_step(e.clean, m0 / kStepRows, m, e.target, lane, 32);
    }
    if (row >= m) return true;
    if (live && (target & 96) == first) {
        const float loss = logit == -INFINITY ? INFINITY : (top - logit) + logf(sum);
        e.row_loss[row] = loss;
        own.loss += loss;
        ++own.counted;
        atomicAdd(&own.targets[target / 128 * 32 + target % 32], 1);
    } else if (!live && share == 0) {
        e.row_loss[row] = 0.0f;
    }
    return true;
}

template <int BN, int DT, int EPI>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads<EPI>, 1)
    gemm_kernel(const __grid_constant__ KernelArgs a) {
    using Cfg = Config<BN>;
    constexpr int S = EPI == kRows ? kRowsStages : Cfg::kStages;
    extern __shared__ __align__(1024) uint8_t ring[];  // at the same address in both CTAs
    constexpr int EW = kEpiWarps<EPI>;
    constexpr int kWarp = EPI == kRows ? kRowsWarpBytes : kWarpBytes + Cfg::kCols * 2;  // of blocks, then the rest
    constexpr int kBlocks = EPI == kRows ? 2 * kRowsBlock : kWarpBytes;
    constexpr int kBufs = EPI == kRows ? 4 : 2;         // of BN columns of TMEM
    uint8_t* blocks_all = ring + S * Cfg::kStageBytes;  // a multiple of 1 KB, as each warp's part is
    uint8_t* own_all = blocks_all + EW * kBlocks;       // per warp its 16-bit bias, or a RowsWarp's columns
    float2* stats = reinterpret_cast<float2*>(own_all + EW * (kWarp - kBlocks));  // kRows: [2][4][kRowsCta]
    uint64_t* bars = reinterpret_cast<uint64_t*>(stats + (EPI == kRows ? kRowsStats / 8 : 0));
    uint64_t* full = bars;           // even CTA's: a stage has landed in both CTAs
    uint64_t* empty = bars + S;      // each CTA's: the products have read a stage
    uint64_t* tfull = bars + 2 * S;  // [kBufs] each CTA's: a tile's sums are complete
    uint64_t* tempty = tfull + 4;    // [kBufs] even CTA's: both CTAs have read them
    uint64_t* done = tempty + 4;     // even CTA's: the last products are complete
    uint64_t* landed = done + 1;     // [EW][2] a warp's residual block has arrived
    uint64_t* told = bars + Cfg::kBarriers;  // kRows: [EW] the warps of its rows have left their statistics
    float* loss_all = reinterpret_cast<float*>(told + (EPI == kRows ? EW : 0));  // kRows: [EW]
    int* count_all = reinterpret_cast<int*>(loss_all + (EPI == kRows ? EW : 0));  // kRows: [EW]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(count_all + (EPI == kRows ? EW : 0));

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(smem_u32(&full[s]), 1);
            mbar_init(smem_u32(&empty[s]), 1);
        }
        for (int i = 0; i < kBufs; ++i) {
            mbar_init(smem_u32(&tfull[i]), 1);
            mbar_init(smem_u32(&tempty[i]), 2 * EW);
        }
        mbar_init(smem_u32(done), 1);
        for (int i = 0; EPI != kRows && i < 2 * EW; ++i) mbar_init(smem_u32(&landed[i]), 1);
        for (int i = 0; EPI == kRows && i < EW; ++i) mbar_init(smem_u32(&told[i]), 4);
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc_pair(smem_u32(tmem_slot), kBufs * BN);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    griddep_launch_dependents();
    griddep_wait();

    const UnitWalk walk(a, pair, pairs);
    const int jobs = a.units[1] > 0 ? 2 : 1;
    if (warp == 0) {
        // Control flow here and in the MMA warp is the whole warp's; one
        // elected lane issues (elect_one).
        int s = 0, round = 0;  // stage, and times around the ring
        int64_t used = 0;
        bool ok = true;
        for (int job = 0; job < jobs && ok; ++job) {
            const Tiling tiling(a.job[job]);
            const bool a_mn = a.job[job].a_mn, b_mn = a.job[job].b_mn;
            // Whether a step of the unit is to be read from b_other, which takes a loop of its
            // own: units without one, nearly all there are, pay nothing for it (chosen step by
            // step in one loop, 1262 us instead of 1223 for 2048 rows of 2048, 65536 classes).
            const uint16_t* use_other = EPI == kStore ? a.job[job].use_other : nullptr;
            int marks_at = -1, marks_to = -1;
            bool marked = false;
            for (int i = 0, unit; ok && (unit = walk.unit(job, i)) >= 0; ++i) {
                const Tile t(tiling, unit, BN);
                const int am = t.m0 + (int)rank * kRowsCta;
                int bn = t.n0 + (int)rank * (BN / 2), kb = t.kb0;
                const int steps = (t.kb1 - t.kb0) * (EPI == kRows ? a.job[0].across : 1);
                const auto produce = [&](const CUtensorMap* tb) {
                    const uint32_t wait = smem_u32(&empty[s]);
                    if (!mbar_wait_warp(wait, (round & 1) ^ 1, a.err, kErrWaitProducer)) return false;
                    const uint32_t bar = map_to_rank(smem_u32(&full[s]), 0);
                    const uint32_t da = smem_u32(ring + s * Cfg::kStageBytes), db = da + Cfg::kABytes;
                    const int k0 = kb * kBK;
                    if (elect_one()) {
                        if (rank == 0) mbar_arrive_expect_tx(smem_u32(&full[s]), 2 * Cfg::kStageBytes);
                        if (a_mn) {
                            tma_load_2d_pair(da, &a.ta[job], bar, am, k0);
                            tma_load_2d_pair(da + 8192, &a.ta[job], bar, am + 64, k0);
                        } else {
                            tma_load_2d_pair(da, &a.ta[job], bar, k0, am);
                        }
                        if (b_mn) {
                            tma_load_2d_pair(db, tb, bar, bn, k0);
                            if (BN == 256) tma_load_2d_pair(db + 8192, tb, bar, bn + 64, k0);
                        } else {
                            tma_load_2d_pair(db, tb, bar, k0, bn);
                        }
                    }
                    ++used;
                    if (++s == S) {
                        s = 0;
                        ++round;
                    }
                    return true;
                };
                if (use_other != nullptr && (t.kb0 != marks_at || t.kb1 != marks_to)) {
                    marks_at = t.kb0;
                    marks_to = t.kb1;
                    uint32_t mine = 0;
#pragma unroll 8
                    for (int x = t.kb0 + lane; x < t.kb1; x += 32) mine |= use_other[x];
                    marked = __any_sync(~0u, mine != 0);
                }
                if (marked) {
                    for (int step = 0; ok && step < steps; ++step, ++kb)
                        ok = produce(use_other[kb] != 0 ? &a.tb_other : &a.tb[job]);
                    continue;
                }
                for (int step = 0; step < steps; ++step, ++kb) {
                    if (EPI == kRows && kb == t.kb1) {
                        kb = t.kb0;
                        bn += BN;
                    }
                    if (!produce(&a.tb[job])) {
                        ok = false;
                        break;
                    }
                }
            }
        }
        // Every load has landed and every stage has been released (the
        // release comes from the peer's commits) before this CTA ends.
        for (int i = 0; i < S && i < used; ++i) {
            if (--s < 0) {
                s = S - 1;
                --round;
            }
            if (rank == 0) mbar_wait_warp(smem_u32(&full[s]), round & 1, a.err, kErrWaitDrain);
            if (ok) mbar_wait_warp(smem_u32(&empty[s]), round & 1, a.err, kErrWaitDrain);
        }
    } else if (warp == 1) {
        if (rank == 0) {
            int s = 0, round = 0, tile = 0;
            bool ok = true;
            for (int job = 0; job < jobs && ok; ++job) {
                const Tiling tiling(a.job[job]);
                const bool a_mn = a.job[job].a_mn, b_mn = a.job[job].b_mn;
                const uint32_t idesc = idesc_f16(kRowsPair, BN, DT == MG_PREC_BF16) | (a_mn ? kIdescAMn : 0) |
                                       (b_mn ? kIdescBMn : 0);
                const uint64_t step_a = a_mn ? 2048 >> 4 : 32 >> 4, step_b = b_mn ? 2048 >> 4 : 32 >> 4;
                const uint32_t ring_at = smem_u32(ring);
                const uint64_t first_a = a_mn ? smem_desc_sw128_mn(ring_at) : smem_desc_sw128(ring_at);
                const uint64_t first_b =
                    b_mn ? smem_desc_sw128_mn(ring_at + Cfg::kABytes) : smem_desc_sw128(ring_at + Cfg::kABytes);
                for (int i = 0, unit; ok && (unit = walk.unit(job, i)) >= 0; ++i) {
                    const Tile t(tiling, unit, BN);
                    // kRows: a part per column tile; kSoftmax: per stretch of K
                    const int chain = EPI == kSoftmax ? a.job[0].chain : t.kb1 - t.kb0;
                    const int parts = EPI == kRows ? a.job[0].across : EPI == kSoftmax ? (t.kb1 + chain - 1) / chain : 1;
                    for (int x = 0; x < parts && ok; ++x) {
                        const int kb0 = EPI == kSoftmax ? x * chain : t.kb0, kb1 = min(t.kb1, kb0 + chain);
                        const int buf = tile % kBufs;
                        if (!mbar_wait_warp(smem_u32(&tempty[buf]), ((tile / kBufs) & 1) ^ 1, a.err, kErrWaitMma)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint32_t acc = tmem_base + buf * BN;
                        for (int kb = kb0; kb < kb1; ++kb) {
                            if (!mbar_wait_warp(smem_u32(&full[s]), round & 1, a.err, kErrWaitMma)) {
                                ok = false;
                                break;
                            }
                            tc_fence_after();
                            const uint64_t xa = first_a + s * (Cfg::kStageBytes >> 4);
                            const uint64_t xb = first_b + s * (Cfg::kStageBytes >> 4);
                            if (elect_one()) {
#pragma unroll
                                for (int kk = 0; kk < kBK / 16; ++kk)
                                    mma_f16_pair(acc, xa + kk * step_a, xb + kk * step_b, idesc, kb > kb0 || kk > 0);
                                mma_commit_pair(smem_u32(&empty[s]));
                                if (kb + 1 == kb1) mma_commit_pair(smem_u32(&tfull[buf]));
                            }
                            if (++s == S) {
                                s = 0;
                                ++round;
                            }
                        }
                        ++tile;
                    }
                }
            }
            // Products still in flight finish before TMEM is freed.
            if (elect_one())
                asm volatile(
                    "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(done))
                    : "memory");
            mbar_wait_warp(smem_u32(done), 0, a.err, kErrWaitDrain);
        }
    } else {
        const int ew = warp - 2, quarter = warp & 3;
        const int c0 = (ew >> 2) * Cfg::kCols;
        // the warp's own copy of its columns' bias: one shared by four warps would
        // need a barrier, which a warp whose wait gave up would leave the others at
        uint16_t* sbias = reinterpret_cast<uint16_t*>(own_all + ew * (kWarp - kBlocks));
        WarpBlocks blocks;
        blocks.blocks = blocks_all + ew * kBlocks;
        blocks.landed = &landed[2 * ew];
        blocks.lane = lane;
        const uint32_t taddr0 = tmem_base + c0 + ((uint32_t)quarter << 21);
        int tile = 0;
        bool ok = true;
        if constexpr (EPI == kRows) {
            const JobArgs& job = a.job[0];
            const RowsEpilogue e = job.r;
            const Tiling tiling(job);
            const int m = job.m, n = job.n, across = job.across, share = ew >> 2;
            RowsWarp own;
            own.blocks = blocks.blocks;
            own.bias = reinterpret_cast<float*>(sbias);
            own.columns = own.bias + kRowsColumnsWarp;
            own.targets = reinterpret_cast<int*>(own.columns + kRowsColumnsWarp);
            for (int t = 0; t < across; ++t) {
                const int col = t * 128 + share * 32 + lane;
                float v = col < n ? 0.0f : -INFINITY;
                if (e.bias != nullptr && col < n) v = Elem<DT>::get(static_cast<const typename Elem<DT>::T*>(e.bias)[col]);
                own.bias[t * 32 + lane] = v;
                own.columns[t * 32 + lane] = 0.0f;
                own.targets[t * 32 + lane] = 0;
            }
            __syncwarp();
            for (int i = 0, unit; ok && (unit = walk.unit(0, i)) >= 0; ++i) {
                const int m0 = Tile(tiling, unit, BN).m0 + (int)rank * kRowsCta + quarter * 32;
                const int target = m0 + lane < m ? (int)e.target.at(m0 + lane) : -1;
                const auto wait = [&](int t) {
                    const int at = tile + t;
                    const bool there =
                        mbar_wait_warp(smem_u32(&tfull[at % kBufs]), at / kBufs & 1, a.err, kErrWaitEpilogue);
                    tc_fence_after();
                    return there;
                };
                const auto release = [&](int t) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(map_to_rank(smem_u32(&tempty[(tile + t) % kBufs]), 0));
                };
                // The statistics lie in buffers by turns: the other warps, which are at most
                // a unit behind, may still read the last ones.
                const auto exchange = [&](float2 mine, float2(&all)[4]) {
                    float2* at = stats + (i & 1) * 4 * kRowsCta + quarter * 32 + lane;
                    at[share * kRowsCta] = mine;
                    __syncwarp();
                    if (lane < 4) mbar_arrive(smem_u32(&told[lane * 4 + (ew & 3)]));
                    if (!mbar_wait_warp(smem_u32(&told[ew]), i & 1, a.err, kErrWaitEpilogue)) return false;
#pragma unroll
                    for (int k = 0; k < 4; ++k) all[k] = at[k * kRowsCta];
                    return true;
                };
                const auto address = [&](int t) {
                    return tmem_base + (tile + t) % kBufs * BN + share * 32 + ((uint32_t)quarter << 21);
                };
                ok = rows_epilogue<DT>(a, e, m, n, across, m0, share, target, lane, own, wait, release, exchange, address);
                tile += across;
            }
#pragma unroll
            for (int d = 16; d > 0; d /= 2) own.loss += __shfl_xor_sync(~0u, own.loss, d);
            own.counted = __reduce_add_sync(~0u, own.counted);
            if (lane == 0) {
                loss_all[ew] = own.loss;
                count_all[ew] = own.counted;
            }
        } else for (int job = 0; job < jobs && ok; ++job) {
            const Tiling tiling(a.job[job]);
            const EpilogueJob j(a.job[job], lane);
            const SoftmaxEpilogue soft = a.job[0].s;
            const void* bias = EPI == kSoftmax ? soft.bias : j.has_out32 ? nullptr : a.job[job].e.bias;
            int bias_at = -1;  // first column of the tile whose bias is there
            for (int i = 0, unit; ok && (unit = walk.unit(job, i)) >= 0; ++i) {
                const Tile t(tiling, unit, BN);
                const int m0 = t.m0 + (int)rank * kRowsCta + quarter * 32;
                // what the tile needs besides its sums is on its way before they are complete
                int target = -1, after_col = -1, after_row = 0;
                if constexpr (EPI == kSoftmax) {
                    if (m0 + lane < j.m) target = soft.target.at(m0 + lane);
                } else if (j.has_res && j.by_tma && !j.has_z) {
                    const auto mine = [&](const Tile& u, int* col, int* row) {
                        *row = u.m0 + (int)rank * kRowsCta + quarter * 32;
                        *col = u.n0 + c0;
                        return *row < j.m && *col < j.n;
                    };
                    int col, row;
                    if (blocks.flying == 0 && mine(t, &col, &row)) {
                        blocks.settle<0>();
                        blocks.start_res(blocks.next, &a.tr, col, row);
                    }
                    const int following = walk.unit(job, i + 1);
                    after_col = -1;
                    if (following >= 0 && mine(Tile(tiling, following, BN), &col, &row)) {
                        after_col = col;
                        after_row = row;
                    }
                }
                if (t.n0 != bias_at) {
                    bias_at = t.n0;
                    __syncwarp();
                    for (int b = lane; b < Cfg::kCols; b += 32) {
                        const int64_t col = t.n0 + c0 + b;
                        // past the last column: nothing, or for the softmax a logit of -inf
                        uint16_t v = EPI == kSoftmax && col >= j.n ? (DT == MG_PREC_BF16 ? 0xff80 : 0xfc00) : 0;
                        if (bias != nullptr && col < j.n) v = static_cast<const uint16_t*>(bias)[col];
                        sbias[b] = v;
                    }
                    __syncwarp();
                }
                // one answer for the warp, which goes on or stops together
                const auto wait = [&](int p) {
                    const int at = tile + p;
                    const bool there = mbar_wait_warp(smem_u32(&tfull[at & 1]), at >> 1 & 1, a.err, kErrWaitEpilogue);
                    tc_fence_after();
                    return there;
                };
                const auto release = [&](int p) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(map_to_rank(smem_u32(&tempty[(tile + p) & 1]), 0));
                };
                if constexpr (EPI == kSoftmax) {
                    const int parts = (t.kb1 + a.job[0].chain - 1) / a.job[0].chain;
                    ok = softmax_epilogue<BN, DT>(a, soft, j.m, j.n, t, m0, c0, target, blocks, sbias, parts, wait, release,
                                                  [&](int p) { return taddr0 + ((tile + p) & 1) * BN; });
                    tile += parts;
                } else {
                    if (!wait(0)) {
                        ok = false;
                        break;
                    }
                    ok = epilogue<BN, DT>(a, job, j, t, m0, c0, taddr0 + (tile & 1) * BN, blocks, sbias, after_col, after_row,
                                          [&] { release(0); });
                    ++tile;
                }
            }
        }
        for (int b = blocks.next; blocks.flying > 0; b ^= 1)  // only after a wait gave up
            blocks.wait_res(b, a.err, kErrWaitDrain);
        if (lane == 0) bulk_wait_all();
        __syncwarp();
    }
    // Neither CTA ends, or frees TMEM, while the other may still read its
    // shared memory or signal its barriers.
    tc_fence_before();
    __syncthreads();
    if constexpr (EPI == kRows) {
        // what the CTA's warps have added up, joined in a fixed order
        const RowsEpilogue& e = a.job[0].r;
        if (threadIdx.x == 0) {
            float loss = 0.0f;
            int count = 0;
            for (int i = 0; i < EW; ++i) {
                loss += loss_all[i];
                count += count_all[i];
            }
            e.loss[blockIdx.x] = loss;
            if (e.counts != nullptr) e.counts[blockIdx.x] = count;
        }
        const int n = a.job[0].n;
        if (e.sums != nullptr && threadIdx.x < n) {
            const int c = threadIdx.x, at = c / 128 * 32 + c % 32;
            float sum = 0.0f;
            int targets = 0;
            for (int i = 0; i < 4; ++i) {
                const float* columns = reinterpret_cast<const float*>(own_all + (c / 32 % 4 * 4 + i) * (kWarp - kBlocks)) +
                                       kRowsColumnsWarp;
                sum += columns[at];
                targets += reinterpret_cast<const int*>(columns + kRowsColumnsWarp)[at];
            }
            e.sums[(int64_t)blockIdx.x * n + c] = sum - (float)targets;
        }
    }
    cluster_sync();
    tc_fence_after();
    if (warp == 1) tmem_dealloc_pair(tmem_base, kBufs * BN);
}

// A tensor map of a dense-enough matrix: `rows` lines of `inner` elements,
// `ld` apart, in boxes of box_rows x box_inner.
void encode(CUtensorMap* map, CUtensorMapDataType type, int elem, const void* base, int64_t inner, int64_t rows,
            int64_t ld, int box_inner, int box_rows, CUtensorMapSwizzle swizzle) {
    static PFN_cuTensorMapEncodeTiled_v12000 enc = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
                       q == cudaDriverEntryPointSuccess
                   ? reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p)
                   : nullptr;
    }();
    if (enc == nullptr) fail(MG_E_CUDA, "cuTensorMapEncodeTiled is unavailable");
    cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)(ld * elem)};
    cuuint32_t box[2] = {(cuuint32_t)box_inner, (cuuint32_t)box_rows};
    cuuint32_t one[2] = {1, 1};
    if (enc(map, type, 2, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        fail(MG_E_CUDA, "cuTensorMapEncodeTiled rejected a tensor map");
}

CUtensorMapDataType map_type(int dtype) {
    return dtype == MG_PREC_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

}  // namespace

// An operand, in boxes of 64 contraction steps (128 bytes, or lines).
void encode_operand(CUtensorMap* map, int dtype, const StagedOperand& s, int64_t rows, int64_t k, int tile_rows) {
    encode(map, map_type(dtype), 2, s.data, s.mn ? rows : k, s.mn ? k : rows, s.ld, 64, s.mn ? kBK : tile_rows,
           CU_TENSOR_MAP_SWIZZLE_128B);
}

namespace {

// A matrix that the epilogue moves in blocks of 32 x 64 16-bit elements.
void encode_blocks(CUtensorMap* map, int dtype, const void* base, int64_t m, int64_t n, int64_t ld) {
    encode(map, map_type(dtype), 2, base, n, m, ld, 64, 32, CU_TENSOR_MAP_SWIZZLE_128B);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
int64_t up8(int64_t v) { return (v + 7) / 8 * 8; }

template <int BN, int DT, int EPI>
void launch_one(const KernelArgs& a, int pairs, Queue& q) {
    check(cudaFuncSetAttribute(gemm_kernel<BN, DT, EPI>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               Config<BN>::kSmem),
          "cudaFuncSetAttribute(gemm_kernel)");
    q.launch("gemm_kernel", gemm_kernel<BN, DT, EPI>, dim3(2 * pairs), kThreads<EPI>, Config<BN>::kSmem, a);
}

void launch_rows(KernelArgs& a, int dtype, Queue& q) {
    a.err = op_status_word();
    const int pairs = std::min(kPairs, a.units[0]);
    const auto kernel = dtype == MG_PREC_BF16 ? gemm_kernel<128, MG_PREC_BF16, kRows> : gemm_kernel<128, MG_PREC_FP16, kRows>;
    check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowsSmem),
          "cudaFuncSetAttribute(gemm_kernel)");
    q.launch("gemm_kernel", kernel, dim3(2 * pairs), kThreads<kRows>, kRowsSmem, a);
}

template <int EPI>
void launch(KernelArgs& a, int bn, int dtype, Queue& q) {
    a.err = op_status_word();
    const int pairs = (int)std::min<int64_t>(kPairs, (int64_t)a.units[0] + a.units[1]);
    if (bn == 256) {
        if (dtype == MG_PREC_BF16) launch_one<256, MG_PREC_BF16, EPI>(a, pairs, q);
        else launch_one<256, MG_PREC_FP16, EPI>(a, pairs, q);
    } else {
        if (dtype == MG_PREC_BF16) launch_one<128, MG_PREC_BF16, EPI>(a, pairs, q);
        else launch_one<128, MG_PREC_FP16, EPI>(a, pairs, q);
    }
}

// Fills in what a job's tiles are, for tiles of bn columns.
template <class Job>
void lay_out(JobArgs& j, const Job& g, int bn) {
    j.m = (int)g.m;
    j.n = (int)g.n;
    j.kblocks = (int)((g.k + kBK - 1) / kBK);
    j.tiles_m = (int)((g.m + kRowsPair - 1) / kRowsPair);
    j.tiles_n = (int)((g.n + bn - 1) / bn);
    j.splits = 1;
    j.kb_split = j.kblocks;
    j.a_mn = g.a.mn;
    j.b_mn = g.b.mn;
    j.m_pad = j.tiles_m * kRowsPair;
    need((int64_t)j.tiles_m * j.tiles_n < (int64_t(1) << 24), "too many tiles");
}

template <class Job>
void encode_operands(KernelArgs& a, int i, int dtype, const Job& g, int bn) {
    encode_operand(&a.ta[i], dtype, g.a, g.m, g.k, kRowsCta);
    encode_operand(&a.tb[i], dtype, g.b, g.n, g.k, bn / 2);
}

void encode_other(KernelArgs& a, int i, int dtype, const GemmJob& g, int bn) {
    need(i == 0 || a.job[0].use_other == nullptr, "one product of a launch reads steps from elsewhere");
    need(g.b_other.mn == g.b.mn, "both copies of an operand lie the same way");
    a.job[i].use_other = g.use_other;
    encode_operand(&a.tb_other, dtype, g.b_other, g.n, g.k, bn / 2);
}

// Narrow tiles where wide ones would leave pairs idle or mostly compute
// padding; a narrow tile costs more than half a wide one, since it reads A
// as often.
template <class Job>
int tile_columns(const Job* jobs, int count) {
    const auto cost = [&](int bn) {
        double work = 0;
        int64_t units = 0;
        for (int i = 0; i < count; ++i) {
            const int64_t t = (jobs[i].m + 255) / 256 * ((jobs[i].n + bn - 1) / bn);
            work += (double)t * (double)jobs[i].k;
            units += t;
        }
        const double waves = std::max(1.0, (double)units / kPairs);
        return work / units * waves * (bn == 256 ? 1.0 : 0.6);
    };
    return cost(128) < cost(256) ? 128 : 256;
}

}  // namespace

StagedOperand stage_operand(Workspace& w, Packs& packs, const GemmOperand& op, int64_t rows, int64_t k) {
    // a dimension of one element has no stride of its own
    const int64_t row = rows == 1 ? up8(std::max(k, op.row)) : op.row;
    const int64_t col = k == 1 ? up8(std::max(rows, op.col)) : op.col;
    const int64_t top = int64_t(1) << 38;
    StagedOperand s;
    s.data = op.data;
    if (op.col == 1 || k == 1) {
        s.ld = row;
        if (row % 8 == 0 && row >= k && row < top && aligned16(op.data)) return s;
    }
    if (op.row == 1 || rows == 1) {
        s.ld = col;
        s.mn = true;
        if (col % 8 == 0 && col >= rows && col < top && aligned16(op.data)) return s;
    }
    // copied along the way it lies, so that reads and writes are both in order
    s.mn = op.row == 1 && op.col != 1;
    PackTask& t = packs.task[packs.count++];
    t.lines = s.mn ? k : rows;
    t.len = s.mn ? rows : k;
    t.line = s.mn ? op.col : op.row;
    t.step = s.mn ? op.row : op.col;
    t.ld = s.ld = up8(t.len);
    t.in = static_cast<const uint16_t*>(op.data);
    t.out = w.take<uint16_t>((size_t)t.lines * t.ld * 2);
    t.blocks = (int)std::min<int64_t>((t.lines * ((t.len + 511) / 512) + 7) / 8, 148 * 6);
    s.data = t.out;
    return s;
}

void gemm(Workspace& w, bool go, int dtype, GemmJob* jobs, int count, Post& post, Queue& q) {
    if (count == 1 && jobs->m <= kSkinnyRows && !jobs->a.mn && !jobs->b.mn && jobs->e.out32 == nullptr &&
        jobs->e.acc32 == nullptr && jobs->e.count.parts == nullptr && jobs->use_other == nullptr) {
        if (go) skinny(dtype, *jobs, q);
        return;
    }
    if (count == 2 && jobs[1].k > jobs[0].k) std::swap(jobs[0], jobs[1]);
    const int bn = tile_columns(jobs, count);
    KernelArgs a{};
    GemmEpilogue finish[2];
    double len[2] = {0, 0};
    int64_t share = 0;  // K steps per pair, a tile's epilogue counted as 8
    for (int i = 0; i < count; ++i) {
        lay_out(a.job[i], jobs[i], bn);
        share += (int64_t)a.job[i].tiles_m * a.job[i].tiles_n * std::max(8, a.job[i].kblocks);
    }
    share = (share + kPairs - 1) / kPairs;
    for (int i = 0; i < count; ++i) {
        JobArgs& j = a.job[i];
        const GemmJob& g = jobs[i];
        j.e = finish[i] = g.e;
        // what tensor maps ask of the outputs and the residual
        j.by_tma = g.e.ld % 8 == 0 && aligned16(g.e.out) && aligned16(g.e.z) &&
                   (g.e.res == nullptr || (aligned16(g.e.res) && g.e.r_col == 1 && g.e.r_row % 8 == 0 &&
                                           g.e.r_row >= g.n && g.e.r_row < int64_t(1) << 38));
        const int64_t tiles = (int64_t)j.tiles_m * j.tiles_n;
        // Few tiles: their K steps are shared out, in units about as long as a pair's share
        // of all the work (of no fewer than 8 steps, which an epilogue's time is worth).
        if (tiles * 2 <= kPairs) j.kb_split = (int)std::min<int64_t>(j.kblocks, std::max<int64_t>(8, share));
        j.splits = (j.kblocks + j.kb_split - 1) / j.kb_split;
        j.kb_split = (j.kblocks + j.splits - 1) / j.splits;
        if (j.splits > 1) {
            j.e = GemmEpilogue{};
            j.e.ld32 = up8(g.n);
            j.e.out32 = w.take<float>((size_t)j.splits * j.m_pad * j.e.ld32 * 4);
        }
        a.units[i] = (int)(tiles * j.splits);
        len[i] = std::max(8, j.kb_split);
    }
    if (!go) return;
    w.require();
    for (int i = 0; i < count; ++i) {
        encode_operands(a, i, dtype, jobs[i], bn);
        if (jobs[i].use_other != nullptr) encode_other(a, i, dtype, jobs[i], bn);
        const JobArgs& j = a.job[i];
        const GemmEpilogue& e = j.e;
        if (e.out32 != nullptr)
            encode(&a.to[i], CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, e.out32, e.ld32, (int64_t)j.splits * j.m_pad, e.ld32,
                   32, 32, CU_TENSOR_MAP_SWIZZLE_128B);
        else if (j.by_tma)
            encode_blocks(&a.to[i], dtype, e.out, j.m, j.n, e.ld);
        if (!j.by_tma || e.out32 != nullptr) continue;
        need(i == 0 || (e.z == nullptr && e.res == nullptr), "z and residual belong to a launch's first product");
        if (e.z != nullptr) encode_blocks(&a.tz, dtype, e.z, j.m, j.n, e.ld);
        if (e.res != nullptr) encode_blocks(&a.tr, dtype, e.res, j.m, j.n, e.r_row);
    }
    a.head_start = count == 2 ? (int)(len[0] / len[1] + 0.5) : 0;
    launch<kStore>(a, bn, dtype, q);
    for (int i = 0; i < count; ++i)
        if (a.job[i].splits > 1)
            post.finish[post.finishes++] = FinishTask{a.job[i].e.out32,  a.job[i].splits, a.job[i].m_pad, jobs[i].m,
                                                      jobs[i].n,         a.job[i].e.ld32, finish[i],      0};
}

namespace {
bool is_skinny(const SoftmaxJob& g) { return g.m <= kSkinnyRows && !g.a.mn && !g.b.mn; }
}  // namespace

SoftmaxBlocks gemm_softmax_blocks(const SoftmaxJob& g, bool even) {
    if (is_skinny(g)) return skinny_blocks(g.m, g.n, g.k, even);
    const int columns = tile_columns(&g, 1) / 2;
    return {columns, (int)((g.n + columns - 1) / columns)};
}

void gemm_softmax(int dtype, const SoftmaxJob& g, int columns, Queue& q) {
    if (is_skinny(g) && (columns == 0 || columns == skinny_blocks(g.m, g.n, g.k, true).columns))
        return skinny_softmax(dtype, g, columns, q);
    const int bn = 2 * columns;
    KernelArgs a{};
    lay_out(a.job[0], g, bn);
    a.job[0].s = g.e;
    a.units[0] = a.job[0].tiles_m * a.job[0].tiles_n;
    a.job[0].chain = kChain;
    encode_operands(a, 0, dtype, g, bn);
    if (g.e.probs != nullptr) encode_blocks(&a.to[0], dtype, g.e.probs, g.m, g.e.probs_ld, g.e.probs_ld);
    launch<kSoftmax>(a, bn, dtype, q);
}

// A pair takes a unit's column tiles one after another, which other pairs
// would share where rows are few; it saves the joining launch, with gradients
// also the pass over the probabilities.  Measured in us (this way, by tiles;
// 362 classes) for rows x dim, with the K steps more on a pair's way:
// gradients 32768 x 256 (0) 49, 63; 256 x 256 (8) 23, 27; 4096 x 1024 (32)
// 38.5, 39.  Loss alone 32768 x 256 (0) 18, 23; 256 x 256 (8) 12.3, 10.8;
// 4096 x 1024 (32) 20, 14.
bool gemm_rows_pays(const SoftmaxJob& g, bool grads) {
    // (chains of products are not cut up there)
    if (g.n > kRowsColumns || g.k > kChain * kBK || is_skinny(g)) return false;
    const int64_t down = (g.m + kRowsPair - 1) / kRowsPair, across = (g.n + 127) / 128, steps = (g.k + kBK - 1) / kBK;
    const int64_t whole = (down + kPairs - 1) / kPairs * across * steps;
    const int64_t tiles = (down * across + kPairs - 1) / kPairs * steps;
    return whole <= tiles + (grads ? 32 : 4);
}

int gemm_rows_ctas(int64_t m) { return (int)std::min<int64_t>(kPairs, (m + kRowsPair - 1) / kRowsPair) * 2; }

void gemm_rows(int dtype, const RowsJob& g, Queue& q) {
    KernelArgs a{};
    JobArgs& j = a.job[0];
    lay_out(j, g, 128);
    j.across = j.tiles_n;
    j.tiles_n = 1;
    j.r = g.e;
    a.units[0] = j.tiles_m;
    encode_operands(a, 0, dtype, g, 128);
    if (g.e.d != nullptr)
        encode(&a.to[0], map_type(dtype), 2, g.e.d, g.e.ld, g.m, g.e.ld, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B);
    launch_rows(a, dtype, q);
}

}  // namespace ops
}  // namespace mgb
