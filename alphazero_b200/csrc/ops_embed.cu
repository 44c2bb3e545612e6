// Embedding lookup with scaling and its gradient (include/minigo_ops.h).
// Both are bound by memory: each moves n rows of dim elements once.
//
// Lookup: a warp (or 8 lanes) per row, pieces of up to 16 bytes, four of them
// in flight per lane.  131072 rows of 1024 bf16 from 65536: 70 us, the 403 MB
// at 88% of the rate of a plain copy.
//
// Gradient: the tokens are sorted (stable, so equal tokens stay in order of
// position), then cut into windows of equal length whatever the tokens are.
// A warp sums a window's rows run by run (a run: equal tokens) for one
// segment of columns.  A run inside one window is written at once; the parts
// of one that crosses windows go to scratch and are added by join_kernel in
// window order.  So a token that makes up a tenth of the batch is spread
// over as many warps as its rows deserve, there are no atomics on sums, and
// the result does not depend on the order in which blocks run.  100003 rows of
// 1000 bf16 into 65536 entries: two digits' sort 26 us, bound by the latency
// of its four launches; the sums 66 us, 5 TB/s of rows read and entries
// written; the join 6 us.
#include "ops_common.cuh"
#include "sorted_search.cuh"

#include <algorithm>

namespace mgb {
namespace ops {
namespace {

// ---- vectors of B bytes ----

template <int B>
struct Bytes;
template <>
struct Bytes<16> {
    using T = uint4;
};
template <>
struct Bytes<8> {
    using T = uint2;
};
template <>
struct Bytes<4> {
    using T = uint32_t;
};
template <>
struct Bytes<2> {
    using T = uint16_t;
};

// The widest access that rows of `row_bytes`, `stride_bytes` apart at p, all allow.
int widest(int elem, int64_t row_bytes, int64_t stride_a, int64_t stride_b, const void* p, const void* q) {
    const uint64_t all = (uint64_t)row_bytes | (uint64_t)stride_a | (uint64_t)stride_b |
                         reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q) | 16;
    return std::max<int>(elem, (int)(all & (~all + 1)));
}

// ---- lookup ----

constexpr int kPerLane = 4;  // pieces of B bytes that a lane has in flight

// LANES lanes per row; pieces = row in pieces of B bytes.  Rows that are not
// whole 16-byte pieces are bound by the issue of instructions, so offsets are
// 32-bit and known when compiled, and a piece is one compare, one load, its
// products and one store.
template <int DT, int B, int LANES>
__global__ void __launch_bounds__(256) embed_kernel(mg_embed_args a, int pieces) {
    using E = Elem<DT>;
    using T = typename E::T;
    using V = typename Bytes<B>::T;
    constexpr int N = B / (int)sizeof(T);
    griddep_wait();
    const int lane = threadIdx.x & (LANES - 1);
    const float scale = a.scale;
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LANES; i < a.n;
         i += (int64_t)gridDim.x * 256 / LANES) {
        const int64_t t = index_at(a.tokens, a.token_bytes, i * a.token_stride, a.vocab);
        const V* row = reinterpret_cast<const V*>(static_cast<const T*>(a.table) + max(t, (int64_t)0) * a.table_row);
        V* out = reinterpret_cast<V*>(static_cast<T*>(a.out) + i * a.dim);
        for (int c = blockIdx.y * (kPerLane * LANES) + lane; c < pieces; c += gridDim.y * (kPerLane * LANES)) {
            const int left = pieces - c;
            alignas(16) V v[kPerLane];
#pragma unroll
            for (int q = 0; q < kPerLane; ++q)
                if (q * LANES < left) v[q] = __ldg(row + c + q * LANES);
#pragma unroll
            for (int q = 0; q < kPerLane; ++q) {
                alignas(16) T e[N];
                *reinterpret_cast<V*>(e) = v[q];
#pragma unroll
                for (int j = 0; j < N; ++j) e[j] = E::put(t < 0 ? 0.0f : E::get(e[j]) * scale);
                if (q * LANES < left) out[c + q * LANES] = *reinterpret_cast<V*>(e);
            }
        }
    }
}

template <int DT, int B>
void embed_with(const mg_embed_args& a, Queue& q) {
    const int64_t pieces = a.dim * elem_bytes(DT) / B;
    need(pieces < (int64_t(1) << 31), "dim is too large");
    const bool narrow = pieces <= 8 * kPerLane;
    const int64_t rows = narrow ? 32 : 8, blocks = (a.n + rows - 1) / rows;
    // a few long rows are cut up to fill the card
    const int64_t segments = (pieces + 32 * kPerLane - 1) / (32 * kPerLane);
    const int64_t cuts = narrow ? 1 : std::clamp<int64_t>(148 * 8 / blocks, 1, std::min<int64_t>(segments, 65535));
    q.launch("embed_kernel", narrow ? embed_kernel<DT, B, 8> : embed_kernel<DT, B, 32>,
             dim3((unsigned)std::min<int64_t>(blocks, 1 << 30), (unsigned)cuts), 256, 0, a, (int)pieces);
}

template <int DT>
void embed(const mg_embed_args& a, Queue& q) {
    const int e = elem_bytes(DT);
    switch (widest(e, a.dim * e, a.table_row * e, 0, a.table, a.out)) {
        case 16: return embed_with<DT, 16>(a, q);
        case 8: return embed_with<DT, 8>(a, q);
        case 4: return embed_with<DT, 4>(a, q);
        default:
            if constexpr (DT != MG_PREC_FP32) embed_with<DT, 2>(a, q);
    }
}

// ---- sort ----
//
// Stable least-significant-digit radix sort of (token, position), padding
// last as token `vocab`: two launches per digit.  rank_kernel gives each
// token its place among its block's tokens of the same digit and counts the
// block's digits; scatter_kernel adds up the counts of smaller digits and
// earlier blocks and moves the tokens.  The moves are scattered 8-byte
// writes, which one SM does at about one a clock: so the sort uses up to 148
// blocks rather than one cluster (16 CTAs: 22 us a digit for 65536 tokens,
// where these two take 12).

constexpr int kSortWarps = 16;
constexpr int kSortThreads = 32 * kSortWarps;
constexpr int kMaxBits = 10;  // of the key per pass
constexpr int kBatch = 4;     // steps of 32 tokens whose loads a warp issues together

struct SortArgs {
    const void* tokens;
    int token_bytes;
    int64_t token_stride, vocab;
    int n, passes, bits;
    int blocks, steps;    // steps of 32 tokens per warp
    uint2* pair[2];       // [n] (token, position); host side
    const uint2* in;      // of this pass (the first reads tokens)
    uint2* out;
    uint32_t* place;      // [n]
    uint32_t* counts;     // [blocks][bins]
};

__device__ __forceinline__ uint32_t sort_key(const SortArgs& a, int pass, int64_t i, uint32_t* pos) {
    if (pass > 0) {
        const uint2 u = a.in[i];
        *pos = u.y;
        return u.x;
    }
    *pos = (uint32_t)i;
    const int64_t t = index_at(a.tokens, a.token_bytes, i * a.token_stride, a.vocab);
    return (uint32_t)(t < 0 ? a.vocab : t);
}

// Equal digits of a warp find one another with match_any, so places follow
// the order of the input.
__global__ void __launch_bounds__(kSortThreads) rank_kernel(SortArgs a, int pass) {
    extern __shared__ uint32_t rows[];  // [warps][bins]
    const int bins = 1 << a.bits, shift = pass * a.bits;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t begin = ((int64_t)blockIdx.x * kSortWarps + warp) * a.steps * 32;
    const int64_t end = min((int64_t)a.n, begin + (int64_t)a.steps * 32);
    uint32_t* mine = rows + warp * bins;
    uint32_t k[kBatch], at[kBatch], pos;
    griddep_launch_dependents();
    for (int b = threadIdx.x; b < kSortWarps * bins; b += kSortThreads) rows[b] = 0;
    __syncthreads();
    griddep_wait();
    const auto load = [&](int64_t i0) {
#pragma unroll
        for (int q = 0; q < kBatch; ++q) {
            const int64_t i = i0 + 32 * q + lane;
            // past the end: a digit of its own
            k[q] = i < end ? sort_key(a, pass, i, &pos) >> shift & (bins - 1) : (uint32_t)bins + lane;
        }
    };
    const auto rank = [&]() {
#pragma unroll
        for (int q = 0; q < kBatch; ++q) {
            const uint32_t peers = __match_any_sync(~0u, k[q]);
            const uint32_t below = __popc(peers & ((1u << lane) - 1));
            const uint32_t before = k[q] < bins ? mine[k[q]] : 0;
            __syncwarp();
            if (k[q] < bins && below == 0) mine[k[q]] = before + __popc(peers);
            __syncwarp();
            at[q] = before + below;
        }
    };
    for (int64_t i0 = begin; i0 < end; i0 += 32 * kBatch) {
        load(i0);
        rank();
#pragma unroll
        for (int q = 0; q < kBatch; ++q)
            if (i0 + 32 * q + lane < end) a.place[i0 + 32 * q + lane] = at[q];
    }
    __syncthreads();
    // per digit: the counts of the warps before each warp, and of the block
    for (int b = threadIdx.x; b < bins; b += kSortThreads) {
        uint32_t s = 0;
#pragma unroll
        for (int w = 0; w < kSortWarps; ++w) {
            const uint32_t c = rows[w * bins + b];
            rows[w * bins + b] = s;
            s += c;
        }
        a.counts[(int64_t)blockIdx.x * bins + b] = s;
    }
    __syncthreads();
    for (int64_t i0 = begin; i0 < end; i0 += 32 * kBatch) {
        if (a.steps > kBatch) load(i0);  // else still in k and at
#pragma unroll
        for (int q = 0; q < kBatch; ++q) {
            const int64_t i = i0 + 32 * q + lane;
            if (i < end) a.place[i] = (a.steps > kBatch ? a.place[i] : at[q]) + mine[k[q]];
        }
    }
}

__global__ void __launch_bounds__(kSortThreads) scatter_kernel(SortArgs a, int pass) {
    extern __shared__ uint32_t rows[];  // [slices][2][bins]: counts of earlier blocks, of all
    __shared__ uint32_t warp_sum[kSortWarps];
    const int bins = 1 << a.bits, shift = pass * a.bits;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    griddep_launch_dependents();
    griddep_wait();
    // four adjacent digits per thread, the blocks in `slices` interleaved shares
    const int quads = bins / 4, slices = max(1, kSortThreads / quads);
    if (threadIdx.x < slices * quads) {
        const int quad = threadIdx.x % quads, slice = threadIdx.x / quads;
        uint4 before = make_uint4(0, 0, 0, 0), all = before;
        for (int b0 = slice; b0 < a.blocks; b0 += 8 * slices) {  // eight loads at once, whatever is left
            uint4 c[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const int b = b0 + q * slices;
                c[q] = b < a.blocks ? *reinterpret_cast<const uint4*>(a.counts + (int64_t)b * bins + quad * 4)
                                    : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                all.x += c[q].x, all.y += c[q].y, all.z += c[q].z, all.w += c[q].w;
                if (b0 + q * slices < blockIdx.x)
                    before.x += c[q].x, before.y += c[q].y, before.z += c[q].z, before.w += c[q].w;
            }
        }
        *reinterpret_cast<uint4*>(rows + (slice * 2) * bins + quad * 4) = before;
        *reinterpret_cast<uint4*>(rows + (slice * 2 + 1) * bins + quad * 4) = all;
    }
    __syncthreads();
    uint32_t carry = 0;
    for (int b0 = 0; b0 < bins; b0 += kSortThreads) {
        const int b = b0 + threadIdx.x;
        uint32_t before = 0, all = 0;
        if (b < bins)
            for (int s = 0; s < slices; ++s) {
                before += rows[s * 2 * bins + b];
                all += rows[(s * 2 + 1) * bins + b];
            }
        uint32_t scan = all;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const uint32_t up = __shfl_up_sync(~0u, scan, d);
            if (lane >= d) scan += up;
        }
        if (lane == 31) warp_sum[warp] = scan;
        __syncthreads();
        uint32_t lower = carry;
#pragma unroll
        for (int w = 0; w < kSortWarps; ++w) {
            if (w < warp) lower += warp_sum[w];
            carry += warp_sum[w];
        }
        if (b < bins) rows[b] = lower + scan - all + before;  // slice 0's counts of earlier blocks are used up
        __syncthreads();
    }
    const int64_t begin = (int64_t)blockIdx.x * a.steps * kSortThreads;
    const int64_t end = min((int64_t)a.n, begin + (int64_t)a.steps * kSortThreads);
    for (int64_t i0 = begin + threadIdx.x; i0 < end; i0 += kBatch * kSortThreads) {
        uint32_t k[kBatch], pos[kBatch], place[kBatch];
#pragma unroll
        for (int q = 0; q < kBatch; ++q) {
            const int64_t i = i0 + q * kSortThreads;
            if (i >= end) continue;
            k[q] = sort_key(a, pass, i, &pos[q]);
            place[q] = a.place[i];
        }
#pragma unroll
        for (int q = 0; q < kBatch; ++q)
            if (i0 + q * kSortThreads < end) a.out[rows[k[q] >> shift & (bins - 1)] + place[q]] = make_uint2(k[q], pos[q]);
    }
}

// Up to kSmallSort tokens: one block sorts (token, position) as one number by
// a bitonic network in shared memory, in one launch (60 tokens: 5.6 us; two
// radix passes 19, but 2048 tokens 30).
constexpr int kSmallSort = 256;

__global__ void __launch_bounds__(kSmallSort / 2) small_sort_kernel(SortArgs a, int padded) {
    __shared__ uint64_t item[kSmallSort];
    griddep_launch_dependents();
    griddep_wait();
    for (int i = threadIdx.x; i < padded; i += kSmallSort / 2) {
        uint32_t pos;
        item[i] = i < a.n ? (uint64_t)sort_key(a, 0, i, &pos) << 32 | (uint32_t)i : ~uint64_t(0);
    }
    __syncthreads();
    for (int size = 2; size <= padded; size *= 2)
        for (int d = size / 2; d > 0; d /= 2) {
            const int p = threadIdx.x;
            if (p < padded / 2) {
                const int lo = 2 * (p & ~(d - 1)) + (p & (d - 1)), hi = lo + d;
                const uint64_t x = item[lo], y = item[hi];
                if ((x > y) == ((lo & size) == 0)) {
                    item[lo] = y;
                    item[hi] = x;
                }
            }
            __syncthreads();
        }
    for (int i = threadIdx.x; i < a.n; i += kSmallSort / 2)
        a.out[i] = make_uint2((uint32_t)(item[i] >> 32), (uint32_t)item[i]);
}

// ---- sums ----

struct SumArgs {
    const uint2* pair;  // sorted (token, position)
    int n, window, windows;
    int64_t segments;
    const void* grad;
    int64_t grad_row, dim, vocab;
    float scale;
    void* d_table;
    float* head;  // [windows][dim] sums of a run that began in an earlier window
    float* tail;  // [windows][dim] sums of one that begins here and goes on
};

// Columns of a segment that a lane has: N (16 bytes), in accesses of B bytes
// that lie 32 lanes apart.
template <int DT, int B>
struct Columns {
    using E = Elem<DT>;
    using T = typename E::T;
    using V = typename Bytes<B>::T;
    static constexpr int N = 16 / (int)sizeof(T);
    static constexpr int kEach = B / (int)sizeof(T);  // columns of an access
    static constexpr int kSegment = 32 * N;
    int c0, left;  // first column; columns from there on (32-bit: one compare each)
    __device__ Columns(int64_t segment, int64_t dim)
        : c0((int)segment * kSegment + kEach * (threadIdx.x & 31)), left((int)dim - c0) {}
    static __device__ __forceinline__ constexpr int col(int i) { return i / kEach * (32 * kEach) + i % kEach; }
    __device__ __forceinline__ void load(const T* row, T (&v)[N]) const {
        row += c0;
#pragma unroll
        for (int i = 0; i < N; i += kEach)
            if (col(i) < left) *reinterpret_cast<V*>(v + i) = __ldg(reinterpret_cast<const V*>(row + col(i)));
    }
    __device__ __forceinline__ void store(T* row, const float (&s)[N], float scale) const {
        alignas(16) T v[N];
        row += c0;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = E::put(s[i] * scale);
#pragma unroll
        for (int i = 0; i < N; i += kEach)
            if (col(i) < left) *reinterpret_cast<V*>(row + col(i)) = *reinterpret_cast<V*>(v + i);
    }
    // fp32 scratch, whose rows are dim long: 16-byte accesses where rows allow
    static constexpr int kWide = B == 16 ? 4 : 1;
    __device__ __forceinline__ void load32(const float* row, float (&s)[N]) const {
        row += c0;
#pragma unroll
        for (int i = 0; i < N; i += kWide)
            if (col(i) < left) {
                if constexpr (kWide == 4) {
                    const float4 f = *reinterpret_cast<const float4*>(row + col(i));
                    s[i] = f.x, s[i + 1] = f.y, s[i + 2] = f.z, s[i + 3] = f.w;
                } else {
                    s[i] = row[col(i)];
                }
            }
    }
    __device__ __forceinline__ void store32(float* row, const float (&s)[N]) const {
        row += c0;
#pragma unroll
        for (int i = 0; i < N; i += kWide)
            if (col(i) < left) {
                if constexpr (kWide == 4)
                    *reinterpret_cast<float4*>(row + col(i)) = make_float4(s[i], s[i + 1], s[i + 2], s[i + 3]);
                else
                    row[col(i)] = s[i];
            }
    }
};

constexpr int kAhead = 8;  // rows in flight per warp

// The sorted tokens, for lower_bound.
struct SortedTokens {
    const uint2* pair;
    __device__ __forceinline__ uint32_t operator()(int i) const { return pair[i].x; }
};

// Zeros to a row of any alignment.
template <int DT>
__device__ __forceinline__ void zero_row(typename Elem<DT>::T* row, int64_t dim, int lane) {
    using T = typename Elem<DT>::T;
    constexpr int N = 16 / (int)sizeof(T);
    const int64_t head = min(dim, (int64_t)((-reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T)));
    const int64_t body = (dim - head) / N, tail = head + body * N;
    if (lane < head) row[lane] = Elem<DT>::put(0.0f);
    uint4* p = reinterpret_cast<uint4*>(row + head);
    for (int64_t i = lane; i < body; i += 32) p[i] = make_uint4(0, 0, 0, 0);
    if (tail + lane < dim) row[tail + lane] = Elem<DT>::put(0.0f);
}

// The first zero_blocks blocks write zeros to the rows, of zero_rows entries
// each, that no token names (first, so that their searches overlap the
// sums); the others sum the windows, a warp per window and segment.
template <int DT, int B>
__global__ void __launch_bounds__(256, 3) sum_kernel(SumArgs a, int64_t zero_blocks, int zero_rows) {
    using C = Columns<DT, B>;
    using T = typename C::T;
    constexpr int N = C::N;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    griddep_launch_dependents();
    griddep_wait();
    if (blockIdx.x < zero_blocks) {
        __shared__ bool empty[256];
        const int64_t v0 = (int64_t)blockIdx.x * zero_rows, v = v0 + threadIdx.x;
        bool none = false;
        if (threadIdx.x < zero_rows && v < a.vocab) {
            const int at = lower_bound(SortedTokens{a.pair}, a.n, (uint32_t)v);
            none = at == a.n || a.pair[at].x != (uint32_t)v;
        }
        empty[threadIdx.x] = none;
        __syncthreads();
        for (int r = warp; r < zero_rows; r += 8)
            if (empty[r]) zero_row<DT>(static_cast<T*>(a.d_table) + (v0 + r) * a.dim, a.dim, lane);
        return;
    }
    const int64_t task = (blockIdx.x - zero_blocks) * 8 + warp;
    const int64_t window = task / a.segments;
    if (window >= a.windows) return;
    const C c(task % a.segments, a.dim);
    const int s0 = (int)window * a.window, s1 = min(a.n, s0 + a.window);
    uint32_t run = a.pair[s0].x;
    const uint32_t before = s0 > 0 ? a.pair[s0 - 1].x : ~0u, after = s1 < a.n ? a.pair[s1].x : ~0u;
    if (run >= a.vocab) return;
    bool from_prev = before == run;
    float sum[N] = {};
    for (int j0 = s0; j0 < s1; j0 += 32) {
        const uint2 u = j0 + lane < s1 ? a.pair[j0 + lane] : make_uint2(~0u, 0);
        const int valid = __popc(__ballot_sync(~0u, u.x < a.vocab));  // padding comes last
        uint32_t up = __shfl_up_sync(~0u, u.x, 1);
        if (lane == 0) up = run;
        const uint32_t starts = __ballot_sync(~0u, u.x != up);
        for (int j = 0; j < valid; j += kAhead) {
            alignas(16) T v[kAhead][N];
#pragma unroll
            for (int q = 0; q < kAhead; ++q) {
                const uint32_t at = __shfl_sync(~0u, u.y, j + q);
                if (j + q < valid) c.load(static_cast<const T*>(a.grad) + at * a.grad_row, v[q]);
            }
#pragma unroll
            for (int q = 0; q < kAhead; ++q) {
                if (j + q >= valid) break;
                if (starts >> (j + q) & 1) {
                    if (from_prev) c.store32(a.head + window * a.dim, sum);
                    else c.store(static_cast<T*>(a.d_table) + run * a.dim, sum, a.scale);
                    from_prev = false;
                    run = __shfl_sync(~0u, u.x, j + q);
#pragma unroll
                    for (int i = 0; i < N; ++i) sum[i] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < N; ++i) sum[i] += C::E::get(v[q][i]);
            }
        }
        if (valid < 32) break;
    }
    if (from_prev) c.store32(a.head + window * a.dim, sum);
    else if (after == run) c.store32(a.tail + window * a.dim, sum);
    else c.store(static_cast<T*>(a.d_table) + run * a.dim, sum, a.scale);
}

// Adds the parts of the runs that begin in windows 8 blockIdx.x .. + 7 and
// go past their end.  A run of up to 32 windows more is its warp's own work;
// for a longer one the block's warps take equal stretches of its windows.
template <int DT, int B>
__global__ void __launch_bounds__(256, 3) join_kernel(SumArgs a) {
    using C = Columns<DT, B>;
    using T = typename C::T;
    constexpr int N = C::N;
    __shared__ float part[8][32][N + 1];
    __shared__ uint32_t runs[8];  // the long ones
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const C c(blockIdx.y, a.dim);
    griddep_wait();
    const auto add_windows = [&](int64_t from, int64_t to, float (&sum)[N]) {
        constexpr int kMore = 32 / N;
        for (int64_t w0 = from; w0 < to; w0 += kMore) {
            float v[kMore][N];
#pragma unroll
            for (int q = 0; q < kMore; ++q)
                if (w0 + q < to) c.load32(a.head + (w0 + q) * a.dim, v[q]);
#pragma unroll
            for (int q = 0; q < kMore; ++q)
                if (w0 + q < to)
#pragma unroll
                    for (int i = 0; i < N; ++i) sum[i] += v[q][i];
        }
    };
    {
        const int64_t w = (int64_t)blockIdx.x * 8 + warp;
        const int64_t s0 = w * a.window, s1 = s0 + a.window;
        uint32_t run = ~0u;
        if (s1 < a.n) {
            const uint32_t k = a.pair[s1 - 1].x, next = a.pair[s1].x, before = s0 > 0 ? a.pair[s0 - 1].x : ~0u;
            if (k < a.vocab && next == k && before != k) run = k;
        }
        // the windows that go on with the run: those whose first token is its own
        const int64_t x = w + 1 + lane;
        const uint32_t first = x < a.windows ? a.pair[x * a.window].x : ~0u;
        const int more = __popc(__ballot_sync(~0u, run != ~0u && first == run));
        if (lane == 0) runs[warp] = more == 32 ? run : ~0u;
        if (run != ~0u && more < 32) {
            float sum[N];
            c.load32(a.tail + w * a.dim, sum);
            add_windows(w + 1, w + 1 + more, sum);
            c.store(static_cast<T*>(a.d_table) + run * a.dim, sum, a.scale);
        }
    }
    __syncthreads();
    for (int r = 0; r < 8; ++r) {
        const uint32_t run = runs[r];
        if (run == ~0u) continue;
        const int64_t window = (int64_t)blockIdx.x * 8 + r;
        int64_t last = window;
        for (int more = 256; more == 256; last += more) {
            const int64_t x = last + 1 + threadIdx.x;
            more = __syncthreads_count(x < a.windows && a.pair[x * a.window].x == run);
        }
        const int64_t per = (last - window + 7) / 8;
        const int64_t from = window + 1 + warp * per;
        float sum[N] = {};
        add_windows(from, min(last + 1, from + per), sum);
#pragma unroll
        for (int i = 0; i < N; ++i) part[warp][lane][i] = sum[i];
        __syncthreads();
        if (warp == 0) {
            c.load32(a.tail + window * a.dim, sum);
            for (int w = 0; w < 8; ++w)
#pragma unroll
                for (int i = 0; i < N; ++i) sum[i] += part[w][lane][i];
            c.store(static_cast<T*>(a.d_table) + run * a.dim, sum, a.scale);
        }
        __syncthreads();
    }
}

template <int DT, int B>
void sum_rows(SumArgs a, Queue& q) {
    const int64_t sum_blocks = ((int64_t)a.windows * a.segments + 7) / 8;
    // as many blocks for the empty rows as fill the card, up to 256 rows each
    const int zero_rows = (int)std::clamp<int64_t>(a.vocab / (148 * 4) / 8 * 8, 8, 256);
    const int64_t zero_blocks = (a.vocab + zero_rows - 1) / zero_rows, blocks = zero_blocks + sum_blocks;
    need(blocks < (int64_t(1) << 31) && a.segments <= 65535, "n times dim is too large");
    q.launch("sum_kernel", sum_kernel<DT, B>, dim3((unsigned)blocks), 256, 0, a, zero_blocks, zero_rows);
    if (a.windows > 1)
        q.launch("join_kernel", join_kernel<DT, B>, dim3((unsigned)((a.windows + 7) / 8), (unsigned)a.segments), 256,
                 0, a);
}

void plan_sort(SortArgs& a) {
    int total = 2;
    while ((int64_t(1) << total) <= a.vocab) ++total;  // vocab itself is a key
    a.passes = (total + kMaxBits - 1) / kMaxBits;
    a.bits = (total + a.passes - 1) / a.passes;
    const int64_t per_step = kSortThreads;
    a.steps = (int)std::max<int64_t>(2, (a.n + 148 * per_step - 1) / (148 * per_step));
    a.blocks = (int)((a.n + a.steps * per_step - 1) / (a.steps * per_step));
}

void sort(SortArgs a, Queue& q) {
    if (a.n <= kSmallSort) {
        a.out = a.pair[a.passes & 1];
        int padded = 2;
        while (padded < a.n) padded *= 2;
        q.launch("small_sort_kernel", small_sort_kernel, dim3(1), kSmallSort / 2, 0, a, padded);
        return;
    }
    const int bins = 1 << a.bits, slices = std::max(1, kSortThreads / (bins / 4));
    const int most = kSortWarps * (4 << kMaxBits);
    check(cudaFuncSetAttribute(rank_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most),
          "cudaFuncSetAttribute(rank_kernel)");
    for (int pass = 0; pass < a.passes; ++pass) {
        a.in = a.pair[pass & 1];
        a.out = a.pair[(pass + 1) & 1];
        q.launch("rank_kernel", rank_kernel, dim3(a.blocks), kSortThreads, kSortWarps * bins * 4, a, pass);
        q.launch("scatter_kernel", scatter_kernel, dim3(a.blocks), kSortThreads, slices * 2 * bins * 4, a, pass);
    }
}

template <int DT>
void embed_backward(const mg_embed_backward_args& a, Workspace& w, bool go, Queue& q) {
    const int e = elem_bytes(DT);
    if (a.n == 0) {
        if (go) q.clear(a.d_table, (size_t)a.vocab * a.dim * e);
        return;
    }
    SortArgs sort_args{};
    sort_args.tokens = a.tokens;
    sort_args.token_bytes = a.token_bytes;
    sort_args.token_stride = a.token_stride;
    sort_args.vocab = a.vocab;
    sort_args.n = (int)a.n;
    plan_sort(sort_args);
    for (int i = 0; i < 2; ++i) sort_args.pair[i] = w.take<uint2>((size_t)a.n * 8);
    sort_args.place = w.take<uint32_t>((size_t)a.n * 4);
    sort_args.counts = w.take<uint32_t>((size_t)sort_args.blocks * 4 << sort_args.bits);
    SumArgs sum{};
    sum.n = (int)a.n;
    const int segment = 32 * 16 / e;
    sum.segments = (a.dim + segment - 1) / segment;
    // Windows long enough that few runs cross them, and as many as the card's warps (24 on
    // each SM) can take in equal rounds: 128 tokens at most and a last round of a few blocks
    // made it 109 us instead of 96 for 100003 tokens of 1000, 73 instead of 60 for 30000 of 2048.
    const int64_t warps = 148 * 24, work = a.n * sum.segments, rounds = (work + warps * 256 - 1) / (warps * 256);
    sum.window = (int)std::max<int64_t>(16, ((work + warps * rounds - 1) / (warps * rounds) + 7) / 8 * 8);
    sum.windows = (int)((a.n + sum.window - 1) / sum.window);
    sum.head = w.take<float>((size_t)sum.windows * a.dim * 4);
    sum.tail = w.take<float>((size_t)sum.windows * a.dim * 4);
    if (!go) return;
    w.require();
    sort(sort_args, q);
    sum.pair = sort_args.pair[sort_args.passes & 1];
    sum.grad = a.grad;
    sum.grad_row = a.grad_row;
    sum.dim = a.dim;
    sum.vocab = a.vocab;
    sum.scale = a.scale;
    sum.d_table = a.d_table;
    switch (widest(e, a.dim * e, a.grad_row * e, 0, a.grad, a.d_table)) {
        case 16: return sum_rows<DT, 16>(sum, q);
        case 8: return sum_rows<DT, 8>(sum, q);
        case 4: return sum_rows<DT, 4>(sum, q);
        default:
            if constexpr (DT != MG_PREC_FP32) sum_rows<DT, 2>(sum, q);
    }
}

void embed_backward(const mg_embed_backward_args& a, Workspace& w, bool go, Queue& q) {
    if (a.dtype == MG_PREC_BF16) embed_backward<MG_PREC_BF16>(a, w, go, q);
    else if (a.dtype == MG_PREC_FP16) embed_backward<MG_PREC_FP16>(a, w, go, q);
    else embed_backward<MG_PREC_FP32>(a, w, go, q);
}

void check_tokens(const void* p, int bytes, int64_t stride, int64_t n) {
    need(bytes == 8 || bytes == 4, "tokens are int64 or int32 (token_bytes 8 or 4)");
    need(n == 0 || p != nullptr, "tokens is null");
    need(stride >= 0, "token_stride is negative");
    need_aligned(p, bytes, "tokens");
}

void check_args(const mg_embed_args& a) {
    need(a.n >= 0 && a.vocab >= 1 && a.dim >= 1, "sizes: n >= 0, vocab >= 1, dim >= 1");
    need(a.vocab < (int64_t(1) << 31), "vocab must be below 2^31");
    need(a.dtype >= MG_PREC_BF16 && a.dtype <= MG_PREC_FP32, "dtype is not an MG_PREC_* value");
    check_tokens(a.tokens, a.token_bytes, a.token_stride, a.n);
    need(a.table_row >= 0, "table_row is negative");
    need(a.n == 0 || (a.table != nullptr && a.out != nullptr), "table or out is null");
    need_aligned(a.table, elem_bytes(a.dtype), "table");
    need_aligned(a.out, elem_bytes(a.dtype), "out");
}

void check_args(const mg_embed_backward_args& a) {
    need(a.n >= 0 && a.vocab >= 1 && a.dim >= 1, "sizes: n >= 0, vocab >= 1, dim >= 1");
    need(a.n < (int64_t(1) << 31) - 1024 && a.vocab < (int64_t(1) << 31) && a.dim < (int64_t(1) << 30),
         "n must be below 2^31 - 1024, vocab below 2^31, dim below 2^30");
    need(a.dtype >= MG_PREC_BF16 && a.dtype <= MG_PREC_FP32, "dtype is not an MG_PREC_* value");
    check_tokens(a.tokens, a.token_bytes, a.token_stride, a.n);
    need(a.grad_row >= 0, "grad_row is negative");
    need(a.d_table != nullptr && (a.n == 0 || a.grad != nullptr), "grad or d_table is null");
    need_aligned(a.grad, elem_bytes(a.dtype), "grad");
    need_aligned(a.d_table, elem_bytes(a.dtype), "d_table");
}

}  // namespace
}  // namespace ops
}  // namespace mgb

using namespace mgb::ops;

extern "C" int mg_embed(const mg_embed_args* args, void* stream) {
    return guarded([&] {
        need(args != nullptr, "args is null");
        check_args(*args);
        if (args->n == 0) return;
        OnDevice on(args->device);
        Queue q(stream);
        if (args->dtype == MG_PREC_BF16) embed<MG_PREC_BF16>(*args, q);
        else if (args->dtype == MG_PREC_FP16) embed<MG_PREC_FP16>(*args, q);
        else embed<MG_PREC_FP32>(*args, q);
    });
}

extern "C" int mg_embed_backward_workspace(const mg_embed_backward_args* args, size_t* bytes) {
    return guarded([&] {
        need(args != nullptr && bytes != nullptr, "args or bytes is null");
        check_args(*args);
        Workspace w;
        Queue q(nullptr);
        embed_backward(*args, w, false, q);
        *bytes = w.used();
    });
}

extern "C" int mg_embed_backward(const mg_embed_backward_args* args, void* workspace,
                                 size_t workspace_bytes, void* stream) {
    return guarded([&] {
        need(args != nullptr, "args is null");
        check_args(*args);
        OnDevice on(args->device);
        Workspace w(workspace, workspace_bytes);
        Queue q(stream);
        embed_backward(*args, w, true, q);
    });
}
