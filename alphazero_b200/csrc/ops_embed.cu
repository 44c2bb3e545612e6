// Embedding lookup with scaling and its gradient (include/minigo_ops.h).
// Both are bound by memory: each moves n rows of dim elements once.
//
// Lookup: a group of lanes per row, up to four independent loads of up to 16
// bytes per lane; rows longer than that are cut into segments on the grid's
// other axis, so that a few long rows still fill the card.
//
// Gradient: the tokens are sorted (stable, so equal tokens stay in order of
// position), then cut into windows of equal length whatever the tokens are.
// A warp sums a window's rows run by run (a run: equal tokens) for one
// segment of columns.  A run inside one window is written at once; the parts
// of one that crosses windows go to scratch and are added by join_kernel in
// window order.  So a token that makes up a tenth of the batch is spread
// over as many warps as its rows deserve, there are no atomics on sums, and
// the result does not depend on the order in which blocks run.
#include "ops_common.cuh"
#include "ptx_sm100.cuh"

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

constexpr int kPerLane = 4;  // vectors of a segment that a lane holds

// `lanes` (a power of two up to 32) per row and segment; chunks = vectors per row.
template <int DT, int B>
__global__ void __launch_bounds__(256) embed_kernel(mg_embed_args a, int64_t chunks, int lanes) {
    using E = Elem<DT>;
    using T = typename E::T;
    using V = typename Bytes<B>::T;
    constexpr int N = B / (int)sizeof(T);
    const int lane = threadIdx.x & (lanes - 1);
    const int64_t c0 = (int64_t)blockIdx.y * (kPerLane * lanes) + lane;
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) / lanes; i < a.n;
         i += (int64_t)gridDim.x * 256 / lanes) {
        const int64_t t = index_at(a.tokens, a.token_bytes, i * a.token_stride, a.vocab);
        const V* row = reinterpret_cast<const V*>(static_cast<const T*>(a.table) + t * a.table_row);
        V* out = reinterpret_cast<V*>(static_cast<T*>(a.out) + i * a.dim);
        alignas(16) V v[kPerLane];
#pragma unroll
        for (int q = 0; q < kPerLane; ++q)
            if (c0 + q * lanes < chunks && t >= 0) v[q] = __ldg(row + c0 + q * lanes);
#pragma unroll
        for (int q = 0; q < kPerLane; ++q) {
            if (c0 + q * lanes >= chunks) continue;
            alignas(16) T e[N];
            *reinterpret_cast<V*>(e) = v[q];
#pragma unroll
            for (int j = 0; j < N; ++j) e[j] = E::put(t < 0 ? 0.0f : E::get(e[j]) * a.scale);
            out[c0 + q * lanes] = *reinterpret_cast<V*>(e);
        }
    }
}

template <int DT, int B>
void embed_with(const mg_embed_args& a, cudaStream_t s) {
    const int64_t chunks = a.dim * elem_bytes(DT) / B;
    int lanes = 1;
    while (lanes < 32 && lanes < chunks) lanes *= 2;
    const int64_t rows_per_block = 256 / lanes, segments = (chunks + kPerLane * lanes - 1) / (kPerLane * lanes);
    const dim3 grid((unsigned)std::min<int64_t>((a.n + rows_per_block - 1) / rows_per_block, 1 << 30),
                    (unsigned)segments);
    need(segments <= 65535, "dim is too large");
    embed_kernel<DT, B><<<grid, 256, 0, s>>>(a, chunks, lanes);
    launched("embed_kernel");
}

template <int DT>
void embed(const mg_embed_args& a, cudaStream_t s) {
    const int e = elem_bytes(DT);
    switch (widest(e, a.dim * e, a.table_row * e, 0, a.table, a.out)) {
        case 16: return embed_with<DT, 16>(a, s);
        case 8: return embed_with<DT, 8>(a, s);
        case 4: return embed_with<DT, 4>(a, s);
        default:
            if constexpr (DT != MG_PREC_FP32) embed_with<DT, 2>(a, s);
    }
}

// ---- sort ----

constexpr int kSortWarps = 32;
constexpr int kSortCtas = 8;   // of the cluster
constexpr int kMaxBits = 10;   // of the key per pass

struct SortArgs {
    const void* tokens;
    int token_bytes;
    int64_t token_stride, vocab;
    int n, passes, bits;
    uint32_t* key[2];
    uint32_t* pos[2];
};

// Stable least-significant-digit radix sort of (token, position), padding
// last as token `vocab`, by one cluster: its barriers order the passes, and
// the digit counts travel through distributed shared memory.  Warp w of CTA
// c has the (32 c + w)-th stretch of the input and its own row of counts,
// which after a scan over digits, CTAs and warps are the places its tokens
// go to.  The result is in key[passes & 1], pos[passes & 1].
__global__ void __launch_bounds__(32 * kSortWarps) sort_kernel(SortArgs a) {
    extern __shared__ uint32_t counts[];  // [warps][bins], then [bins] sums of the CTA
    const int bins = 1 << a.bits;
    uint32_t* total = counts + kSortWarps * bins;
    __shared__ uint32_t warp_sum[kSortWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    uint32_t ctas;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
    const int64_t per = ((int64_t)a.n + ctas * kSortWarps * 32 - 1) / (ctas * kSortWarps * 32) * 32;
    const int64_t begin = min((int64_t)a.n, ((int64_t)rank * kSortWarps + warp) * per);
    const int64_t end = min((int64_t)a.n, begin + per);
    uint32_t* mine = counts + warp * bins;

    for (int pass = 0; pass < a.passes; ++pass) {
        const uint32_t* kin = a.key[pass & 1];
        const uint32_t* pin = a.pos[pass & 1];
        uint32_t* kout = a.key[(pass + 1) & 1];
        uint32_t* pout = a.pos[(pass + 1) & 1];
        const int shift = pass * a.bits;
        const auto key_at = [&](int64_t i) -> uint32_t {
            if (pass > 0) return __ldcg(kin + i);
            const int64_t t = index_at(a.tokens, a.token_bytes, i * a.token_stride, a.vocab);
            return (uint32_t)(t < 0 ? a.vocab : t);
        };
        for (int b = threadIdx.x; b < kSortWarps * bins; b += blockDim.x) counts[b] = 0;
        __syncthreads();
#pragma unroll 4
        for (int64_t i = begin + lane; i < end; i += 32) atomicAdd(&mine[key_at(i) >> shift & (bins - 1)], 1u);
        __syncthreads();
        // bin `threadIdx.x`: counts of the warps before each warp, sum of the CTA
        if (threadIdx.x < bins) {
            uint32_t s = 0;
            for (int w = 0; w < kSortWarps; ++w) {
                const uint32_t c = counts[w * bins + threadIdx.x];
                counts[w * bins + threadIdx.x] = s;
                s += c;
            }
            total[threadIdx.x] = s;
        }
        cluster_sync();
        uint32_t before = 0, all = 0;
        if (threadIdx.x < bins)
            for (uint32_t r = 0; r < ctas; ++r) {
                uint32_t c;
                asm volatile("ld.shared::cluster.u32 %0, [%1];"
                             : "=r"(c)
                             : "r"(map_to_rank(smem_u32(&total[threadIdx.x]), r))
                             : "memory");
                if (r < rank) before += c;
                all += c;
            }
        uint32_t scan = all;
        for (int d = 1; d < 32; d *= 2) {
            const uint32_t up = __shfl_up_sync(~0u, scan, d);
            if (lane >= d) scan += up;
        }
        if (lane == 31) warp_sum[warp] = scan;
        __syncthreads();
        if (warp == 0) {
            uint32_t v = warp_sum[lane], inc = v;
            for (int d = 1; d < 32; d *= 2) {
                const uint32_t up = __shfl_up_sync(~0u, inc, d);
                if (lane >= d) inc += up;
            }
            warp_sum[lane] = inc - v;
        }
        __syncthreads();
        if (threadIdx.x < bins) {
            const uint32_t base = warp_sum[warp] + scan - all + before;
            for (int w = 0; w < kSortWarps; ++w) counts[w * bins + threadIdx.x] += base;
        }
        __syncthreads();
        for (int64_t i0 = begin; i0 < end; i0 += 32) {
            const int64_t i = i0 + lane;
            const bool in = i < end;
            const uint32_t k = in ? key_at(i) : 0;
            const uint32_t p = !in ? 0 : pass > 0 ? __ldcg(pin + i) : (uint32_t)i;
            const uint32_t digit = in ? k >> shift & (bins - 1) : (uint32_t)bins + lane;
            const uint32_t peers = __match_any_sync(~0u, digit);
            const uint32_t below = __popc(peers & ((1u << lane) - 1));
            const uint32_t to = in ? mine[digit] + below : 0;
            __syncwarp();
            if (in && below == 0) mine[digit] += __popc(peers);
            __syncwarp();
            if (in) {
                kout[to] = k;
                pout[to] = p;
            }
        }
        cluster_sync();  // before the next pass reads what this one wrote (and reuses the counts)
    }
}

// ---- sums ----

struct SumArgs {
    const uint32_t* key;  // sorted
    const uint32_t* pos;
    int n, window, windows;
    int64_t segments;
    const void* grad;
    int64_t grad_row, dim, vocab;
    float scale;
    void* d_table;
    float* head;  // [windows][dim] sums of a run that began in an earlier window
    float* tail;  // [windows][dim] sums of one that begins here and goes on
};

// Columns of a segment that a lane has: N adjacent ones with 16-byte
// accesses, otherwise N of them 32 apart.
template <int DT, bool VEC>
struct Columns {
    using E = Elem<DT>;
    using T = typename E::T;
    static constexpr int N = 16 / (int)sizeof(T);
    static constexpr int kSegment = 32 * N;
    int64_t c0, dim;
    __device__ Columns(int64_t segment, int64_t dim) : c0(segment * kSegment + (VEC ? N : 1) * (threadIdx.x & 31)), dim(dim) {}
    __device__ __forceinline__ int64_t col(int i) const { return c0 + (VEC ? i : 32 * i); }
    __device__ __forceinline__ void load(const T* row, T (&v)[N]) const {
        if constexpr (VEC) {
            if (c0 < dim) *reinterpret_cast<uint4*>(v) = __ldg(reinterpret_cast<const uint4*>(row + c0));
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (col(i) < dim) v[i] = row[col(i)];
        }
    }
    __device__ __forceinline__ void store(T* row, const float (&s)[N], float scale) const {
        alignas(16) T v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = E::put(s[i] * scale);
        if constexpr (VEC) {
            if (c0 < dim) *reinterpret_cast<uint4*>(row + c0) = *reinterpret_cast<uint4*>(v);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (col(i) < dim) row[col(i)] = v[i];
        }
    }
    __device__ __forceinline__ void load32(const float* row, float (&s)[N]) const {
#pragma unroll
        for (int i = 0; i < N; i += VEC ? 4 : 1)
            if (col(i) < dim) {
                if constexpr (VEC) {
                    const float4 f = *reinterpret_cast<const float4*>(row + col(i));
                    s[i] = f.x, s[i + 1] = f.y, s[i + 2] = f.z, s[i + 3] = f.w;
                } else {
                    s[i] = row[col(i)];
                }
            }
    }
    __device__ __forceinline__ void store32(float* row, const float (&s)[N]) const {
#pragma unroll
        for (int i = 0; i < N; i += VEC ? 4 : 1)
            if (col(i) < dim) {
                if constexpr (VEC)
                    *reinterpret_cast<float4*>(row + col(i)) = make_float4(s[i], s[i + 1], s[i + 2], s[i + 3]);
                else
                    row[col(i)] = s[i];
            }
    }
};

constexpr int kAhead = 8;  // rows in flight per warp

// First place in the sorted keys whose key is at least v.
__device__ __forceinline__ int lower_bound(const uint32_t* key, int n, uint32_t v) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (key[mid] < v) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// Blocks [0, sum_blocks) sum the windows, a warp per window and segment; the
// others write zeros to the rows of 256 entries each that no token names.
template <int DT, bool VEC>
__global__ void __launch_bounds__(256) sum_kernel(SumArgs a, int64_t sum_blocks) {
    using C = Columns<DT, VEC>;
    using T = typename C::T;
    constexpr int N = C::N;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (blockIdx.x >= sum_blocks) {
        __shared__ bool empty[256];
        const int64_t v0 = (blockIdx.x - sum_blocks) * 256, v = v0 + threadIdx.x;
        bool none = false;
        if (v < a.vocab) {
            const int at = lower_bound(a.key, a.n, (uint32_t)v);
            none = at == a.n || a.key[at] != (uint32_t)v;
        }
        empty[threadIdx.x] = none;
        __syncthreads();
        const float zero[N] = {};
        for (int r = warp; r < 256; r += 8)
            if (empty[r])
                for (int64_t s = 0; s < a.segments; ++s)
                    C(s, a.dim).store(static_cast<T*>(a.d_table) + (v0 + r) * a.dim, zero, 1.0f);
        return;
    }
    const int64_t task = (int64_t)blockIdx.x * 8 + warp;
    const int64_t window = task / a.segments;
    if (window >= a.windows) return;
    const C c(task % a.segments, a.dim);
    const int s0 = (int)window * a.window, s1 = min(a.n, s0 + a.window);
    uint32_t run = a.key[s0];
    bool from_prev = s0 > 0 && a.key[s0 - 1] == run;
    float sum[N] = {};
    const auto flush = [&](bool to_next) {
        if (from_prev) c.store32(a.head + window * a.dim, sum);
        else if (to_next) c.store32(a.tail + window * a.dim, sum);
        else c.store(static_cast<T*>(a.d_table) + (int64_t)run * a.dim, sum, a.scale);
    };
    for (int j0 = s0; j0 < s1 && run < a.vocab; j0 += 32) {
        const int have = min(32, s1 - j0);
        const uint32_t k = lane < have ? a.key[j0 + lane] : ~0u;
        const uint32_t p = lane < have ? a.pos[j0 + lane] : 0;
        for (int j = 0; j < have; j += kAhead) {
            alignas(16) T v[kAhead][N];
#pragma unroll
            for (int q = 0; q < kAhead; ++q) {
                const uint32_t at = __shfl_sync(~0u, p, j + q), key = __shfl_sync(~0u, k, j + q);
                if (key < a.vocab) c.load(static_cast<const T*>(a.grad) + (int64_t)at * a.grad_row, v[q]);
            }
#pragma unroll
            for (int q = 0; q < kAhead; ++q) {
                const uint32_t key = __shfl_sync(~0u, k, j + q);
                if (key >= a.vocab && key != run && j + q >= have) continue;  // past the window
                if (key != run) {
                    if (run < a.vocab) flush(false);
                    run = key;
                    from_prev = false;
#pragma unroll
                    for (int i = 0; i < N; ++i) sum[i] = 0.0f;
                }
                if (key < a.vocab)
#pragma unroll
                    for (int i = 0; i < N; ++i) sum[i] += C::E::get(v[q][i]);
            }
        }
    }
    if (run < a.vocab) flush(s1 < a.n && a.key[s1] == run);
}

// Adds the parts of the run that begins in window blockIdx.x and goes past
// its end; the block's warps take equal stretches of its windows.
template <int DT, bool VEC>
__global__ void __launch_bounds__(256) join_kernel(SumArgs a) {
    using C = Columns<DT, VEC>;
    using T = typename C::T;
    constexpr int N = C::N;
    const int64_t window = blockIdx.x;
    const int s0 = (int)window * a.window, s1 = s0 + a.window;
    if (s1 >= a.n) return;
    const uint32_t run = a.key[s1 - 1];
    if (run >= a.vocab || a.key[s1] != run) return;                                // ends here
    if (a.key[s0] == run && s0 > 0 && a.key[s0 - 1] == run) return;                // began earlier
    const int warp = threadIdx.x >> 5;
    __shared__ float part[8][32][N + 1];
    const int64_t last = (lower_bound(a.key + s1, a.n - s1, run + 1) + s1 - 1) / a.window;
    const int64_t per = (last - window + 7) / 8;
    const C c(blockIdx.y, a.dim);
    float sum[N] = {};
    const int64_t from = window + 1 + warp * per, to = min(last + 1, from + per);
    for (int64_t w0 = from; w0 < to; w0 += kAhead) {
        float v[kAhead][N];
#pragma unroll
        for (int q = 0; q < kAhead; ++q)
            if (w0 + q < to) c.load32(a.head + (w0 + q) * a.dim, v[q]);
#pragma unroll
        for (int q = 0; q < kAhead; ++q)
            if (w0 + q < to)
#pragma unroll
                for (int i = 0; i < N; ++i) sum[i] += v[q][i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) part[warp][threadIdx.x & 31][i] = sum[i];
    __syncthreads();
    if (warp > 0) return;
    c.load32(a.tail + window * a.dim, sum);
    for (int w = 0; w < 8; ++w)
#pragma unroll
        for (int i = 0; i < N; ++i) sum[i] += part[w][threadIdx.x][i];
    c.store(static_cast<T*>(a.d_table) + (int64_t)run * a.dim, sum, a.scale);
}

template <int DT, bool VEC>
void sum_rows(SumArgs a, cudaStream_t s) {
    const int64_t sum_blocks = ((int64_t)a.windows * a.segments + 7) / 8;
    const int64_t blocks = sum_blocks + (a.vocab + 255) / 256;
    need(blocks < (int64_t(1) << 31) && a.segments <= 65535, "n times dim is too large");
    sum_kernel<DT, VEC><<<(unsigned)blocks, 256, 0, s>>>(a, sum_blocks);
    launched("sum_kernel");
    if (a.windows > 1) {
        join_kernel<DT, VEC><<<dim3((unsigned)a.windows, (unsigned)a.segments), 256, 0, s>>>(a);
        launched("join_kernel");
    }
}

void sort(SortArgs& a, cudaStream_t s) {
    int total = 1;
    while ((int64_t(1) << total) <= a.vocab) ++total;  // vocab itself is a key
    a.passes = (total + kMaxBits - 1) / kMaxBits;
    a.bits = (total + a.passes - 1) / a.passes;
    const int smem = (kSortWarps + 1) * (4 << a.bits);
    check(cudaFuncSetAttribute(sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               (kSortWarps + 1) * (4 << kMaxBits)),
          "cudaFuncSetAttribute(sort_kernel)");
    cudaLaunchConfig_t cfg{};
    // one CTA while each of its warps has at most a few steps of 32 tokens
    const unsigned ctas = a.n <= 4096 ? 1 : kSortCtas;
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(32 * kSortWarps);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = ctas;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    check(cudaLaunchKernelEx(&cfg, sort_kernel, a), "sort_kernel");
}

template <int DT>
void embed_backward(const mg_embed_backward_args& a, Workspace& w, bool go, cudaStream_t s) {
    const int e = elem_bytes(DT);
    if (a.n == 0) {
        if (go) check(cudaMemsetAsync(a.d_table, 0, (size_t)a.vocab * a.dim * e, s), "cudaMemsetAsync");
        return;
    }
    SortArgs sort_args{};
    sort_args.tokens = a.tokens;
    sort_args.token_bytes = a.token_bytes;
    sort_args.token_stride = a.token_stride;
    sort_args.vocab = a.vocab;
    sort_args.n = (int)a.n;
    for (int i = 0; i < 2; ++i) {
        sort_args.key[i] = w.take<uint32_t>((size_t)a.n * 4);
        sort_args.pos[i] = w.take<uint32_t>((size_t)a.n * 4);
    }
    const bool vec = widest(e, a.dim * e, a.grad_row * e, 0, a.grad, a.d_table) == 16;
    SumArgs sum{};
    sum.n = (int)a.n;
    const int segment = 32 * 16 / e;
    sum.segments = (a.dim + segment - 1) / segment;
    // windows long enough that few runs cross them, short enough for 24 warps per SM
    sum.window = (int)std::clamp<int64_t>(a.n * sum.segments / (148 * 24) / 8 * 8, 16, 128);
    sum.windows = (int)((a.n + sum.window - 1) / sum.window);
    sum.head = w.take<float>((size_t)sum.windows * a.dim * 4);
    sum.tail = w.take<float>((size_t)sum.windows * a.dim * 4);
    if (!go) return;
    w.require();
    sort(sort_args, s);
    sum.key = sort_args.key[sort_args.passes & 1];
    sum.pos = sort_args.pos[sort_args.passes & 1];
    sum.grad = a.grad;
    sum.grad_row = a.grad_row;
    sum.dim = a.dim;
    sum.vocab = a.vocab;
    sum.scale = a.scale;
    sum.d_table = a.d_table;
    if (vec) sum_rows<DT, true>(sum, s);
    else sum_rows<DT, false>(sum, s);
}

void embed_backward(const mg_embed_backward_args& a, Workspace& w, bool go, cudaStream_t s) {
    if (a.dtype == MG_PREC_BF16) embed_backward<MG_PREC_BF16>(a, w, go, s);
    else if (a.dtype == MG_PREC_FP16) embed_backward<MG_PREC_FP16>(a, w, go, s);
    else embed_backward<MG_PREC_FP32>(a, w, go, s);
}

void check_tokens(const void* p, int bytes, int64_t stride, int64_t n) {
    need(bytes == 8 || bytes == 4, "tokens are int64 or int32 (token_bytes 8 or 4)");
    need(n == 0 || p != nullptr, "tokens is null");
    need(stride >= 0, "token_stride is negative");
}

void check_args(const mg_embed_args& a) {
    need(a.n >= 0 && a.vocab >= 1 && a.dim >= 1, "sizes: n >= 0, vocab >= 1, dim >= 1");
    need(a.vocab < (int64_t(1) << 31), "vocab must be below 2^31");
    need(a.dtype >= MG_PREC_BF16 && a.dtype <= MG_PREC_FP32, "dtype is not an MG_PREC_* value");
    check_tokens(a.tokens, a.token_bytes, a.token_stride, a.n);
    need(a.table_row >= 0, "table_row is negative");
    need(a.n == 0 || (a.table != nullptr && a.out != nullptr), "table or out is null");
}

void check_args(const mg_embed_backward_args& a) {
    need(a.n >= 0 && a.vocab >= 1 && a.dim >= 1, "sizes: n >= 0, vocab >= 1, dim >= 1");
    need(a.n < (int64_t(1) << 31) && a.vocab < (int64_t(1) << 31), "n and vocab must be below 2^31");
    need(a.dtype >= MG_PREC_BF16 && a.dtype <= MG_PREC_FP32, "dtype is not an MG_PREC_* value");
    check_tokens(a.tokens, a.token_bytes, a.token_stride, a.n);
    need(a.grad_row >= 0, "grad_row is negative");
    need(a.d_table != nullptr && (a.n == 0 || a.grad != nullptr), "grad or d_table is null");
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
        auto s = static_cast<cudaStream_t>(stream);
        if (args->dtype == MG_PREC_BF16) embed<MG_PREC_BF16>(*args, s);
        else if (args->dtype == MG_PREC_FP16) embed<MG_PREC_FP16>(*args, s);
        else embed<MG_PREC_FP32>(*args, s);
    });
}

extern "C" int mg_embed_backward_workspace(const mg_embed_backward_args* args, size_t* bytes) {
    return guarded([&] {
        need(args != nullptr && bytes != nullptr, "args or bytes is null");
        check_args(*args);
        Workspace w;
        embed_backward(*args, w, false, nullptr);
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
        embed_backward(*args, w, true, static_cast<cudaStream_t>(stream));
    });
}
