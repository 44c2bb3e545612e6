// Shared by the training operators (include/minigo_ops.h): element types,
// argument checks, workspace layout and errors.
#pragma once

#include "../../include/minigo_ops.h"

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <exception>
#include <new>
#include <string>

#include "ptx_sm100.cuh"

namespace mgb {
namespace ops {

// ---- element types ----

template <int DT>
struct Elem;
template <>
struct Elem<MG_PREC_BF16> {
    using T = __nv_bfloat16;
    static __device__ __forceinline__ float get(T v) { return __bfloat162float(v); }
    static __device__ __forceinline__ T put(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Elem<MG_PREC_FP16> {
    using T = __half;
    static __device__ __forceinline__ float get(T v) { return __half2float(v); }
    static __device__ __forceinline__ T put(float v) { return __float2half_rn(v); }
};
template <>
struct Elem<MG_PREC_FP32> {
    using T = float;
    static __device__ __forceinline__ float get(T v) { return v; }
    static __device__ __forceinline__ T put(float v) { return v; }
};

inline int elem_bytes(int dtype) { return dtype == MG_PREC_FP32 ? 4 : 2; }

// A token or target, or -1 where it lies outside [0, limit).
__device__ __forceinline__ int64_t index_at(const void* p, int bytes, int64_t i, int64_t limit) {
    const int64_t t = bytes == 8 ? static_cast<const int64_t*>(p)[i]
                                 : (int64_t)static_cast<const int32_t*>(p)[i];
    return t >= 0 && t < limit ? t : -1;
}

// Targets (or any indices) as the caller keeps them.
struct Indices {
    const void* data = nullptr;
    int64_t stride = 0, limit = 0;
    int bytes = 8;
    __device__ __forceinline__ int at(int64_t i) const { return (int)index_at(data, bytes, i * stride, limit); }
    Indices from(int64_t first) const {
        Indices r = *this;
        r.data = static_cast<const char*>(data) + first * stride * bytes;
        return r;
    }
};

// Eight 16-bit elements from p on, which is element `at` of memory that holds
// elements [0, span); what lies past it comes back as anything.  16 bytes at
// any alignment by 32-bit loads, as far as those stay inside.
__device__ __forceinline__ uint4 load8_unaligned(const uint16_t* p, int64_t at, int64_t span) {
    const bool odd = (reinterpret_cast<uintptr_t>(p) & 2) != 0;
    uint32_t w[5];
    if (at >= odd && at + 8 + odd <= span) {
        const uint32_t* q = reinterpret_cast<const uint32_t*>(p - odd);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __ldg(q + i);
        w[4] = odd ? __ldg(q + 4) : 0;
    } else {
        uint32_t h[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = at + i < span ? p[i] : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = odd ? __byte_perm(i ? h[2 * i - 1] : 0, h[2 * i], 0x5410)
                                              : __byte_perm(h[2 * i], h[2 * i + 1], 0x5410);
        w[4] = h[7];
    }
    if (!odd) return make_uint4(w[0], w[1], w[2], w[3]);
    return make_uint4(__byte_perm(w[0], w[1], 0x5432), __byte_perm(w[1], w[2], 0x5432),
                      __byte_perm(w[2], w[3], 0x5432), __byte_perm(w[3], w[4], 0x5432));
}

// ---- host side ----

struct OpFailure {
    int code;
    std::string what;
};
[[noreturn]] inline void fail(int code, const std::string& what) { throw OpFailure{code, what}; }
inline void need(bool ok, const char* what) {
    if (!ok) fail(MG_E_ARG, what);
}
// Kernels read and write whole elements.
inline void need_aligned(const void* p, int bytes, const char* name) {
    if (reinterpret_cast<uintptr_t>(p) % bytes != 0)
        fail(MG_E_ARG, std::string(name) + " is not aligned to its elements");
}
inline void check(cudaError_t e, const char* where) {
    if (e != cudaSuccess) fail(MG_E_CUDA, std::string(where) + ": " + cudaGetErrorString(e));
}

// The launches of one call, in order.  All but the first may begin while the
// one before is finishing (programmatic dependent launch), so every kernel
// that goes through here calls griddep_wait() in every thread before it
// touches global memory; the first is launched in the ordinary way, after
// everything the stream holds.
class Queue {
public:
    explicit Queue(void* stream) : stream_(static_cast<cudaStream_t>(stream)) {}
    template <class... P, class... A>
    void launch(const char* name, void (*kernel)(P...), dim3 grid, int block, int smem, A... args) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = grid;
        cfg.blockDim = dim3((unsigned)block);
        cfg.dynamicSmemBytes = (size_t)smem;
        cfg.stream = stream_;
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr.val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = begun_ ? 1 : 0;
        check(cudaLaunchKernelEx(&cfg, kernel, P(args)...), name);
        begun_ = true;
    }
    void clear(void* p, size_t bytes) {
        check(cudaMemsetAsync(p, 0, bytes, stream_), "cudaMemsetAsync");
        begun_ = false;  // what follows a memset waits for it in the ordinary way
    }

private:
    cudaStream_t stream_;
    bool begun_ = false;
};

// Makes args->device current for one call.
class OnDevice {
public:
    explicit OnDevice(int device) {
        check(cudaGetDevice(&prev_), "cudaGetDevice");
        if (prev_ != device) check(cudaSetDevice(device), "cudaSetDevice");
        now_ = device;
    }
    ~OnDevice() {
        if (prev_ != now_) cudaSetDevice(prev_);
    }

private:
    int prev_ = 0, now_ = 0;
};

// Lays buffers out one after another.  With a null base it only adds up the
// bytes, so the size query and the call run the same code.
class Workspace {
public:
    Workspace() = default;
    Workspace(void* base, size_t bytes) : base_(static_cast<char*>(base)), bytes_(bytes) {}
    template <class T = void>
    T* take(size_t bytes) {
        const size_t at = used_;
        used_ += (bytes + 255) & ~size_t(255);
        return base_ ? reinterpret_cast<T*>(base_ + at) : nullptr;
    }
    size_t used() const { return used_; }
    void require() const {
        need(used_ == 0 || base_ != nullptr, "workspace is null");
        need((reinterpret_cast<uintptr_t>(base_) & 255) == 0, "workspace is not 256-byte aligned");
        need(used_ <= bytes_, "workspace is smaller than the matching *_workspace call reports");
    }

private:
    char* base_ = nullptr;
    size_t bytes_ = 0, used_ = 0;
};

std::string& last_op_error();  // of the calling thread

// Leaves a message, or where there is no memory for one, none.
inline int failed(int code, const char* what) noexcept {
    try {
        last_op_error().clear();
        last_op_error() = what;
    } catch (...) {
    }
    return code;
}

// Runs a C entry's body: any failure becomes a code and a message.
template <class F>
int guarded(F&& body) noexcept {
    try {
        body();
        return MG_OK;
    } catch (const OpFailure& f) {
        return failed(f.code, f.what.c_str());
    } catch (const std::bad_alloc&) {
        return failed(MG_E_STATE, "out of host memory");
    } catch (const std::exception& e) {
        return failed(MG_E_STATE, e.what());
    } catch (...) {
        return failed(MG_E_STATE, "unknown exception");
    }
}

// The device status word of these kernels (0, or a DeviceError of
// ptx_sm100.cuh from a wait that gave up) on the current device.
int* op_status_word();

}  // namespace ops
}  // namespace mgb
