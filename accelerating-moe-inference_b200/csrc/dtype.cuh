// Element types of the 4-bit operators' activations (MoeDtype) and what their
// host entry points share.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <exception>
#include <string>

#include "moe_b200.h"

namespace moe {

int report_error(int code, const std::string& msg);  // capi.cu

// Memory of a handle on `device`, which is current; 1024-byte aligned.  handle_free
// waits for the current device (handle_memory.cu).
cudaError_t handle_alloc(int device, size_t bytes, void** out);
void handle_free(void* p) noexcept;

template <class T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }

// One rounding to the output type (to nearest even).
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// n / d for 0 <= n < 2^31 by a multiplication: with 2^s >= d the
// smallest such power, q = floor(n m / 2^(31 + s)) for m = ceil(2^(31 + s) / d),
// since n (m d - 2^(31 + s)) < 2^31 d <= 2^(31 + s).
struct FastDiv {
    unsigned long long mul;
    int shift, d;
    FastDiv() = default;
    explicit FastDiv(int div) : d(div) {
        shift = 31;
        while ((1ll << (shift - 31)) < div) ++shift;
        mul = ((1ull << shift) + div - 1) / div;
    }
    __device__ __forceinline__ int div(int n) const { return (int)((unsigned)n * mul >> shift); }
};

inline bool valid_dtype(int32_t t) { return t >= MOE_DTYPE_F32 && t <= MOE_DTYPE_F16; }
inline size_t dtype_bytes(int32_t t) { return t == MOE_DTYPE_F32 ? 4 : 2; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline bool aligned_to(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Makes `dev` current for a scope; the caller's device comes back at its end.
struct OnDevice {
    int prev = -1;
    bool ok = true;
    explicit OnDevice(int dev) {
        if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
        if (prev != dev) ok = cudaSetDevice(dev) == cudaSuccess;
        else prev = -1;
    }
    ~OnDevice() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

// A launch sequence's error as a status.  An error that an earlier call of
// the caller's left behind is not this operator's: entry points launch
// through cudaLaunchKernelEx and pass its own result here.
inline int launch_status(cudaError_t e, const char* what) {
    return e == cudaSuccess ? MOE_OK
                            : report_error(MOE_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

// Runs an entry point's body; nothing that it throws (an allocation of the
// host's) passes the C boundary.
template <class F> int guarded(const char* what, F&& body) noexcept {
    try {
        return body();
    } catch (const std::exception& e) {
        try {
            return report_error(MOE_ERR_OOM, std::string(what) + ": " + e.what());
        } catch (...) {
        }
    } catch (...) {
    }
    return MOE_ERR_OOM;
}

// kernel<<<grid, block, smem, s>>>(args...), returning its own error.
template <class... P, class... A>
cudaError_t launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, bool dependent,
                   A&&... args) {
    cudaLaunchConfig_t c{};
    c.gridDim = grid;
    c.blockDim = block;
    c.dynamicSmemBytes = smem;
    c.stream = s;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    if (dependent) {
        c.attrs = &at;
        c.numAttrs = 1;
    }
    return cudaLaunchKernelEx(&c, kernel, P(args)...);
}

}  // namespace moe
