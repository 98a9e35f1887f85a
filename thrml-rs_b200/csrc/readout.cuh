// What the readout's translation units share: element types, rows read in 16-byte pieces, block reductions, and the host
// side's call frame (device guard, no exception past the C boundary).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <new>
#include <string>
#include <type_traits>

#include "ctx.h"
#include "tables.h"

namespace thrml {
namespace readout {

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <class T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// One element of an array whose type is a run-time argument (short arrays only: ids, teacher logits, histories).
__device__ __forceinline__ float load_as_float(const void* p, int32_t type, int64_t i) {
    if (type == THRML_F32) return static_cast<const float*>(p)[i];
    if (type == THRML_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ int64_t load_as_int(const void* p, int32_t type, int64_t i) {
    return type == THRML_I64 ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

template <class T>
constexpr int VEC = 16 / static_cast<int>(sizeof(T));
template <int N>
using Count = std::integral_constant<int, N>;

__device__ __forceinline__ bool on_16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <class T>
__device__ __forceinline__ void unpack_16(const uint4& raw, float (&v)[VEC<T>]) {
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < VEC<T>; ++i) v[i] = to_float(e[i]);
}
template <class T>
__device__ __forceinline__ uint4 pack_16(const float* v) {
    uint4 raw;
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int i = 0; i < VEC<T>; ++i) e[i] = from_float<T>(v[i]);
    return raw;
}
// n values of a row to dst (16 bytes at once where dst allows it).
template <class T, int N>
__device__ __forceinline__ void store_n(T* dst, const float* v, Count<N>) {
    if (N == VEC<T> && on_16(dst)) {
        *reinterpret_cast<uint4*>(dst) = pack_16<T>(v);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) dst[i] = from_float<T>(v[i]);
    }
}
// f(index, values, Count) over row[0 .. n): up to the first 16-byte boundary one by one, then 16 bytes at a time, then one by
// one.  Thread `tid` of `threads` takes its share; every thread calls f for its own elements only.
template <class T, class F>
__device__ __forceinline__ void for_row(const T* row, int32_t n, int tid, int threads, F f) {
    const int32_t ahead = min(n, static_cast<int32_t>((-reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T)));
    const int32_t vecs = (n - ahead) / VEC<T>, behind = ahead + vecs * VEC<T>;
    if (tid < ahead) {
        const float v[1] = {to_float(row[tid])};
        f(tid, v, Count<1>{});
    }
    for (int32_t i = tid; i < vecs; i += threads) {
        float v[VEC<T>];
        unpack_16<T>(*reinterpret_cast<const uint4*>(row + ahead + i * VEC<T>), v);
        f(ahead + i * VEC<T>, v, Count<VEC<T>>{});
    }
    if (behind + tid < n) {
        const float v[1] = {to_float(row[behind + tid])};
        f(behind + tid, v, Count<1>{});
    }
}

struct MaxOp {
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
    static constexpr float none = -INFINITY;
};
struct SumOp {
    __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
    static constexpr float none = 0.0f;
};
// All threads of the block get the result; `scratch` holds 32 floats.  The order of the additions is fixed.
template <class Op>
__device__ __forceinline__ float block_reduce(float x, float* scratch) {
    const Op op;
#pragma unroll
    for (int d = 16; d; d >>= 1) x = op(x, __shfl_xor_sync(0xffffffffu, x, d));
    __syncthreads();  // the scratch may still be read from an earlier reduction
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = x;
    __syncthreads();
    x = (threadIdx.x & 31) < (blockDim.x >> 5) ? scratch[threadIdx.x & 31] : Op::none;
#pragma unroll
    for (int d = 16; d; d >>= 1) x = op(x, __shfl_xor_sync(0xffffffffu, x, d));
    return x;
}

// ---- host side
inline bool is_float_type(int32_t t) { return t == THRML_F32 || t == THRML_BF16 || t == THRML_F16; }
inline bool is_index_type(int32_t t) { return t == THRML_I32 || t == THRML_I64; }
inline size_t type_size(int32_t t) { return t == THRML_F32 || t == THRML_I32 ? 4 : t == THRML_I64 ? 8 : 2; }
inline bool aligned_to(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// The context's device for the length of a call; the caller's current device comes back.
class OnDevice {
public:
    explicit OnDevice(int device) {
        if (cudaGetDevice(&before_) != cudaSuccess) before_ = device;
        if (before_ != device) status_ = cudaSetDevice(device);
        changed_ = before_ != device;
    }
    ~OnDevice() {
        if (changed_) cudaSetDevice(before_);
    }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;
    cudaError_t status() const { return status_; }

private:
    int before_ = 0;
    bool changed_ = false;
    cudaError_t status_ = cudaSuccess;
};

// Body of an entry point: reports a wait that ran out in an earlier call, and turns exceptions into a status.
template <class F>
int32_t guarded(thrml_ctx* ctx, F body) noexcept {
    try {
        if (!ctx) return fail(THRML_ERR_INVALID_ARG, "null context");
        if (int32_t rc = ctx->check_waits()) return rc;
        OnDevice on(ctx->device);
        CU_TRY(on.status());
        return body();
    } catch (const std::bad_alloc&) {
        return THRML_ERR_OOM;  // no message: making one would allocate
    } catch (...) {
        return THRML_ERR_INVALID_ARG;
    }
}

// f(element of the type) for one of the three float types.
template <class F>
int32_t for_type(int32_t type, F f) {
    if (type == THRML_F32) return f(float{});
    if (type == THRML_BF16) return f(__nv_bfloat16{});
    return f(__half{});
}

}  // namespace readout
}  // namespace thrml
