// What the readout's translation units share: element types, rows read in 16-byte pieces, and the host
// side's call frame (device guard, no exception past the C boundary).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
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
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, float>::value) v[i] = __uint_as_float(w[i]);
        else if constexpr (std::is_same<T, __half>::value) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            v[2 * i] = f.x, v[2 * i + 1] = f.y;
        } else {
            // a bf16 is the upper half of its f32: shift and mask, where the conversion instruction would run on the pipe that
            // the exponentials need
            v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
}
template <class T>
__device__ __forceinline__ uint4 pack_16(const float* v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, float>::value) w[i] = __float_as_uint(v[i]);
        else if constexpr (std::is_same<T, __half>::value) {
            const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);  // two conversions in one instruction
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// Two f32 operations in one instruction.
__device__ __forceinline__ float2 fma_2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add_2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 mul_2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// 16 bytes to shared memory without passing through registers; the thread that asked for them may read them after its own
// wait_copies<N>(), which leaves its last N groups in flight.
__device__ __forceinline__ void copy_16_async(void* to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))), "l"(from) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A row by positions, counted from the last 16-byte boundary at or before its first element: position = element + ahead.  A
// piece is 16 bytes at a multiple of VEC positions; the row's first and last may hold fewer elements of it.
template <class T>
struct Pieces {
    const T* row;
    int32_t ahead, end;  // first and last + 1 of the row's positions
    __device__ __forceinline__ Pieces(const T* r, int32_t cols) : row(r) {
        ahead = static_cast<int32_t>((reinterpret_cast<uintptr_t>(r) & 15u) / sizeof(T));
        end = cols + ahead;
    }
    __device__ __forceinline__ bool whole(int32_t at) const { return at >= ahead && at + VEC<T> <= end; }
    // The piece at `at` into `slot`, zeros for what lies outside the row; a whole one is on its way until wait_copies.
    __device__ __forceinline__ void fetch(uint4* slot, int32_t at) const {
        if (whole(at)) {
            copy_16_async(slot, row + (at - ahead));
        } else {
            *slot = make_uint4(0u, 0u, 0u, 0u);
            for (int j = 0; j < VEC<T>; ++j)
                if (at + j >= ahead && at + j < end) reinterpret_cast<T*>(slot)[j] = row[at + j - ahead];
        }
    }
    // The piece to the same place of another row (16 bytes at once where `wide`), except the elements marked in `skip`.
    __device__ __forceinline__ void store(T* to, int32_t at, const uint4& raw, bool wide, uint32_t skip) const {
        if (wide && whole(at) && !skip) {
            *reinterpret_cast<uint4*>(to + (at - ahead)) = raw;
        } else {
#pragma unroll
            for (int j = 0; j < VEC<T>; ++j)
                if (at + j >= ahead && at + j < end && !((skip >> j) & 1u)) to[at + j - ahead] = reinterpret_cast<const T*>(&raw)[j];
        }
    }
    // Whether pieces of `to` lie on 16-byte boundaries as the row's do.
    __device__ __forceinline__ bool same_phase(const T* to) const { return ((reinterpret_cast<uintptr_t>(to) ^ reinterpret_cast<uintptr_t>(row)) & 15u) == 0; }
};

// One CTA's share of a row: whole pieces of 16 bytes from `first` on, and up to VEC - 1 elements before and behind them.
template <class T>
struct Share {
    const T* row;
    int32_t head, first, pieces, tail, stop;  // elements [head, first), pieces from first, elements [tail, stop)
    __device__ __forceinline__ Share(const T* r, int32_t cols, int32_t from, int32_t share) : row(r) {
        const Pieces<T> p(r, cols);
        const int32_t to = min(p.end, from + share);
        head = max(from - p.ahead, 0);
        stop = max(to - p.ahead, head);
        first = min(from < p.ahead ? from + VEC<T> - p.ahead : head, stop);
        pieces = (stop - first) / VEC<T>;
        tail = first + pieces * VEC<T>;
    }
    __device__ __forceinline__ uint4 piece(int32_t i) const { return *reinterpret_cast<const uint4*>(row + first + i * VEC<T>); }
};

// ---- host side
inline bool is_float_type(int32_t t) { return t == THRML_F32 || t == THRML_BF16 || t == THRML_F16; }
inline bool is_index_type(int32_t t) { return t == THRML_I32 || t == THRML_I64; }
inline size_t type_size(int32_t t) { return t == THRML_F32 || t == THRML_I32 ? 4 : t == THRML_I64 ? 8 : 2; }
inline bool aligned_to(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Rows of `width` elements `pitch` apart, by their bytes.
struct Area {
    uintptr_t at;
    int64_t rows, width, pitch;
    Area(const void* p, size_t size, int64_t r, int64_t w, int64_t pitch_) : at(reinterpret_cast<uintptr_t>(p)), rows(r), width(w * static_cast<int64_t>(size)), pitch(pitch_ * static_cast<int64_t>(size)) {}
};
// Whether two areas share bytes (rows of one pitch may lie beside each other in one buffer; of two pitches, they are taken to share).
inline bool overlap(const Area& a, const Area& b) {
    using Wide = __int128;
    if (!a.at || !b.at || a.rows < 1 || b.rows < 1 || a.width < 1 || b.width < 1) return false;
    const Wide a_end = static_cast<Wide>(a.at) + static_cast<Wide>(a.rows - 1) * a.pitch + a.width, b_end = static_cast<Wide>(b.at) + static_cast<Wide>(b.rows - 1) * b.pitch + b.width;
    if (a.at >= b_end || b.at >= a_end) return false;
    if (a.rows > 1 && b.rows > 1 && a.pitch != b.pitch) return true;
    const int64_t pitch = a.rows > 1 ? a.pitch : b.pitch;
    if ((a.rows == 1 && b.rows == 1) || pitch < 1) return true;
    const Wide apart = static_cast<Wide>(b.at) - static_cast<Wide>(a.at);
    const Wide behind = ((apart % pitch) + pitch) % pitch;  // of b's rows behind a's
    return behind < a.width || behind + b.width > pitch;
}

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

// Body of an entry point: refuses while a wait that ran out in an earlier call is reported, and turns exceptions into a status.
template <class F>
int32_t guarded(thrml_ctx* ctx, F body) noexcept {
    try {
        if (!ctx) return fail(THRML_ERR_INVALID_ARG, "null context");
        if (int32_t rc = ctx->check_waits()) return rc;
        OnDevice on(ctx->device);
        CU_TRY(on.status());
        const int32_t rc = body();
        if (rc == THRML_ERR_CUDA) cudaGetLastError();  // a refused launch is reported here, not by whoever asks next
        return rc;
    } catch (const std::bad_alloc&) {
        return THRML_ERR_OOM;  // no message: making one would allocate
    } catch (...) {
        return THRML_ERR_INVALID_ARG;
    }
}

// Lets a kernel have more than 48 KB of dynamic shared memory, once for each device (threads that come at once do it twice).
template <auto KERNEL>
int32_t allow_shared(const thrml_ctx* ctx, size_t bytes) {
    static std::atomic<bool> done[64];
    if (ctx->device < 64 && done[ctx->device].load(std::memory_order_acquire)) return THRML_OK;
    CU_TRY(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
    if (ctx->device < 64) done[ctx->device].store(true, std::memory_order_release);
    return THRML_OK;
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
