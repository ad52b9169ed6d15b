// Rows of bf16 / fp16 / f32 read and written as vectors of 16, 8, 4 or 2 bytes, whichever every row's start allows.
#pragma once

#include "vmoe_common.cuh"

#include <type_traits>

namespace vmoe {

template <int BYTES> struct RawVec;
template <> struct RawVec<16> { using type = uint4; };
template <> struct RawVec<8>  { using type = uint2; };
template <> struct RawVec<4>  { using type = uint32_t; };
template <> struct RawVec<2>  { using type = uint16_t; };

__device__ __forceinline__ float elem_float(float v) { return v; }
__device__ __forceinline__ float elem_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float elem_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void elem_store(float& d, float v) { d = v; }
__device__ __forceinline__ void elem_store(__half& d, float v) { d = __float2half_rn(v); }
__device__ __forceinline__ void elem_store(__nv_bfloat16& d, float v) { d = __float2bfloat16_rn(v); }

// BYTES_ bytes of a row of T_ elements; element access by value, so the vector stays in registers.
template <typename T_, int BYTES_>
struct RowVec {
    using T = T_;
    using Raw = typename RawVec<BYTES_>::type;
    static constexpr int BYTES = BYTES_, N = BYTES_ / (int)sizeof(T_);
    union { Raw raw; uint16_t half[BYTES_ / 2]; };
    __device__ __forceinline__ RowVec() {}
    __device__ __forceinline__ void load(const void* row, long long c) { raw = static_cast<const Raw*>(row)[c]; }
    __device__ __forceinline__ void store(void* row, long long c) const { static_cast<Raw*>(row)[c] = raw; }
    __device__ __forceinline__ float get(int k) const { return elem_float(reinterpret_cast<const T_*>(half)[k]); }
    // Largest magnitude so far, joined with this vector's; a NaN stays.  16-bit elements are compared two at a time: `top`
    // then holds two of them.  magnitude(top) is the result as an f32's bits.
    __device__ __forceinline__ uint32_t join(uint32_t top) const {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(half);
        if constexpr (sizeof(T_) == 4) {
#pragma unroll
            for (int k = 0; k < N; ++k)
                asm("max.NaN.f32 %0, %1, %2;" : "=r"(top) : "r"(top), "r"(w[k] & 0x7fffffffu));
        } else {
#pragma unroll
            for (int k = 0; k < (BYTES + 3) / 4; ++k) {
                const uint32_t v = (BYTES >= 4 ? w[k] : half[0]) & 0x7fff7fffu;
                if constexpr (std::is_same<T_, __half>::value) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(top) : "r"(top), "r"(v));
                else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(top) : "r"(top), "r"(v));
            }
        }
        return top;
    }
    __device__ static __forceinline__ uint32_t magnitude(uint32_t top) {
        if constexpr (sizeof(T_) == 4) return top & 0x7fffffffu;
        const uint16_t m = (uint16_t)max(top & 0x7fffu, (top >> 16) & 0x7fffu);      // ordered as integers: NaN > infinity > finite
        return __float_as_uint(elem_float(*reinterpret_cast<const T_*>(&m))) & 0x7fffffffu;
    }
    __device__ __forceinline__ void set(int k, float v) { elem_store(reinterpret_cast<T_*>(half)[k], v); }
};

// The widest vector that divides every address, stride and length or-ed together here.
inline int vector_bytes(uintptr_t addresses, long long lengths) {
    const unsigned long long all = (unsigned long long)addresses | (unsigned long long)lengths;
    return all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 2;
}

// A launch's status.  A refused launch must not leave its error for the next call's cudaGetLastError.
inline int launch_status(cudaError_t e) {
    if (e != cudaSuccess) cudaGetLastError();
    return cuda_status(e);
}

// More than 48 KB of dynamic shared memory have to be allowed once per device and kernel; `done` is the caller's, one for each.
struct SmemAllowed { bool on[64] = {}; };
template <typename F>
inline cudaError_t allow_smem(F* kernel, size_t bytes, SmemAllowed& done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev < 64 && done.on[dev])) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess && dev < 64) done.on[dev] = true;
    if (e != cudaSuccess) cudaGetLastError();
    return e;
}

// f(RowTag) for the wanted type and width
template <typename T_, int BYTES_>
struct RowTag {
    using T = T_;
    static constexpr int BYTES = BYTES_, N = BYTES_ / (int)sizeof(T_);
};
template <typename T_, typename F>
inline int with_width(int bytes, F f) {
    if (bytes == 16) return f(RowTag<T_, 16>{});
    if (bytes == 8) return f(RowTag<T_, 8>{});
    if (bytes == 4) return f(RowTag<T_, 4>{});
    if constexpr (sizeof(T_) == 2) return f(RowTag<T_, 2>{});
    return VMOE_ERR_ALIGN;
}
template <typename F>
inline int with_rows(int dtype, int bytes, F f) {
    switch (dtype) {
        case VMOE_BF16: return with_width<__nv_bfloat16>(bytes, f);
        case VMOE_F16:  return with_width<__half>(bytes, f);
        case VMOE_F32:  return with_width<float>(bytes, f);
    }
    return VMOE_ERR_SHAPE;
}

}  // namespace vmoe
