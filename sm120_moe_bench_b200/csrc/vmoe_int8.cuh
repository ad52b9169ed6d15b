// The 8-bit integer product as its kernels see it:
//   out[m, n] = (sum_k a[m, k] * w[e][n, k]) * a_scale[m] * w_scale[e][n],   e = the expert of row m (0 when dense)
// The sum is exact in int32 (K <= I8_MAX_K); it becomes f32 once and takes the two scales in that order.  swiglu: w has
// 2 N rows per expert, gate rows first, and out[m, n] = silu(gate[m, n]) * up[m, n].
#pragma once

#include "vmoe_rows.cuh"

namespace vmoe {

constexpr int I8_MAX_K = 131071;       // 128 * 128 * K stays below 2^31

struct I8Problem {
    const int8_t* a; long long a_stride; const float* a_scale;
    const int8_t* w; long long w_stride, w_expert_stride; const float* w_scale;      // w_scale [E, wrows]
    void* out; long long out_stride;                                                  // in elements
    const int32_t* offsets;                                                           // [E + 1] device, NULL = dense
    int M, N, K, E, wrows, swiglu, out_dtype, zero_tail;                              // wrows = N or 2 N
};

__device__ __forceinline__ float i8_scaled(int acc, float sa, float sw) { return (__int2float_rn(acc) * sa) * sw; }

// Above 20 the denominator rounds to 1 (and an infinite gate must not meet the quotient's correction step).
__device__ __forceinline__ float i8_silu(float x) { return x > 20.f ? x : silu(x); }

__device__ __forceinline__ void i8_store(void* out, long long at, int dtype, float v) {
    if (dtype == VMOE_F32) static_cast<float*>(out)[at] = v;
    else if (dtype == VMOE_BF16) static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
    else static_cast<__half*>(out)[at] = __float2half_rn(v);
}

// tensor-core kernels (vmoe_int8_tc.cu)
constexpr int I8_TC_MAX_EXPERTS = 16384;                 // their tables lie in shared memory
bool i8_tc_ok(const I8Problem& p);                       // addresses and strides are multiples of 16 bytes
int  launch_i8_tc(const I8Problem& p, cudaStream_t st);
int  launch_i8_split(const I8Problem& p, cudaStream_t st);   // dense only

}  // namespace vmoe
