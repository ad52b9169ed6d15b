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

// ---------------------------------------------------------------------------------
// Row quantiser: scale = max|x| / 127, code = rint(127 x / max|x|), ties to even -- the code of the exact quotient, not of
// a rounded one.  inv = 127 * RN(1 / max|x|) and y = x * inv carry three roundings, so y is off by less than 127 * 3 * 2^-24 <
// 2.3e-5: only vectors with a y within 2.5e-5 of a border between two codes are decided in 64 bits.  A row of zeros has
// scale 0 and codes 0; a row with an infinity or a NaN has scale NaN and codes 0, so that its outputs are NaN and no other
// row's are.  Rounding adds 1.5 * 2^23: the sum's low byte is the code, and taking the constant off again gives the
// rounded value.
// ---------------------------------------------------------------------------------
constexpr float I8_ROUND = 12582912.f;
constexpr float I8_BORDER = 0.5f - 2.5e-5f;

// (kept out of line: a rare path with long 64-bit divisions)
static __device__ __noinline__ float i8_exact_code(float x, float amax) { return (float)rint(127.0 * (double)x / (double)amax); }

struct I8RowScale {
    float scale, amax, up, inv;          // inv = 0: every code is 0
    // top: the largest magnitude of the row as an integer, which orders NaN > infinity > finite
    __device__ __forceinline__ explicit I8RowScale(uint32_t top) {
        const bool finite = top < 0x7f800000u;
        amax = __uint_as_float(top);
        // by rcp.rn and a correction, exact for this divisor (Divider) while nothing underflows
        scale = !finite ? __uint_as_float(0x7fc00000u) : amax >= 0x1p-100f ? Divider(127.f)(amax) : amax / 127.f;
        up = amax < 0x1p-100f ? 0x1p100f : amax > 0x1p100f ? 0x1p-100f : 1.f;     // keeps 1 / max|x| a normal number; exact
        amax *= up;
        float r;
        asm("rcp.rn.f32 %0, %1;" : "=f"(r) : "f"(amax));
        inv = finite && amax > 0.f ? 127.f * r : 0.f;
    }
    // neither a row of zeros nor one that needs `up`: almost every row
    __device__ __forceinline__ bool plain() const { return up == 1.f && inv != 0.f; }
    __device__ __forceinline__ float exact(float x) const { return i8_exact_code(x * up, amax); }
    __device__ __forceinline__ int code(float x) const {
        if (inv == 0.f) return 0;
        const float y = x * up * inv, r = rintf(y);
        return (int)(fabsf(y - r) > I8_BORDER ? exact(x) : r);
    }
    // the codes of a vector, four to a word
    template <typename R>
    __device__ __forceinline__ void codes(const R& v, uint32_t (&w)[2]) const {
        if (plain()) put<R, true>(v, w);
        else if (inv != 0.f) put<R, false>(v, w);
        else w[0] = w[1] = 0;
    }
private:
    template <typename R, bool PLAIN>
    __device__ __forceinline__ void put(const R& v, uint32_t (&w)[2]) const {
        float t[R::N], far = 0.f;
#pragma unroll
        for (int k = 0; k < R::N; ++k) {
            const float y = (PLAIN ? v.get(k) : v.get(k) * up) * inv;
            t[k] = y + I8_ROUND;
            far = fmaxf(far, fabsf(y - (t[k] - I8_ROUND)));
        }
        if (far > I8_BORDER) {
#pragma unroll
            for (int k = 0; k < R::N; ++k) t[k] = I8_ROUND + exact(v.get(k));
        }
#pragma unroll
        for (int h = 0; h < (R::N + 3) / 4; ++h) {
            uint32_t b[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) b[k] = 4 * h + k < R::N ? __float_as_uint(t[4 * h + k < R::N ? 4 * h + k : 0]) : 0u;
            w[h] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
        }
    }
};

// A few rows (vmoe_int8_gemv.cu): x, when not NULL, holds them as bf16 / fp16 / f32 and p.a is not read.
constexpr int I8_GEMV_ROWS = 8;
bool i8_gemv_ok(const I8Problem& p);
int  launch_i8_gemv(const I8Problem& p, const void* x, long long x_stride_bytes, int x_dtype, cudaStream_t st);

// tensor-core kernels (vmoe_int8_tc.cu)
constexpr int I8_TC_MAX_EXPERTS = 16384;                 // their tables lie in shared memory
bool i8_tc_ok(const I8Problem& p);                       // addresses and strides are multiples of 16 bytes
int  launch_i8_tc(const I8Problem& p, cudaStream_t st);
int  launch_i8_split(const I8Problem& p, cudaStream_t st);   // dense only

}  // namespace vmoe
