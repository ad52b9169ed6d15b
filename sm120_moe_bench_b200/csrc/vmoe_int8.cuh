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

// x / (1 + exp(-x)): approximate reciprocal, one Newton-Raphson step, one Markstein correction of the quotient (as Divider, whose
// reciprocal is the rounded one: with that the epilogue of 8192 x 4096 x (4096 gate + 4096 up) took 293 us a product, so 193).
//   The step leaves r within 2^-24 + 2^-45 of 1 / d, the product q within 2^-23 of the quotient, and the correction, whose
//   residual is off by less than 2^-46 of x, q within 2^-24 + 2^-44: half a step.  With expf's 2 ulp (2^-22) and the rounded sum
//   (2^-24) the result is within 6 * 2^-24 of silu.
// Above 20 the denominator rounds to 1 (and an infinite x must not meet the correction).  It is kept below 1e38; from 2^126 on,
// x below -87.33, the reciprocal is flushed and the result is 0 where silu is above -1.04e-36.
__device__ __forceinline__ float i8_silu(float x) {
    const float d = fminf(1.f + expf(-x), 1e38f);
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    r = fmaf(fmaf(-d, r, 1.f), r, r);
    const float q = x * r;
    return x > 20.f ? x : fmaf(fmaf(-d, q, x), r, q);
}

__device__ __forceinline__ void i8_store(void* out, long long at, int dtype, float v) {
    if (dtype == VMOE_F32) static_cast<float*>(out)[at] = v;
    else if (dtype == VMOE_BF16) static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
    else static_cast<__half*>(out)[at] = __float2half_rn(v);
}

// ---------------------------------------------------------------------------------
// Row quantiser: scale = max|x| / 127, code = rint(127 x / max|x|), ties to even -- the code of the exact quotient, not of
// a rounded one.  A row of zeros has scale 0 and codes 0; a row with an infinity or a NaN has scale NaN and codes 0, so that
// its outputs are NaN and no other row's are.  Rounding adds 1.5 * 2^23: the sum's low byte is the code.
//   16-bit elements: n = 127 x is exact in f32 (7 + 11 bits), q = n * RN(1 / max|x|) with one correction q + (n - q max|x|) r is
//   the correctly rounded quotient, exact at a tie; a quotient that is no tie is at least y / (254 * 2047) away from one
//   (its numerator is a whole number of units), f32's half step y * 2^-24 is less, so rounding q rounds the quotient.
//   f32 elements: inv = 127 * RN(1 / max|x|) and y = x * inv carry three roundings, so y is off by less than
//   127 * 3 * 2^-24 < 2.3e-5; vectors with a y within 2.5e-5 of a border between two codes are decided in 64 bits.
// Rows whose largest magnitude is below 2^-100 or above 2^100 are decided in 64 bits throughout: 1 / max|x| and the
// residual stay normal numbers otherwise.
// ---------------------------------------------------------------------------------
constexpr float I8_ROUND = 12582912.f;
constexpr float I8_BORDER = 0.5f - 2.5e-5f;

// (kept out of line: a rare path with long 64-bit divisions)
static __device__ __noinline__ float i8_exact_code(float x, float amax) { return (float)rint(127.0 * (double)x / (double)amax); }

struct I8RowScale {
    float scale, amax, r, inv;           // r = RN(1 / amax), inv = 127 r; plain: these are good for the whole row
    bool plain;
    // top: the largest magnitude of the row as an integer, which orders NaN > infinity > finite
    __device__ __forceinline__ explicit I8RowScale(uint32_t top) {
        amax = __uint_as_float(top);
        plain = amax >= 0x1p-100f && amax <= 0x1p100f;
        // by rcp.rn and a correction, exact for this divisor (Divider) while nothing underflows
        scale = plain ? Divider(127.f)(amax) : top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : amax / 127.f;
        asm("rcp.rn.f32 %0, %1;" : "=f"(r) : "f"(amax));
        inv = 127.f * r;
    }
    __device__ __forceinline__ float exact(float x) const {
        return amax > 0.f && amax < __uint_as_float(0x7f800000u) ? i8_exact_code(x, amax) : 0.f;
    }
    __device__ __forceinline__ int code(float x) const {
        const float y = x * inv, t = rintf(y);
        return (int)(plain && fabsf(y - t) < I8_BORDER ? t : exact(x));
    }
    // the codes of a vector, four to a word
    template <typename R>
    __device__ __forceinline__ void codes(const R& v, uint32_t (&w)[2]) const {
        float t[R::N];
        bool good = plain;
        if constexpr (sizeof(typename R::T) == 2) {
#pragma unroll
            for (int k = 0; k < R::N; ++k) {
                const float n = 127.f * v.get(k), q = n * r;
                t[k] = fmaf(fmaf(-amax, q, n), r, q) + I8_ROUND;
            }
        } else {
            float far = 0.f;
#pragma unroll
            for (int k = 0; k < R::N; ++k) {
                const float y = v.get(k) * inv;
                t[k] = y + I8_ROUND;
                far = fmaxf(far, fabsf(y - (t[k] - I8_ROUND)));
            }
            good = good && far < I8_BORDER;
        }
        if (!good) {
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
bool i8_gemv_fits(const I8Problem& p);                   // it can take the product
bool i8_gemv_ok(const I8Problem& p);                     // and is the better kernel for it
int  launch_i8_gemv(const I8Problem& p, const void* x, long long x_stride_bytes, int x_dtype, cudaStream_t st);

// tensor-core kernels (vmoe_int8_tc.cu)
constexpr int I8_TC_MAX_EXPERTS = 16384;                 // their tables lie in shared memory
bool i8_tc_ok(const I8Problem& p);                       // addresses and strides are multiples of 16 bytes
int  launch_i8_tc(const I8Problem& p, cudaStream_t st);
int  launch_i8_split(const I8Problem& p, cudaStream_t st);   // dense only

}  // namespace vmoe
