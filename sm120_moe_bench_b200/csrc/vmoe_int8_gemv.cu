// The 8-bit product for a few rows (decode of one to eight tokens), in one launch: the rows are quantised inside.
//
// Bound by reading the weights once, and at these sizes by latency: a warp owns one channel (with swiglu its gate and up
// rows), requests the first 4 KB of it before anything else, and quantises the rows -- every CTA for itself, 8 KB from
// L2 -- while they are on their way.  Codes lie in shared memory; four products per dp4a, integer sums joined by one
// warp reduction, so the result is the other kernels' bit for bit.
#include "vmoe_int8.cuh"

namespace vmoe {

constexpr int I8G_THREADS = 256;
constexpr int I8G_SMEM = 64 * 1024;                       // codes of all rows

// VB = 16: the weights' rows start on 16-byte boundaries.  VB = 4: anywhere; a word is joined from the two aligned ones that
// hold it, the second of which is read only where the row reaches into it.
template <int VB> struct I8Word;
template <> struct I8Word<16> { using type = uint4; };
template <> struct I8Word<4>  { using type = uint32_t; };

__device__ __forceinline__ int i8_dot(uint4 a, uint4 b, int s) {
    s = __dp4a((int)a.x, (int)b.x, s);
    s = __dp4a((int)a.y, (int)b.y, s);
    s = __dp4a((int)a.z, (int)b.z, s);
    return __dp4a((int)a.w, (int)b.w, s);
}
__device__ __forceinline__ int i8_dot(uint32_t a, uint32_t b, int s) { return __dp4a((int)a, (int)b, s); }

__device__ __forceinline__ uint4 i8_weights(const uint4* row, int c, int, int) { return row[c]; }
__device__ __forceinline__ uint32_t i8_weights(const uint32_t* row, int c, int shift, int K) {      // shift: the row starts so many bytes into row[0]
    const uint32_t lo = row[c];
    if (shift == 0) return lo;
    const uint32_t hi = 4 * (c + 1) - shift < K ? row[c + 1] : 0u;
    return __funnelshift_r(lo, hi, 8 * shift);
}

// One row into shared memory: its codes (padded with zeros to `pitch`) and scale, by the whole CTA.
template <typename T_>
__device__ __forceinline__ void i8_row_codes(const T_* x, int K, int pitch, uint8_t* codes, float* scale, uint32_t* s_max) {
    const int tid = threadIdx.x;
    uint32_t top = 0;
    for (int k = tid; k < K; k += I8G_THREADS) top = max(top, __float_as_uint(elem_float(x[k])) & 0x7fffffffu);
    top = __reduce_max_sync(0xffffffffu, top);
    __syncthreads();                                      // the row before has been read out of s_max
    if ((tid & 31) == 0) s_max[tid >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < I8G_THREADS / 32; ++w) top = max(top, s_max[w]);
    const I8RowScale r(top);
    if (tid == 0) *scale = r.scale;
    for (int k = tid; k < pitch; k += I8G_THREADS) codes[k] = k < K ? (uint8_t)r.code(elem_float(x[k])) : 0;
}
// The same for rows of whole 16-byte vectors.
template <typename T_>
__device__ __forceinline__ void i8_row_codes_vec(const T_* x, int K, int pitch, uint8_t* codes, float* scale, uint32_t* s_max) {
    using R = RowVec<T_, 16>;
    const int tid = threadIdx.x, vecs = K / R::N;
    constexpr int KEPT = 4;
    uint32_t top = 0;
    R keep[KEPT];
#pragma unroll
    for (int i = 0; i < KEPT; ++i)
        if (tid + i * I8G_THREADS < vecs) keep[i].load(x, tid + i * I8G_THREADS);
#pragma unroll
    for (int i = 0; i < KEPT; ++i)
        if (tid + i * I8G_THREADS < vecs) top = keep[i].join(top);
    for (int c = tid + KEPT * I8G_THREADS; c < vecs; c += I8G_THREADS) {
        R v;
        v.load(x, c);
        top = v.join(top);
    }
    top = __reduce_max_sync(0xffffffffu, R::magnitude(top));
    __syncthreads();
    if ((tid & 31) == 0) s_max[tid >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < I8G_THREADS / 32; ++w) top = max(top, s_max[w]);
    const I8RowScale r(top);
    if (tid == 0) *scale = r.scale;
    auto put = [&](const R& v, int c) {
        uint32_t w[2] = {0, 0};
        r.codes(v, w);
        if (R::N == 8) *reinterpret_cast<uint2*>(codes + c * 8) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint32_t*>(codes + c * 4) = w[0];
    };
#pragma unroll
    for (int i = 0; i < KEPT; ++i)
        if (tid + i * I8G_THREADS < vecs) put(keep[i], tid + i * I8G_THREADS);
    for (int c = tid + KEPT * I8G_THREADS; c < vecs; c += I8G_THREADS) {
        R v;
        v.load(x, c);
        put(v, c);
    }
    for (int k = K + tid; k < pitch; k += I8G_THREADS) codes[k] = 0;
}
__device__ __forceinline__ void i8_row_copy(const int8_t* a, int K, int pitch, uint8_t* codes) {
    const int tid = threadIdx.x;
    if (((uintptr_t)a & 15) == 0) {
        for (int k = tid * 16; k < K / 16 * 16; k += I8G_THREADS * 16) *reinterpret_cast<uint4*>(codes + k) = *reinterpret_cast<const uint4*>(a + k);
        for (int k = K / 16 * 16 + tid; k < pitch; k += I8G_THREADS) codes[k] = k < K ? (uint8_t)a[k] : 0;
    } else {
        for (int k = tid; k < pitch; k += I8G_THREADS) codes[k] = k < K ? (uint8_t)a[k] : 0;
    }
}

// x_dtype < 0: p.a / p.a_scale hold the rows; else x does.
template <int VB, int ROWS, bool SWIGLU>
__global__ void __launch_bounds__(I8G_THREADS)
i8_gemv_kernel(const I8Problem p, const uint8_t* x, long long x_stride, int x_dtype, int x_vec) {
    using W = typename I8Word<VB>::type;
    constexpr int AHEAD = VB == 16 ? 8 : 16, SETS = SWIGLU ? 2 : 1;
    extern __shared__ __align__(16) uint8_t codes[];
    __shared__ uint32_t s_max[I8G_THREADS / 32];
    __shared__ float s_scale[ROWS];
    pdl_begin();
    const int lane = threadIdx.x & 31, n = blockIdx.x * (I8G_THREADS / 32) + (threadIdx.x >> 5);
    const int K = p.K, pitch = (K + 15) & ~15, words = (K + VB - 1) / VB;
    const bool on = n < p.N;
    const W* w[SETS];
    int shift[SETS];
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
        const uintptr_t at = (uintptr_t)(p.w + (long long)(s * p.N + (on ? n : 0)) * p.w_stride);
        shift[s] = VB == 4 ? (int)(at & 3) : 0;
        w[s] = reinterpret_cast<const W*>(at - shift[s]);
    }
    W have[SETS][AHEAD];
#pragma unroll
    for (int s = 0; s < SETS; ++s)
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            have[s][i] = W{};
            if (lane + 32 * i < words) have[s][i] = i8_weights(w[s], lane + 32 * i, shift[s], K);
        }
    for (int m = 0; m < p.M; ++m) {
        uint8_t* dst = codes + (size_t)m * pitch;
        if (x_dtype < 0) {
            i8_row_copy(p.a + m * p.a_stride, K, pitch, dst);
            if (threadIdx.x == 0) s_scale[m] = p.a_scale[m];
        } else {
            const uint8_t* src = x + m * x_stride;
#define VMOE_I8_ROW(T) (x_vec ? i8_row_codes_vec(reinterpret_cast<const T*>(src), K, pitch, dst, &s_scale[m], s_max) \
                              : i8_row_codes(reinterpret_cast<const T*>(src), K, pitch, dst, &s_scale[m], s_max))
            if (x_dtype == VMOE_BF16) VMOE_I8_ROW(__nv_bfloat16);
            else if (x_dtype == VMOE_F16) VMOE_I8_ROW(__half);
            else VMOE_I8_ROW(float);
#undef VMOE_I8_ROW
        }
    }
    __syncthreads();
    if (!on) return;
    int acc[SETS][ROWS] = {};
    for (int c0 = 0; c0 < words; c0 += 32 * AHEAD) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int c = c0 + lane + 32 * i;
            if (c < words) {
                // bytes behind K meet zero codes
#pragma unroll
                for (int m = 0; m < ROWS; ++m) {
                    if (m >= p.M) break;
                    const W a = *reinterpret_cast<const W*>(codes + (size_t)m * pitch + (size_t)c * VB);
#pragma unroll
                    for (int s = 0; s < SETS; ++s) acc[s][m] = i8_dot(have[s][i], a, acc[s][m]);
                }
            }
        }
#pragma unroll
        for (int s = 0; s < SETS; ++s)
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int c = c0 + 32 * AHEAD + lane + 32 * i;
                if (c < words) have[s][i] = i8_weights(w[s], c, shift[s], K);
            }
    }
    float mine = 0.f;
#pragma unroll
    for (int m = 0; m < ROWS; ++m) {
        if (m >= p.M) break;
        float v = i8_scaled(__reduce_add_sync(0xffffffffu, acc[0][m]), s_scale[m], p.w_scale[n]);
        if (SWIGLU) v = i8_scaled(__reduce_add_sync(0xffffffffu, acc[SETS - 1][m]), s_scale[m], p.w_scale[p.N + n]) * i8_silu(v);
        if (lane == m) mine = v;
    }
    if (lane < p.M) i8_store(p.out, lane * p.out_stride + n, p.out_dtype, mine);
}

bool i8_gemv_ok(const I8Problem& p) {
    return p.E == 1 && !p.offsets && p.M <= I8_GEMV_ROWS && p.K > 0 && p.w_stride >= p.K && (long long)p.M * ((p.K + 15) & ~15) <= I8G_SMEM;
}

template <int VB, int ROWS, bool SWIGLU>
static int launch_gemv(const I8Problem& p, const void* x, long long x_stride, int x_dtype, int x_vec, cudaStream_t st) {
    const size_t smem = (size_t)p.M * ((p.K + 15) & ~15);
    if (smem > 40 * 1024 && cudaFuncSetAttribute(i8_gemv_kernel<VB, ROWS, SWIGLU>, cudaFuncAttributeMaxDynamicSharedMemorySize, I8G_SMEM) != cudaSuccess)
        return VMOE_ERR_CUDA;
    return cuda_status(launch_pdl(i8_gemv_kernel<VB, ROWS, SWIGLU>, (unsigned)((p.N + 7) / 8), (unsigned)I8G_THREADS, smem, st, p,
                                  static_cast<const uint8_t*>(x), x_stride, x_dtype, x_vec));
}
template <int VB, bool SWIGLU>
static int launch_gemv_rows(const I8Problem& p, const void* x, long long x_stride, int x_dtype, int x_vec, cudaStream_t st) {
    if (p.M == 1) return launch_gemv<VB, 1, SWIGLU>(p, x, x_stride, x_dtype, x_vec, st);
    if (p.M == 2) return launch_gemv<VB, 2, SWIGLU>(p, x, x_stride, x_dtype, x_vec, st);
    if (p.M <= 4) return launch_gemv<VB, 4, SWIGLU>(p, x, x_stride, x_dtype, x_vec, st);
    return launch_gemv<VB, 8, SWIGLU>(p, x, x_stride, x_dtype, x_vec, st);
}
int launch_i8_gemv(const I8Problem& p, const void* x, long long x_stride_bytes, int x_dtype, cudaStream_t st) {
    const int el = x_dtype == VMOE_F32 ? 4 : 2;
    const int x_vec = x && (((uintptr_t)x | (unsigned long long)x_stride_bytes | (unsigned long long)p.K * el) & 15) == 0;
    const bool wide = (((uintptr_t)p.w | (unsigned long long)p.w_stride) & 15) == 0;
    if (!x) x_dtype = -1;
    if (wide) return p.swiglu ? launch_gemv_rows<16, true>(p, x, x_stride_bytes, x_dtype, x_vec, st)
                              : launch_gemv_rows<16, false>(p, x, x_stride_bytes, x_dtype, x_vec, st);
    return p.swiglu ? launch_gemv_rows<4, true>(p, x, x_stride_bytes, x_dtype, x_vec, st)
                    : launch_gemv_rows<4, false>(p, x, x_stride_bytes, x_dtype, x_vec, st);
}

}  // namespace vmoe
