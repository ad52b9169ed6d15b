// The 8-bit product for a few rows (decode of one to eight tokens), in one launch: the rows are quantised inside.  One token,
// N = 2048, K = 4096: 4.5 us (8.4 MB of weights: 1.9 TB/s, a launch alone is 2 us); N = 8192: 8.9 us (3.8 TB/s); N = 131072:
// 83 us (6.5 TB/s).
//
// Bound by reading the weights once, and at these sizes by latency: a warp requests the first 4 KB of its first channel
// (with swiglu of its gate and up rows) before anything else and quantises the rows -- every CTA for itself, 8 KB from L2
// -- while they are on their way; from then on each vector it uses is replaced at once by the one that comes next, of the
// same channel or of the warp's next one.  Codes lie in shared memory; four products per dp4a, integer sums joined by
// one warp reduction, so the result is the other kernels' bit for bit.  With swiglu two channels' vectors are under way and
// 192 to 232 bytes a thread spill at 128 registers (two CTAs an SM); its 8192 rows of weights take 8.2 us.
#include "vmoe_int8.cuh"
#include "vmoe_tc_common.cuh"

namespace vmoe {

constexpr int I8G_THREADS = 256;
constexpr int I8G_SMEM = 64 * 1024;                       // codes of all rows

// VB = 16: the weights' rows start on 16-byte boundaries; the bytes behind a row's last whole vector go to a lane each, so that
// nothing behind the row is read.  VB = 4: anywhere; a word is joined from the two aligned ones that hold it.  Only aligned words
// with a byte of the row in them are read, so a row's first and last may bring up to three bytes beside it.
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

// The rows into shared memory as codes (padded with zeros to `pitch`) and scales, all at once: the CTA's warps share the
// ROWS rows out.  Rows of whole 16-byte vectors; a thread keeps up to eight of its vectors between the two passes.
template <typename T_, int ROWS>
__device__ __forceinline__ void i8_rows_vec(const uint8_t* x, long long x_stride, int M, int K, int pitch, uint8_t* codes, float* scales, uint32_t* s_max) {
    using R = RowVec<T_, 16>;
    constexpr int WPR = 8 / ROWS, STEP = WPR * 32, KEPT = 8;
    const int warp = threadIdx.x >> 5, m = warp / WPR, part = (warp % WPR) * 32 + (threadIdx.x & 31), vecs = K / R::N;
    const uint8_t* src = x + m * x_stride;
    uint32_t top = 0;
    R keep[KEPT];
    if (m < M) {
#pragma unroll
        for (int i = 0; i < KEPT; ++i)
            if (part + i * STEP < vecs) keep[i].load(src, part + i * STEP);
#pragma unroll
        for (int i = 0; i < KEPT; ++i)
            if (part + i * STEP < vecs) top = keep[i].join(top);
        for (int c = part + KEPT * STEP; c < vecs; c += STEP) {
            R v;
            v.load(src, c);
            top = v.join(top);
        }
    }
    top = __reduce_max_sync(0xffffffffu, R::magnitude(top));
    if ((threadIdx.x & 31) == 0) s_max[warp] = top;
    __syncthreads();
    if (m >= M) return;
#pragma unroll
    for (int w = 0; w < WPR; ++w) top = max(top, s_max[m * WPR + w]);
    const I8RowScale r(top);
    uint8_t* dst = codes + (size_t)m * pitch;
    if (part == 0) scales[m] = r.scale;
    auto put = [&](const R& v, int c) {
        uint32_t w[2] = {0, 0};
        r.codes(v, w);
        if (R::N == 8) *reinterpret_cast<uint2*>(dst + c * 8) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint32_t*>(dst + c * 4) = w[0];
    };
#pragma unroll
    for (int i = 0; i < KEPT; ++i)
        if (part + i * STEP < vecs) put(keep[i], part + i * STEP);
    for (int c = part + KEPT * STEP; c < vecs; c += STEP) {
        R v;
        v.load(src, c);
        put(v, c);
    }
    for (int k = K + part; k < pitch; k += STEP) dst[k] = 0;
}
// The same for rows of any length and alignment.
template <typename T_, int ROWS>
__device__ __forceinline__ void i8_rows(const uint8_t* x, long long x_stride, int M, int K, int pitch, uint8_t* codes, float* scales, uint32_t* s_max) {
    constexpr int WPR = 8 / ROWS, STEP = WPR * 32;
    const int warp = threadIdx.x >> 5, m = warp / WPR, part = (warp % WPR) * 32 + (threadIdx.x & 31);
    const T_* src = reinterpret_cast<const T_*>(x + m * x_stride);
    uint32_t top = 0;
    if (m < M) {
#pragma unroll 4
        for (int k = part; k < K; k += STEP) top = max(top, __float_as_uint(elem_float(src[k])) & 0x7fffffffu);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) s_max[warp] = top;
    __syncthreads();
    if (m >= M) return;
#pragma unroll
    for (int w = 0; w < WPR; ++w) top = max(top, s_max[m * WPR + w]);
    const I8RowScale r(top);
    uint8_t* dst = codes + (size_t)m * pitch;
    if (part == 0) scales[m] = r.scale;
#pragma unroll 4
    for (int k = part; k < pitch; k += STEP) dst[k] = k < K ? (uint8_t)r.code(elem_float(src[k])) : 0;
}
// Rows that are codes already.
__device__ __forceinline__ void i8_rows_copy(const int8_t* a, long long a_stride, int M, int K, int pitch, uint8_t* codes) {
    const int vecs = pitch / 16;
    const bool aligned = (((uintptr_t)a | (unsigned long long)a_stride) & 15) == 0;
#pragma unroll 4
    for (int i = threadIdx.x; i < M * vecs; i += I8G_THREADS) {
        const int m = i / vecs, k = (i - m * vecs) * 16;
        const int8_t* src = a + m * a_stride + k;
        uint4 v;
        if (aligned && k + 16 <= K) {
            v = *reinterpret_cast<const uint4*>(src);
        } else {
            uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (k + j < K) w[j >> 2] |= (uint32_t)(uint8_t)src[j] << (8 * (j & 3));
            v = make_uint4(w[0], w[1], w[2], w[3]);
        }
        *reinterpret_cast<uint4*>(codes + (size_t)m * pitch + k) = v;
    }
}

// x_dtype < 0: p.a / p.a_scale hold the rows; else x does.
template <int VB, int ROWS, bool SWIGLU>
__global__ void __launch_bounds__(I8G_THREADS, 2)
i8_gemv_kernel(const I8Problem p, const uint8_t* x, long long x_stride, int x_dtype, int x_vec) {
    using W = typename I8Word<VB>::type;
    constexpr int AHEAD = VB == 16 ? 8 : 16, SETS = SWIGLU ? 2 : 1;
    extern __shared__ __align__(16) uint8_t codes[];
    __shared__ uint32_t s_max[I8G_THREADS / 32];
    __shared__ float s_scale[ROWS];
    pdl_begin();
    const int lane = threadIdx.x & 31, stride = gridDim.x * (I8G_THREADS / 32);
    int n = blockIdx.x * (I8G_THREADS / 32) + (threadIdx.x >> 5);
    const int K = p.K, pitch = (K + 15) & ~15, words = VB == 16 ? K / 16 : (K + 3) / 4, over = VB == 16 ? K & 15 : 0;
    const W* w[SETS];
    int shift[SETS];
    float scale[SETS] = {};                               // of the channel whose vectors come next: requested with them
    auto channel = [&](int c) {
#pragma unroll
        for (int s = 0; s < SETS; ++s) {
            scale[s] = p.w_scale[s * p.N + c];
            const uintptr_t at = (uintptr_t)(p.w + (long long)(s * p.N + c) * p.w_stride);
            shift[s] = VB == 4 ? (int)(at & 3) : 0;
            w[s] = reinterpret_cast<const W*>(at - shift[s]);
        }
    };
    W have[SETS][AHEAD];
    if (n < p.N) channel(n);
#pragma unroll
    for (int s = 0; s < SETS; ++s)
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            have[s][i] = W{};
            if (n < p.N && lane + 32 * i < words) have[s][i] = i8_weights(w[s], lane + 32 * i, shift[s], K);
        }
    if (x_dtype < 0) {
        i8_rows_copy(p.a, p.a_stride, p.M, K, pitch, codes);
        if (threadIdx.x < p.M) s_scale[threadIdx.x] = p.a_scale[threadIdx.x];
    } else {
#define VMOE_I8_ROWS(T) (x_vec ? i8_rows_vec<T, ROWS>(x, x_stride, p.M, K, pitch, codes, s_scale, s_max) \
                               : i8_rows<T, ROWS>(x, x_stride, p.M, K, pitch, codes, s_scale, s_max))
        if (x_dtype == VMOE_BF16) VMOE_I8_ROWS(__nv_bfloat16);
        else if (x_dtype == VMOE_F16) VMOE_I8_ROWS(__half);
        else VMOE_I8_ROWS(float);
#undef VMOE_I8_ROWS
    }
    __syncthreads();
    for (; n < p.N; n += stride) {
        int acc[SETS][ROWS] = {};
        float sw[SETS];
#pragma unroll
        for (int s = 0; s < SETS; ++s) sw[s] = scale[s];
        for (int c0 = 0; c0 == 0 || c0 < words; c0 += 32 * AHEAD) {       // once at least: it brings the next channel
            const bool last = c0 + 32 * AHEAD >= words;
            const int next = last ? 0 : c0 + 32 * AHEAD;
            const bool more = !last || n + stride < p.N;
            if (last && more) channel(n + stride);
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int c = c0 + lane + 32 * i;
                if (c < words) {
                    // (of a row's last word) bytes behind K meet zero codes
#pragma unroll
                    for (int m = 0; m < ROWS; ++m) {
                        if (m >= p.M) break;
                        const W a = *reinterpret_cast<const W*>(codes + (size_t)m * pitch + (size_t)c * VB);
#pragma unroll
                        for (int s = 0; s < SETS; ++s) acc[s][m] = i8_dot(have[s][i], a, acc[s][m]);
                    }
                }
                const int cn = next + lane + 32 * i;
                if (more && cn < words) {
#pragma unroll
                    for (int s = 0; s < SETS; ++s) have[s][i] = i8_weights(w[s], cn, shift[s], K);
                }
            }
        }
        if (lane < over) {
            int tail[SETS];
#pragma unroll
            for (int s = 0; s < SETS; ++s) tail[s] = p.w[(long long)(s * p.N + n) * p.w_stride + K - over + lane];
#pragma unroll
            for (int m = 0; m < ROWS; ++m) {
                if (m >= p.M) break;
                const int a = static_cast<int8_t>(codes[(size_t)m * pitch + K - over + lane]);
#pragma unroll
                for (int s = 0; s < SETS; ++s) acc[s][m] += tail[s] * a;
            }
        }
        float mine = 0.f;
#pragma unroll
        for (int m = 0; m < ROWS; ++m) {
            if (m >= p.M) break;
            float v = i8_scaled(__reduce_add_sync(0xffffffffu, acc[0][m]), s_scale[m], sw[0]);
            if (SWIGLU) v = i8_scaled(__reduce_add_sync(0xffffffffu, acc[SETS - 1][m]), s_scale[m], sw[SETS - 1]) * i8_silu(v);
            if (lane == m) mine = v;
        }
        if (lane < p.M) i8_store(p.out, lane * p.out_stride + n, p.out_dtype, mine);
    }
}

// When this kernel is the better one, against quantiser + tensor-core product (weights that no copy can read: + packing).
// A channel costs it 0.27 ns (1 row) to 0.5 (8 rows) however short it is, a KB of weights 0.14 ns (1 row, HBM speed), 0.17, 0.2
// and 0.22 (4 rows), and the rows are quantised in every block; the others cost 3 to 5 us more to begin with.  us:
//   K = 1024   8192 channels, 1 / 4 / 8 rows   5.4 / 6.8 / 8.8 against 9.3      16384, 1 / 2 / 4   7.8 / 8.5 / 10.0 against 9.0
//              131072, 1 / 4   42 / 59 against 28 (K = 256: 37 / 53 against 12)
//   K = 4096   8192, 1 / 3 / 4   8.9 / 11.4 / 12.5 against 13.0                 16384, 2 / 3 / 4   15.2 / 17.1 / 18.7 against 17.5
//              32768, 1 / 2 / 3  24.4 / 26.1 / 29.4 against 26.8                131072, 1 / 2 / 4  83 / 92 / 112 against 87
//   K = 8192   1024, 4 / 8       10.5 / 17.1 against 9.9                        8192, 1 / 2 / 3    14.6 / 16.6 / 20.1 against 18.9
//   rows of words (K = 1000)     4096, 1 / 8   5.3 / 9.5 against 10.4           16384, 1 / 4 / 8   11.9 / 17.5 / 24 against 16.2
//                 (K = 4088)     4096, 1 / 4 / 8   10.8 / 15.8 / 23.8 against 15.9
//   of bytes (K = 1001)          1024, 1 / 4 / 8   6.1 / 9.2 / 12.5 against 8.4     4096, 1 / 8   13.5 / 21.1 against 11.2
//            (K = 4095)          4096, 1 / 8       43 / 71 against 21
// A call on its own takes 10 us of the host with one launch and 17 to 20 with two or three, so near a draw it is this one.
static bool i8_few_rows(long long M, long long wrows, long long K, int align) {
    const long long MB = 1 << 20, bytes = wrows * K;
    if (align < 4) return bytes <= (M <= 4 ? 2 * MB : MB);
    if (M > 4) return bytes <= 8 * MB && (align < 16 || (K <= 4096 && wrows <= 8192));
    if (align < 16) return true;
    if (K < 2048) return wrows <= (M <= 2 && K >= 1024 ? 16384 : 8192);
    return M == 1 || bytes <= (M == 2 ? 128 * MB : M == 3 ? 32 * MB : 24 * MB);
}
static int i8_row_align(unsigned long long address_or_stride) { return address_or_stride % 16 == 0 ? 16 : address_or_stride % 4 == 0 ? 4 : 1; }
static bool i8_gemv_takes(long long M, long long K) { return M <= I8_GEMV_ROWS && K > 0 && M * ((K + 15) & ~15LL) <= I8G_SMEM; }

bool i8_gemv_fits(const I8Problem& p) { return p.E == 1 && !p.offsets && p.w_stride >= p.K && i8_gemv_takes(p.M, p.K); }
bool i8_gemv_ok(const I8Problem& p) {
    return i8_gemv_fits(p) && i8_few_rows(p.M, p.wrows, p.K, i8_row_align((unsigned long long)(uintptr_t)p.w | (unsigned long long)p.w_stride));
}

template <int VB, int ROWS, bool SWIGLU>
static int launch_gemv(const I8Problem& p, const void* x, long long x_stride, int x_dtype, int x_vec, cudaStream_t st) {
    const size_t smem = (size_t)p.M * ((p.K + 15) & ~15);
    static SmemAllowed done;
    if (allow_smem(i8_gemv_kernel<VB, ROWS, SWIGLU>, I8G_SMEM, done) != cudaSuccess) return VMOE_ERR_CUDA;
    // two CTAs an SM, every warp the same number of channels
    const long long warps = 2LL * tc_sm_count() * (I8G_THREADS / 32), rounds = (p.N + warps - 1) / warps;
    const unsigned grid = (unsigned)((p.N + rounds * (I8G_THREADS / 32) - 1) / (rounds * (I8G_THREADS / 32)));
    return launch_status(launch_pdl(i8_gemv_kernel<VB, ROWS, SWIGLU>, grid, (unsigned)I8G_THREADS, smem, st, p,
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

extern "C" int vmoe_int8_one_launch(int32_t M, int32_t weight_rows, int32_t K, int32_t align) {
    return M > 0 && weight_rows > 0 && align > 0 && vmoe::i8_gemv_takes(M, K) &&
           vmoe::i8_few_rows(M, weight_rows, K, vmoe::i8_row_align((unsigned long long)align));
}
