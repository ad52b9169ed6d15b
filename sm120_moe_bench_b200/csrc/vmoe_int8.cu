// 8-bit integer rows: the row quantiser and the product's entry point.  (No pointer is __restrict__: see vmoe_sort.cu.)
#include "vmoe_int8.cuh"

namespace vmoe {

// ---------------------------------------------------------------------------------
// Row quantiser: scale = max|x| / 127, code = rint(127 x / max|x|), ties to even -- the code of the exact quotient, not of
// a rounded one.  y = x * RN(127 / max|x|) is off by at most 127 * 2^-23 < 2e-5, so only vectors with a y within 1e-4 of a
// border between two codes are decided in 64 bits.  A row of zeros has scale 0 and codes 0; a row with an infinity or a NaN has
// scale NaN and codes 0, so that its outputs are NaN and no other row's are.
// WPR warps per row, eight per CTA.  With row_of_pair a row is a token and its codes go to the token's T sorted rows.
// A thread keeps up to four vectors of the row in registers, so that rows of up to 4 * 32 * WPR vectors are read once.
// Rounding adds 1.5 * 2^23: the sum's low byte is the code, and taking the constant off again gives the rounded value.
// ---------------------------------------------------------------------------------
constexpr float I8_ROUND = 12582912.f;
constexpr int I8_KEPT = 4;

template <typename R>
__device__ __forceinline__ void i8_codes(const R& v, float up, float inv, float amax, uint32_t (&w)[2]) {
    float t[R::N], far = 0.f;
#pragma unroll
    for (int k = 0; k < R::N; ++k) {
        const float y = v.get(k) * up * inv;
        t[k] = y + I8_ROUND;
        far = fmaxf(far, fabsf(y - (t[k] - I8_ROUND)));
    }
    if (far > 0.5f - 1e-4f) {                            // next to a border
#pragma unroll
        for (int k = 0; k < R::N; ++k) t[k] = I8_ROUND + (float)rint(127.0 * (double)(v.get(k) * up) / (double)amax);
    }
#pragma unroll
    for (int h = 0; h < (R::N + 3) / 4; ++h) {
        uint32_t b[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) b[k] = 4 * h + k < R::N ? __float_as_uint(t[4 * h + k < R::N ? 4 * h + k : 0]) : 0u;
        w[h] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    }
}

template <typename T_, int VB, int WPR>
__global__ void __launch_bounds__(256)
i8_quantize_kernel(const uint8_t* x, long long x_stride, long long rows, int vecs, int T, const int32_t* row_of_pair,
                   const int32_t* live, int8_t* q, long long q_stride, float* scales) {
    using R = RowVec<T_, VB>;
    __shared__ uint32_t s_max[8];
    pdl_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long m = (long long)blockIdx.x * (8 / WPR) + warp / WPR;
    const int part = (warp % WPR) * 32 + lane;
    const bool on = m < rows && (!live || m < *live);
    const uint8_t* src = x + m * x_stride;
    uint32_t top = 0;                                    // magnitudes ordered as integers: NaN > infinity > finite
    R keep[I8_KEPT];
    if (on) {
#pragma unroll
        for (int i = 0; i < I8_KEPT; ++i)
            if (part + i * WPR * 32 < vecs) keep[i].load(src, part + i * WPR * 32);
#pragma unroll
        for (int i = 0; i < I8_KEPT; ++i)
            if (part + i * WPR * 32 < vecs) {
#pragma unroll
                for (int k = 0; k < R::N; ++k) top = max(top, __float_as_uint(keep[i].get(k)) & 0x7fffffffu);
            }
        for (int c = part + I8_KEPT * WPR * 32; c < vecs; c += WPR * 32) {
            R v;
            v.load(src, c);
#pragma unroll
            for (int k = 0; k < R::N; ++k) top = max(top, __float_as_uint(v.get(k)) & 0x7fffffffu);
        }
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (WPR > 1) {
        if (lane == 0) s_max[warp] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WPR; ++w) top = max(top, s_max[warp / WPR * WPR + w]);
    }
    if (!on) return;
    const bool finite = top < 0x7f800000u;
    float amax = __uint_as_float(top);
    const float scale = finite ? amax / 127.f : __uint_as_float(0x7fc00000u);
    const float up = amax < 0x1p-100f ? 0x1p100f : 1.f;  // keeps 127 / max|x| in range; exact
    amax *= up;
    const float inv = finite && amax > 0.f ? 127.f / amax : 0.f;
    const int copies = row_of_pair ? T : 1;
    if (part == 0)
        for (int t = 0; t < copies; ++t) {
            const long long r = row_of_pair ? row_of_pair[m * T + t] : m;
            if (r >= 0) scales[r] = scale;
        }
    auto put = [&](const R& v, int c) {
        uint32_t w[2] = {0, 0};
        if (inv > 0.f) i8_codes(v, up, inv, amax, w);
        for (int t = 0; t < copies; ++t) {
            const long long r = row_of_pair ? row_of_pair[m * T + t] : m;
            if (r < 0) continue;
            int8_t* dst = q + r * q_stride + (long long)c * R::N;
            if (R::N == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
            else if (R::N == 4) *reinterpret_cast<uint32_t*>(dst) = w[0];
            else if (R::N == 2) *reinterpret_cast<uint16_t*>(dst) = (uint16_t)w[0];
            else *dst = (int8_t)w[0];
        }
    };
#pragma unroll
    for (int i = 0; i < I8_KEPT; ++i)
        if (part + i * WPR * 32 < vecs) put(keep[i], part + i * WPR * 32);
    for (int c = part + I8_KEPT * WPR * 32; c < vecs; c += WPR * 32) {
        R v;
        v.load(src, c);
        put(v, c);
    }
}

// ---------------------------------------------------------------------------------
// Product, any stride and alignment: 64 x 64 outputs per CTA, four by four per thread, 64 bytes of K at a time through
// shared memory, four products per dp4a.
// ---------------------------------------------------------------------------------
constexpr int I8_TILE = 64, I8_WORDS = 16, I8_PITCH = I8_WORDS + 1;

__device__ __forceinline__ uint32_t i8_word(const int8_t* row, int k, int K, bool aligned) {
    if (aligned && k + 4 <= K) return *reinterpret_cast<const uint32_t*>(row + k);
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (k + i < K) w |= (uint32_t)(uint8_t)row[k + i] << (8 * i);
    return w;
}

template <bool SWIGLU>
__global__ void __launch_bounds__(256)
i8_tile_kernel(const I8Problem p, int aligned_a, int aligned_w) {
    __shared__ uint32_t sa[I8_TILE][I8_PITCH], sw[SWIGLU ? 2 : 1][I8_TILE][I8_PITCH];
    pdl_begin();
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int e = blockIdx.y, n0 = blockIdx.x * I8_TILE;
    const int first = p.offsets ? p.offsets[e] : 0, end = p.offsets ? p.offsets[e + 1] : p.M;
    const int8_t* w = p.w + e * p.w_expert_stride;
    const float* wscale = p.w_scale + (long long)e * p.wrows;
    for (long long m0 = first + (long long)blockIdx.z * I8_TILE; m0 < end; m0 += (long long)gridDim.z * I8_TILE) {
        int acc[SWIGLU ? 2 : 1][4][4] = {};
        for (int k0 = 0; k0 < p.K; k0 += 4 * I8_WORDS) {
            __syncthreads();
            for (int i = tid; i < I8_TILE * I8_WORDS; i += 256) {
                const int r = i / I8_WORDS, c = i % I8_WORDS, k = k0 + 4 * c;
                sa[r][c] = m0 + r < end ? i8_word(p.a + (m0 + r) * p.a_stride, k, p.K, aligned_a) : 0u;
#pragma unroll
                for (int h = 0; h < (SWIGLU ? 2 : 1); ++h)
                    sw[h][r][c] = n0 + r < p.N ? i8_word(w + (long long)(h * p.N + n0 + r) * p.w_stride, k, p.K, aligned_w) : 0u;
            }
            __syncthreads();
#pragma unroll
            for (int c = 0; c < I8_WORDS; ++c) {
                uint32_t av[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) av[i] = sa[ty * 4 + i][c];
#pragma unroll
                for (int h = 0; h < (SWIGLU ? 2 : 1); ++h)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t wv = sw[h][tx + 16 * j][c];
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[h][i][j] = __dp4a((int)av[i], (int)wv, acc[h][i][j]);
                    }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const long long m = m0 + ty * 4 + i;
            if (m >= end) continue;
            const float s = p.a_scale[m];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int n = n0 + tx + 16 * j;
                if (n >= p.N) continue;
                float v = i8_scaled(acc[0][i][j], s, wscale[n]);
                if (SWIGLU) v = i8_scaled(acc[SWIGLU ? 1 : 0][i][j], s, wscale[p.N + n]) * i8_silu(v);
                i8_store(p.out, m * p.out_stride + n, p.out_dtype, v);
            }
        }
    }
    if (p.offsets && p.zero_tail) {
        const long long block = blockIdx.x + (long long)gridDim.x * (blockIdx.y + (long long)gridDim.y * blockIdx.z);
        const long long blocks = (long long)gridDim.x * gridDim.y * gridDim.z;
        for (long long m = p.offsets[p.E] + block; m < p.M; m += blocks)
            for (int n = tid; n < p.N; n += 256) i8_store(p.out, m * p.out_stride + n, p.out_dtype, 0.f);
    }
}

static int launch_i8_tile(const I8Problem& p, cudaStream_t st) {
    const long long tiles = ((long long)p.M + I8_TILE - 1) / I8_TILE;
    const unsigned z = (unsigned)(tiles < 1 ? 1 : p.E > 1 ? (tiles < 4 ? tiles : 4) : (tiles < 65535 ? tiles : 65535));
    const bool aa = ((uintptr_t)p.a | (unsigned long long)p.a_stride) % 4 == 0;
    const bool aw = ((uintptr_t)p.w | (unsigned long long)p.w_stride | (unsigned long long)p.w_expert_stride) % 4 == 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((p.N + I8_TILE - 1) / I8_TILE), (unsigned)p.E, z); cfg.blockDim = dim3(256); cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 1;
    return cuda_status(p.swiglu ? cudaLaunchKernelEx(&cfg, i8_tile_kernel<true>, p, (int)aa, (int)aw)
                                : cudaLaunchKernelEx(&cfg, i8_tile_kernel<false>, p, (int)aa, (int)aw));
}

}  // namespace vmoe

using namespace vmoe;

extern "C" {

int vmoe_int8_quantize(const void* x, int64_t x_stride, int32_t dtype, int32_t rows, int32_t K, int32_t T, const int32_t* row_of_pair,
                       const int32_t* live_rows, int8_t* q, int64_t q_stride, float* scales, void* stream) {
    if (rows < 0 || K < 0 || dtype < VMOE_BF16 || dtype > VMOE_F32 || x_stride < 0 || q_stride < K) return VMOE_ERR_SHAPE;
    if (row_of_pair && (T <= 0 || T > MAX_TOPK)) return VMOE_ERR_SHAPE;
    if (rows == 0) return VMOE_OK;
    if (!scales || (K > 0 && (!x || !q))) return VMOE_ERR_NULL;
    const long long el = dtype == VMOE_F32 ? 4 : 2, xs = x_stride * el;
    if ((uintptr_t)x & (el - 1)) return VMOE_ERR_ALIGN;
    // a vector of n elements becomes n bytes: both sides have to allow it
    int vb = vector_bytes((uintptr_t)x, xs | K * el);
    const int qb = vector_bytes((uintptr_t)q, q_stride);
    const int q_odd = (((uintptr_t)q | (unsigned long long)q_stride) & 1) != 0;
    const int most = (q_odd ? 1 : qb > 8 ? 8 : qb) * (int)el;
    if (vb > most) vb = most;
    return with_rows(dtype, vb, [&](auto r) {
        using R = decltype(r);
        const int vecs = K / R::N;
        const auto a = static_cast<const uint8_t*>(x);
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        if (vecs <= 64)
            return cuda_status(launch_pdl(i8_quantize_kernel<typename R::T, R::BYTES, 1>, (unsigned)((rows + 7LL) / 8), 256u, 0, st, a, xs,
                                          (long long)rows, vecs, T, row_of_pair, live_rows, q, q_stride, scales));
        if (vecs <= 256)
            return cuda_status(launch_pdl(i8_quantize_kernel<typename R::T, R::BYTES, 2>, (unsigned)((rows + 3LL) / 4), 256u, 0, st, a, xs,
                                          (long long)rows, vecs, T, row_of_pair, live_rows, q, q_stride, scales));
        if (vecs <= 512)
            return cuda_status(launch_pdl(i8_quantize_kernel<typename R::T, R::BYTES, 4>, (unsigned)((rows + 1LL) / 2), 256u, 0, st, a, xs,
                                          (long long)rows, vecs, T, row_of_pair, live_rows, q, q_stride, scales));
        return cuda_status(launch_pdl(i8_quantize_kernel<typename R::T, R::BYTES, 8>, (unsigned)rows, 256u, 0, st, a, xs, (long long)rows,
                                      vecs, T, row_of_pair, live_rows, q, q_stride, scales));
    });
}

int vmoe_int8_matmul(const int8_t* a, int64_t a_stride, const float* a_scale, int32_t M, const int8_t* w, int64_t w_stride,
                     int64_t w_expert_stride, const float* w_scale, int32_t N, int32_t K, int32_t E, const int32_t* expert_offsets,
                     int32_t swiglu, int32_t zero_tail, void* out, int64_t out_stride, int32_t out_dtype, void* stream) {
    if (M < 0 || N <= 0 || K < 0 || E <= 0 || out_dtype < VMOE_BF16 || out_dtype > VMOE_F32) return VMOE_ERR_SHAPE;
    if (a_stride < 0 || w_stride < 0 || w_expert_stride < 0 || out_stride < N || (!expert_offsets && E != 1)) return VMOE_ERR_SHAPE;
    if (K > I8_MAX_K || E > 65535 || N > (1 << 30)) return VMOE_ERR_LIMIT;
    if (M == 0) return VMOE_OK;
    if (!a_scale || !w_scale || !out || (K > 0 && (!a || !w))) return VMOE_ERR_NULL;
    if ((uintptr_t)out & (out_dtype == VMOE_F32 ? 3 : 1)) return VMOE_ERR_ALIGN;
    I8Problem p;
    p.a = a; p.a_stride = a_stride; p.a_scale = a_scale;
    p.w = w; p.w_stride = w_stride; p.w_expert_stride = w_expert_stride; p.w_scale = w_scale;
    p.out = out; p.out_stride = out_stride; p.offsets = expert_offsets;
    p.M = M; p.N = N; p.K = K; p.E = E; p.wrows = swiglu ? 2 * N : N; p.swiglu = swiglu; p.out_dtype = out_dtype; p.zero_tail = zero_tail;
    if (M == 1) p.a_stride = (K + 15) / 16 * 16;             // the stride of a single row says nothing
    if (p.wrows == 1) p.w_stride = (K + 15) / 16 * 16;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!i8_tc_ok(p) || E > I8_TC_MAX_EXPERTS) return launch_i8_tile(p, st);
    if (!expert_offsets) {
        const long long items = (M + 127LL) / 128 * ((N + (swiglu ? 127LL : 255LL)) / (swiglu ? 128 : 256));
        if (items < 148) return launch_i8_split(p, st);
    }
    return launch_i8_tc(p, st);
}

}  // extern "C"
