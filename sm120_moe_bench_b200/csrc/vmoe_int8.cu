// 8-bit integer rows: the row quantiser and the product's entry point.  (No pointer is __restrict__: see vmoe_sort.cu.)
#include "vmoe_int8.cuh"

namespace vmoe {

// ---------------------------------------------------------------------------------
// Rows to codes (the arithmetic: I8RowScale).  WPR warps per row, eight per CTA; a thread keeps up to eight vectors of the
// row in registers, so that rows of up to 8 * 32 * WPR vectors are read once.  With row_of_pair a row is a token and its
// codes go to the token's T sorted rows.  8192 x 4096 bf16: 21 us (4.8 TB/s; at a copy's rate 15.4): four CTAs an SM leave 64
// registers, and the 16-byte instances for 16-bit rows spill up to 36 bytes a thread.
// ---------------------------------------------------------------------------------
constexpr int I8_KEPT = 8;

template <typename T_, int VB, int WPR, bool SORTED>
__global__ void __launch_bounds__(256, 4)
i8_quantize_kernel(const uint8_t* x, long long x_stride, long long rows, int vecs, int T, const int32_t* row_of_pair,
                   const int32_t* live, int8_t* q, long long q_stride, float* scales) {
    using R = RowVec<T_, VB>;
    constexpr int STEP = WPR * 32;
    __shared__ uint32_t s_max[8];
    pdl_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long m = (long long)blockIdx.x * (8 / WPR) + warp / WPR;
    const int part = (warp % WPR) * 32 + lane;
    const bool on = m < rows && (!live || m < *live);
    const uint8_t* src = x + m * x_stride;
    uint32_t top = 0;
    R keep[I8_KEPT];
    if (on) {
#pragma unroll
        for (int i = 0; i < I8_KEPT; ++i)
            if (part + i * STEP < vecs) keep[i].load(src, part + i * STEP);
#pragma unroll
        for (int i = 0; i < I8_KEPT; ++i)
            if (part + i * STEP < vecs) top = keep[i].join(top);
        for (int c = part + I8_KEPT * STEP; c < vecs; c += STEP) {
            R v;
            v.load(src, c);
            top = v.join(top);
        }
    }
    top = __reduce_max_sync(0xffffffffu, R::magnitude(top));
    if (WPR > 1) {
        if (lane == 0) s_max[warp] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WPR; ++w) top = max(top, s_max[warp / WPR * WPR + w]);
    }
    if (!on) return;
    const I8RowScale rs(top);
    // a sorted row's place; outside the rows there are (a table not made by vmoe_plan_tokens): dropped
    auto place = [&](int t) { const int r = row_of_pair[m * T + t]; return r < rows * T ? r : -1; };
    if (SORTED) {
        for (int t = part; t < T; t += STEP)
            if (place(t) >= 0) scales[place(t)] = rs.scale;
    } else if (part == 0) {
        scales[m] = rs.scale;
    }
    auto store = [&](long long r, int c, const uint32_t (&w)[2]) {
        int8_t* dst = q + r * q_stride + (long long)c * R::N;
        if (R::N == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
        else if (R::N == 4) *reinterpret_cast<uint32_t*>(dst) = w[0];
        else if (R::N == 2) *reinterpret_cast<uint16_t*>(dst) = (uint16_t)w[0];
        else *dst = (int8_t)w[0];
    };
    auto put = [&](const R& v, int c) {
        uint32_t w[2];
        rs.codes(v, w);
        if (SORTED) {
            for (int t = 0; t < T; ++t) {
                const int r = place(t);
                if (r >= 0) store(r, c, w);
            }
        } else {
            store(m, c, w);
        }
    };
#pragma unroll
    for (int i = 0; i < I8_KEPT; ++i)
        if (part + i * STEP < vecs) put(keep[i], part + i * STEP);
    for (int c = part + I8_KEPT * STEP; c < vecs; c += STEP) {
        R v;
        v.load(src, c);
        put(v, c);
    }
}

template <typename T_, int VB, int WPR>
static int launch_quantize_rows(const void* x, long long xs, long long rows, int vecs, int T, const int32_t* row_of_pair, const int32_t* live,
                                int8_t* q, long long q_stride, float* scales, cudaStream_t st) {
    const unsigned grid = (unsigned)((rows + 8 / WPR - 1) / (8 / WPR));
    const auto a = static_cast<const uint8_t*>(x);
    return launch_status(row_of_pair
        ? launch_pdl(i8_quantize_kernel<T_, VB, WPR, true>, grid, 256u, 0, st, a, xs, rows, vecs, T, row_of_pair, live, q, q_stride, scales)
        : launch_pdl(i8_quantize_kernel<T_, VB, WPR, false>, grid, 256u, 0, st, a, xs, rows, vecs, T, row_of_pair, live, q, q_stride, scales));
}

// ---------------------------------------------------------------------------------
// Small batches of the expert layer: plan and quantiser in one launch.  A CTA per token counts, over all ids, the pairs in
// front of each of its own (a smaller expert, or the same and an earlier pair): that is the pair's row, with no word from any
// other CTA.  One more CTA counts the experts' offsets.  The counting grows with the pairs squared, so there is a limit.  The
// whole layer, plan + quantiser -> this (us; K, N, experts, top-k):
//   10 pairs    4096, 256, 16, 2: 32.0 -> 27.7     4096, 64, 512, 10: 45.2 -> 37.0     512, 256, 64, 10: 21.1 -> 18.4
//   1000 pairs  4096, 256, 16, 2: 43.4 -> 39.3     4096, 64, 512, 10: 144  -> 139      512, 256, 64, 10: 28.8 -> 24.9
// Limits of 2048 and 4096 cost the small sizes 0.5 and 2 us (more ids per thread) and give 2 us or nothing above 1024, and the
// largest lose: 4000 pairs of 1024, 256, 32, 1: 43 -> 53.
// ---------------------------------------------------------------------------------
constexpr int FRONT_THREADS = 256, FRONT_PAIRS = 1024, FRONT_IDS = FRONT_PAIRS / FRONT_THREADS;

template <typename T_, int VB>
__global__ void __launch_bounds__(FRONT_THREADS)
i8_front_kernel(const uint8_t* x, long long x_stride, int M, int vecs, int T, const int32_t* ids, const int32_t* expert_map, int map_len,
                int E, int32_t* offsets, int32_t* row_of_pair, int8_t* q, long long q_stride, float* scales) {
    using R = RowVec<T_, VB>;
    constexpr int WARPS = FRONT_THREADS / 32, KEPT = 4;
    extern __shared__ int s_count[];                     // [E], the offsets' CTA only
    __shared__ uint32_t s_max[WARPS];
    __shared__ int s_expert[MAX_TOPK], s_part[WARPS][MAX_TOPK], s_row[MAX_TOPK];
    pdl_begin();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, m = blockIdx.x, P = M * T;
    auto expert = [&](int p) {
        int e = ids[p];
        if (expert_map) e = e >= 0 && e < map_len ? expert_map[e] : -1;
        return e >= 0 && e < E ? e : -1;
    };
    int other[FRONT_IDS];                                // -1: dropped, or behind the last pair
#pragma unroll
    for (int i = 0; i < FRONT_IDS; ++i) {
        other[i] = -1;
        if (tid + i * FRONT_THREADS < P) other[i] = expert(tid + i * FRONT_THREADS);
    }
    if (m == M) {
        for (int e = tid; e < E; e += FRONT_THREADS) s_count[e] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < FRONT_IDS; ++i)
            if (other[i] >= 0) atomicAdd(&s_count[other[i]], 1);
        __syncthreads();
        const int per = (E + FRONT_THREADS - 1) / FRONT_THREADS;     // every thread a contiguous run of experts
        int sum = 0;
        for (int k = 0; k < per; ++k) { const int e = tid * per + k; if (e < E) sum += s_count[e]; }
        int incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= o) incl += v; }
        if (lane == 31) s_part[warp][0] = incl;
        __syncthreads();
        int at = incl - sum;
        for (int w = 0; w < warp; ++w) at += s_part[w][0];
        for (int k = 0; k < per; ++k) {
            const int e = tid * per + k;
            if (e < E) { offsets[e] = at; at += s_count[e]; }
        }
        if (tid == FRONT_THREADS - 1) offsets[E] = at;   // the last run ends behind the last expert
        return;
    }
    const uint8_t* src = x + m * x_stride;
    R keep[KEPT];
#pragma unroll
    for (int i = 0; i < KEPT; ++i)
        if (tid + i * FRONT_THREADS < vecs) keep[i].load(src, tid + i * FRONT_THREADS);
    if (tid < T) s_expert[tid] = expert(m * T + tid);
    __syncthreads();
    for (int t = 0; t < T; ++t) {
        const int e = s_expert[t], p = m * T + t;
        int front = 0;
#pragma unroll
        for (int i = 0; i < FRONT_IDS; ++i)
            front += other[i] >= 0 && (other[i] < e || (other[i] == e && tid + i * FRONT_THREADS < p)) ? 1 : 0;
        front = __reduce_add_sync(0xffffffffu, front);
        if (lane == 0) s_part[warp][t] = front;
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < KEPT; ++i)
        if (tid + i * FRONT_THREADS < vecs) top = keep[i].join(top);
    for (int c = tid + KEPT * FRONT_THREADS; c < vecs; c += FRONT_THREADS) {
        R v;
        v.load(src, c);
        top = v.join(top);
    }
    top = __reduce_max_sync(0xffffffffu, R::magnitude(top));
    if (lane == 0) s_max[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = max(top, s_max[w]);
    const I8RowScale rs(top);
    if (tid < T) {
        int row = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) row += s_part[w][tid];
        if (s_expert[tid] < 0) row = -1;
        s_row[tid] = row;
        row_of_pair[m * T + tid] = row;
        if (row >= 0) scales[row] = rs.scale;
    }
    __syncthreads();
    auto put = [&](const R& v, int c) {
        uint32_t w[2];
        rs.codes(v, w);
        for (int t = 0; t < T; ++t) {
            const long long r = s_row[t];
            if (r < 0) continue;
            int8_t* dst = q + r * q_stride + (long long)c * R::N;
            if (R::N == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
            else if (R::N == 4) *reinterpret_cast<uint32_t*>(dst) = w[0];
            else if (R::N == 2) *reinterpret_cast<uint16_t*>(dst) = (uint16_t)w[0];
            else *dst = (int8_t)w[0];
        }
    };
#pragma unroll
    for (int i = 0; i < KEPT; ++i)
        if (tid + i * FRONT_THREADS < vecs) put(keep[i], tid + i * FRONT_THREADS);
    for (int c = tid + KEPT * FRONT_THREADS; c < vecs; c += FRONT_THREADS) {
        R v;
        v.load(src, c);
        put(v, c);
    }
}

static int launch_i8_front(const void* x, long long x_stride, int dtype, int M, int T, int K, const int32_t* ids, const int32_t* expert_map,
                           int map_len, int E, int32_t* offsets, int32_t* row_of_pair, int8_t* q, long long q_stride, float* scales,
                           cudaStream_t st) {
    const long long el = dtype == VMOE_F32 ? 4 : 2, xs = x_stride * el;
    if ((uintptr_t)x & (el - 1)) return VMOE_ERR_ALIGN;
    return with_rows(dtype, vector_bytes((uintptr_t)x, xs | K * el), [&](auto r) {     // the codes' rows start on 16-byte boundaries
        using R = decltype(r);
        return launch_status(launch_pdl(i8_front_kernel<typename R::T, R::BYTES>, (unsigned)M + 1, (unsigned)FRONT_THREADS, (size_t)E * sizeof(int),
                                        st, static_cast<const uint8_t*>(x), xs, M, K / R::N, T, ids, expert_map, map_len, E, offsets,
                                        row_of_pair, q, q_stride, scales));
    });
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
    const int first = p.offsets ? max(p.offsets[e], 0) : 0, end = p.offsets ? min(p.offsets[e + 1], p.M) : p.M;
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
        for (long long m = max(p.offsets[p.E], 0) + block; m < p.M; m += blocks)
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
    return launch_status(p.swiglu ? cudaLaunchKernelEx(&cfg, i8_tile_kernel<true>, p, (int)aa, (int)aw)
                                : cudaLaunchKernelEx(&cfg, i8_tile_kernel<false>, p, (int)aa, (int)aw));
}

// Both operands of a product, rows of any alignment, to rows that start on 16-byte boundaries: one thread per 16 codes,
// first those of a [M], then those of w [E][wrows].  Columns behind K become zero.
__global__ void __launch_bounds__(256)
i8_pack_kernel(const I8Problem p, int pack_a, int8_t* a, int8_t* w) {
    pdl_begin();
    const int K = p.K, vecs = (K + 15) / 16;
    const long long in_a = pack_a ? (long long)p.M * vecs : 0;
    long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    const int8_t* src;
    int8_t* dst;
    int k;
    if (i < in_a) {
        const long long r = i / vecs;
        k = (int)(i - r * vecs) * 16;
        src = p.a + r * p.a_stride + k;
        dst = a + r * vecs * 16 + k;
    } else {
        i -= in_a;
        const long long r = i / vecs, e = r / p.wrows;
        if (!w || e >= p.E) return;
        k = (int)(i - r * vecs) * 16;
        src = p.w + e * p.w_expert_stride + (r - e * p.wrows) * p.w_stride + k;
        dst = w + r * vecs * 16 + k;
    }
    const bool aligned = ((uintptr_t)src & 3) == 0;
    uint4 v;
    v.x = i8_word(src, 0, K - k, aligned); v.y = i8_word(src, 4, K - k, aligned);
    v.z = i8_word(src, 8, K - k, aligned); v.w = i8_word(src, 12, K - k, aligned);
    *reinterpret_cast<uint4*>(dst) = v;
}

static int i8_pitch(int K) { return (K + 15) / 16 * 16; }
static size_t i8_align(size_t n) { return (n + 255) & ~(size_t)255; }

static int i8_problem(I8Problem* p, const int8_t* a, long long a_stride, const float* a_scale, int M, const int8_t* w, long long w_stride,
                      long long w_expert_stride, const float* w_scale, int N, int K, int E, const int32_t* expert_offsets, int swiglu,
                      int zero_tail, void* out, long long out_stride, int out_dtype) {
    if (M < 0 || N <= 0 || K < 0 || E <= 0 || out_dtype < VMOE_BF16 || out_dtype > VMOE_F32) return VMOE_ERR_SHAPE;
    if (a_stride < 0 || w_stride < 0 || w_expert_stride < 0 || out_stride < N || (!expert_offsets && E != 1)) return VMOE_ERR_SHAPE;
    if (K > I8_MAX_K || E > 65535 || N > (1 << 30) || M > 0x7fffffff - 1024) return VMOE_ERR_LIMIT;
    if (M == 0) return VMOE_OK;
    if (!w_scale || !out || (K > 0 && !w)) return VMOE_ERR_NULL;
    if ((uintptr_t)out & (out_dtype == VMOE_F32 ? 3 : 1)) return VMOE_ERR_ALIGN;
    p->a = a; p->a_stride = M == 1 ? i8_pitch(K) : a_stride; p->a_scale = a_scale;      // the stride of a single row says nothing
    p->wrows = swiglu ? 2 * N : N;
    p->w = w; p->w_stride = p->wrows == 1 ? i8_pitch(K) : w_stride; p->w_expert_stride = w_expert_stride; p->w_scale = w_scale;
    p->out = out; p->out_stride = out_stride; p->offsets = expert_offsets;
    p->M = M; p->N = N; p->K = K; p->E = E; p->swiglu = swiglu; p->out_dtype = out_dtype; p->zero_tail = zero_tail;
    return VMOE_OK;
}

// The kernel of a product, by its sizes and the alignment of its operands.  Dense, split against persistent, K = N = 4096:
// 48 rows (16 items of 128 tokens) 8.8 against 14.4 us, 256 rows (32) 14.7 against 14.6, 384 rows (48) 18.6 against 14.8.  Longer
// reductions gain more by the split (1024 channels of 8192, 48 rows: 8.4 against 23.8), shorter ones lose (2048 x 2048: 11.8 against
// 9.2; 8192 channels of 1024: 8.6 against 7.2), which the rule does not look at.
static int i8_product(const I8Problem& p, cudaStream_t st) {
    if (i8_gemv_ok(p)) return launch_i8_gemv(p, nullptr, 0, 0, st);
    if (!i8_tc_ok(p) || p.E > I8_TC_MAX_EXPERTS) return i8_gemv_fits(p) ? launch_i8_gemv(p, nullptr, 0, 0, st) : launch_i8_tile(p, st);
    if (!p.offsets) {
        const long long items = (p.M + 127LL) / 128 * ((p.N + (p.swiglu ? 127LL : 255LL)) / (p.swiglu ? 128 : 256));
        if (items < 48) return launch_i8_split(p, st);
    }
    return launch_i8_tc(p, st);
}

static size_t i8_pack_bytes(long long M, long long wrows, int K, int E) {
    return i8_align((size_t)M * i8_pitch(K)) + (size_t)E * wrows * i8_pitch(K);
}

// The product of operands of any alignment: with room for it, unaligned ones are packed first.  Measured, K = 1001, in place
// against packed: 12 rows x 2048 channels 37 against 13 us, 64 matrices of 1024 channels with 4 rows each 117 against 53 us,
// with 64 rows 183 against 56 us.  Packing reads every matrix and reading in place only those with rows, so below about one
// row per matrix a caller leaves the room out.
static int i8_product_any(I8Problem p, void* room, size_t bytes, cudaStream_t st) {
    if (room && p.M > 0 && p.K > 0 && p.E <= I8_TC_MAX_EXPERTS && !i8_gemv_ok(p) && !i8_tc_ok(p) &&
        bytes >= i8_pack_bytes(p.M, p.wrows, p.K, p.E) && !((uintptr_t)room & 15)) {
        I8Problem q = p;
        int8_t* a = static_cast<int8_t*>(room);
        int8_t* w = a + i8_align((size_t)p.M * i8_pitch(p.K));
        const bool pack_a = (((uintptr_t)p.a | (unsigned long long)p.a_stride) & 15) != 0 || p.a_stride < p.K;
        if (pack_a) { q.a = a; q.a_stride = i8_pitch(p.K); }
        const bool pack_w = !i8_tc_ok(q);
        if (pack_w) { q.w = w; q.w_stride = i8_pitch(p.K); q.w_expert_stride = (long long)p.wrows * i8_pitch(p.K); }
        const long long vecs = (long long)(i8_pitch(p.K) / 16) * ((pack_a ? p.M : 0) + (pack_w ? (long long)p.E * p.wrows : 0));
        if ((vecs + 255) / 256 > 0x7fffffffLL) return VMOE_ERR_LIMIT;
        const int rc = launch_status(launch_pdl(i8_pack_kernel, (unsigned)((vecs + 255) / 256), 256u, 0, st, p, (int)pack_a, a,
                                                pack_w ? w : (int8_t*)nullptr));
        if (rc) return rc;
        p = q;
    }
    return i8_product(p, st);
}

struct I8ExpertsScratch { size_t offsets, row_of_pair, pair_of_row, counts, counts_bytes, scale, q1, h, q2, y, room13, room2, room13_bytes, room2_bytes, total; };
// false: sizes the plan does not take.  The f32 rows of the second product (y) take the place of the first one's operands.
static bool i8_experts_scratch(int M, int T, int E, int K, int N, int pack, I8ExpertsScratch* s) {
    if (M < 0 || T <= 0 || T > MAX_TOPK || E <= 0 || E > 8192 || K <= 0 || N <= 0 || (long long)M * T > 0x7fffffffLL - 1024) return false;
    const size_t P = (size_t)M * T;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t here = at; at += i8_align(bytes); return here; };
    s->offsets = take(((size_t)E + 1) * 4);
    s->row_of_pair = take(P * 4);
    s->pair_of_row = take(P * 4);
    s->counts_bytes = vmoe_plan_scratch_bytes(M, T, E);
    s->counts = take(s->counts_bytes);
    s->scale = take(P * 4);
    s->q2 = take(P * i8_pitch(N));
    s->y = s->q1 = take(P * i8_pitch(K));
    s->h = take(P * N * 4);
    const size_t y_end = s->y + i8_align(P * K * 4);
    if (at < y_end) at = y_end;
    s->room13_bytes = pack ? i8_pack_bytes(P, 2LL * N, K, E) : 0;      // the rows are packed already; only the weights may be copied
    s->room2_bytes = pack ? i8_pack_bytes(P, K, N, E) : 0;
    s->room13 = s->room2 = take(s->room13_bytes > s->room2_bytes ? s->room13_bytes : s->room2_bytes);
    s->total = at;
    return true;
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
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        // Many rows: eight vectors a thread, so that the row's own work (its largest magnitude, its scale) is spread over
        // them.  Few rows: as many warps a row as find a vector for each lane.
        const bool many = rows >= 2048;
        if (vecs <= (many ? 256 : 32)) return launch_quantize_rows<typename R::T, R::BYTES, 1>(x, xs, rows, vecs, T, row_of_pair, live_rows, q, q_stride, scales, st);
        if (vecs <= (many ? 512 : 64)) return launch_quantize_rows<typename R::T, R::BYTES, 2>(x, xs, rows, vecs, T, row_of_pair, live_rows, q, q_stride, scales, st);
        if (vecs <= (many ? 1024 : 128)) return launch_quantize_rows<typename R::T, R::BYTES, 4>(x, xs, rows, vecs, T, row_of_pair, live_rows, q, q_stride, scales, st);
        return launch_quantize_rows<typename R::T, R::BYTES, 8>(x, xs, rows, vecs, T, row_of_pair, live_rows, q, q_stride, scales, st);
    });
}

size_t vmoe_int8_pack_bytes(int32_t M, int32_t weight_rows, int32_t K, int32_t E) {
    return M <= 0 || weight_rows <= 0 || K <= 0 || E <= 0 || K > I8_MAX_K ? 0 : i8_pack_bytes(M, weight_rows, K, E);
}

int vmoe_int8_matmul(const int8_t* a, int64_t a_stride, const float* a_scale, int32_t M, const int8_t* w, int64_t w_stride,
                     int64_t w_expert_stride, const float* w_scale, int32_t N, int32_t K, int32_t E, const int32_t* expert_offsets,
                     int32_t swiglu, int32_t zero_tail, void* out, int64_t out_stride, int32_t out_dtype, void* scratch,
                     size_t scratch_bytes, void* stream) {
    I8Problem p;
    const int rc = i8_problem(&p, a, a_stride, a_scale, M, w, w_stride, w_expert_stride, w_scale, N, K, E, expert_offsets, swiglu,
                              zero_tail, out, out_stride, out_dtype);
    if (rc || M == 0) return rc;
    if (!a_scale || (K > 0 && !a)) return VMOE_ERR_NULL;
    return i8_product_any(p, scratch, scratch_bytes, static_cast<cudaStream_t>(stream));
}

size_t vmoe_int8_linear_scratch_bytes(int32_t M, int32_t K) {
    if (M <= 0 || K < 0 || K > I8_MAX_K) return 0;
    return i8_align((size_t)M * i8_pitch(K)) + i8_align((size_t)M * sizeof(float));
}

int vmoe_int8_linear(const void* x, int64_t x_stride, int32_t dtype, int32_t M, const int8_t* w, int64_t w_stride, const float* w_scale,
                     int32_t N, int32_t K, int32_t swiglu, void* out, int64_t out_stride, int32_t out_dtype, void* scratch,
                     size_t scratch_bytes, void* stream) {
    if (dtype < VMOE_BF16 || dtype > VMOE_F32 || x_stride < 0) return VMOE_ERR_SHAPE;
    uint8_t* const base = static_cast<uint8_t*>(scratch);
    I8Problem p;
    const int pitch = i8_pitch(K > 0 && K <= I8_MAX_K ? K : 0);
    int rc = i8_problem(&p, nullptr, pitch, nullptr, M, w, w_stride, 0, w_scale, N, K, 1, nullptr, swiglu, 0, out, out_stride, out_dtype);
    if (rc || M == 0) return rc;
    if (K > 0 && !x) return VMOE_ERR_NULL;
    const long long el = dtype == VMOE_F32 ? 4 : 2;
    if ((uintptr_t)x & (el - 1)) return VMOE_ERR_ALIGN;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const size_t need = vmoe_int8_linear_scratch_bytes(M, K);
    const bool room = scratch && scratch_bytes >= need;
    if (i8_gemv_ok(p) || (!room && i8_gemv_fits(p))) return launch_i8_gemv(p, x, x_stride * el, dtype, st);
    if (!room) return VMOE_ERR_WORKSPACE;
    if ((uintptr_t)scratch & 15) return VMOE_ERR_ALIGN;
    int8_t* q = reinterpret_cast<int8_t*>(base);
    float* scale = reinterpret_cast<float*>(base + i8_align((size_t)M * pitch));
    if ((rc = vmoe_int8_quantize(x, x_stride, dtype, M, K, 0, nullptr, nullptr, q, pitch, scale, stream))) return rc;
    p.a = q; p.a_scale = scale;
    return i8_product_any(p, base + need, scratch_bytes - need, st);
}

size_t vmoe_int8_experts_scratch_bytes(int32_t M, int32_t T, int32_t E, int32_t K, int32_t N, int32_t pack) {
    I8ExpertsScratch s;
    return i8_experts_scratch(M, T, E, K, N, pack, &s) ? s.total : 0;
}

int vmoe_int8_experts(const void* x, int64_t x_stride, int32_t dtype, int32_t M, int32_t T, int32_t E, int32_t K, int32_t N,
                      const int32_t* topk_ids, const float* topk_weights, const int32_t* expert_map, int32_t map_len,
                      const int8_t* w13, int64_t w13_stride, int64_t w13_expert_stride, const float* w13_scale,
                      const int8_t* w2, int64_t w2_stride, int64_t w2_expert_stride, const float* w2_scale,
                      void* out, int64_t out_stride, int32_t out_dtype, void* scratch, size_t scratch_bytes, void* stream) {
    if (dtype < VMOE_BF16 || dtype > VMOE_F32 || x_stride < 0 || K <= 0 || N <= 0) return VMOE_ERR_SHAPE;
    if (M < 0 || T <= 0 || E <= 0) return VMOE_ERR_SHAPE;
    if (K > I8_MAX_K || N > I8_MAX_K) return VMOE_ERR_LIMIT;
    I8ExpertsScratch L;
    if (!i8_experts_scratch(M, T, E, K, N, 1, &L)) return VMOE_ERR_LIMIT;
    const bool pack = scratch_bytes >= L.total;
    if (!pack) i8_experts_scratch(M, T, E, K, N, 0, &L);
    if (M == 0) return VMOE_OK;
    if (!x || !topk_ids || !topk_weights || !w13 || !w2 || !w13_scale || !w2_scale || !out) return VMOE_ERR_NULL;
    if (!scratch || scratch_bytes < L.total) return VMOE_ERR_WORKSPACE;
    if ((uintptr_t)scratch & 15) return VMOE_ERR_ALIGN;
    uint8_t* const b = static_cast<uint8_t*>(scratch);
    int32_t* offsets = reinterpret_cast<int32_t*>(b + L.offsets);
    int32_t* row_of_pair = reinterpret_cast<int32_t*>(b + L.row_of_pair);
    float* scale = reinterpret_cast<float*>(b + L.scale);
    int8_t* q1 = reinterpret_cast<int8_t*>(b + L.q1);
    float* h = reinterpret_cast<float*>(b + L.h);
    int8_t* q2 = reinterpret_cast<int8_t*>(b + L.q2);
    float* y = reinterpret_cast<float*>(b + L.y);
    void* room = pack ? b + L.room13 : nullptr;
    const int P = M * T;
    int rc;
    if (expert_map && map_len < 0) return VMOE_ERR_SHAPE;
    if (P <= FRONT_PAIRS) {
        if ((rc = launch_i8_front(x, x_stride, dtype, M, T, K, topk_ids, expert_map, map_len, E, offsets, row_of_pair, q1, i8_pitch(K), scale,
                                  static_cast<cudaStream_t>(stream)))) return rc;
    } else {
        if ((rc = vmoe_plan_tokens(topk_ids, expert_map, map_len, M, T, E, offsets, row_of_pair, reinterpret_cast<int32_t*>(b + L.pair_of_row),
                                   b + L.counts, L.counts_bytes, stream))) return rc;
        if ((rc = vmoe_int8_quantize(x, x_stride, dtype, M, K, T, row_of_pair, nullptr, q1, i8_pitch(K), scale, stream))) return rc;
    }
    if ((rc = vmoe_int8_matmul(q1, i8_pitch(K), scale, P, w13, w13_stride, w13_expert_stride, w13_scale, N, K, E, offsets, 1, 0, h, N, VMOE_F32,
                               room, L.room13_bytes, stream))) return rc;
    if ((rc = vmoe_int8_quantize(h, N, VMOE_F32, P, N, 0, nullptr, offsets + E, q2, i8_pitch(N), scale, stream))) return rc;
    if ((rc = vmoe_int8_matmul(q2, i8_pitch(N), scale, P, w2, w2_stride, w2_expert_stride, w2_scale, K, N, E, offsets, 0, 0, y, K, VMOE_F32,
                               room, L.room2_bytes, stream))) return rc;
    return vmoe_unsort_tokens(y, K, VMOE_F32, M, T, K, row_of_pair, topk_weights, out, out_stride, out_dtype, stream);
}

}  // extern "C"
