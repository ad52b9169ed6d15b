// Token rows sorted by expert and back, for rows of bf16 / fp16 / f32, with the gradients of both directions.
//
//   plan    pairs p = m * T + t with a local expert, ordered by (expert, p):  offsets, row_of_pair, pair_of_row
//   sort    rows[r] = x[pair_of_row[r] / T]
//   unsort  y[m]    = sum_t w[m, t] * rows[row_of_pair[m, t]]          (w = 1: the gradient of sort)
//   grad    drows[row_of_pair[m, t]] = w[m, t] * dy[m],   dw[m, t] = <rows[row_of_pair[m, t]], dy[m]>
//
// Unlike the tables inside the layer's workspace (vmoe_phases.cuh: one bit per expert and token) a token may name an
// expert twice here; each pair has its own row.  All sums run over t in ascending order in f32 and are rounded once;
// nothing is summed with atomics, so every result is reproducible bit for bit.
//
// No pointer is __restrict__: these kernels may start while the kernel that writes their inputs still runs
// (pdl_begin), and loads through the non-coherent path are only defined for data that does not change meanwhile.
#include "vmoe_common.cuh"
#include "vmoe_rows.cuh"

namespace vmoe {

// ---------------------------------------------------------------------------------
// Plan: a stable counting sort.  Each warp owns a contiguous run of pairs.  Pass 1 counts them per expert into the warp's
// own row of counters; sums over warps, CTAs and experts turn the counters into the first row of (expert, warp); pass 2
// walks the run again, 32 pairs at a time: __match_any_sync gives a pair's rank among the lanes with its expert.
// Up to 4096 pairs one CTA does it all.  Above, every CTA needs the others' counts: a first launch leaves them in the
// caller's scratch [CTAs][E], the second reads them (a few times E words each) and places its own run.
// ---------------------------------------------------------------------------------
constexpr int PLAN_MAX_EXPERTS = 8192;
constexpr int PLAN_ONE_CTA_PAIRS = 4096;
constexpr int PLAN_PAIRS_PER_CTA = 1024;        // 4096: placing them takes 9500 cycles of a CTA's 19700
constexpr int PLAN_KEPT = 4;                 // experts of a lane's first pairs stay in registers between the passes
constexpr int PLAN_MAX_CTAS = 148;
constexpr int PLAN_SMEM = 200 * 1024;

static int plan_ctas(long long pairs) {
    if (pairs <= PLAN_ONE_CTA_PAIRS) return 1;
    const long long n = (pairs + PLAN_PAIRS_PER_CTA - 1) / PLAN_PAIRS_PER_CTA;
    return (int)(n < PLAN_MAX_CTAS ? n : PLAN_MAX_CTAS);
}

__device__ __forceinline__ int plan_expert(const int32_t* ids, const int32_t* expert_map, int map_len, int E, long long p, long long end) {
    if (p >= end) return -1;
    int e = ids[p];
    if (expert_map) e = (e >= 0 && e < map_len) ? expert_map[e] : -1;
    return (e >= 0 && e < E) ? e : -1;
}

__global__ void __launch_bounds__(1024)
plan_count_kernel(const int32_t* ids, const int32_t* expert_map, int map_len, int P, int E, int per_cta,
                  int32_t* counts) {
    extern __shared__ int s_plan[];
    for (int e = threadIdx.x; e < E; e += blockDim.x) s_plan[e] = 0;
    __syncthreads();
    pdl_begin();
    const long long first = (long long)blockIdx.x * per_cta, end = min(first + per_cta, (long long)P);
    for (long long p = first + threadIdx.x; p < end; p += blockDim.x) {
        const int e = plan_expert(ids, expert_map, map_len, E, p, end);
        if (e >= 0) atomicAdd(&s_plan[e], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += blockDim.x) counts[(size_t)blockIdx.x * E + e] = s_plan[e];
}

template <bool MANY>
__global__ void __launch_bounds__(1024)
plan_kernel(const int32_t* ids, const int32_t* expert_map, int map_len, int P, int E, int run,
            const int32_t* counts, int32_t* offsets, int32_t* row_of_pair, int32_t* pair_of_row) {
    extern __shared__ int s_plan[];
    __shared__ int s_warp[33];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x, warps = threads >> 5;
    int* count = s_plan;                      // [warps][E]
    int* start = count + (size_t)warps * E;   // [E] all CTAs' pairs, then the first row of this CTA's pairs
    int* before = start + E;                  // [E] pairs of the CTAs in front
    const int rank = (int)blockIdx.x, ctas = (int)gridDim.x;
    for (int i = tid; i < (warps + (MANY ? 2 : 0)) * E; i += threads) count[i] = 0;       // start and before lie behind count
    __syncthreads();
    pdl_begin();

    int* mine = count + (size_t)warp * E;
    const long long first = ((long long)rank * warps + warp) * run;
    const long long end = min(first + run, (long long)P);
    int kept_e[PLAN_KEPT];
#pragma unroll
    for (int i = 0; i < PLAN_KEPT; ++i) kept_e[i] = plan_expert(ids, expert_map, map_len, E, first + 32 * i + lane, end);
    if (MANY) {                               // the CTAs' counts, while the ids are on their way: `parts` threads per expert
        const int parts = threads >= 2 * E ? threads / E : 1;
        for (int i = tid; i < parts * E; i += threads) {
            const int e = i % E, part = i / E;
            int all = 0, front = 0;
            for (int r0 = part; r0 < ctas; r0 += 16 * parts) {           // sixteen loads in flight
                int n[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) n[k] = r0 + k * parts < ctas ? counts[(size_t)(r0 + k * parts) * E + e] : 0;
#pragma unroll
                for (int k = 0; k < 16; ++k) { all += n[k]; front += r0 + k * parts < rank ? n[k] : 0; }
            }
            atomicAdd(&start[e], all);
            atomicAdd(&before[e], front);
        }
    }
#pragma unroll
    for (int i = 0; i < PLAN_KEPT; ++i)
        if (kept_e[i] >= 0) atomicAdd(&mine[kept_e[i]], 1);
    for (long long b = first + 32 * PLAN_KEPT; b < end; b += 32) {
        const int e = plan_expert(ids, expert_map, map_len, E, b + lane, end);
        if (e >= 0) atomicAdd(&mine[e], 1);
    }
    __syncthreads();
    if (!MANY) {
        for (int e = tid; e < E; e += threads) {
            int all = 0;
#pragma unroll 8
            for (int w = 0; w < warps; ++w) all += count[(size_t)w * E + e];
            start[e] = all;
            before[e] = 0;
        }
        __syncthreads();
    }
    // exclusive prefix over the experts: every thread a contiguous run of them
    const int per = (E + threads - 1) / threads;
    int sum = 0;
    for (int k = 0; k < per; ++k) { const int e = tid * per + k; if (e < E) sum += start[e]; }
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= o) incl += v; }
    if (lane == 31) s_warp[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        const int v = lane < warps ? s_warp[lane] : 0;
        int in = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int u = __shfl_up_sync(0xffffffffu, in, o); if (lane >= o) in += u; }
        s_warp[lane] = in - v;
        if (lane == 31) s_warp[32] = in;
    }
    __syncthreads();
    int at = s_warp[warp] + incl - sum;
    for (int k = 0; k < per; ++k) {
        const int e = tid * per + k;
        if (e < E) {
            const int n = start[e];
            if (rank == 0) offsets[e] = at;
            start[e] = at + before[e];
            at += n;
        }
    }
    const int kept = s_warp[32];
    if (rank == 0 && tid == 0) offsets[E] = kept;
    __syncthreads();
    for (int e = tid; e < E; e += threads) {
        int row = start[e];
        for (int w0 = 0; w0 < warps; w0 += 8) {               // eight loads in flight
            int n[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) n[k] = w0 + k < warps ? count[(size_t)(w0 + k) * E + e] : 0;
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (w0 + k < warps) { count[(size_t)(w0 + k) * E + e] = row; row += n[k]; }
        }
    }
    __syncthreads();
    auto place = [&](long long p, int e) {               // one pair per lane, the whole warp
        const uint32_t same = __match_any_sync(0xffffffffu, e);
        const int rank_in = __popc(same & ((1u << lane) - 1));
        const int row = e >= 0 ? mine[e] + rank_in : -1;
        __syncwarp();
        if (e >= 0 && rank_in == 0) mine[e] += __popc(same);
        __syncwarp();
        if (p < end) {
            row_of_pair[p] = row;
            if (row >= 0) pair_of_row[row] = (int)p;
        }
    };
#pragma unroll
    for (int i = 0; i < PLAN_KEPT; ++i)
        if (first + 32 * i < end) place(first + 32 * i + lane, kept_e[i]);
    for (long long b = first + 32 * PLAN_KEPT; b < end; b += 32) place(b + lane, plan_expert(ids, expert_map, map_len, E, b + lane, end));
    for (long long r = (long long)kept + rank * threads + tid; r < P; r += (long long)ctas * threads) pair_of_row[r] = -1;
}

// A pair's row, or -1: dropped, or (in a table that vmoe_plan_tokens did not make) outside the rows there are.
__device__ __forceinline__ int pair_row(const int32_t* row_of_pair, long long pair, long long rows) {
    const int r = row_of_pair[pair];
    return r < rows ? r : -1;
}

// i = m * vecs + c
__device__ __forceinline__ void row_and_vector(long long i, long long vecs, long long& m, long long& c) {
    if (i <= 0xffffffffLL && vecs <= 0xffffffffLL) {
        const uint32_t q = (uint32_t)i / (uint32_t)vecs;
        m = q;
        c = (uint32_t)i - q * (uint32_t)vecs;
    } else {
        m = i / vecs;
        c = i - m * vecs;
    }
}

// Rows from `first` on become zero: a warp per row, all warps of the grid in turn.
template <typename V>
__device__ __forceinline__ void zero_rows(uint8_t* rows, long long stride, long long first, long long end, long long vecs) {
    const long long warps = (long long)gridDim.x * (blockDim.x >> 5);
    for (long long r = max(first, 0LL) + (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); r < end; r += warps) {
        V* row = reinterpret_cast<V*>(rows + r * stride);
        for (long long c = threadIdx.x & 31; c < vecs; c += 32) row[c] = V{};
    }
}

// Which vectors of which token a thread owns.  U = 1: vector i of all tokens' vectors in a row.  U > 1 (rows that only allow
// narrow vectors): a warp owns 32 U neighbours of one token, a lane every 32nd of them, so that a thread has as many bytes in
// flight as with one wide vector.
template <int U>
struct Share {
    long long m, c;
    bool on;
    __device__ __forceinline__ Share(long long vecs, int M) {
        const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
        if (U == 1) {
            on = i < (long long)M * vecs;
            if (on) row_and_vector(i, vecs, m, c);
        } else {
            const long long tiles = (vecs + 32 * U - 1) / (32 * U);
            on = (i >> 5) < M * tiles;
            if (on) {
                row_and_vector(i >> 5, tiles, m, c);
                c = c * 32 * U + (i & 31);
            }
        }
    }
    __device__ __forceinline__ bool has(int u, long long vecs) const { return U == 1 || c + 32 * u < vecs; }
};
static unsigned share_blocks(long long vecs, int M, int U) {
    const long long threads = U == 1 ? M * vecs : 32LL * M * ((vecs + 32 * U - 1) / (32 * U));
    return (unsigned)((threads + 255) / 256);
}
// Narrow vectors: as many as make 16 bytes, where a row has enough of them.
static constexpr int share_of(int vector_bytes, long long vecs) { return vector_bytes < 16 && vecs >= 64 ? 16 / vector_bytes : 1; }

// ---------------------------------------------------------------------------------
// Sort: a thread reads its vectors of one token and stores them to the token's T rows, so a token is read once and the
// rest of the traffic is the rows' own writes.  Rows nobody owns (dropped pairs leave them behind the last kept row)
// are zeroed when the caller wants every row defined.  Bound by the writes: 8192 x 10 rows of 4096 bf16 6.1 TB/s (0.93 of a
// copy's); rows of 1021 f32 (4-byte vectors) 3.6 TB/s with one vector a thread, 6.6 (part of it L2) with four.
// ---------------------------------------------------------------------------------
constexpr int SORT_BATCH = 4;

template <typename V, int U>
__global__ void __launch_bounds__(256)
sort_kernel(const uint8_t* x, long long x_stride, uint8_t* rows, long long rows_stride, long long vecs,
            int M, int T, const int32_t* row_of_pair, const int32_t* kept, int zero_tail) {
    pdl_begin();
    if (zero_tail) zero_rows<V>(rows, rows_stride, *kept, (long long)M * T, vecs);
    const Share<U> s(vecs, M);
    if (!s.on) return;
    V v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (s.has(u, vecs)) v[u] = reinterpret_cast<const V*>(x + s.m * x_stride)[s.c + 32 * u];
    const long long pairs = (long long)M * T;
    for (int t0 = 0; t0 < T; t0 += SORT_BATCH) {
        int r[SORT_BATCH];
#pragma unroll
        for (int j = 0; j < SORT_BATCH; ++j) r[j] = t0 + j < T ? pair_row(row_of_pair, s.m * T + t0 + j, pairs) : -1;
#pragma unroll
        for (int j = 0; j < SORT_BATCH; ++j)
            if (r[j] >= 0) {
                V* dst = reinterpret_cast<V*>(rows + r[j] * rows_stride) + s.c;
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (s.has(u, vecs)) dst[32 * u] = v[u];
            }
    }
}

// ---------------------------------------------------------------------------------
// Unsort: a thread sums its vectors of one token over the token's pairs in order; BATCH rows are requested at a time.
// Bound by reading the rows.  BATCH divides T as evenly as up to five rows allow: with 4 for every T, 10 choices of 4096
// bf16 reach 5.6 TB/s and 8 choices 6.0; with 5, 6.0 and 5.6.  Rows in f32 may leave as bf16 / fp16: the expert layer's
// rows stay in f32 until they are summed.
// ---------------------------------------------------------------------------------
template <typename T_, int VB, typename O_, int BATCH, int U>
__global__ void __launch_bounds__(256)
unsort_kernel(const uint8_t* rows, long long rows_stride, uint8_t* out, long long out_stride, long long vecs,
              int M, int T, const int32_t* row_of_pair, const float* weights) {
    using R = RowVec<T_, VB>;
    pdl_begin();
    const Share<U> s(vecs, M);
    if (!s.on) return;
    float acc[U][R::N];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < R::N; ++k) acc[u][k] = 0.f;
    const long long pairs = (long long)M * T;
    for (int t0 = 0; t0 < T; t0 += BATCH) {
        R v[BATCH][U];
        int r[BATCH];
        float w[BATCH];
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
            r[j] = t0 + j < T ? pair_row(row_of_pair, s.m * T + t0 + j, pairs) : -1;
            w[j] = r[j] >= 0 && weights ? weights[s.m * T + t0 + j] : 1.f;
            if (r[j] >= 0) {
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (s.has(u, vecs)) v[j][u].load(rows + r[j] * rows_stride, s.c + 32 * u);
            }
        }
#pragma unroll
        for (int j = 0; j < BATCH; ++j)
            if (r[j] >= 0) {
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int k = 0; k < R::N; ++k) acc[u][k] = fmaf(w[j], v[j][u].get(k), acc[u][k]);
            }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (s.has(u, vecs)) {
            RowVec<O_, R::N * (int)sizeof(O_)> o;
#pragma unroll
            for (int k = 0; k < R::N; ++k) o.set(k, acc[u][k]);
            o.store(out + s.m * out_stride, s.c + 32 * u);
        }
}

// ---------------------------------------------------------------------------------
// Gradient of unsort: WPT warps per token, eight warps per CTA.  Four pairs at a time: their rows are read for the
// dot products with dy[m] and their gradients written in the same pass.  Order of a dot product: a thread's vectors
// in ascending order, the warp's xor tree, the warps in order.
// ---------------------------------------------------------------------------------
constexpr int UNSORT_BATCH = 4;

template <typename T_, int VB, int WPT>
__global__ void __launch_bounds__(256)
unsort_grad_kernel(const uint8_t* dy, long long dy_stride, const uint8_t* rows, long long rows_stride,
                   uint8_t* drows, long long drows_stride, float* dw, int vecs, int M, int T,
                   const int32_t* row_of_pair, const float* weights, const int32_t* kept) {
    using R = RowVec<T_, VB>;
    __shared__ float s_dot[8][MAX_TOPK];
    pdl_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long m = (long long)blockIdx.x * (8 / WPT) + warp / WPT;
    const int part = (warp % WPT) * 32 + lane;
    if (m < M) {
        const long long pairs = (long long)M * T;
        for (int t0 = 0; t0 < T; t0 += UNSORT_BATCH) {
            int r[UNSORT_BATCH];
            float w[UNSORT_BATCH], dot[UNSORT_BATCH];
#pragma unroll
            for (int j = 0; j < UNSORT_BATCH; ++j) {
                r[j] = t0 + j < T ? pair_row(row_of_pair, m * T + t0 + j, pairs) : -1;
                w[j] = r[j] >= 0 && weights ? weights[m * T + t0 + j] : 1.f;
                dot[j] = 0.f;
            }
            constexpr int U = VB < 16 ? 8 / VB < 2 ? 2 : 8 / VB : 1;         // narrow vectors: several in flight
            for (int c0 = part; c0 < vecs; c0 += WPT * 32 * U) {
                R g[U], v[UNSORT_BATCH][U];
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (c0 + WPT * 32 * u < vecs) g[u].load(dy + m * dy_stride, c0 + WPT * 32 * u);
                if (dw) {
#pragma unroll
                    for (int j = 0; j < UNSORT_BATCH; ++j)
#pragma unroll
                        for (int u = 0; u < U; ++u)
                            if (r[j] >= 0 && c0 + WPT * 32 * u < vecs) v[j][u].load(rows + r[j] * rows_stride, c0 + WPT * 32 * u);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int c = c0 + WPT * 32 * u;
                    if (c >= vecs) break;
#pragma unroll
                    for (int j = 0; j < UNSORT_BATCH; ++j)
                        if (r[j] >= 0) {
                            if (dw) {
#pragma unroll
                                for (int k = 0; k < R::N; ++k) dot[j] = fmaf(v[j][u].get(k), g[u].get(k), dot[j]);
                            }
                            if (drows) {
                                R o;
#pragma unroll
                                for (int k = 0; k < R::N; ++k) o.set(k, w[j] * g[u].get(k));
                                o.store(drows + r[j] * drows_stride, c);
                            }
                        }
                }
            }
            if (dw) {
#pragma unroll
                for (int j = 0; j < UNSORT_BATCH; ++j) {
                    float d = dot[j];
#pragma unroll
                    for (int o = 16; o; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
                    if (lane == 0 && t0 + j < T) s_dot[warp][t0 + j] = d;
                }
            }
        }
    }
    if (dw) {
        __syncthreads();
        const int tok = threadIdx.x / MAX_TOPK, t = threadIdx.x % MAX_TOPK;
        const long long mm = (long long)blockIdx.x * (8 / WPT) + tok;
        if (tok < 8 / WPT && mm < M && t < T) {
            float d = 0.f;
#pragma unroll
            for (int w = 0; w < WPT; ++w) d += s_dot[tok * WPT + w][t];
            dw[mm * T + t] = d;
        }
    }
    if (drows) zero_rows<typename R::Raw>(drows, drows_stride, *kept, (long long)M * T, vecs);      // rows nobody owns
}

static int launch_plan(const int32_t* ids, const int32_t* expert_map, int map_len, int M, int T, int E, int32_t* offsets,
                       int32_t* row_of_pair, int32_t* pair_of_row, int32_t* scratch, cudaStream_t st) {
    const int P = M * T, ctas = plan_ctas(P);
    int warps = (PLAN_SMEM / 4 - 2 * E) / E;
    const int need = (int)(((long long)P + 32 * ctas - 1) / (32 * ctas));
    if (warps > 32) warps = 32;
    if (warps > need) warps = need > 0 ? need : 1;
    int run = (int)(((long long)P + (long long)ctas * warps - 1) / ((long long)ctas * warps));
    run = (run + 31) / 32 * 32;
    const size_t smem = (size_t)4 * E * (warps + 2);
    if (ctas == 1) {
        static SmemAllowed one;
        if (allow_smem(plan_kernel<false>, PLAN_SMEM, one) != cudaSuccess) return VMOE_ERR_CUDA;
        return launch_status(launch_pdl(plan_kernel<false>, 1u, (unsigned)warps * 32, smem, st, ids, expert_map, map_len, P, E, run,
                                      (const int32_t*)nullptr, offsets, row_of_pair, pair_of_row));
    }
    static SmemAllowed many;
    if (allow_smem(plan_kernel<true>, PLAN_SMEM, many) != cudaSuccess) return VMOE_ERR_CUDA;
    const cudaError_t e = launch_pdl(plan_count_kernel, (unsigned)ctas, 1024u, (size_t)4 * E, st, ids, expert_map, map_len, P, E, run * warps, scratch);
    if (e != cudaSuccess) return launch_status(e);
    return launch_status(launch_pdl(plan_kernel<true>, (unsigned)ctas, (unsigned)warps * 32, smem, st, ids, expert_map, map_len, P, E, run,
                                  (const int32_t*)scratch, offsets, row_of_pair, pair_of_row));
}

template <typename T_, int VB, typename O_>
static int launch_unsort(const uint8_t* rows, long long rs, uint8_t* out, long long os, long long vecs, int M, int T, const int32_t* rp,
                         const float* w, cudaStream_t st) {
    auto go = [&](auto kernel, int U) { return launch_status(launch_pdl(kernel, share_blocks(vecs, M, U), 256u, 0, st, rows, rs, out, os, vecs, M, T, rp, w)); };
    if constexpr (VB == 16) {
        const int batches = (T + 4) / 5;
        switch ((T + batches - 1) / batches) {
            case 1: return go(unsort_kernel<T_, VB, O_, 1, 1>, 1);
            case 2: return go(unsort_kernel<T_, VB, O_, 2, 1>, 1);
            case 3: return go(unsort_kernel<T_, VB, O_, 3, 1>, 1);
            case 4: return go(unsort_kernel<T_, VB, O_, 4, 1>, 1);
            default: return go(unsort_kernel<T_, VB, O_, 5, 1>, 1);
        }
    } else {
        constexpr int U = share_of(VB, 1 << 20);
        if (share_of(VB, vecs) > 1) return go(unsort_kernel<T_, VB, O_, 4, U>, U);
        return go(unsort_kernel<T_, VB, O_, 4, 1>, 1);
    }
}

template <typename V>
static int launch_sort(const uint8_t* x, long long xs, uint8_t* rows, long long rs, long long vecs, int M, int T, const int32_t* rp,
                       const int32_t* kept, int zero_tail, cudaStream_t st) {
    constexpr int U = share_of(sizeof(V), 1 << 20);
    auto go = [&](auto kernel, int u) { return launch_status(launch_pdl(kernel, share_blocks(vecs, M, u), 256u, 0, st, x, xs, rows, rs, vecs, M, T, rp, kept, zero_tail)); };
    if (share_of(sizeof(V), vecs) > 1) return go(sort_kernel<V, U>, U);
    return go(sort_kernel<V, 1>, 1);
}

template <typename T_, int VB>
static int launch_grad(const void* dy, long long dys, const void* rows, long long rs, void* drows, long long drs, float* dw, int K,
                       int M, int T, const int32_t* rp, const float* w, const int32_t* kept, cudaStream_t st) {
    const int vecs = (int)((long long)K * sizeof(T_) / VB);
    const auto a = static_cast<const uint8_t*>(dy), b = static_cast<const uint8_t*>(rows);
    const auto o = static_cast<uint8_t*>(drows);
    if (vecs <= 64)
        return launch_status(launch_pdl(unsort_grad_kernel<T_, VB, 1>, (unsigned)((M + 7) / 8), 256u, 0, st, a, dys, b, rs, o, drs, dw, vecs, M, T, rp, w, kept));
    if (vecs <= 256)
        return launch_status(launch_pdl(unsort_grad_kernel<T_, VB, 4>, (unsigned)((M + 1) / 2), 256u, 0, st, a, dys, b, rs, o, drs, dw, vecs, M, T, rp, w, kept));
    return launch_status(launch_pdl(unsort_grad_kernel<T_, VB, 8>, (unsigned)M, 256u, 0, st, a, dys, b, rs, o, drs, dw, vecs, M, T, rp, w, kept));
}

static int check_rows(int32_t M, int32_t T, int32_t E, int32_t K, int32_t dtype) {
    if (M < 0 || T <= 0 || K < 0 || E <= 0 || dtype < VMOE_BF16 || dtype > VMOE_F32) return VMOE_ERR_SHAPE;
    if (T > MAX_TOPK || E > PLAN_MAX_EXPERTS || (long long)M * T > 0x7fffffffLL - 1024) return VMOE_ERR_LIMIT;
    // one thread per vector (at least one element), 256 threads per block
    if ((long long)M * K / 256 >= 0x7fffffffLL) return VMOE_ERR_LIMIT;
    return VMOE_OK;
}

}  // namespace vmoe

using namespace vmoe;

extern "C" {

size_t vmoe_plan_scratch_bytes(int32_t M, int32_t T, int32_t E) {
    if (check_rows(M, T, E, 0, VMOE_BF16) != VMOE_OK) return 0;
    const int ctas = plan_ctas((long long)M * T);
    return ctas > 1 ? (size_t)ctas * E * sizeof(int32_t) : 0;
}

int vmoe_plan_tokens(const int32_t* topk_ids, const int32_t* expert_map, int32_t map_len, int32_t M, int32_t T, int32_t E,
                     int32_t* expert_offsets, int32_t* row_of_pair, int32_t* pair_of_row, void* scratch, size_t scratch_bytes,
                     void* stream) {
    const int rc = check_rows(M, T, E, 0, VMOE_BF16);
    if (rc) return rc;
    if (!expert_offsets || (M > 0 && (!topk_ids || !row_of_pair || !pair_of_row))) return VMOE_ERR_NULL;
    if (expert_map && map_len < 0) return VMOE_ERR_SHAPE;
    const size_t need = vmoe_plan_scratch_bytes(M, T, E);
    if (need && (!scratch || scratch_bytes < need)) return VMOE_ERR_WORKSPACE;
    return launch_plan(topk_ids, expert_map, map_len, M, T, E, expert_offsets, row_of_pair, pair_of_row, static_cast<int32_t*>(scratch),
                       static_cast<cudaStream_t>(stream));
}

int vmoe_sort_tokens(const void* x, int64_t x_stride, int32_t dtype, int32_t M, int32_t T, int32_t E, int32_t K,
                     const int32_t* expert_offsets, const int32_t* row_of_pair, int32_t zero_tail, void* rows, int64_t rows_stride,
                     void* stream) {
    const int rc = check_rows(M, T, E, K, dtype);
    if (rc) return rc;
    if (M == 0 || K == 0) return VMOE_OK;
    if (!x || !expert_offsets || !row_of_pair || !rows) return VMOE_ERR_NULL;
    if (rows_stride < K || x_stride < 0) return VMOE_ERR_SHAPE;
    const long long el = dtype == VMOE_F32 ? 4 : 2, xs = x_stride * el, rs = rows_stride * el;
    if (((uintptr_t)x | (uintptr_t)rows) & (el - 1)) return VMOE_ERR_ALIGN;
    const int vb = vector_bytes((uintptr_t)x | (uintptr_t)rows, xs | rs | K * el);
    const long long vecs = K * el / vb;
    const auto a = static_cast<const uint8_t*>(x);
    const auto o = static_cast<uint8_t*>(rows);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int32_t* kept = expert_offsets + E;
    if (vb == 16) return launch_sort<uint4>(a, xs, o, rs, vecs, M, T, row_of_pair, kept, zero_tail, st);
    if (vb == 8) return launch_sort<uint2>(a, xs, o, rs, vecs, M, T, row_of_pair, kept, zero_tail, st);
    if (vb == 4) return launch_sort<uint32_t>(a, xs, o, rs, vecs, M, T, row_of_pair, kept, zero_tail, st);
    return launch_sort<uint16_t>(a, xs, o, rs, vecs, M, T, row_of_pair, kept, zero_tail, st);
}

int vmoe_unsort_tokens(const void* rows, int64_t rows_stride, int32_t dtype, int32_t M, int32_t T, int32_t K,
                       const int32_t* row_of_pair, const float* weights, void* out, int64_t out_stride, int32_t out_dtype,
                       void* stream) {
    const int rc = check_rows(M, T, 1, K, dtype);
    if (rc) return rc;
    if (out_dtype != dtype && (dtype != VMOE_F32 || out_dtype < VMOE_BF16 || out_dtype > VMOE_F32)) return VMOE_ERR_SHAPE;
    if (M == 0 || K == 0) return VMOE_OK;
    if (!rows || !row_of_pair || !out) return VMOE_ERR_NULL;
    if (out_stride < K || rows_stride < 0) return VMOE_ERR_SHAPE;
    const long long el = dtype == VMOE_F32 ? 4 : 2, ol = out_dtype == VMOE_F32 ? 4 : 2, rs = rows_stride * el, os = out_stride * ol;
    if (((uintptr_t)rows & (el - 1)) || ((uintptr_t)out & (ol - 1))) return VMOE_ERR_ALIGN;
    // a vector of n row elements becomes n output elements: both sides have to allow it
    int vb = vector_bytes((uintptr_t)rows, rs | K * el);
    const int ob = vector_bytes((uintptr_t)out, os) / (int)ol * (int)el;
    if (vb > ob) vb = ob;
    const auto a = static_cast<const uint8_t*>(rows);
    const auto o = static_cast<uint8_t*>(out);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return with_rows(dtype, vb, [&](auto r) {
        using R = decltype(r);
        using T_ = typename R::T;
        const long long vecs = (long long)K / R::N;
        if constexpr (sizeof(T_) == 4) {
            if (out_dtype == VMOE_BF16) return launch_unsort<T_, R::BYTES, __nv_bfloat16>(a, rs, o, os, vecs, M, T, row_of_pair, weights, st);
            if (out_dtype == VMOE_F16) return launch_unsort<T_, R::BYTES, __half>(a, rs, o, os, vecs, M, T, row_of_pair, weights, st);
        }
        return launch_unsort<T_, R::BYTES, T_>(a, rs, o, os, vecs, M, T, row_of_pair, weights, st);
    });
}

int vmoe_unsort_tokens_grad(const void* dout, int64_t dout_stride, const void* rows, int64_t rows_stride, int32_t dtype, int32_t M,
                            int32_t T, int32_t E, int32_t K, const int32_t* expert_offsets, const int32_t* row_of_pair,
                            const float* weights, void* drows, int64_t drows_stride, float* dweights, void* stream) {
    const int rc = check_rows(M, T, E, K, dtype);
    if (rc) return rc;
    if (M == 0 || (!drows && !dweights)) return VMOE_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (K > 0 && (!dout || !expert_offsets || !row_of_pair || (dweights && !rows))) return VMOE_ERR_NULL;
    if (dout_stride < 0 || (dweights && rows_stride < 0) || (drows && drows_stride < K)) return VMOE_ERR_SHAPE;
    if (K == 0)
        return dweights ? launch_status(cudaMemsetAsync(dweights, 0, (size_t)M * T * sizeof(float), st)) : VMOE_OK;
    const long long el = dtype == VMOE_F32 ? 4 : 2, ds = dout_stride * el;
    const long long rs = dweights ? rows_stride * el : 0, gs = drows ? drows_stride * el : 0;
    const uintptr_t ptrs = (uintptr_t)dout | (dweights ? (uintptr_t)rows : 0) | (uintptr_t)drows;
    if (ptrs & (el - 1)) return VMOE_ERR_ALIGN;
    const int vb = vector_bytes(ptrs, ds | rs | gs | K * el);
    return with_rows(dtype, vb, [&](auto r) {
        using R = decltype(r);
        return launch_grad<typename R::T, R::BYTES>(dout, ds, rows, rs, drows, gs, dweights, K, M, T, row_of_pair, weights,
                                                    expert_offsets + E, st);
    });
}

}  // extern "C"
