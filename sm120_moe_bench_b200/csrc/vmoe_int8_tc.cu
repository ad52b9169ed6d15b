// The 8-bit integer product on the tensor cores (tcgen05.mma kind::i8, s8 x s8 -> s32, accumulators in tensor memory).
//
// In both kernels the MMA's rows (operand A) are output channels and its columns (operand B) are tokens, so the number of
// tokens of an item is free in steps of 16 or 32: an expert with 5 rows costs 16 columns, one with 320 costs 2 x 160, and a
// decode batch streams every weight once.  A thread of the epilogue owns a channel; 32 lanes store 32 neighbours of a row.
//
//   i8_tc_kernel      persistent, grouped or large: 256 weight rows x up to 256 tokens per item
//   i8_split_kernel   dense products too small to fill the GPU that way: 128 channels x up to 128 tokens per CTA, the
//                     reduction split over a cluster, partial sums met in distributed shared memory (exact: integers)
#include "vmoe_int8.cuh"
#include "vmoe_tc_common.cuh"

#include <atomic>
#include <string.h>

namespace vmoe {

// A wait that ran out leaves its status here (read and cleared by vmoe_int8_read_status).
__device__ int g_i8_status;
// Limit of a wait in microseconds; 0: the producers hold their first copies back until a wait has run out
// (vmoe_int8_set_wait_limit).
static std::atomic<int> g_i8_wait_us{(int)(MBAR_WAIT_LIMIT_NS / 1000)};

// When a wait runs out: the role that gave up sets the CTA's flag and the status word and ends its loop; the others follow by
// their own limits.  Behind the barrier that ends the roles, a CTA with its flag set waits, with mbar_wait's limit, for the
// copies and MMAs that nobody waited for (i8_unwind): nothing of it is under way when it leaves.
__device__ __forceinline__ bool i8_wait(uint64_t* bar, uint32_t parity, unsigned long long limit_ns) {
    if (mbar_try_wait(bar, parity)) return true;
    const unsigned long long t0 = global_timer_ns();
    for (uint32_t i = 1;; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 63u) == 0 && global_timer_ns() - t0 > limit_ns) return false;
    }
}
// No copy for now, for tests: until the CTA's flag is set, or mbar_wait's limit has passed.
static __device__ __noinline__ void i8_hold(const int* abort_flag) {
    const unsigned long long t0 = global_timer_ns();
    while (*reinterpret_cast<const volatile int*>(abort_flag) == 0 && global_timer_ns() - t0 < MBAR_WAIT_LIMIT_NS) {}
    __syncwarp();
}

__device__ __forceinline__ void i8_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t i8_cluster_addr(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void i8_load_3d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void i8_mma(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n"
                 ::"r"(d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ uint32_t i8_idesc(int m, int n) {
    // accumulator s32 (2), operands signed 8-bit (1), both K-major
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

constexpr int I8_KB = 128;                                // bytes of K per stage: one swizzled row
constexpr int I8_A_BYTES = 128 * I8_KB;                   // 128 channels
constexpr int I8_BOX_BIG = 64, I8_BOX_SMALL = 16;         // token rows per copy

// ----------------------------------------------------------------------------------------------------- persistent
// An item is 256 weight rows (two MMA row tiles: 256 channels, or 128 gate rows and the 128 matching up rows, so that a lane
// of the epilogue has both) times at most P.tokens tokens of one expert.  A stage of U tokens is 32 KB + U * 128 bytes
// for 8 MMAs of U columns: at 64 bytes per clock an SM ingests it in 512 + 2 U cycles, the tensor pipe needs 4 U -- the
// two meet at 256 tokens.  Items of up to 128 tokens leave room in tensor memory for two accumulator sets, so that the
// epilogue of one runs under the MMAs of the next; above there is one set.
constexpr int I8P_MAX_STAGES = 8;
constexpr int I8P_EPI_WARPS = 16;
constexpr int I8P_THREADS = 64 + 32 * I8P_EPI_WARPS;
constexpr int I8P_ROWS = 256;                             // weight rows per item
constexpr int I8P_TOKENS = 256;                           // tokens per item at most (UMMA N)

struct I8Shared {
    uint64_t full[I8P_MAX_STAGES], empty[I8P_MAX_STAGES];
    uint64_t tmem_full[2], tmem_empty[2], done;           // done: every MMA has completed
    uint32_t tmem_base;
    int abort_flag;
    int blocks;                                           // token blocks of all experts
    int pad;
    alignas(16) float row_scale[I8P_EPI_WARPS][I8P_TOKENS / 2];       // of the item in hand, each epilogue warp its own tokens
};

struct I8TcParams {
    CUtensorMap map_w;                                    // [E, weight rows, K]
    CUtensorMap map_a64, map_a16;                         // token rows [M, K] in boxes of 64 and 16 (split: of the tile's tokens)
    I8Problem p;
    unsigned long long wait_ns;                           // limit of a wait
    int kblocks, ctiles, stages, tokens;                  // tokens: most of an item
    int hold;                                             // the first copies come when a wait has run out
};

struct I8Item { int expert, ctile, row0, rows, n; };
__device__ __forceinline__ int i8_blocks(int count, int most) { return (max(count, 0) + most - 1) / most; }
__device__ __forceinline__ I8Item i8_item(const I8TcParams& P, const int* s_pref, const int* s_off, long long item) {
    I8Item r;
    const int block = (int)(item / P.ctiles);
    r.ctile = (int)(item - (long long)block * P.ctiles);
    int lo = 0, hi = P.p.E;                               // s_pref[lo] <= block < s_pref[lo + 1]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_pref[mid] <= block) lo = mid; else hi = mid;
    }
    r.expert = lo;
    const int count = s_off[lo + 1] - s_off[lo], nb = s_pref[lo + 1] - s_pref[lo], j = block - s_pref[lo];
    r.n = min(((count + nb - 1) / nb + 15) & ~15, P.tokens);      // the expert's rows in equal blocks
    if (r.n > 16) r.n = (r.n + 31) & ~31;
    r.row0 = s_off[lo] + j * r.n;
    r.rows = min(r.n, max(s_off[lo + 1] - r.row0, 0));
    return r;
}

__device__ __forceinline__ void i8_abort(int* flag) {
    atomicExch(&g_i8_status, VMOE_ERR_TIMEOUT);
    atomicExch(flag, 1);
}
// issued: the producer's stages; committed: `done` stands for all MMAs already.  The whole CTA calls it.
static __device__ __noinline__ void i8_unwind(uint64_t* full, uint32_t issued, int stages, uint64_t* done, bool committed, bool leader) {
    const int warp = threadIdx.x >> 5;
    if (warp == 0) {
        for (uint32_t g = issued > (uint32_t)stages ? issued - stages : 0; g < issued; ++g) mbar_wait(&full[g % stages], (g / stages) & 1);
    } else if (warp == 1) {
        if (leader && !committed) tc_commit(done);
        __syncwarp();
        mbar_wait(done, 0);
    }
    __syncwarp();
    __syncthreads();
}

template <typename O_> __device__ __forceinline__ void i8_put(O_* at, float v);
template <> __device__ __forceinline__ void i8_put<float>(float* at, float v) { *at = v; }
template <> __device__ __forceinline__ void i8_put<__nv_bfloat16>(__nv_bfloat16* at, float v) { *at = __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ void i8_put<__half>(__half* at, float v) { *at = __float2half_rn(v); }

template <bool SWIGLU, typename O_>
__global__ void __launch_bounds__(I8P_THREADS, 1)
i8_tc_kernel(const __grid_constant__ I8TcParams P) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int stage_bytes = 2 * I8_A_BYTES + P.tokens * I8_KB;
    I8Shared* sh = reinterpret_cast<I8Shared*>(smem + (size_t)P.stages * stage_bytes);
    int* s_pref = reinterpret_cast<int*>(sh + 1);         // [E + 1] token blocks of the experts in front
    int* s_off = s_pref + P.p.E + 1;                      // [E + 1] first row of each expert
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const I8Problem& p = P.p;
    const int stages = P.stages;
    const bool two = P.tokens <= I8P_TOKENS / 2;          // two accumulator sets
    const uint32_t second = two ? I8P_TOKENS / 2 : I8P_TOKENS;    // column of the second row tile's accumulator

    if (tid == 0) {
        for (int i = 0; i < stages; ++i) { mbar_init(&sh->full[i], 1); mbar_init(&sh->empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&sh->tmem_full[i], 1); mbar_init(&sh->tmem_empty[i], I8P_EPI_WARPS); }
        mbar_init(&sh->done, 1);
        sh->abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh->tmem_base)), "r"(TC_TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh->tmem_base;
    pdl_begin();

    const int E = p.E;
    for (int e = tid; e <= E; e += I8P_THREADS) s_off[e] = p.offsets ? min(max(p.offsets[e], 0), p.M) : (e ? p.M : 0);
    __syncthreads();
    if (warp == 0) {                  // exclusive prefix of the experts' token blocks
        const int per = (E + 31) / 32;
        int sum = 0;
        for (int k = 0; k < per; ++k) { const int e = lane * per + k; if (e < E) sum += i8_blocks(s_off[e + 1] - s_off[e], P.tokens); }
        int incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int t = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= o) incl += t; }
        int run = incl - sum;
        for (int k = 0; k < per; ++k) {
            const int e = lane * per + k;
            if (e < E) { s_pref[e] = run; run += i8_blocks(s_off[e + 1] - s_off[e], P.tokens); }
        }
        if (lane == 31) { s_pref[E] = incl; sh->blocks = incl; }
    }
    __syncthreads();
    const long long total = (long long)sh->blocks * P.ctiles;
    const int kblocks = P.kblocks;
    uint32_t g = 0;                                       // stages of the producer, of the MMA warp
    bool leader = false;

    if (warp == 0) {
        // ------------------------------------------------------------- producer: the item's weight rows and token rows
        leader = elect_one();
        bool ok = true;
        int gone = 0;                                     // the flag, as of the last stage
        if (P.hold && blockIdx.x < total) i8_hold(&sh->abort_flag);
        for (long long item = blockIdx.x; item < total && ok; item += gridDim.x) {
            const I8Item u = i8_item(P, s_pref, s_off, item);
            const int ch = u.ctile * (SWIGLU ? 128 : I8P_ROWS);
            for (int kb = 0; kb < kblocks; ++kb) {
                const int slot = g % stages;
                bool w = true;
                if (g >= (uint32_t)stages) w = i8_wait(&sh->empty[slot], ((g / stages) - 1) & 1, P.wait_ns);
                if (!__all_sync(0xffffffffu, w && !gone)) { ok = false; break; }
                uint8_t* st = smem + (size_t)slot * stage_bytes;
                uint64_t* bar = &sh->full[slot];
                if (leader) {
                    mbar_arrive_expect_tx(bar, 2 * I8_A_BYTES + u.n * I8_KB);
                    i8_load_3d(st, &P.map_w, kb * I8_KB, ch, u.expert, bar);
                    if (SWIGLU) i8_load_3d(st + I8_A_BYTES, &P.map_w, kb * I8_KB, p.N + ch, u.expert, bar);
                    int r = 0;
                    for (; r + I8_BOX_BIG <= u.n; r += I8_BOX_BIG)
                        tma_load_2d(st + 2 * I8_A_BYTES + r * I8_KB, &P.map_a64, kb * I8_KB, u.row0 + r, bar);
                    for (; r < u.n; r += I8_BOX_SMALL)
                        tma_load_2d(st + 2 * I8_A_BYTES + r * I8_KB, &P.map_a16, kb * I8_KB, u.row0 + r, bar);
                }
                gone = *reinterpret_cast<volatile int*>(&sh->abort_flag);
                __syncwarp();
                ++g;
            }
        }
        if (!ok && leader) i8_abort(&sh->abort_flag);
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------------- MMA issuer (warp-uniform loop, one elected lane issues)
        leader = elect_one();
        uint32_t it = 0;
        bool ok = true;
        const uint32_t smem16 = smem_u32(smem) >> 4;
        for (long long item = blockIdx.x; item < total && ok; item += gridDim.x) {
            const I8Item u = i8_item(P, s_pref, s_off, item);
            const uint32_t idesc = i8_idesc(128, u.n);
            const uint32_t buf = two ? it & 1 : 0, use = two ? it >> 1 : it, acc = tmem + buf * I8P_TOKENS;
            bool w = true;
            if (use >= 1) w = i8_wait(&sh->tmem_empty[buf], (use - 1) & 1, P.wait_ns);
            if (!__all_sync(0xffffffffu, w)) { ok = false; break; }
            for (int kb = 0; kb < kblocks; ++kb) {
                const int slot = g % stages;
                if (!__all_sync(0xffffffffu, i8_wait(&sh->full[slot], (g / stages) & 1, P.wait_ns))) { ok = false; break; }
                tc_fence_after();
                const uint32_t st16 = smem16 + slot * (stage_bytes >> 4);
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint64_t da = make_desc(st16 + ((t * I8_A_BYTES + j * 32) >> 4) + DESC_SW128_LBO, DESC_SW128_HI);
                        const uint64_t db = make_desc(st16 + ((2 * I8_A_BYTES + j * 32) >> 4) + DESC_SW128_LBO, DESC_SW128_HI);
                        if (leader) i8_mma(acc + t * second, da, db, idesc, (kb | j) ? 1u : 0u);
                    }
                if (leader) tc_commit(&sh->empty[slot]);
                ++g;
            }
            if (!ok) break;
            if (leader) tc_commit(&sh->tmem_full[buf]);
            ++it;
        }
        if (!ok && leader) i8_abort(&sh->abort_flag);
        __syncwarp();
    } else {
        // ------------------------------------------------------------- epilogue: a lane is a channel; the four warps of a
        // lane quadrant take the item's units (16 tokens of one row tile, with swiglu of both) in turn
        const int quad = warp & 3, sub = (warp - 2) >> 2, et = tid - 64;
        O_* const out = static_cast<O_*>(p.out);
        if (p.offsets && p.zero_tail) {
            for (long long m = (long long)s_off[E] + blockIdx.x; m < p.M; m += gridDim.x)
                for (int n = et; n < p.N; n += 32 * I8P_EPI_WARPS) i8_put(out + m * p.out_stride + n, 0.f);
        }
        float* const rs = sh->row_scale[warp - 2];
        uint32_t it = 0;
        for (long long item = blockIdx.x; item < total; item += gridDim.x, ++it) {
            const I8Item u = i8_item(P, s_pref, s_off, item);
            const uint32_t buf = two ? it & 1 : 0, use = two ? it >> 1 : it;
            const int units = SWIGLU ? u.n >> 4 : u.n >> 3;
            __syncwarp();
            for (int k = sub * 16 + (lane & 15), slot = lane; ; k += 64, slot += 16) {      // scales of unit (k >> 4)
                if ((k >> 4) >= units) break;
                const int c = (SWIGLU ? k >> 4 : k >> 5) * 16 + (k & 15);
                if (lane < 16) rs[slot] = c < u.rows ? p.a_scale[u.row0 + c] : 0.f;
            }
            __syncwarp();
            const int ch = u.ctile * (SWIGLU ? 128 : I8P_ROWS) + quad * 32 + lane;
            const float* wsc = p.w_scale + (long long)u.expert * p.wrows;
            const int ch2 = SWIGLU ? p.N + ch : ch + 128;
            const float sw0 = ch < p.N ? wsc[ch] : 0.f;
            const float sw1 = (SWIGLU ? ch : ch2) < p.N ? wsc[ch2] : 0.f;
            const bool w = i8_wait(&sh->tmem_full[buf], use & 1, P.wait_ns);
            if (!__all_sync(0xffffffffu, w)) { if (lane == 0) i8_abort(&sh->abort_flag); break; }
            tc_fence_after();
            const uint32_t tacc = tmem + buf * I8P_TOKENS + ((uint32_t)(quad * 32) << 16);
            for (int k = sub, slot = 0; k < units; k += 4, slot += 16) {
                const int c = (SWIGLU ? k : k >> 1) * 16, left = u.rows - c;
                float cs[16];
#pragma unroll
                for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(cs + i) = *reinterpret_cast<const float4*>(rs + slot + i);
                uint32_t v[16], v2[SWIGLU ? 16 : 1];
                __syncwarp();
                if (SWIGLU) {
                    tc_ld16(tacc + c, v);
                    tc_ld16(tacc + second + c, reinterpret_cast<uint32_t (&)[16]>(v2));
                } else {
                    tc_ld16(tacc + (k & 1) * second + c, v);
                }
                tc_ld_wait();
                const float sw = SWIGLU || !(k & 1) ? sw0 : sw1;
                auto value = [&](int i) {
                    float x = i8_scaled((int)v[i], cs[i], sw);
                    if (SWIGLU) x = i8_scaled((int)v2[SWIGLU ? i : 0], cs[i], sw1) * i8_silu(x);
                    return x;
                };
                const int chn = SWIGLU || !(k & 1) ? ch : ch2;
                O_* o = out + (long long)(u.row0 + c) * p.out_stride + chn;
                // Straight from the lanes: 32 of them make 64 or 128 bytes of a row.  (Through shared memory, for 16-byte stores, the
                // bf16 product of 8192 x 4096 x 4096 takes 113 us instead of 99: the MMA's operands need that bandwidth.)
                if (chn < p.N) {
                    if (left >= 16) {
#pragma unroll
                        for (int i = 0; i < 16; ++i, o += p.out_stride) i8_put(o, value(i));
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i, o += p.out_stride) {
                            if (i >= left) break;
                            i8_put(o, value(i));
                        }
                    }
                }
            }
            __syncwarp();
            tc_fence_before();
            if (lane == 0) mbar_arrive(&sh->tmem_empty[buf]);
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (sh->abort_flag) i8_unwind(sh->full, g, stages, &sh->done, false, leader);
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TC_TMEM_COLS) : "memory");
    }
}

// -------------------------------------------------------------------------------------------------------- split
constexpr int I8S_THREADS = 192;                          // producer, MMA issuer, four epilogue warps
constexpr int I8S_TOKENS = 128;                           // tokens per tile at most
constexpr int I8S_MAX_STAGES = 8;
constexpr int I8S_SMEM = 200 * 1024;
constexpr size_t I8S_SMEM_LEAST = 116 * 1024;

struct I8SplitShared {
    uint64_t full[I8S_MAX_STAGES], empty[I8S_MAX_STAGES];
    uint64_t done;
    uint32_t tmem_base;
    int abort_flag;
};

__device__ __forceinline__ int4 i8_ld_peer(uint32_t addr) {
    int4 r;
    asm volatile("ld.shared::cluster.v4.s32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(addr) : "memory");
    return r;
}

constexpr int I8_NOTHING = -0x7fffffff - 1;               // stands for the partial sums of a CTA whose waits ran out; no sum of
                                                          // I8_MAX_K products of codes has this value
template <bool SWIGLU>
__global__ void __launch_bounds__(I8S_THREADS, 1)
i8_split_kernel(const __grid_constant__ I8TcParams P) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ I8SplitShared sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const I8Problem& p = P.p;
    const int split = (int)gridDim.x, rank = (int)blockIdx.x, n = P.tokens, stages = P.stages;
    const int stage_bytes = I8_A_BYTES + n * I8_KB;
    const int ch0 = (int)blockIdx.y * (SWIGLU ? 64 : 128), tok0 = (int)blockIdx.z * n;
    const int kb0 = (int)((long long)P.kblocks * rank / split), kb1 = (int)((long long)P.kblocks * (rank + 1) / split);

    if (tid == 0) {
        for (int i = 0; i < stages; ++i) { mbar_init(&sh.full[i], 1); mbar_init(&sh.empty[i], 1); }
        mbar_init(&sh.done, 1);
        sh.abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)), "r"(I8S_TOKENS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem_base;
    bool ok = true, leader = false;
    uint32_t issued = 0;

    if (warp == 0) {
        leader = elect_one();
        if (P.hold) i8_hold(&sh.abort_flag);
        for (int kb = kb0; kb < kb1; ++kb) {
            const int g = kb - kb0, slot = g % stages;
            bool w = true;
            if (g >= stages) w = i8_wait(&sh.empty[slot], ((g / stages) - 1) & 1, P.wait_ns);
            if (!__all_sync(0xffffffffu, w)) { ok = false; break; }
            uint8_t* st = smem + (size_t)slot * stage_bytes;
            if (leader) {
                mbar_arrive_expect_tx(&sh.full[slot], stage_bytes);
                if (SWIGLU) {
#pragma unroll
                    for (int b = 0; b < 2; ++b)           // 64 gate rows, then the 64 matching up rows
                        i8_load_3d(st + b * 64 * I8_KB, &P.map_w, kb * I8_KB, b * p.N + ch0, 0, &sh.full[slot]);
                } else {
                    i8_load_3d(st, &P.map_w, kb * I8_KB, ch0, 0, &sh.full[slot]);
                }
                tma_load_2d(st + I8_A_BYTES, &P.map_a64, kb * I8_KB, tok0, &sh.full[slot]);
            }
            ++issued;
        }
        if (!ok && leader) i8_abort(&sh.abort_flag);
    } else if (warp == 1) {
        leader = elect_one();
        const uint32_t smem16 = smem_u32(smem) >> 4, idesc = i8_idesc(128, n);
        for (int kb = kb0; kb < kb1; ++kb) {
            const int g = kb - kb0, slot = g % stages;
            if (!__all_sync(0xffffffffu, i8_wait(&sh.full[slot], (g / stages) & 1, P.wait_ns))) { ok = false; break; }
            tc_fence_after();
            const uint32_t st16 = smem16 + slot * (stage_bytes >> 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint64_t da = make_desc(st16 + ((j * 32) >> 4) + DESC_SW128_LBO, DESC_SW128_HI);
                const uint64_t db = make_desc(st16 + ((I8_A_BYTES + j * 32) >> 4) + DESC_SW128_LBO, DESC_SW128_HI);
                if (leader) i8_mma(tmem, da, db, idesc, (g | j) ? 1u : 0u);
            }
            if (leader) tc_commit(&sh.empty[slot]);
        }
        if (ok && leader) tc_commit(&sh.done);
        if (!ok && leader) i8_abort(&sh.abort_flag);
    } else {
        // partial sums to shared memory, [token][channel]; the stages are free once every MMA has completed
        const int quad = warp & 3;
        if (!__all_sync(0xffffffffu, i8_wait(&sh.done, 0, P.wait_ns))) {
            if (lane == 0) i8_abort(&sh.abort_flag);
        } else {
            tc_fence_after();
            int* part = reinterpret_cast<int*>(smem) + quad * 32 + lane;
            for (int c = 0; c < n; c += 16) {
                uint32_t v[16];
                tc_ld16(tmem + c + ((uint32_t)(quad * 32) << 16), v);
                tc_ld_wait();
#pragma unroll
                for (int i = 0; i < 16; ++i) part[(c + i) * 128] = (int)v[i];
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (sh.abort_flag) {
        i8_unwind(sh.full, issued, stages, &sh.done, ok, leader);
        for (int i = tid; i < n * 128; i += I8S_THREADS) reinterpret_cast<int*>(smem)[i] = I8_NOTHING;
        __syncthreads();                                  // (alone in its cluster it reads them itself)
    }
    if (split > 1) i8_cluster_sync();
    // The CTAs of the cluster share the tile's tokens out; a thread owns four neighbouring channels of a token.
    const uint32_t base = smem_u32(smem);
    const int rows = min(n, p.M - tok0), per = (n + split - 1) / split;
    const int t_end = min(rows, (rank + 1) * per);
    constexpr int QUADS = SWIGLU ? 16 : 32;               // groups of four channels per token
    const bool vec = ((uintptr_t)p.out & 15) == 0 && p.out_stride % 8 == 0 && p.N % 4 == 0;
    for (int i = tid + rank * per * QUADS; i < t_end * QUADS; i += I8S_THREADS) {
        const int t = i / QUADS, c = (i % QUADS) * 4, ch = ch0 + c;
        if (ch >= p.N) continue;
        int s0[4] = {0, 0, 0, 0}, s1[4] = {0, 0, 0, 0}, low = 0;
        const uint32_t at = base + (uint32_t)(t * 128 + c) * 4;
        for (int r = 0; r < split; ++r) {
            const uint32_t a = i8_cluster_addr(at, r);
            const int4 x = i8_ld_peer(a);
            low = min(low, x.x);
            s0[0] += x.x; s0[1] += x.y; s0[2] += x.z; s0[3] += x.w;
            if (SWIGLU) {
                const int4 y = i8_ld_peer(a + 64 * 4);
                s1[0] += y.x; s1[1] += y.y; s1[2] += y.z; s1[3] += y.w;
            }
        }
        const float sa = p.a_scale[tok0 + t];
        float o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int n_ = min(ch + k, p.N - 1);
            o[k] = i8_scaled(s0[k], sa, p.w_scale[n_]);
            if (SWIGLU) o[k] = i8_scaled(s1[k], sa, p.w_scale[p.N + n_]) * i8_silu(o[k]);
        }
        if (low == I8_NOTHING) continue;
        const long long at_out = (long long)(tok0 + t) * p.out_stride + ch;
        if (vec && p.out_dtype == VMOE_F32) {
            *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at_out) = make_float4(o[0], o[1], o[2], o[3]);
        } else if (vec) {
            union { uint2 w; __nv_bfloat16 b[4]; __half h[4]; } q;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (p.out_dtype == VMOE_BF16) q.b[k] = __float2bfloat16_rn(o[k]); else q.h[k] = __float2half_rn(o[k]);
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at_out) = q.w;
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (ch + k < p.N) i8_store(p.out, at_out + k, p.out_dtype, o[k]);
        }
    }
    __syncthreads();
    if (split > 1) i8_cluster_sync();                     // nobody leaves while its partial sums are read
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(I8S_TOKENS) : "memory");
    }
}

// -------------------------------------------------------------------------------------------------------- host
static int i8_map_w(CUtensorMap* map, const I8Problem& p, uint32_t box_rows) {
    const unsigned long long dims[3] = {(unsigned long long)p.K, (unsigned long long)p.wrows, (unsigned long long)p.E};
    const unsigned long long experts = p.E > 1 ? (unsigned long long)p.w_expert_stride : (unsigned long long)p.w_stride * p.wrows;
    const unsigned long long strides[2] = {(unsigned long long)p.w_stride, experts};
    const uint32_t box[3] = {I8_KB, box_rows, 1};
    return encode_byte_map(map, p.w, 3, dims, strides, box);
}
static int i8_map_a(CUtensorMap* map, const I8Problem& p, uint32_t box_rows) {
    const unsigned long long dims[2] = {(unsigned long long)p.K, (unsigned long long)p.M};
    const unsigned long long strides[1] = {(unsigned long long)p.a_stride};
    const uint32_t box[2] = {I8_KB, box_rows};
    return encode_byte_map(map, p.a, 2, dims, strides, box);
}

// Whether the copies of the tensor-core kernels can read the operands as they are.
bool i8_tc_ok(const I8Problem& p) {
    const unsigned long long all = (unsigned long long)(uintptr_t)p.a | (unsigned long long)p.a_stride | (unsigned long long)(uintptr_t)p.w |
                                   (unsigned long long)p.w_stride | (p.E > 1 ? (unsigned long long)p.w_expert_stride : 0ULL);
    if (all & 15) return false;
    if (p.K < 1 || p.a_stride < p.K || p.w_stride < p.K) return false;
    return p.E == 1 || p.w_expert_stride >= p.w_stride * p.wrows;
}

constexpr size_t I8P_SMEM = 227 * 1024;
// Shared memory of the persistent kernel; an item size goes with a number of experts if two stages fit.
static constexpr size_t i8_tc_smem(int tokens, int E, int stages) {
    return (size_t)stages * (2 * I8_A_BYTES + (size_t)tokens * I8_KB) + sizeof(I8Shared) + 2 * ((size_t)E + 1) * sizeof(int) + 1024;
}
static_assert(i8_tc_smem(64, I8_TC_MAX_EXPERTS, 2) <= I8P_SMEM, "the smallest items go with every number of experts");

// Tokens per item.  Grouped: from the average rows per expert (the counts are on the device); 64 experts, N = 1024, K = 4096,
// items of 64 / 128 / 256 tokens: 16 rows each 46 / 47 / 48 us, 100 rows 64 / 56 / 57, 160 rows 85 / 75 / 66, 320 rows
// 134 / 111 / 103.  Dense: the size whose last round of items over the SMs wastes least -- a k-block costs the larger of 4 U
// (tensor pipe) and 512 + 2 U cycles (ingest), an item of more than 128 tokens its epilogue on top (about 20 cycles a
// token); 8192 x 4096 x 4096: 224 tokens (the choice) 92.5 us, 128 107, 192 101, 256 97.
static int i8_tokens(const I8Problem& p, int kblocks, int ctiles) {
    if (p.offsets) {
        const long long per = p.M / p.E;
        int u = per <= 32 ? 64 : per <= 128 ? 128 : I8P_TOKENS;
        while (u > 64 && i8_tc_smem(u, p.E, 2) > I8P_SMEM) u /= 2;       // from 11496 and 15592 experts on
        return u;
    }
    int best = 128;
    long long least = -1;
    for (int u = 64; u <= I8P_TOKENS; u += 32) {
        const long long rounds = ((p.M + u - 1LL) / u * ctiles + tc_sm_count() - 1) / tc_sm_count();
        const int kb = 4 * u > 512 + 2 * u ? 4 * u : 512 + 2 * u;
        const long long cost = rounds * ((long long)kblocks * kb + (u > 128 ? 20 * u : 0));
        if (least < 0 || cost <= least) { least = cost; best = u; }
    }
    return best;
}

static void i8_limits(I8TcParams* P) {
    const int us = g_i8_wait_us.load(std::memory_order_relaxed);
    P->hold = us == 0;
    P->wait_ns = us ? 1000ull * (unsigned)us : 1000000ull;
}

template <bool SWIGLU, typename O_>
static int launch_i8_tc_t(const I8Problem& p, cudaStream_t st) {
    I8TcParams P;
    memset(&P, 0, sizeof(P));
    P.p = p;
    i8_limits(&P);
    P.kblocks = (p.K + I8_KB - 1) / I8_KB;
    P.ctiles = SWIGLU ? (p.N + 127) / 128 : (p.N + I8P_ROWS - 1) / I8P_ROWS;
    P.tokens = i8_tokens(p, P.kblocks, P.ctiles);
    P.stages = I8P_MAX_STAGES;
    while (P.stages > 2 && i8_tc_smem(P.tokens, p.E, P.stages) > I8P_SMEM) --P.stages;
    const size_t smem = i8_tc_smem(P.tokens, p.E, P.stages);
    if (smem > I8P_SMEM) return VMOE_ERR_LIMIT;
    int rc;
    if ((rc = i8_map_w(&P.map_w, p, SWIGLU ? 128 : I8P_ROWS))) return rc;
    if ((rc = i8_map_a(&P.map_a64, p, I8_BOX_BIG))) return rc;
    if ((rc = i8_map_a(&P.map_a16, p, I8_BOX_SMALL))) return rc;
    // one CTA per SM (tc_sm_count), but no more than there can be items
    const long long blocks = ((long long)p.M + P.tokens - 1) / P.tokens + (p.E > 1 ? (p.E < p.M ? p.E : p.M) : 0);
    const long long items = blocks * P.ctiles;
    const unsigned grid = (unsigned)(items < tc_sm_count() ? items : tc_sm_count());
    static SmemAllowed done;
    if (allow_smem(i8_tc_kernel<SWIGLU, O_>, I8P_SMEM, done) != cudaSuccess) return VMOE_ERR_CUDA;
    return launch_status(launch_pdl(i8_tc_kernel<SWIGLU, O_>, grid, (unsigned)I8P_THREADS, smem, st, P));
}
int launch_i8_tc(const I8Problem& p, cudaStream_t st) {
    if (p.swiglu)
        return p.out_dtype == VMOE_F32 ? launch_i8_tc_t<true, float>(p, st) : p.out_dtype == VMOE_BF16 ? launch_i8_tc_t<true, __nv_bfloat16>(p, st)
                                                                                                         : launch_i8_tc_t<true, __half>(p, st);
    return p.out_dtype == VMOE_F32 ? launch_i8_tc_t<false, float>(p, st) : p.out_dtype == VMOE_BF16 ? launch_i8_tc_t<false, __nv_bfloat16>(p, st)
                                                                                                      : launch_i8_tc_t<false, __half>(p, st);
}

template <bool SWIGLU>
static int launch_i8_split_t(const I8Problem& p, cudaStream_t st) {
    I8TcParams P;
    memset(&P, 0, sizeof(P));
    P.p = p;
    i8_limits(&P);
    P.kblocks = (p.K + I8_KB - 1) / I8_KB;
    P.ctiles = SWIGLU ? (p.N + 63) / 64 : (p.N + 127) / 128;
    const int ttiles = (p.M + I8S_TOKENS - 1) / I8S_TOKENS;
    P.tokens = ((p.M + ttiles - 1) / ttiles + 15) & ~15;
    if (P.ctiles > 65535 || ttiles > 65535) return VMOE_ERR_LIMIT;
    const long long tiles = (long long)P.ctiles * ttiles;
    int split = 1;
    while (split < 8 && 2 * split * tiles <= 148 && 2 * split <= P.kblocks) split *= 2;
    const size_t stage = I8_A_BYTES + (size_t)P.tokens * I8_KB;
    const int per = (P.kblocks + split - 1) / split;
    P.stages = (int)((I8S_SMEM - 1024) / stage);
    if (P.stages > I8S_MAX_STAGES) P.stages = I8S_MAX_STAGES;
    if (P.stages > per) P.stages = per;
    size_t smem = P.stages * stage;
    const size_t part = (size_t)P.tokens * 128 * sizeof(int);
    if (smem < part) smem = part;
    smem += 1024;
    // More than half of an SM's shared memory: one CTA per SM.  CTAs that wait for tensor memory which a CTA of another
    // cluster holds, while that one waits for its own cluster, could otherwise wait in a circle.
    if (smem < I8S_SMEM_LEAST) smem = I8S_SMEM_LEAST;
    int rc;
    if ((rc = i8_map_w(&P.map_w, p, SWIGLU ? 64 : 128))) return rc;
    if ((rc = i8_map_a(&P.map_a64, p, (uint32_t)P.tokens))) return rc;
    static SmemAllowed done;
    if (allow_smem(i8_split_kernel<SWIGLU>, I8S_SMEM, done) != cudaSuccess) return VMOE_ERR_CUDA;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)split, (unsigned)P.ctiles, (unsigned)ttiles); cfg.blockDim = dim3(I8S_THREADS);
    cfg.dynamicSmemBytes = smem; cfg.stream = st;
    // in plain stream order: a cluster kernel here neither starts under its predecessor nor lets its successor start early
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)split; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = 1;
    return launch_status(cudaLaunchKernelEx(&cfg, i8_split_kernel<SWIGLU>, P));
}
int launch_i8_split(const I8Problem& p, cudaStream_t st) { return p.swiglu ? launch_i8_split_t<true>(p, st) : launch_i8_split_t<false>(p, st); }

}  // namespace vmoe

extern "C" int vmoe_int8_set_wait_limit(int32_t microseconds) {
    if (microseconds < 0) return VMOE_ERR_SHAPE;
    vmoe::g_i8_wait_us.store(microseconds, std::memory_order_relaxed);
    return VMOE_OK;
}

extern "C" int vmoe_int8_read_status(void* stream) {
    int v = 0;
    const int zero = 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (cudaMemcpyFromSymbolAsync(&v, vmoe::g_i8_status, sizeof(v), 0, cudaMemcpyDeviceToHost, st) != cudaSuccess ||
        cudaStreamSynchronize(st) != cudaSuccess) {
        cudaGetLastError();                               // not left for the next launch's check
        return VMOE_ERR_CUDA;
    }
    if (v != 0) cudaMemcpyToSymbolAsync(vmoe::g_i8_status, &zero, sizeof(zero), 0, cudaMemcpyHostToDevice, st);
    return v;
}
