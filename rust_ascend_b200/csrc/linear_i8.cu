// Linear on 8-bit integers: y[m, n] = (sum_k x[m, k] w[n, k]) * (sx[m] * sw[n]) (+ bias[n]) on the tensor cores (tcgen05 kind::i8, 32-bit
// integer accumulators in TMEM), both operands K-major in 128-byte-swizzled shared memory, fed by TMA.
//
// The integer sum is exact, so splitting K over CTAs and adding the parts in any order gives the same bits; every output is
// rounded to FP32 once (the conversion of the sum), multiplied by the product of the two scales, biased, and rounded to y's type.
//
// Orientation: the tensor core's M rows are rows of W and its N columns are tokens.  A decoding step then fills the 128 rows with
// weights and pays for as many columns as there are tokens (16 at least), and an output row y[m, ..] is stored by neighbouring lanes,
// so no N needs alignment.
//
// Three kernels:
//   * one or two tokens, and up to four over short rows: a warp per weight row (or several), 16-byte loads and dot products of four bytes; no
//     set-up but the launch.
//   * few tokens: one tile of 128 weight rows x TOKENS tokens per cluster, K split over the cluster's CTAs so that all SMs stream
//     weights; the parts are added through distributed shared memory.  Bound: the bytes of W.
//   * many tokens: CTA pairs (cta_group::2) on 256 x 256 tiles, persistent, two accumulators in TMEM so that the store of one tile runs
//     under the products of the next.  Bound: the tensor cores.
#include "common.cuh"

#include "linear_plan.h"
#include "schedule.h"
#include "sm100.cuh"

namespace {

using namespace sm100;
using bf = __nv_bfloat16;

constexpr int ROWS = RB_LINEAR_ROWS;        // weight rows per CTA (TMEM lanes)
constexpr int BK = RB_LINEAR_BK;            // K per stage: one 128-byte swizzle row
constexpr int UMMA_K = 32;       // 32 bytes
constexpr int A_BYTES = ROWS * BK;
constexpr int THREADS = 192;     // producer, issuer, four epilogue warps

struct LinearParams {
    uint32_t m, n, num_kb;
    uint32_t tiles_t, tiles_n;       // token tiles, weight tiles
    uint32_t tokens;                 // pair kernel: tokens of a whole tile, 128 or 256
    uint32_t split, items;           // pair kernel: whole tiles, all work items (see rb_gemm_plan)
    const float* sx; const float* sw; const float* bias;
    void* y;
    uint32_t* status;
};

// tcgen05.mma.kind::i8 instruction descriptor: D = S32 (bits 4-5 = 2), A and B signed (bits 7-9, 10-12 = 1), both K-major.
__host__ __device__ constexpr uint32_t idesc_i8(uint32_t m, uint32_t n) { return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24); }

__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(tmem_d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void umma_i8_pair(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(tmem_d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, uint64_t* bar, int32_t x, int32_t y) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, uint32_t bar_cluster, int32_t x, int32_t y) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(bar_cluster) : "memory");
}
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(taddr) : "memory");
}
__device__ __forceinline__ int32_t ld_cluster_s32(uint32_t addr) {
    int32_t v; asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory"); return v;
}

template <typename Out> __device__ __forceinline__ Out rounded(float v);
template <> __device__ __forceinline__ float rounded<float>(float v) { return v; }
template <> __device__ __forceinline__ bf rounded<bf>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half rounded<__half>(float v) { return __float2half_rn(v); }

// N tokens of one output column, `count` of which exist: y[(token + j) * n + col] for the sums acc[j].  sx: the tokens' scales in shared
// memory.  Lanes are neighbouring columns, so each store is one row segment.  The whole block of values is formed before the first
// store: a branch inside the loop costs the epilogue its instruction-level parallelism (measured: 16 us instead of 3 per 256 x 256 tile).
template <typename Out, int N>
__device__ __forceinline__ void put(const LinearParams& p, uint32_t token, uint32_t col, const uint32_t (&acc)[N], const float* sx, float sw, float bias, uint32_t count) {
    float v[N];
#pragma unroll
    for (int j = 0; j < N; j += 4) {
        const float4 s = *reinterpret_cast<const float4*>(sx + j);
        v[j] = __fmul_rn(__int2float_rn((int32_t)acc[j]), __fmul_rn(s.x, sw));
        v[j + 1] = __fmul_rn(__int2float_rn((int32_t)acc[j + 1]), __fmul_rn(s.y, sw));
        v[j + 2] = __fmul_rn(__int2float_rn((int32_t)acc[j + 2]), __fmul_rn(s.z, sw));
        v[j + 3] = __fmul_rn(__int2float_rn((int32_t)acc[j + 3]), __fmul_rn(s.w, sw));
    }
    if (p.bias) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = __fadd_rn(v[j], bias);
    }
    if (col >= p.n) return;
    Out* at = static_cast<Out*>(p.y) + (size_t)token * p.n;
    if (count >= (uint32_t)N) {
#pragma unroll
        for (int j = 0; j < N; ++j) at[(size_t)j * p.n + col] = rounded<Out>(v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) if ((uint32_t)j < count) at[(size_t)j * p.n + col] = rounded<Out>(v[j]);
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// One to four tokens: bound by the bytes of W and, for small layers, by latency.  A warp reads R rows of W, so that a load of x (from
// L1) serves R times, and has four to eight vectors of 16 bytes a lane in flight: the next step's loads leave before this step's
// products.  6144 x 4096, one token, recorded: 5.9 us = 4.2 TB/s with the launch; 14336 x 4096: 10.8 us = 5.4 TB/s.
template <typename Out, int M, int R>
__global__ void __launch_bounds__(128) linear_i8_row_kernel(const int8_t* x, const int8_t* w, const LinearParams p, const uint32_t k) {
    constexpr int UNROLL = 4 / R;
    const uint32_t lane = threadIdx.x & 31, row0 = (blockIdx.x * 4 + (threadIdx.x >> 5)) * R;
    rb::predecessor_done();
    if (row0 >= p.n) return;                            // a whole warp
    const uint32_t vectors = k / 16;
    const uint4* at[R];
#pragma unroll
    for (int r = 0; r < R; ++r) at[r] = reinterpret_cast<const uint4*>(w + (size_t)(row0 + r < p.n ? row0 + r : p.n - 1) * k);
    auto load = [&](uint32_t base, uint4 (&a)[R][UNROLL]) {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const uint32_t i = base + u * 32;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                a[r][u] = make_uint4(0, 0, 0, 0);       // behind the row: adds nothing
                if (i < vectors) asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(a[r][u].x), "=r"(a[r][u].y), "=r"(a[r][u].z), "=r"(a[r][u].w) : "l"(at[r] + i));
            }
        }
    };
    int32_t acc[R][M] = {};
    uint4 a[R][UNROLL], ahead[R][UNROLL];
    load(lane, a);
    load(lane + 32 * UNROLL, ahead);
    for (uint32_t base = lane; base - lane < vectors; base += 32 * UNROLL) {      // the same number of rounds for every lane
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const uint32_t i = base + u * 32 < vectors ? base + u * 32 : 0;
#pragma unroll
            for (int t = 0; t < M; ++t) {
                const uint4 b = reinterpret_cast<const uint4*>(x + (size_t)((uint32_t)t < p.m ? t : 0) * k)[i];      // a missing token repeats the first
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    acc[r][t] = __dp4a((int)a[r][u].x, (int)b.x, acc[r][t]);
                    acc[r][t] = __dp4a((int)a[r][u].y, (int)b.y, acc[r][t]);
                    acc[r][t] = __dp4a((int)a[r][u].z, (int)b.z, acc[r][t]);
                    acc[r][t] = __dp4a((int)a[r][u].w, (int)b.w, acc[r][t]);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) a[r][u] = ahead[r][u];
        load(base + 64 * UNROLL, ahead);
    }
    // lane r * M + t ends with row r, token t
    int32_t mine = 0;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < M; ++t) { const int32_t sum = __reduce_add_sync(0xffffffffu, acc[r][t]); if (lane == (uint32_t)(r * M + t)) mine = sum; }
    const uint32_t r = lane / M, t = lane - r * M, col = row0 + r;
    if (r < (uint32_t)R && t < p.m && col < p.n) {
        float v = __fmul_rn(__int2float_rn(mine), __fmul_rn(p.sx[t], p.sw[col]));
        if (p.bias) v = __fadd_rn(v, p.bias[col]);
        static_cast<Out*>(p.y)[(size_t)t * p.n + col] = rounded<Out>(v);
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// Few tokens.  Stages are sized so that two CTAs share an SM (one streams while the other starts or stores).  17 x 4096 x 14336, recorded: 13.2 us =
// 4.4 TB/s of weights; about 4 us of any call are the launch, the first load's latency and the join of the parts.
template <int TOKENS> struct Few {
    static constexpr int B_BYTES = TOKENS * BK;
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int STAGES = TOKENS == 16 ? 6 : TOKENS == 32 ? 5 : TOKENS == 64 ? 4 : 3;
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 /*alignment*/ + 128 /*barriers*/ + TOKENS * 4 /*scales*/;
    static constexpr int TMEM_COLS = TOKENS < 32 ? 32 : TOKENS;
    static_assert(TOKENS * ROWS * 4 <= STAGES * STAGE_BYTES, "the parts of a split K are exchanged in the stage buffers");
};

template <typename Out, int TOKENS>
__global__ void __launch_bounds__(THREADS, 2)
linear_i8_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const LinearParams p) {
    using C = Few<TOKENS>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + C::STAGES * C::STAGE_BYTES);
    uint64_t* empty_bar = full_bar + C::STAGES;
    uint64_t* done_bar = empty_bar + C::STAGES;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done_bar + 1);
    volatile uint32_t* abort_word = tmem_slot + 1;
    float* sx = reinterpret_cast<float*>(smem + C::STAGES * C::STAGE_BYTES + 128);

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t parts; asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(parts));
    const uint32_t rank = cluster_ctarank();
    const uint32_t tile = blockIdx.x / parts, tn = tile / p.tiles_t, tt = tile - tn * p.tiles_t;   // neighbours share the weight rows
    const uint32_t row0 = tn * ROWS, token0 = tt * TOKENS;
    const uint32_t kb0 = (uint32_t)((uint64_t)p.num_kb * rank / parts), kb1 = (uint32_t)((uint64_t)p.num_kb * (rank + 1) / parts);
    const uint32_t tokens = p.m - token0 < (uint32_t)TOKENS ? p.m - token0 : TOKENS;

    auto fetch = [&](uint32_t kb, uint32_t stage) {
        uint8_t* sa = smem + stage * C::STAGE_BYTES;
        mbar_expect_tx(&full_bar[stage], C::STAGE_BYTES);
        tma_load_2d(sa, &map_w, &full_bar[stage], (int32_t)(kb * BK), (int32_t)row0);
        tma_load_2d(sa + A_BYTES, &map_x, &full_bar[stage], (int32_t)(kb * BK), (int32_t)token0);
    };
    // The first stages are on their way before anything else is set up: the thread that makes the barriers fills the ring.
    const uint32_t ahead = kb1 - kb0 < (uint32_t)C::STAGES ? kb1 - kb0 : C::STAGES;
    if (threadIdx.x == 0) {
        prefetch_tmap(&map_w); prefetch_tmap(&map_x);
        for (int s = 0; s < C::STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
        mbar_init(done_bar, 1);
        *abort_word = 0;
        fence_barrier_init();
    }
    rb::predecessor_done();
    if (threadIdx.x == 0) for (uint32_t i = 0; i < ahead; ++i) fetch(kb0 + i, i);
    // Blocks of the kernel behind may be on the SM by now.  Shared memory lets two such CTAs share it (at most 256 of the 512 columns)
    // and none of the pair kernel's, so nobody that waits for this kernel can hold what it waits for here.
    if (warp == 1) { tmem_alloc(tmem_slot, C::TMEM_COLS); tmem_relinquish(); }
    for (uint32_t j = threadIdx.x; j < (uint32_t)TOKENS; j += THREADS) sx[j] = j < tokens ? p.sx[token0 + j] : 0.f;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    bool ok = true;
    if (warp == 0) {
        if (threadIdx.x == 0) {
            uint32_t stage = 0, phase = 0;           // the next fill of stage s waits for its (phase + 1)-th release
            for (uint32_t kb = kb0 + ahead; kb < kb1; ++kb) {
                if (!(ok = mbar_wait(&empty_bar[stage], phase, abort_word))) break;
                fetch(kb, stage);
                if (++stage == C::STAGES) { stage = 0; phase ^= 1; }
            }
            if (!ok)   // a wait ran out: a bounded time for the copies in flight to land before the CTA retires
                for (uint32_t i = 0; i < (1u << 22); ++i) __nanosleep(32);
        }
    } else if (warp == 1) {
        if (elect_one()) {
            uint32_t stage = 0, phase = 0;
            for (uint32_t kb = kb0; kb < kb1; ++kb) {
                if (!(ok = mbar_wait(&full_bar[stage], phase, abort_word))) break;
                tc_fence_after();
                uint8_t* sa = smem + stage * C::STAGE_BYTES;
                const uint64_t da = make_kmajor_sw128_desc(smem_u32(sa)), db = make_kmajor_sw128_desc(smem_u32(sa + A_BYTES));
#pragma unroll
                for (uint32_t k = 0; k < BK / UMMA_K; ++k) umma_i8(tmem, da + 2 * k, db + 2 * k, idesc_i8(ROWS, TOKENS), kb != kb0 || k != 0);
                umma_commit(&empty_bar[stage]);
                if (++stage == C::STAGES) { stage = 0; phase ^= 1; }
            }
            if (ok) umma_commit(done_bar);
        }
    } else {
        const uint32_t quarter = warp & 3, row = quarter * 32 + lane, col = row0 + row;
        const float sw = col < p.n ? p.sw[col] : 0.f, bias = p.bias && col < p.n ? p.bias[col] : 0.f;
        ok = mbar_wait(done_bar, 0, abort_word);
        ok = __all_sync(0xffffffffu, ok);
        int32_t* part = reinterpret_cast<int32_t*>(smem);       // [TOKENS][ROWS], over the stages: every product has been read
        if (ok) {
            tc_fence_after();
            for (uint32_t c = 0; c < tokens; c += 16) {
                uint32_t r[16];
                tmem_ld_32x16(tmem + ((quarter * 32) << 16) + c, r);
                tmem_wait_ld();
                if (parts == 1) put<Out, 16>(p, token0 + c, col, r, sx + c, sw, bias, tokens - c);
                else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) part[(c + j) * ROWS + row] = (int32_t)r[j];
                }
            }
            tc_fence_before();
        }
        if (parts > 1) {
            // Every CTA of the cluster adds up its share of the tokens from all parts, in groups of four.  All threads of the cluster
            // meet at the two barriers, whatever happened before; after a wait that ran out the sums are wrong and the status word
            // says so.
            __syncwarp();
            cluster_sync_all();
            const uint32_t groups = (tokens + 3) / 4, first = groups * rank / parts, last = groups * (rank + 1) / parts;
#pragma unroll 2
            for (uint32_t g = first; g < last; ++g) {
                uint32_t acc[4] = {0, 0, 0, 0};
                const uint32_t at = smem_u32(part) + (g * 4 * ROWS + row) * 4;
#pragma unroll 4
                for (uint32_t s = 0; s < parts; ++s) {
                    const uint32_t from = mapa_shared(at, s);
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[j] += (uint32_t)ld_cluster_s32(from + j * ROWS * 4);
                }
                put<Out, 4>(p, token0 + g * 4, col, acc, sx + g * 4, sw, bias, tokens - g * 4);
            }
            __syncwarp();
            cluster_sync_all();      // nobody leaves while its part is being read
        }
    }
    if (warp < 2 && parts > 1) { __syncwarp(); cluster_sync_all(); cluster_sync_all(); }

    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && *abort_word) atomicExch(p.status, 1u);
    if (warp == 1) { __syncwarp(); tc_fence_after(); tmem_dealloc(tmem, C::TMEM_COLS); }
}

// ---------------------------------------------------------------------------------------------------------------------
// Many tokens: pairs of CTAs on tiles of 256 weight rows x 256 tokens.  Each CTA keeps 128 of the weight rows in its TMEM and loads
// its weight rows and half of the tokens; rank 0 issues the products and every completion reaches the barriers of both.
// Every CTA fetches its own tiles.  A last round that would use at most half of the pairs runs as tiles of 128 tokens.
// 4096 x 14336 x 4096: tensor pipe busy in 88 % of all cycles, 143 us = 3.4 POP/s from a cool start, 170 us = 2.8 in a loop under the power cap.
// Rows that do not start on cache lines (K not a multiple of 128) cost about 1.4 times as much: each 128-byte row of a copy then
// takes two lines through the SM's port to L2 (1003 x 5001: 22 us at K = 4096, 30 at 4112).
constexpr int PAIR_TOKENS = 256;
constexpr int PAIR_STAGES = 6;
constexpr int PAIR_B_BYTES = (PAIR_TOKENS / 2) * BK;
constexpr int PAIR_STAGE_BYTES = A_BYTES + PAIR_B_BYTES;
constexpr int PAIR_SMEM_BYTES = PAIR_STAGES * PAIR_STAGE_BYTES + 1024 + 256 + 4 * 2 * PAIR_TOKENS * 4;
constexpr int GROUP = 8;         // raster: weight tiles walked together, so that their operands stay in L2

struct Item { uint32_t row0, token0, tokens; };
__device__ __forceinline__ Item item_of(uint32_t item, const LinearParams& p) {
    uint32_t t, half, batch, tn, tt;
    rb_gemm_item(item, p.split, t, half);
    rb_tile_coords(t, p.tiles_n, p.tiles_t, GROUP, batch, tn, tt);
    const uint32_t tokens = half == 2 ? p.tokens : p.tokens / 2;
    return {tn * 2 * ROWS, tt * p.tokens + (half == 2 ? 0 : half * tokens), tokens};
}

template <typename Out>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
linear_i8_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_xh, const LinearParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + PAIR_STAGES * PAIR_STAGE_BYTES);   // used in the leader only
    uint64_t* empty_bar = full_bar + PAIR_STAGES;
    uint64_t* tmem_full = empty_bar + PAIR_STAGES;
    uint64_t* tmem_empty = tmem_full + 2;                                                       // used in the leader only: 256 arrivals
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tmem_empty + 2);
    volatile uint32_t* abort_word = tmem_slot + 1;
    float* sx_smem = reinterpret_cast<float*>(smem + PAIR_STAGES * PAIR_STAGE_BYTES + 256);

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < PAIR_STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
        for (int a = 0; a < 2; ++a) { mbar_init(&tmem_full[a], 1); mbar_init(&tmem_empty[a], 256); }
        *abort_word = 0;
        fence_barrier_init();
        prefetch_tmap(&map_w); prefetch_tmap(&map_x); if (p.items > p.split) prefetch_tmap(&map_xh);
    }
    if (warp == 1) { tmem_alloc_pair(tmem_slot, 2 * PAIR_TOKENS); tmem_relinquish_pair(); }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    rb::predecessor_done();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    bool ok = true;
    if (warp == 0) {
        if (elect_one()) {
            uint32_t stage = 0, phase = 0;
            for (uint32_t t = pair; ok && t < p.items; t += pairs) {
                const Item it = item_of(t, p);
                const uint32_t rows = it.tokens / 2;
                const CUtensorMap* mx = it.tokens == p.tokens ? &map_x : &map_xh;
                for (uint32_t kb = 0; kb < p.num_kb; ++kb) {
                    if (!(ok = mbar_wait(&empty_bar[stage], phase ^ 1, abort_word))) break;
                    uint8_t* sa = smem + stage * PAIR_STAGE_BYTES;
                    const uint32_t leader = mapa_shared(smem_u32(&full_bar[stage]), 0);
                    if (rank == 0) mbar_expect_tx(&full_bar[stage], 2 * (A_BYTES + rows * BK));   // the bytes of both CTAs
                    tma_load_2d_pair(sa, &map_w, leader, (int32_t)(kb * BK), (int32_t)(it.row0 + rank * ROWS));
                    tma_load_2d_pair(sa + A_BYTES, mx, leader, (int32_t)(kb * BK), (int32_t)(it.token0 + rank * rows));
                    if (++stage == PAIR_STAGES) { stage = 0; phase ^= 1; }
                }
            }
            if (!ok)   // a wait ran out: a bounded time for the copies in flight to land before the CTA retires
                for (uint32_t i = 0; i < (1u << 22); ++i) __nanosleep(32);
        }
    } else if (warp == 1) {
        if (rank == 0 && elect_one()) {
            uint32_t stage = 0, phase = 0, iter = 0;
            for (uint32_t t = pair; ok && t < p.items; t += pairs, ++iter) {
                const uint32_t acc = iter & 1, acc_phase = (iter >> 1) & 1;
                const uint32_t idesc = idesc_i8(2 * ROWS, t < p.split ? p.tokens : p.tokens / 2);
                if (!(ok = mbar_wait(&tmem_empty[acc], acc_phase ^ 1, abort_word))) break;
                tc_fence_after();
                const uint32_t tmem_d = tmem_base + acc * PAIR_TOKENS;
                for (uint32_t kb = 0; kb < p.num_kb; ++kb) {
                    if (!(ok = mbar_wait(&full_bar[stage], phase, abort_word))) break;
                    tc_fence_after();
                    uint8_t* sa = smem + stage * PAIR_STAGE_BYTES;
                    const uint64_t da = make_kmajor_sw128_desc(smem_u32(sa)), db = make_kmajor_sw128_desc(smem_u32(sa + A_BYTES));
#pragma unroll
                    for (uint32_t k = 0; k < BK / UMMA_K; ++k) umma_i8_pair(tmem_d, da + 2 * k, db + 2 * k, idesc, (kb | k) != 0);
                    umma_commit_pair(&empty_bar[stage]);
                    if (++stage == PAIR_STAGES) { stage = 0; phase ^= 1; }
                }
                if (ok) umma_commit_pair(&tmem_full[acc]);
            }
        }
    } else {
        const uint32_t quarter = warp & 3;
        uint32_t iter = 0;
        for (uint32_t t = pair; ok && t < p.items; t += pairs, ++iter) {
            const uint32_t acc = iter & 1, acc_phase = (iter >> 1) & 1;
            const Item it = item_of(t, p);
            const uint32_t col = it.row0 + rank * ROWS + quarter * 32 + lane;
            const float sw = col < p.n ? p.sw[col] : 0.f, bias = p.bias && col < p.n ? p.bias[col] : 0.f;
            // each warp stages the tokens' scales for itself, so no CTA barrier can be left waiting
            float* sx = sx_smem + (quarter * 2 + acc) * PAIR_TOKENS;
            for (uint32_t j = lane; j < it.tokens; j += 32) sx[j] = it.token0 + j < p.m ? p.sx[it.token0 + j] : 0.f;
            __syncwarp();
            ok = mbar_wait(&tmem_full[acc], acc_phase, abort_word);
            if (!(ok = __all_sync(0xffffffffu, ok))) break;
            tc_fence_after();
            for (uint32_t c = 0; c < it.tokens; c += 32) {
                if (it.token0 + c >= p.m) break;     // warp-uniform
                uint32_t r[32];
                tmem_ld_32x32(tmem_base + acc * PAIR_TOKENS + ((quarter * 32) << 16) + c, r);
                tmem_wait_ld();
                put<Out, 32>(p, it.token0 + c, col, r, sx + c, sw, bias, p.m - it.token0 - c);
            }
            tc_fence_before();
            mbar_arrive_cluster(mapa_shared(smem_u32(&tmem_empty[acc]), 0));   // 128 arrivals from each CTA of the pair
        }
    }

    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && *abort_word) atomicExch(p.status, 1u);
    cluster_sync_all();            // nothing may still report to this CTA's barriers when its shared memory goes away
    if (warp == 1) { __syncwarp(); tc_fence_after(); tmem_dealloc_pair(tmem_base, 2 * PAIR_TOKENS); }
}

// ---- host ------------------------------------------------------------------------------------------------------------
// [rows, k] bytes, boxes of BK columns x box_rows rows with the 128-byte swizzle; what a box reaches outside reads as zero.
bool byte_map(CUtensorMap* map, const void* base, uint64_t rows, uint64_t k, uint32_t box_rows) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return false;
    const cuuint64_t dims[2] = {k, rows}, strides[1] = {k};
    const cuuint32_t box[2] = {BK, box_rows}, steps[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename Out, int TOKENS>
int32_t launch_few(rb_ctx* ctx, LinearParams& p, const void* w, const void* x, uint32_t k, uint32_t parts) {
    auto* kernel = linear_i8_few_kernel<Out, TOKENS>;
    static rb::OncePerDevice once;
    const cudaError_t configured = once.run(ctx, [kernel](int&) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Few<TOKENS>::SMEM_BYTES); });
    if (configured != cudaSuccess) return rb::fail(RB_STATUS, "cudaFuncSetAttribute(8-bit linear) failed with CUDA status %d (%s)", (int)configured, cudaGetErrorString(configured));
    CUtensorMap mw, mx;
    if (!byte_map(&mw, w, p.n, k, ROWS) || !byte_map(&mx, x, p.m, k, TOKENS)) return rb::fail(RB_STATUS, "cuTensorMapEncodeTiled failed for the 8-bit linear (m=%u n=%u k=%u)", p.m, p.n, k);
    p.tiles_n = (p.n + ROWS - 1) / ROWS; p.tiles_t = (p.m + TOKENS - 1) / TOKENS;
    rb::launch_behind(ctx, kernel, (uint64_t)p.tiles_n * p.tiles_t * parts, THREADS, Few<TOKENS>::SMEM_BYTES, parts, true, mw, mx, p);
    return rb::after_launch(ctx, "8-bit linear (few tokens)");
}

// CTA pairs that can be resident at once (not every SM can be paired), capped by the context's SM limit; 0 after a failure.
uint32_t resident_pairs(rb_ctx* ctx) {
    static rb::OncePerDevice once;
    const int sms = ctx->sm_count;
    const cudaError_t e = once.run(ctx, [sms](int& clusters) {
        for (auto* kernel : {linear_i8_pair_kernel<float>, linear_i8_pair_kernel<bf>, linear_i8_pair_kernel<__half>}) {
            const cudaError_t set = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PAIR_SMEM_BYTES);
            if (set != cudaSuccess) return set;
        }
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(2 * (unsigned)sms); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = PAIR_SMEM_BYTES;
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeClusterDimension; attr.val.clusterDim.x = 2; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
        cfg.attrs = &attr; cfg.numAttrs = 1;
        return cudaOccupancyMaxActiveClusters(&clusters, linear_i8_pair_kernel<bf>, &cfg);
    });
    if (e != cudaSuccess) return 0;
    uint32_t pairs = (uint32_t)once.value[ctx->device];
    if (ctx->sm_limit > 0 && (uint32_t)ctx->sm_limit / 2 < pairs) pairs = (uint32_t)ctx->sm_limit < 2 ? 1 : (uint32_t)ctx->sm_limit / 2;      // at least one pair
    return pairs;
}

template <typename Out>
int32_t launch_pair(rb_ctx* ctx, LinearParams& p, const void* w, const void* x, uint32_t k, uint32_t pairs, uint32_t tokens) {
    p.tokens = tokens;
    p.tiles_n = (p.n + 2 * ROWS - 1) / (2 * ROWS); p.tiles_t = (p.m + tokens - 1) / tokens;
    rb_gemm_plan(p.tiles_n * p.tiles_t, pairs, true, p.split, p.items);
    if (p.items < pairs) pairs = p.items;
    CUtensorMap mw, mx, mxh;
    if (!byte_map(&mw, w, p.n, k, ROWS) || !byte_map(&mx, x, p.m, k, tokens / 2) || !byte_map(&mxh, x, p.m, k, tokens / 4))
        return rb::fail(RB_STATUS, "cuTensorMapEncodeTiled failed for the 8-bit linear (m=%u n=%u k=%u)", p.m, p.n, k);
    rb::launch_behind(ctx, linear_i8_pair_kernel<Out>, 2 * pairs, THREADS, PAIR_SMEM_BYTES, 0, true, mw, mx, mxh, p);
    return rb::after_launch(ctx, "8-bit linear (CTA pairs)");
}

template <typename Out>
int32_t launch_rows(rb_ctx* ctx, const LinearParams& p, const void* w, const void* x, uint32_t k, uint32_t rows) {
    const int8_t* xp = static_cast<const int8_t*>(x); const int8_t* wp = static_cast<const int8_t*>(w);
#define RB_ROWS(M, R) rb::launch_behind(ctx, linear_i8_row_kernel<Out, M, R>, (p.n + 4 * R - 1) / (4 * R), 128, 0, 0, true, xp, wp, p, k)
    if (p.m == 1) { if (rows == 1) RB_ROWS(1, 1); else RB_ROWS(1, 2); }
    else if (p.m == 2) { if (rows == 1) RB_ROWS(2, 1); else RB_ROWS(2, 2); }
    else { if (rows == 2) RB_ROWS(4, 2); else RB_ROWS(4, 4); }
#undef RB_ROWS
    return rb::after_launch(ctx, "8-bit linear (rows)");
}

template <typename Out>
int32_t launch(rb_ctx* ctx, LinearParams& p, const void* w, const void* x, uint32_t k, const rb_linear_plan& plan, uint32_t pairs) {
    if (plan.tokens == 0) return launch_rows<Out>(ctx, p, w, x, k, plan.rows);
    if (plan.parts == 0) return launch_pair<Out>(ctx, p, w, x, k, pairs, plan.tokens);
    switch (plan.tokens) {
        case 16: return launch_few<Out, 16>(ctx, p, w, x, k, plan.parts);
        case 32: return launch_few<Out, 32>(ctx, p, w, x, k, plan.parts);
        case 64: return launch_few<Out, 64>(ctx, p, w, x, k, plan.parts);
        default: return launch_few<Out, 128>(ctx, p, w, x, k, plan.parts);
    }
}

}  // namespace

using namespace rb;

extern "C" {

int32_t rb_linear_i8(rb_ctx* ctx, const rb_tensor* x, const rb_tensor* x_scales, const rb_tensor* w, const rb_tensor* w_scales,
                     const rb_tensor* bias, const rb_tensor* y) {
    const char* what = "8-bit linear";
    RB_TRY(check_ctx(ctx));
    void *px, *psx, *pw, *psw, *pb, *py;
    RB_TRY(resolve(ctx, x, what, &px)); RB_TRY(resolve(ctx, x_scales, what, &psx)); RB_TRY(resolve(ctx, w, what, &pw)); RB_TRY(resolve(ctx, w_scales, what, &psw));
    RB_TRY(resolve(ctx, bias, what, &pb, true)); RB_TRY(resolve(ctx, y, what, &py));
    if (x->dtype != RB_I8 || w->dtype != RB_I8) return fail(RB_INVALID_TENSOR, "%s requires I8 operands", what);
    if (x_scales->dtype != RB_F32 || w_scales->dtype != RB_F32 || (bias && bias->dtype != RB_F32)) return fail(RB_INVALID_TENSOR, "%s: scales and bias must be FP32", what);
    if (y->dtype != RB_F32 && y->dtype != RB_BF16 && y->dtype != RB_F16) return fail(RB_INVALID_TENSOR, "%s: the output must be F32, BF16 or F16", what);
    uint64_t m, k, ym, n; rows_width(x, &m, &k); rows_width(y, &ym, &n);
    bool ok = w->rank == 2 && w->shape[0] == n && w->shape[1] == k && ym == m && y->rank == x->rank && elements(x_scales) == m && elements(w_scales) == n && (!bias || elements(bias) == n);
    for (uint32_t i = 0; ok && i + 1 < x->rank; ++i) ok = x->shape[i] == y->shape[i];
    if (!ok) return fail(RB_INVALID_TENSOR, "%s: shapes do not agree: x [.., K] with one scale per row, w [N, K] with N scales, bias [N], y [.., N]", what);
    if (k == 0 || k % 16 || k > 131056) return fail(RB_INVALID_TENSOR, "%s: K must be a positive multiple of 16 within 131056", what);
    if (n == 0 || n > 0x7fffff00ull || m > 0x7fffff00ull || ((n + 127) / 128) * ((m + 15) / 16) > 0x0fffffffull) return fail(RB_INVALID_TENSOR, "%s: N must be positive, and M x N within the launch limits", what);
    const uint64_t yb = m * n * dtype_size(y->dtype);
    RB_TRY(no_overlap(py, yb, px, m * k, what)); RB_TRY(no_overlap(py, yb, pw, n * k, what)); RB_TRY(no_overlap(py, yb, psx, m * 4, what));
    RB_TRY(no_overlap(py, yb, psw, n * 4, what)); RB_TRY(no_overlap(py, yb, pb, n * 4, what));
    if (m == 0) return empty_call(ctx);
    DeviceGuard device(ctx);
    LinearParams p{};
    p.m = (uint32_t)m; p.n = (uint32_t)n; p.num_kb = (uint32_t)((k + BK - 1) / BK);
    p.sx = (const float*)psx; p.sw = (const float*)psw; p.bias = (const float*)pb; p.y = py;
    RB_TRY(kernel_status_word(ctx, &p.status));
    const uint32_t pairs = resident_pairs(ctx);
    if (pairs == 0) return fail(RB_STATUS, "%s: configuring the kernel failed", what);
    const bool limited = ctx->sm_limit > 0 && ctx->sm_limit < ctx->sm_count;
    const rb_linear_plan plan = rb_linear_plan_of(p.m, p.n, (uint32_t)k, (uint32_t)(limited ? ctx->sm_limit : ctx->sm_count), pairs, limited);
    if (y->dtype == RB_F32) return launch<float>(ctx, p, pw, px, (uint32_t)k, plan, pairs);
    if (y->dtype == RB_BF16) return launch<bf>(ctx, p, pw, px, (uint32_t)k, plan, pairs);
    return launch<__half>(ctx, p, pw, px, (uint32_t)k, plan, pairs);
}

}  // extern "C"
