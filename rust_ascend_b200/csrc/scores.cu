// Scores of single tokens from a row of logits: log probability of a given id, log-sum-exp, entropy and the largest alternatives, and
// the gradient of the first two with respect to the logits.
//
// With z = scale * x and M = max x every row needs S = sum 2^d and T = sum 2^d d over d = (x - M) scale log2(e):
//     lse = scale M + ln S,   log p = scale (x - M) - ln S,   H = ln S - ln2 T / S.
// One pass holds them against a running maximum: when a chunk raises it, S and T are moved to the new one,
//     f = 2^((m - m') scale log2(e)),   T <- f (T + S (m - m') scale log2(e)),   S <- f S.
// d is held at -1000 and above (2^-1000 is 0 in FP32), which makes a logit of -inf, and a thread that has seen nothing else, count as
// probability 0 without a special case; maxima are taken so that a NaN stays.
//
// HBM-bound: the row is read once.  The top_k largest need no second pass over it either.  A row is split into the slices of the
// block's threads; the k-th largest slice maximum is a lower bound of the k-th largest element, so every element of the answer
// lies in a slice whose maximum reaches that bound (about k of them), and only those are read again (they hit L2).
#include "common.cuh"

namespace {

using bf = __nv_bfloat16;

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int CANDIDATES = 1024;      // elements at or above the bound that a block can hold; more (ties, hostile rows) take the exact search
constexpr int UNROLL = 4;             // 16-byte vectors a thread has in flight

template <typename T> struct Traits;
// KEY_SHIFT: low bits of the FP32 pattern that a value of the storage type never uses
template <> struct Traits<float> { static constexpr int PER = 4, KEY_SHIFT = 0; };
template <> struct Traits<bf> { static constexpr int PER = 8, KEY_SHIFT = 16; };
template <> struct Traits<__half> { static constexpr int PER = 8, KEY_SHIFT = 13; };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_f32(float v, float& o) { o = v; }
__device__ __forceinline__ void from_f32(float v, bf& o) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f32(float v, __half& o) { o = __float2half_rn(v); }

template <typename T> struct __align__(16) Vec { T v[Traits<T>::PER]; };

__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float max_nan(float a, float b) { float y; asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b)); return y; }

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr float LEAST = -1000.0f;

// Integer that orders values as the top list does: larger value, larger key; both zeros alike; every NaN on top.
template <typename T>
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    const uint32_t k = x != x ? 0xffffffffu : ((u & 0x80000000u) ? ~u : u | 0x80000000u);
    return k >> Traits<T>::KEY_SHIFT;
}

struct Stats { float m, s, t; };

// (m, s, t) of two disjoint sets of elements, joined.
__device__ __forceinline__ Stats join(const Stats& a, const Stats& b, float c2) {
    const float m = max_nan(a.m, b.m);
    const float da = fmaxf((a.m - m) * c2, LEAST), db = fmaxf((b.m - m) * c2, LEAST);
    const float fa = ex2(da), fb = ex2(db);
    return {m, fa * a.s + fb * b.s, fa * (a.t + a.s * da) + fb * (b.t + b.s * db)};
}

template <int N>
__device__ __forceinline__ void take(Stats& st, const float (&x)[N], float c2) {
    float top = x[0];
#pragma unroll
    for (int j = 1; j < N; ++j) top = max_nan(top, x[j]);
    top = max_nan(top, st.m);
    if (!(top == st.m)) {
        const float d = fmaxf((st.m - top) * c2, LEAST), f = ex2(d);
        st.t = f * (st.t + st.s * d); st.s *= f; st.m = top;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const float d = fmaxf((x[j] - st.m) * c2, LEAST), e = ex2(d);
        st.s += e;
        st.t = fmaf(e, d, st.t);
    }
}

struct ScoreArgs {
    const void* logits; uint64_t ld;
    const void* ids; uint32_t wide_ids; int64_t ignore;
    float scale;
    float* log_probs; float* lse; float* entropy; float* top_values; int32_t* top_ids;
    uint32_t k, vocab; uint64_t rows;
    int* bad;                         // set when an id is outside the vocabulary; may be null
};

// A row as aligned 16-byte vectors with up to PER - 1 elements in front and behind.
template <typename T> struct RowView {
    const T* p; uint32_t head, vectors, vocab;
    __device__ __forceinline__ RowView(const T* row, uint32_t v) : p(row), vocab(v) {
        const uint32_t off = (uint32_t)((16u - (reinterpret_cast<uintptr_t>(row) & 15u)) & 15u) / (uint32_t)sizeof(T);
        head = off < v ? off : v;
        vectors = (v - head) / Traits<T>::PER;
    }
    __device__ __forceinline__ const Vec<T>* vec() const { return reinterpret_cast<const Vec<T>*>(p + head); }
};

__device__ __forceinline__ uint32_t ld_cluster_u32(const void* at, uint32_t rank) {
    uint32_t a, v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(at)), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory"); }

struct Shared {
    Stats warp[WARPS];
    Stats mine;                          // this block's part, read by the cluster's first block
    uint32_t key[CANDIDATES], at[CANDIDATES];
    uint32_t list_key[RB_MAX_TOP], list_at[RB_MAX_TOP];
    uint32_t winners[THREADS];
    uint32_t found, winner_count, list_count;
    uint32_t tie_warp[WARPS];
};

__device__ __forceinline__ void push(Shared& sh, uint32_t key, uint32_t at) {
    const uint32_t i = atomicAdd(&sh.found, 1u);
    if (i < CANDIDATES) { sh.key[i] = key; sh.at[i] = at; }
}

// Candidates -> sorted list of the first `want`.  Every (key, index) is distinct, so the number of candidates in front of one is its
// place.
__device__ __forceinline__ void rank_candidates(Shared& sh, uint32_t count, uint32_t want) {
    for (uint32_t i = threadIdx.x; i < count; i += THREADS) {
        const uint32_t key = sh.key[i], at = sh.at[i];
        uint32_t place = 0;
        for (uint32_t j = 0; j < count; ++j) { const uint32_t kj = sh.key[j]; place += kj > key || (kj == key && sh.at[j] < at); }
        if (place < want) { sh.list_key[place] = key; sh.list_at[place] = at; }
    }
}

// The k-th largest of one key per thread, bit by bit from the top.
template <typename T>
__device__ __forceinline__ uint32_t kth_of_block(uint32_t key, uint32_t k) {
    uint32_t bound = 0;
    for (int bit = 31 - Traits<T>::KEY_SHIFT; bit >= 0; --bit) {
        const uint32_t trial = bound | (1u << bit);
        if ((uint32_t)__syncthreads_count(key >= trial) >= k) bound = trial;
    }
    return bound;
}

// Elements [first, last) of the row that are > bound (or >=), counted by the whole block.
template <typename T>
__device__ uint32_t count_in_block(Shared& sh, const T* row, uint32_t first, uint32_t last, uint32_t bound, bool or_equal) {
    __syncthreads();
    if (threadIdx.x == 0) sh.found = 0;
    __syncthreads();
    uint32_t n = 0;
    for (uint32_t i = first + threadIdx.x; i < last; i += THREADS) { const uint32_t key = order_key<T>(to_f32(row[i])); n += key > bound || (or_equal && key == bound); }
    n = __reduce_add_sync(0xffffffffu, n);
    if ((threadIdx.x & 31) == 0) atomicAdd(&sh.found, n);
    __syncthreads();
    return sh.found;
}

// Rows on which the bound lets too many elements through: many equal ones (a masked vocabulary, a constant row) or a hostile order.
// Takes the elements above the bound, after tightening it to the exact k-th value where they would not fit, then fills up with the
// equal ones of lowest index.
template <typename T>
__device__ __noinline__ void exact_candidates(Shared& sh, const T* row, uint32_t first, uint32_t last, uint32_t bound, uint32_t want) {
    if (count_in_block<T>(sh, row, first, last, bound, false) > CANDIDATES) {
        bound = 0;
        for (int bit = 31 - Traits<T>::KEY_SHIFT; bit >= 0; --bit) {
            const uint32_t trial = bound | (1u << bit);
            if (count_in_block<T>(sh, row, first, last, trial, true) >= want) bound = trial;
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) sh.found = 0;
    __syncthreads();
    for (uint32_t i = first + threadIdx.x; i < last; i += THREADS) { const uint32_t key = order_key<T>(to_f32(row[i])); if (key > bound) push(sh, key, i); }
    __syncthreads();
    uint32_t have = sh.found;                         // at most CANDIDATES by the search above; want - 1 at most where it tightened the bound
    for (uint32_t base = first; base < last && have < want; base += THREADS) {      // all threads see the same `have`
        const uint32_t i = base + threadIdx.x;
        const bool tie = i < last && order_key<T>(to_f32(row[i])) == bound;
        const uint32_t ballot = __ballot_sync(0xffffffffu, tie);
        __syncthreads();                              // the counts of the round before have been read
        if ((threadIdx.x & 31) == 0) sh.tie_warp[threadIdx.x >> 5] = __popc(ballot);
        __syncthreads();
        uint32_t before = 0, total = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) { if (w < (int)(threadIdx.x >> 5)) before += sh.tie_warp[w]; total += sh.tie_warp[w]; }
        const uint32_t place = have + before + __popc(ballot & ((1u << (threadIdx.x & 31)) - 1));
        if (tie && place < want) { sh.key[place] = bound; sh.at[place] = i; }
        have += total;
    }
    __syncthreads();
    if (threadIdx.x == 0 && sh.found < want) sh.found = have < want ? have : want;
    __syncthreads();
}

// One row per cluster of `parts` blocks (one block where parts is 1), rows in a grid-stride loop.
template <typename T>
__global__ void __launch_bounds__(THREADS, 4) token_scores_kernel(const ScoreArgs a, const uint32_t parts) {
    constexpr int PER = Traits<T>::PER;
    __shared__ Shared sh;
    const uint32_t tid = threadIdx.x, lane = tid & 31, rank = parts > 1 ? blockIdx.x % parts : 0;
    const uint64_t clusters = gridDim.x / parts;
    const float c2 = a.scale * LOG2E;
    for (uint64_t r = blockIdx.x / parts; r < a.rows; r += clusters) {
        const T* row = static_cast<const T*>(a.logits) + r * a.ld;
        const RowView<T> view(row, a.vocab);
        const uint32_t v0 = (uint32_t)((uint64_t)view.vectors * rank / parts), v1 = (uint32_t)((uint64_t)view.vectors * (rank + 1) / parts);
        // this block's elements are [first, last): its vectors, the elements in front in the first block, those behind in the last
        const uint32_t first = rank == 0 ? 0 : view.head + v0 * PER, last = rank + 1 == parts ? a.vocab : view.head + v1 * PER;
        const uint32_t front = view.head + v0 * PER - first, loose = front + (last - (view.head + v1 * PER));
        const uint32_t loose_at = tid < front ? first + tid : view.head + v1 * PER + (tid - front);   // valid for tid < loose

        int64_t id = a.ignore;
        float chosen = 0.f;
        if (tid == 0 && rank == 0) {
            id = a.wide_ids ? static_cast<const int64_t*>(a.ids)[r] : (int64_t) static_cast<const int32_t*>(a.ids)[r];
            if (id != a.ignore && (id < 0 || id >= (int64_t)a.vocab)) { if (a.bad) atomicExch(a.bad, 1); id = a.ignore; }
            if (id != a.ignore && id >= 0 && id < (int64_t)a.vocab) chosen = to_f32(row[id]);
        }

        Stats st{-INFINITY, 0.f, 0.f};
        const Vec<T>* vec = view.vec();
        for (uint32_t v = v0 + tid; v < v1; v += THREADS * UNROLL) {
            Vec<T> got[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) if (v + u * THREADS < v1) got[u] = vec[v + u * THREADS];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                float x[PER];
#pragma unroll
                for (int j = 0; j < PER; ++j) x[j] = v + u * THREADS < v1 ? to_f32(got[u].v[j]) : -INFINITY;
                take<PER>(st, x, c2);
            }
        }
        if (tid < loose) { const float x[1] = {to_f32(row[loose_at])}; take<1>(st, x, c2); }
        const uint32_t slice_key = order_key<T>(st.m);

#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            const Stats o{__shfl_xor_sync(0xffffffffu, st.m, d), __shfl_xor_sync(0xffffffffu, st.s, d), __shfl_xor_sync(0xffffffffu, st.t, d)};
            st = join(st, o, c2);
        }
        if (lane == 0) sh.warp[tid >> 5] = st;
        if (tid == 0) { sh.found = 0; sh.winner_count = 0; }
        __syncthreads();
        st = sh.warp[0];
#pragma unroll
        for (int w = 1; w < WARPS; ++w) st = join(st, sh.warp[w], c2);

        uint32_t want = 0;
        if (a.k) {
            want = a.k < last - first ? a.k : last - first;
            const uint32_t bound = kth_of_block<T>(slice_key, a.k);
            if (slice_key >= bound) sh.winners[atomicAdd(&sh.winner_count, 1u)] = tid;
            if (tid < loose) { const uint32_t key = order_key<T>(to_f32(row[loose_at])); if (key >= bound) push(sh, key, loose_at); }
            __syncthreads();
            const uint32_t winners = sh.winner_count, steps = (v1 - v0 + THREADS - 1) / THREADS;
            for (uint32_t i = tid; i < winners * steps; i += THREADS) {
                const uint32_t v = v0 + sh.winners[i % winners] + (i / winners) * THREADS;
                if (v < v1) {
                    const Vec<T> got = vec[v];
#pragma unroll
                    for (int j = 0; j < PER; ++j) { const uint32_t key = order_key<T>(to_f32(got.v[j])); if (key >= bound) push(sh, key, view.head + v * PER + j); }
                }
            }
            __syncthreads();
            if (sh.found > CANDIDATES) exact_candidates<T>(sh, row, first, last, bound, want);
            rank_candidates(sh, sh.found, want);
        }
        if (parts > 1) {
            if (tid == 0) { sh.mine = st; sh.list_count = want; }
            cluster_sync();
            if (rank == 0) {
                for (uint32_t s = 1; s < parts; ++s) {
                    const Stats o{__uint_as_float(ld_cluster_u32(&sh.mine.m, s)), __uint_as_float(ld_cluster_u32(&sh.mine.s, s)), __uint_as_float(ld_cluster_u32(&sh.mine.t, s))};
                    st = join(st, o, c2);
                }
                if (a.k) {
                    uint32_t count = 0;
                    for (uint32_t s = 0; s < parts; ++s) {
                        const uint32_t n = ld_cluster_u32(&sh.list_count, s);
                        if (tid < n) { sh.key[count + tid] = ld_cluster_u32(&sh.list_key[tid], s); sh.at[count + tid] = ld_cluster_u32(&sh.list_at[tid], s); }
                        count += n;
                    }
                    __syncthreads();
                    rank_candidates(sh, count, a.k);
                }
            }
        }
        if (rank == 0) {
            const float logs = logf(st.s);
            if (tid == 0) {
                a.lse[r] = fmaf(st.m, a.scale, logs);
                a.log_probs[r] = id == a.ignore ? 0.f : fmaf(chosen - st.m, a.scale, -logs);
                if (a.entropy) { const float h = logs - LN2 * (st.t / st.s); a.entropy[r] = h < 0.f ? 0.f : h; }
            }
            if (a.k) {
                __syncthreads();
                if (tid < a.k) {
                    const uint32_t at = sh.list_at[tid];
                    a.top_ids[r * a.k + tid] = (int32_t)at;
                    a.top_values[r * a.k + tid] = fmaf(to_f32(row[at]) - st.m, a.scale, -logs);
                }
            }
        }
        if (parts > 1) cluster_sync();       // the lists of this row have been read
        else __syncthreads();
    }
}

// ---- gradient ---------------------------------------------------------------------------------------------------------------
struct GradArgs {
    const void* logits; uint64_t ld;
    void* out; uint64_t ldo;
    const void* ids; uint32_t wide_ids; int64_t ignore;
    float scale;
    const float* lse; const float* entropy; const float* g; const float* h;
    uint32_t vocab, segments; uint64_t rows;
};

// -(g + h (log p + H)) p scale, with log p = z - lse held above a value whose exponential is 0 (a NaN stays)
__device__ __forceinline__ float gradient(float x, float scale, float lse, float g, float h, float hh) {
    const float lp = max_nan(fmaf(x, scale, -lse), LEAST);
    return -ex2(lp * LOG2E) * fmaf(h, lp, g + hh);
}

// One block per row segment of THREADS * UNROLL vectors.  Reads and writes each logit once: HBM-bound.
template <typename T>
__global__ void __launch_bounds__(THREADS) token_scores_grad_kernel(const GradArgs a) {
    constexpr int PER = Traits<T>::PER;
    const uint64_t r = blockIdx.x / a.segments;
    const uint32_t seg = (uint32_t)(blockIdx.x % a.segments);
    const T* row = static_cast<const T*>(a.logits) + r * a.ld;
    T* out = static_cast<T*>(a.out) + r * a.ldo;
    int64_t id = a.wide_ids ? static_cast<const int64_t*>(a.ids)[r] : (int64_t) static_cast<const int32_t*>(a.ids)[r];
    const bool scored = id != a.ignore && id >= 0 && id < (int64_t)a.vocab;
    const float g = scored ? a.g[r] * a.scale : 0.f, h = a.h ? a.h[r] * a.scale : 0.f, hh = a.h ? h * a.entropy[r] : 0.f;
    // from 2^22 on FP32 steps by half and more: z - lse would not be a log probability
    const float lse = fabsf(a.lse[r]) < 4194304.0f ? a.lse[r] : __int_as_float(0x7fc00000);
    const uint32_t hot = scored ? (uint32_t)id : 0xffffffffu;
    const bool idle = g == 0.f && h == 0.f;      // an unscored row (whose logits may be anything) or no upstream: zeros
    auto one = [&](uint32_t i, float x) { if (idle) return 0.f; float d = gradient(x, a.scale, lse, g, h, hh); return i == hot ? d + g : d; };
    const RowView<T> view(row, a.vocab);
    if (((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15u) != 0) {
        // the rows are aligned differently: single elements, neighbouring threads on neighbouring elements
        const uint32_t span = THREADS * UNROLL * PER, first = seg * span;
        for (uint32_t i = first + threadIdx.x; i < a.vocab && i - first < span; i += THREADS) from_f32(one(i, to_f32(row[i])), out[i]);
        return;
    }
    const uint32_t first = seg * THREADS * UNROLL + threadIdx.x;
    const Vec<T>* in = view.vec();
    Vec<T>* o = reinterpret_cast<Vec<T>*>(out + view.head);
    Vec<T> got[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) if (first + u * THREADS < view.vectors) got[u] = in[first + u * THREADS];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const uint32_t v = first + u * THREADS;
        if (v >= view.vectors) break;
        const uint32_t at = view.head + v * PER;
        Vec<T> d;
#pragma unroll
        for (int j = 0; j < PER; ++j) from_f32(one(at + j, to_f32(got[u].v[j])), d.v[j]);
        o[v] = d;
    }
    if (seg == 0) {      // the elements around the vectors
        const uint32_t loose = a.vocab - view.vectors * PER;
        if (threadIdx.x < loose) {
            const uint32_t i = threadIdx.x < view.head ? threadIdx.x : view.vectors * PER + threadIdx.x;
            from_f32(one(i, to_f32(row[i])), out[i]);
        }
    }
}

bool is_float(uint32_t dtype) { return dtype == RB_F32 || dtype == RB_BF16 || dtype == RB_F16; }

template <typename T>
void launch_scores(rb_ctx* ctx, const ScoreArgs& a) {
    // A row is one block's work where the rows alone fill the GPU; fewer rows are split over clusters of up to eight blocks, as
    // long as each thread keeps a few vectors.
    const uint64_t slots = (uint64_t)ctx->sm_count * 4;
    uint32_t parts = 1;
    while (parts < 8 && a.rows * parts * 2 <= slots && a.vocab / Traits<T>::PER >= parts * 2 * THREADS * 2) parts *= 2;
    const uint64_t clusters = a.rows < slots / parts ? a.rows : slots / parts;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(clusters * parts)); cfg.blockDim = dim3(THREADS); cfg.stream = ctx->stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension; attr.val.clusterDim.x = parts; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cfg.attrs = &attr; cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, token_scores_kernel<T>, a, parts);       // a failure is what after_launch reports
}

}  // namespace

using namespace rb;

namespace {

struct Scored { Rows logits; void* ids = nullptr; };

int32_t check_logits(rb_ctx* ctx, const rb_tensor* logits, const rb_tensor* ids, float scale, const char* what, Scored* out) {
    RB_TRY(resolve_rows(ctx, logits, what, &out->logits)); RB_TRY(resolve(ctx, ids, what, &out->ids));
    if (!is_float(logits->dtype)) return fail(RB_INVALID_TENSOR, "%s: logits must be F32, BF16 or F16", what);
    if (ids->dtype != RB_I32 && ids->dtype != RB_I64) return fail(RB_INVALID_TENSOR, "%s: ids must be INT32 or INT64", what);
    if (out->logits.width == 0 || out->logits.width > 0x7fffffffull) return fail(RB_INVALID_TENSOR, "%s requires a positive vocabulary within INT32_MAX", what);
    if (elements(ids) != out->logits.rows) return fail(RB_INVALID_TENSOR, "%s: one id per row of logits", what);
    if (!(scale > 0.0f) || !(scale <= 3.402823466e38f)) return fail(RB_INVALID_TENSOR, "%s: the scale must be positive and finite", what);
    return RB_OK;
}

int32_t per_row(rb_ctx* ctx, const rb_tensor* t, uint64_t values, uint32_t dtype, const char* what, const char* name, void** p, bool nullable = false) {
    RB_TRY(resolve(ctx, t, what, p, nullable));
    if (t && (t->dtype != dtype || elements(t) != values)) return fail(RB_INVALID_TENSOR, "%s: %s must be %s with %llu values", what, name, dtype_name(dtype), (unsigned long long)values);
    return RB_OK;
}

}  // namespace

extern "C" {

int32_t rb_token_log_probs(rb_ctx* ctx, const rb_tensor* logits, const rb_tensor* ids, float scale, int64_t ignore_index,
                           const rb_tensor* log_probs, const rb_tensor* lse, const rb_tensor* entropy, uint32_t top_k,
                           const rb_tensor* top_values, const rb_tensor* top_ids) {
    const char* what = "token log probabilities";
    RB_TRY(check_ctx(ctx));
    Scored in;
    RB_TRY(check_logits(ctx, logits, ids, scale, what, &in));
    const uint64_t rows = in.logits.rows;
    if (top_k > RB_MAX_TOP || top_k > in.logits.width) return fail(RB_INVALID_TENSOR, "%s: top_k must be within 0..%d and the vocabulary", what, RB_MAX_TOP);
    if ((top_k != 0) != (top_values != nullptr) || (top_k != 0) != (top_ids != nullptr)) return fail(RB_INVALID_TENSOR, "%s: top_values and top_ids come with a positive top_k", what);
    void* out[5];
    RB_TRY(per_row(ctx, log_probs, rows, RB_F32, what, "log_probs", &out[0])); RB_TRY(per_row(ctx, lse, rows, RB_F32, what, "lse", &out[1]));
    RB_TRY(per_row(ctx, entropy, rows, RB_F32, what, "entropy", &out[2], true)); RB_TRY(per_row(ctx, top_values, rows * top_k, RB_F32, what, "top_values", &out[3], true));
    RB_TRY(per_row(ctx, top_ids, rows * top_k, RB_I32, what, "top_ids", &out[4], true));
    const uint64_t sizes[5] = {rows * 4, rows * 4, rows * 4, rows * top_k * 4, rows * top_k * 4};
    for (int i = 0; i < 5; ++i) {
        RB_TRY(no_overlap(out[i], sizes[i], in.logits.ptr, in.logits.extent_bytes, what));
        RB_TRY(no_overlap(out[i], sizes[i], in.ids, rows * dtype_size(ids->dtype), what));
        for (int j = 0; j < i; ++j) RB_TRY(no_overlap(out[i], sizes[i], out[j], sizes[j], what));
    }
    if (rows == 0) return empty_call(ctx);
    DeviceGuard device(ctx);
    ScoreArgs a{in.logits.ptr, in.logits.ld, in.ids, ids->dtype == RB_I64, ignore_index, scale, (float*)out[0], (float*)out[1], (float*)out[2], (float*)out[3], (int32_t*)out[4],
                top_k, (uint32_t)in.logits.width, rows, nullptr};
    if (ctx->synchronous) {          // reports an id outside the vocabulary, as the other indexed operators do
        RB_TRY(ensure_workspace(ctx, 256));
        a.bad = static_cast<int*>(ctx->workspace);
        RB_CUDA(ctx, "cudaMemsetAsync", cudaMemsetAsync(a.bad, 0, 4, ctx->stream));
    }
    if (logits->dtype == RB_F32) launch_scores<float>(ctx, a);
    else if (logits->dtype == RB_BF16) launch_scores<bf>(ctx, a);
    else launch_scores<__half>(ctx, a);
    RB_TRY(after_launch(ctx, what));
    if (a.bad) {
        int h = 0;
        RB_CUDA(ctx, "cudaMemcpy", cudaMemcpy(&h, a.bad, sizeof(int), cudaMemcpyDeviceToHost));
        if (h) return fail(RB_INVALID_TENSOR, "%s: an id is outside [0, vocabulary)", what);
    }
    return RB_OK;
}

int32_t rb_token_log_probs_backward(rb_ctx* ctx, const rb_tensor* logits, const rb_tensor* ids, float scale, int64_t ignore_index,
                                    const rb_tensor* lse, const rb_tensor* entropy, const rb_tensor* grad_log_probs,
                                    const rb_tensor* grad_entropy, const rb_tensor* dlogits) {
    const char* what = "token log probabilities backward";
    RB_TRY(check_ctx(ctx));
    Scored in;
    RB_TRY(check_logits(ctx, logits, ids, scale, what, &in));
    const uint64_t rows = in.logits.rows;
    void *pl, *pe, *pg, *ph;
    RB_TRY(per_row(ctx, lse, rows, RB_F32, what, "lse", &pl)); RB_TRY(per_row(ctx, entropy, rows, RB_F32, what, "entropy", &pe, true));
    RB_TRY(per_row(ctx, grad_log_probs, rows, RB_F32, what, "grad_log_probs", &pg)); RB_TRY(per_row(ctx, grad_entropy, rows, RB_F32, what, "grad_entropy", &ph, true));
    if (grad_entropy && !entropy) return fail(RB_INVALID_TENSOR, "%s: a gradient of the entropy needs the saved entropy", what);
    Rows o;
    RB_TRY(resolve_rows(ctx, dlogits, what, &o));
    if (!same_shape(logits, dlogits) || dlogits->dtype != logits->dtype) return fail(RB_INVALID_TENSOR, "%s: dlogits must have the logits' shape and type", what);
    if (rows > 1 && o.ld < o.width) return fail(RB_INVALID_TENSOR, "%s: rows of dlogits overlap", what);
    const bool in_place = o.ptr == in.logits.ptr && o.ld == in.logits.ld;
    if (!in_place) RB_TRY(no_overlap(o.ptr, o.extent_bytes, in.logits.ptr, in.logits.extent_bytes, what));
    const void* small[] = {in.ids, pl, pe, pg, ph};
    for (int i = 0; i < 5; ++i) RB_TRY(no_overlap(o.ptr, o.extent_bytes, small[i], rows * (i == 0 ? dtype_size(ids->dtype) : 4), what));
    if (rows == 0) return empty_call(ctx);
    DeviceGuard device(ctx);
    const uint64_t per = 16 / dtype_size(logits->dtype), span = THREADS * UNROLL * per, segments = in.logits.width / span ? in.logits.width / span + (in.logits.width % span != 0) : 1;
    if (rows * segments > 0x7fffffffull) return fail(RB_INVALID_TENSOR, "%s: too many rows for one launch", what);
    GradArgs a{in.logits.ptr, in.logits.ld, o.ptr, o.ld, in.ids, ids->dtype == RB_I64, ignore_index, scale, (const float*)pl, (const float*)pe, (const float*)pg, (const float*)ph,
               (uint32_t)in.logits.width, (uint32_t)segments, rows};
    const unsigned grid = (unsigned)(rows * segments);
    if (logits->dtype == RB_F32) token_scores_grad_kernel<float><<<grid, THREADS, 0, ctx->stream>>>(a);
    else if (logits->dtype == RB_BF16) token_scores_grad_kernel<bf><<<grid, THREADS, 0, ctx->stream>>>(a);
    else token_scores_grad_kernel<__half><<<grid, THREADS, 0, ctx->stream>>>(a);
    return after_launch(ctx, what);
}

}  // extern "C"
