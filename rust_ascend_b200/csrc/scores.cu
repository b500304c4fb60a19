// Scores of single tokens from a row of logits: log probability of a given id, log-sum-exp, entropy and the largest alternatives, and
// the gradient of the first two with respect to the logits.
//
// In units of log 2, with c = scale log2(e) and a reference m (the largest c x, rounded), every row needs S = sum 2^d and T = sum 2^d d
// over d = c x - m:
//     lse = ln2 (m + log2 S),   log p = ln2 (c x - m - log2 S),   H = ln2 (log2 S - T / S).
// d is one fused product, and m's own rounding cancels in log p.  One pass holds S and T against a running reference: when a chunk
// raises it, they are moved to the new one, with f = 2^(m - m'):   T <- f (T + S (m - m')),   S <- f S.
// Logits below `low` (masks: -inf, the type's lowest value) are lifted to it, from where 2^d is 0, and the reference starts at half
// of it; a row that never rises above that start, holds a NaN or an infinity, or has products beyond 2^20, is done again by
// careful_row.
//
// Bounds: DRAM (the row is read once), then the exponential unit (one 2^d an element, 16 a clock and SM) and the issue slots: under
// eight instructions an element (the plain form took thirteen), from packed maxima, products and sums.
//
// The top_k largest need no second pass over the row either.  A row is split into the slices of the block's threads; the k-th largest
// slice maximum is a lower bound of the k-th largest element, so every element of the answer lies in a slice whose maximum reaches
// that bound (about k of them).  Threads note the maxima of up to 16 chunks of their slice, and only the chunks that reach the bound
// are read again (they hit L2).  (The least over the warps of each warp's k/8-th largest slice maximum is a cheaper bound, but lets
// several times as many elements through: slower at every k above 5.  Asking L2 for the next rounds ahead of the loads: slower.)
#include "common.cuh"

#include <cmath>
#include <type_traits>

namespace {

using bf = __nv_bfloat16;

constexpr int THREADS = 256;          // of a block of the gradient
constexpr int CANDIDATES = 1024;      // elements at or above the bound that a block can hold; more (ties, hostile rows) take the exact search
constexpr int AGAIN = 512;            // chunks that may be read again before a row takes the exact search
constexpr int UNROLL = 4;             // 16-byte vectors a thread of the gradient has in flight
constexpr int CHUNKS = 16;            // parts of a thread's slice whose maxima are kept

constexpr int LOG_ROUND = 3;          // log2 of the 16-byte vectors a thread of the scores has in flight (2048 x 64000 BF16, 5 alternatives: 52.7 us, at four vectors 57.5)
// Where the search for the bound of the top list ends: a step of 2^-7 of a value lets few more elements through (2048 x 32000 FP32: 54 us, with
// eight more bits 56), rows that lie closer together take eight steps all the same.
constexpr int LEAST_BIT = 16, BOUND_STEPS = 8;

template <typename T> struct Traits { static constexpr int PER = 16 / sizeof(T); };

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
constexpr float LEAST = -1000.0f;       // 2^-1000 is 0
constexpr float SMALLEST_NORMAL = 1.17549435e-38f, LARGEST = 3.402823466e38f;

// Integer that orders values as the top list does: larger value, larger key; both zeros alike; every NaN on top.
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return x != x ? 0xffffffffu : ((u & 0x80000000u) ? ~u : u | 0x80000000u);
}

typedef unsigned long long Entry;         // order key above, complement of the index below: larger is earlier in the top list, no two are equal
__device__ __forceinline__ Entry entry_of(uint32_t key, uint32_t at) { return (Entry)key << 32 | (uint32_t)~at; }
__device__ __forceinline__ uint32_t index_of(Entry e) { return ~(uint32_t)e; }
__device__ __forceinline__ float value_of(Entry e) {      // order_key the other way round
    const uint32_t k = (uint32_t)(e >> 32);
    return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}

// Two FP32 operations in one instruction, each rounded as the single one is.
__device__ __forceinline__ void add2(float& a, float& b, float x, float y) {
    asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tadd.rn.f32x2 p, p, q;\n\tmov.b64 {%0, %1}, p;\n\t}" : "+f"(a), "+f"(b) : "f"(x), "f"(y));
}
__device__ __forceinline__ void fma2(float& c, float& d, float a, float b, float x, float y) {      // (c, d) += (a x, b y)
    asm("{\n\t.reg .b64 p, q, r;\n\tmov.b64 p, {%2, %3};\n\tmov.b64 q, {%4, %5};\n\tmov.b64 r, {%0, %1};\n\tfma.rn.f32x2 r, p, q, r;\n\tmov.b64 {%0, %1}, r;\n\t}"
        : "+f"(c), "+f"(d) : "f"(a), "f"(b), "f"(x), "f"(y));
}
__device__ __forceinline__ void mul2(float& a, float& b, float x, float y) {
    asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tmul.rn.f32x2 p, p, q;\n\tmov.b64 {%0, %1}, p;\n\t}" : "+f"(a), "+f"(b) : "f"(x), "f"(y));
}
__device__ __forceinline__ float max3(float a, float b, float c) { float d; asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c)); return d; }

// S and T against the reference m (log2 units); t is always kept as the sum over d <= 0.
struct Stats { float m, s, t; };

__device__ __forceinline__ void move_to(Stats& a, float m) {
    const float d = fmaxf(a.m - m, LEAST), f = ex2(d);
    a.t = f * (a.t + a.s * d); a.s *= f; a.m = m;
}
// Over the lanes of a warp whose numbers differ below `span` (lanes span apart hold the same): one maximum, one move, then two sums.
__device__ __forceinline__ Stats join_lanes(Stats st, int span) {
    move_to(st, value_of((Entry)__reduce_max_sync(0xffffffffu, order_key(st.m)) << 32));
#pragma unroll
    for (int d = 16; d > 0; d >>= 1)
        if (d < span) { st.s += __shfl_xor_sync(0xffffffffu, st.s, d); st.t += __shfl_xor_sync(0xffffffffu, st.t, d); }
    return st;
}

struct ScoreArgs {
    const void* logits; uint64_t ld;
    const void* ids; uint32_t wide_ids; int64_t ignore;
    float scale, c, low, start;       // c = scale log2(e); logits below `low` count as masked; the reference starts at `start` = c low / 2
    uint32_t careful;                 // the scale is so far from one that careful_row has to do every row
    float* log_probs; float* lse; float* entropy; float* top_values; int32_t* top_ids;
    uint32_t k, vocab; uint64_t rows;
    int* bad;                         // set when an id is outside the vocabulary; may be null
};

// Read or written once: first to leave the caches (with plain accesses 182 us).
template <typename T> __device__ __forceinline__ Vec<T> load_streaming(const Vec<T>* p) { const uint4 t = __ldcs(reinterpret_cast<const uint4*>(p)); Vec<T> v; memcpy(&v, &t, 16); return v; }
template <typename T> __device__ __forceinline__ void store_streaming(Vec<T>* p, const Vec<T>& v) { uint4 t; memcpy(&t, &v, 16); __stcs(reinterpret_cast<uint4*>(p), t); }

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

template <typename T> __device__ __forceinline__ Vec<T> filled(float v) {
    Vec<T> x;
#pragma unroll
    for (int j = 0; j < Traits<T>::PER; ++j) from_f32(v, x.v[j]);
    return x;
}

// Largest element of U vectors, in the storage type where it has a packed maximum; a NaN stays.
template <typename T, int U>
__device__ __forceinline__ float largest(const Vec<T> (&x)[U]) {
    if constexpr (sizeof(T) == 4) {
        float top = x[0].v[0];
#pragma unroll
        for (int u = 0; u < U; ++u) { top = max3(top, x[u].v[0], x[u].v[1]); top = max3(top, x[u].v[2], x[u].v[3]); }
        return top;
    } else {
        typedef typename std::conditional<std::is_same<T, bf>::value, __nv_bfloat162, __half2>::type T2;
        T2 top = *reinterpret_cast<const T2*>(&x[0].v[0]);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < 8; j += 2) top = __hmax2_nan(top, *reinterpret_cast<const T2*>(&x[u].v[j]));
        return max_nan(to_f32(top.x), to_f32(top.y));
    }
}
// Two neighbouring elements, lifted to `low` (NaN too: the reference has it), as FP32.  `low` rounds down into the storage type: rounded up it
// could pass the row's own largest element (steps of 4096 at a million in BF16).
template <typename T>
__device__ __forceinline__ void lifted(const T* p, float low, float& a, float& b) {
    if constexpr (sizeof(T) == 4) { a = fmaxf(p[0], low); b = fmaxf(p[1], low); }
    else if constexpr (std::is_same<T, bf>::value) {
        const __nv_bfloat162 x = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(p), __bfloat162bfloat162(__float2bfloat16_rd(low)));
        const uint32_t w = *reinterpret_cast<const uint32_t*>(&x);
        a = __uint_as_float(w << 16); b = __uint_as_float(w & 0xffff0000u);
    } else {
        const float2 f = __half22float2(__hmax2(*reinterpret_cast<const __half2*>(p), __half2half2(__float2half_rd(low))));
        a = f.x; b = f.y;
    }
}
// Adds U vectors to a thread's S and T (as two sums each) and keeps its largest element.
struct Running { float m, s0, s1, t0, t1, most; };
template <typename T, int U>
__device__ __forceinline__ float take(Running& r, const Vec<T> (&x)[U], const ScoreArgs& a) {
    const float top = largest<T, U>(x);
    r.most = max_nan(r.most, top);
    const float m = max_nan(r.m, top * a.c);
    if (!(m == r.m)) {
        Stats st{r.m, r.s0 + r.s1, r.t0 + r.t1};
        move_to(st, m);
        r.m = m; r.s0 = st.s; r.s1 = 0.f; r.t0 = st.t; r.t1 = 0.f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < Traits<T>::PER; j += 2) {
            float xa, xb, da = -r.m, db = -r.m;
            lifted<T>(&x[u].v[j], a.low, xa, xb);
            fma2(da, db, xa, xb, a.c, a.c);
            const float ea = ex2(da), eb = ex2(db);
            add2(r.s0, r.s1, ea, eb);
            fma2(r.t0, r.t1, ea, eb, da, db);
        }
    return top;
}

__device__ __forceinline__ Entry ld_cluster_u64(const void* at, uint32_t rank) {
    uint32_t a; Entry v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(at)), "r"(rank));
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t ld_cluster_u32(const void* at, uint32_t rank) {
    uint32_t a, v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(at)), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory"); }

template <int THREADS> struct Shared {
    static constexpr int WARPS = THREADS / 32;
    Entry entry[CANDIDATES];
    Entry list[RB_MAX_TOP];
    Stats warp[WARPS];
    float most[WARPS];
    Stats mine;                          // this block's part, read by the cluster's first block
    float chunk[CHUNKS][THREADS];        // largest element of each thread's chunks
    uint16_t again[AGAIN];               // chunks to read again: thread + 256 * chunk (at most 256 threads)
    uint32_t all[WARPS], any[WARPS];     // of the slices' keys
    uint32_t found, again_count;
    uint32_t tie_warp[WARPS];
};

template <int THREADS>
__device__ __forceinline__ void push(Shared<THREADS>& sh, uint32_t key, uint32_t at) {
    const uint32_t i = atomicAdd(&sh.found, 1u);
    if (i < CANDIDATES) sh.entry[i] = entry_of(key, at);
}

// Candidates -> sorted list of the first `want`.  The number of candidates in front of one is its place; eight lanes count for each.
template <int THREADS>
__device__ __forceinline__ void rank_candidates(Shared<THREADS>& sh, uint32_t count, uint32_t want) {
    const uint32_t part = threadIdx.x & 7;
    for (uint32_t base = 0; base < count; base += THREADS / 8) {
        const uint32_t i = base + (threadIdx.x >> 3);
        const Entry e = i < count ? sh.entry[i] : 0;
        uint32_t place = 0;
#pragma unroll 4
        for (uint32_t j = part; j < count; j += 8) place += sh.entry[j] > e;
#pragma unroll
        for (int d = 4; d > 0; d >>= 1) place += __shfl_xor_sync(0xffffffffu, place, d);
        if (part == 0 && i < count && place < want) sh.list[place] = e;
    }
}
// Sorted lists of k entries, one after the other in sh.entry, into one sorted list of k.  An entry's place is its place in its own list
// and the number of larger entries in each other one, found by halving.  Empty entries (0) are behind all others and never placed.
template <int THREADS>
__device__ __forceinline__ void merge_lists(Shared<THREADS>& sh, uint32_t lists, uint32_t k) {
    for (uint32_t i = threadIdx.x; i < lists * k; i += THREADS) {
        const uint32_t own = i / k;
        const Entry e = sh.entry[i];
        uint32_t place = i - own * k;
        for (uint32_t l = 0; l < lists; ++l) {
            if (l == own) continue;
            uint32_t lo = 0, hi = k;                      // entries [0, lo) are larger than e, entries [hi, k) are not
            while (lo < hi) { const uint32_t mid = (lo + hi) / 2; if (sh.entry[l * k + mid] > e) lo = mid + 1; else hi = mid; }
            place += lo;
        }
        if (place < k && e != 0) sh.list[place] = e;
    }
}

// The largest bound that k of the block's keys (one per thread) reach, bit by bit from the first in which the keys differ, down to the last
// one (EXACT) or to LEAST_BIT, but at least BOUND_STEPS of them; `all` and `any` are their conjunction and disjunction.
template <bool EXACT>
__device__ __forceinline__ uint32_t kth_of_block(uint32_t key, uint32_t k, uint32_t all, uint32_t any) {
    const int top = 31 - __clz((int)(all ^ any));             // -1: all alike
    uint32_t bound = top < 0 ? any : any & ~(0xffffffffu >> (31 - top));
    const int least = EXACT ? 0 : max(0, min(LEAST_BIT, top + 1 - BOUND_STEPS));
#pragma unroll 1
    for (int bit = top; bit >= least; --bit) {
        const uint32_t trial = bound | (1u << bit);
        if ((uint32_t)__syncthreads_count(key >= trial) >= k) bound = trial;
    }
    return bound;
}

// Elements [first, last) of the row that are > bound (or >=), counted by the whole block.
template <typename T, int THREADS>
__device__ uint32_t count_in_block(Shared<THREADS>& sh, const T* row, uint32_t first, uint32_t last, uint32_t bound, bool or_equal) {
    __syncthreads();
    if (threadIdx.x == 0) sh.found = 0;
    __syncthreads();
    uint32_t n = 0;
    for (uint32_t i = first + threadIdx.x; i < last; i += THREADS) { const uint32_t key = order_key(to_f32(row[i])); n += key > bound || (or_equal && key == bound); }
    n = __reduce_add_sync(0xffffffffu, n);
    if ((threadIdx.x & 31) == 0) atomicAdd(&sh.found, n);
    __syncthreads();
    return sh.found;
}

// Rows on which the bound lets too many elements through: many equal ones (a masked vocabulary, a constant row) or a hostile order.
// `bound` is the k-th largest slice maximum itself, so that equal elements are equal to it.  Takes the elements above it, after tightening it to the exact k-th value where they would not fit, then fills up with the
// equal ones of lowest index.
template <typename T, int THREADS>
__device__ __noinline__ void exact_candidates(Shared<THREADS>& sh, const T* row, uint32_t first, uint32_t last, uint32_t bound, uint32_t want) {
    constexpr int WARPS = THREADS / 32;
    if (count_in_block<T, THREADS>(sh, row, first, last, bound, false) > CANDIDATES) {
        bound = 0;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t trial = bound | (1u << bit);
            if (count_in_block<T, THREADS>(sh, row, first, last, trial, true) >= want) bound = trial;
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) sh.found = 0;
    __syncthreads();
    for (uint32_t i = first + threadIdx.x; i < last; i += THREADS) { const uint32_t key = order_key(to_f32(row[i])); if (key > bound) push(sh, key, i); }
    __syncthreads();
    // At most CANDIDATES by the count above, want - 1 where it tightened the bound.  Held to that for a row that somebody writes meanwhile,
    // whose scores mean nothing but whose count must not leave the table.
    uint32_t have = sh.found < (uint32_t)CANDIDATES ? sh.found : CANDIDATES;
    for (uint32_t base = first; base < last && have < want; base += THREADS) {      // all threads see the same `have`
        const uint32_t i = base + threadIdx.x;
        const bool tie = i < last && order_key(to_f32(row[i])) == bound;
        const uint32_t ballot = __ballot_sync(0xffffffffu, tie);
        __syncthreads();                              // the counts of the round before have been read
        if ((threadIdx.x & 31) == 0) sh.tie_warp[threadIdx.x >> 5] = __popc(ballot);
        __syncthreads();
        uint32_t before = 0, total = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) { if (w < (int)(threadIdx.x >> 5)) before += sh.tie_warp[w]; total += sh.tie_warp[w]; }
        const uint32_t place = have + before + __popc(ballot & ((1u << (threadIdx.x & 31)) - 1));
        if (tie && place < want) sh.entry[place] = entry_of(bound, i);
        have += total;
    }
    __syncthreads();
    if (threadIdx.x == 0) sh.found = sh.found < want ? (have < want ? have : want) : (sh.found < (uint32_t)CANDIDATES ? sh.found : CANDIDATES);
    __syncthreads();
}

// A whole row by one block, for the rows that the fast form does not answer: nothing but masks, infinities, NaN, scales far from one.
// The exponent is (x - M) c with M the largest element itself, held at -1000 and above, where a logit of -inf then counts as 0.
// m of the result is M, not its product with c.  Where c = scale log2(e) leaves FP32's normal range the scale and log2(e) are multiplied in
// one after the other, and a difference that leaves it (two finite logits under a scale below 2^-120) is formed from halves.
template <typename T, int THREADS>
__device__ __noinline__ Stats careful_row(Shared<THREADS>& sh, const T* row, uint32_t vocab, float scale, float c) {
    constexpr int WARPS = THREADS / 32;
    float most = -INFINITY;
    for (uint32_t i = threadIdx.x; i < vocab; i += THREADS) most = max_nan(most, to_f32(row[i]));
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, d));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.most[threadIdx.x >> 5] = most;
    __syncthreads();
    for (int w = 0; w < WARPS; ++w) most = max_nan(most, sh.most[w]);
    const bool normal = c >= SMALLEST_NORMAL && c <= LARGEST;
    auto take_one = [&](uint32_t i, float& s, float& t) {
        const float x = to_f32(row[i]), gap = x - most;
        float d = normal ? gap * c : gap * scale * LOG2E;
        if (gap < -LARGEST) d = (0.5f * x - 0.5f * most) * scale * (2.f * LOG2E);
        d = fmaxf(d, LEAST);
        const float e = ex2(d);
        s += e; t = fmaf(e, d, t);
    };
    // two sums a thread, as in the fast form: with 128 threads one sum would be V / 128 roundings long
    float s = 0.f, t = 0.f, s1 = 0.f, t1 = 0.f;
    for (uint32_t i = threadIdx.x; i < vocab; i += 2 * THREADS) {
        take_one(i, s, t);
        if (vocab - i > THREADS) take_one(i + THREADS, s1, t1);
    }
    s += s1; t += t1;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) { s += __shfl_xor_sync(0xffffffffu, s, d); t += __shfl_xor_sync(0xffffffffu, t, d); }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.warp[threadIdx.x >> 5] = {most, s, t};
    __syncthreads();
    s = 0.f; t = 0.f;
    for (int w = 0; w < WARPS; ++w) { s += sh.warp[w].s; t += sh.warp[w].t; }
    return {most, s, t};
}

// One row per cluster of 2^log_parts blocks, rows in a grid-stride loop; TOP: with alternatives.  2048 x 128000 BF16: 84 us = 6.2 TB/s; 2048 x
// 32000 FP32: 41 us = 6.4 TB/s, with 5 alternatives 47 (each row's search for them is a chain of barriers and one L2 round trip, which
// the other blocks of the SM hide in part).
template <typename T, int THREADS, bool TOP>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) token_scores_kernel(const ScoreArgs a, const uint32_t log_parts) {
    constexpr int PER = Traits<T>::PER, ROUND = 1 << LOG_ROUND, WARPS = THREADS / 32;
    __shared__ Shared<THREADS> sh;
    const uint32_t tid = threadIdx.x, lane = tid & 31, rank = blockIdx.x & ((1u << log_parts) - 1);
    const uint32_t clusters = gridDim.x >> log_parts;
    rb::predecessor_done();
    for (uint64_t r = blockIdx.x >> log_parts; r < a.rows; r += clusters) {
        const T* row = static_cast<const T*>(a.logits) + r * a.ld;
        const RowView<T> view(row, a.vocab);
        const uint32_t v0 = (uint32_t)((uint64_t)view.vectors * rank >> log_parts), v1 = (uint32_t)((uint64_t)view.vectors * (rank + 1) >> log_parts);
        // this block's elements are [first, last): its vectors, the elements in front in the first block, those behind in the last
        const uint32_t first = rank == 0 ? 0 : view.head + v0 * PER, last = rank + 1 == 1u << log_parts ? a.vocab : view.head + v1 * PER;
        const uint32_t front = view.head + v0 * PER - first, loose = front + (last - (view.head + v1 * PER));
        const uint32_t loose_at = tid < front ? first + tid : view.head + v1 * PER + (tid - front);   // valid for tid < loose

        int64_t id = a.ignore;      // asked for here, looked at when the row has been read: the first warp does not wait for it
        if (tid == 0 && rank == 0) id = a.wide_ids ? static_cast<const int64_t*>(a.ids)[r] : (int64_t) static_cast<const int32_t*>(a.ids)[r];

        Running run{a.start, 0.f, 0.f, 0.f, 0.f, -INFINITY};
        const Vec<T>* vec = view.vec();
        // a chunk is 2^chunk_shift rounds of ROUND vectors, so that CHUNKS of them cover the slice
        const uint32_t rounds = (v1 - v0 + THREADS * ROUND - 1) / (THREADS * ROUND);
        uint32_t chunk_shift = 0;
        while ((CHUNKS << chunk_shift) < (int)rounds) ++chunk_shift;
        uint32_t v = v0 + tid, round = 0;
        float chunk_top = -INFINITY;
        auto note = [&](float top) {
            if constexpr (TOP) {
                chunk_top = max_nan(chunk_top, top);
                sh.chunk[round >> chunk_shift][tid] = chunk_top;
                if ((++round & ((1u << chunk_shift) - 1)) == 0) chunk_top = -INFINITY;
            }
        };
        for (; v - lane + 31 + (ROUND - 1) * THREADS < v1; v += THREADS * ROUND) {      // whole warps: none waits for DRAM once on either side
            Vec<T> got[ROUND];
#pragma unroll
            for (int u = 0; u < ROUND; ++u) got[u] = vec[v + u * THREADS];
            note(take<T, ROUND>(run, got, a));
        }
        if (v < v1) {
            Vec<T> got[ROUND];
#pragma unroll
            for (int u = 0; u < ROUND; ++u) got[u] = v + u * THREADS < v1 ? vec[v + u * THREADS] : filled<T>(-INFINITY);
            note(take<T, ROUND>(run, got, a));
        }
        if (tid < loose) {
            Vec<T> got[1] = {filled<T>(-INFINITY)};
            got[0].v[0] = row[loose_at];
            take<T, 1>(run, got, a);
        }
        float chosen = 0.f;
        if (tid == 0 && rank == 0) {
            if (id != a.ignore && (id < 0 || id >= (int64_t)a.vocab)) { if (a.bad) atomicExch(a.bad, 1); id = a.ignore; }
            if (id != a.ignore && id >= 0 && id < (int64_t)a.vocab) chosen = to_f32(row[id]);
        }
        const uint32_t slice_key = order_key(run.most);

        Stats st = join_lanes({run.m, run.s0 + run.s1, run.t0 + run.t1}, 32);
        if (lane == 0) sh.warp[tid >> 5] = st;
        if constexpr (TOP) {
            const uint32_t all = __reduce_and_sync(0xffffffffu, slice_key), any = __reduce_or_sync(0xffffffffu, slice_key);
            if (lane == 0) { sh.all[tid >> 5] = all; sh.any[tid >> 5] = any; }
        }
        if (tid == 0) { sh.found = 0; sh.again_count = 0; }
        __syncthreads();
        if (tid < 32) st = join_lanes(sh.warp[lane % WARPS], WARPS);

        uint32_t want = 0;
        if constexpr (TOP) {
            want = a.k < last - first ? a.k : last - first;
            const uint32_t all = __reduce_and_sync(0xffffffffu, sh.all[lane % WARPS]), any = __reduce_or_sync(0xffffffffu, sh.any[lane % WARPS]);
            const uint32_t bound = kth_of_block<false>(slice_key, a.k, all, any);
            if (slice_key >= bound) {
                const uint32_t mine = (round + (1u << chunk_shift) - 1) >> chunk_shift;
                for (uint32_t c = 0; c < mine; ++c)
                    if (order_key(sh.chunk[c][tid]) >= bound) { const uint32_t i = atomicAdd(&sh.again_count, 1u); if (i < AGAIN) sh.again[i] = (uint16_t)(tid | c << 8); }
            }
            if (tid < loose) { const uint32_t key = order_key(to_f32(row[loose_at])); if (key >= bound) push(sh, key, loose_at); }
            __syncthreads();
            const uint32_t again = sh.again_count;
            if (again <= AGAIN) {
                const uint32_t per = LOG_ROUND + chunk_shift;        // log2 of a chunk's vectors
                for (uint32_t i = tid; i < again << per; i += THREADS) {
                    const uint32_t which = sh.again[i >> per], at = v0 + (which & 255) + ((which >> 8 << per) + (i & ((1u << per) - 1))) * THREADS;
                    if (at < v1) {
                        const Vec<T> got = vec[at];
                        uint32_t hits = 0;
#pragma unroll
                        for (int j = 0; j < PER; ++j) hits |= (uint32_t)(order_key(to_f32(got.v[j])) >= bound) << j;
                        if (hits) {
                            uint32_t i = atomicAdd(&sh.found, (uint32_t)__popc(hits));
#pragma unroll
                            for (int j = 0; j < PER; ++j) if ((hits >> j & 1) && i++ < CANDIDATES) sh.entry[i - 1] = entry_of(order_key(to_f32(got.v[j])), view.head + at * PER + j);
                        }
                    }
                }
            }
            __syncthreads();
            if (again > AGAIN || sh.found > CANDIDATES) exact_candidates<T, THREADS>(sh, row, first, last, kth_of_block<true>(slice_key, a.k, all, any), want);
            rank_candidates(sh, sh.found, want);
        }
        if (log_parts) {
            const uint32_t parts = 1u << log_parts;
            if (tid == 0) sh.mine = st;
            if (TOP && tid >= want && tid < a.k) sh.list[tid] = 0;      // fewer elements than entries
            cluster_sync();
            if (rank == 0) {
                // one part per lane of the first warp; one list entry per thread
                if (tid < 32) {
                    const uint32_t from = lane % parts;      // parts is 2, 4 or 8
                    st = join_lanes({__uint_as_float(ld_cluster_u32(&sh.mine.m, from)), __uint_as_float(ld_cluster_u32(&sh.mine.s, from)),
                                     __uint_as_float(ld_cluster_u32(&sh.mine.t, from))}, (int)parts);
                }
                if constexpr (TOP) {
                    for (uint32_t i = tid; i < parts * a.k; i += THREADS) sh.entry[i] = ld_cluster_u64(&sh.list[i % a.k], i / a.k);
                    __syncthreads();
                    merge_lists(sh, parts, a.k);
                }
            }
        }
        if (rank == 0) {
            // the joined result is with the first warp; every thread learns whether it stands
            if (tid == 0) sh.mine = st;
            __syncthreads();
            st = sh.mine;
            const bool fast = !a.careful && st.m > a.start && fabsf(st.m) < 1048576.0f;      // beyond 2^20 the rounding of m itself would be felt in d
            float reference, logs;               // log p of x is ln2 (c x - reference) - logs, or scale (x - reference) - logs
            if (fast) { reference = st.m; logs = LN2 * log2f(st.s); }
            else { st = careful_row<T, THREADS>(sh, row, a.vocab, a.scale, a.c); reference = st.m; logs = logf(st.s); }
            const float lse = fast ? fmaf(LN2, reference, logs) : fmaf(reference, a.scale, logs);
            auto log_p = [&](float x) {
                if (!fast) {
                    const float gap = x - reference;
                    return gap < -LARGEST ? fmaf((0.5f * x - 0.5f * reference) * a.scale, 2.f, -logs) : fmaf(gap, a.scale, -logs);
                }
                return x < a.low ? fmaf(x, a.scale, -lse) : fmaf(LN2, fmaf(x, a.c, -reference), -logs);      // c x of a mask's lowest value would overflow
            };
            if (tid == 0) {
                a.lse[r] = lse;
                a.log_probs[r] = id == a.ignore ? 0.f : log_p(chosen);
                if (a.entropy) { const float h = logs - LN2 * (st.t / st.s); a.entropy[r] = h < 0.f ? 0.f : h; }
            }
            if (TOP && tid < a.k) {
                const Entry e = sh.list[tid];
                a.top_ids[r * a.k + tid] = (int32_t)index_of(e);
                a.top_values[r * a.k + tid] = log_p(value_of(e));
            }
        }
        if (log_parts) cluster_sync();       // the lists of this row have been read
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

// -(g + h (log p + H)) p, and g more at the row's token, with log p = z - lse held above a value whose exponential is 0 (a NaN stays); the
// scale comes last, so that a product that leaves FP32's range before it meets p does no harm.
__device__ __forceinline__ float gradient(float x, float scale, float lse, float g, float h, float entropy, bool hot) {
    const float lp = max_nan(fmaf(x, scale, -lse), LEAST);
    const float f = -ex2(lp * LOG2E) * fmaf(h, lp + entropy, g);
    return (hot ? f + g : f) * scale;
}

template <typename T>
__device__ __forceinline__ Vec<T> narrowed(const float (&f)[Traits<T>::PER]) {
    Vec<T> v;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v.v[j] = f[j];
    } else {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (std::is_same<T, bf>::value) { const __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]); w[j] = *reinterpret_cast<const uint32_t*>(&p); }
            else { const __half2 p = __floats2half2_rn(f[2 * j], f[2 * j + 1]); w[j] = *reinterpret_cast<const uint32_t*>(&p); }
        }
        memcpy(&v, w, 16);
    }
    return v;
}

// One block per row segment of THREADS * UNROLL vectors.  Reads and writes each logit once: HBM-bound.  2048 x 128000 BF16: 158 us =
// 6.7 TB/s.
template <typename T>
__global__ void __launch_bounds__(THREADS, 5) token_scores_grad_kernel(const GradArgs a) {
    constexpr int PER = Traits<T>::PER;
    const uint64_t r = blockIdx.x / a.segments;
    rb::predecessor_done();
    const uint32_t seg = (uint32_t)(blockIdx.x % a.segments);
    const T* row = static_cast<const T*>(a.logits) + r * a.ld;
    T* out = static_cast<T*>(a.out) + r * a.ldo;
    int64_t id = a.wide_ids ? static_cast<const int64_t*>(a.ids)[r] : (int64_t) static_cast<const int32_t*>(a.ids)[r];
    const bool scored = id != a.ignore && id >= 0 && id < (int64_t)a.vocab;
    const float g0 = scored ? a.g[r] : 0.f, h0 = a.h ? a.h[r] : 0.f, entropy = a.h ? a.entropy[r] : 0.f;
    const float g = __fmul_rn(g0, a.scale), h = __fmul_rn(h0, a.scale), hh = __fmul_rn(h, entropy);
    // from 2^22 on FP32 steps by half and more: z - lse would not be a log probability
    const float lse = fabsf(a.lse[r]) < 4194304.0f ? a.lse[r] : __int_as_float(0x7fc00000);
    const uint32_t hot = scored ? (uint32_t)id : 0xffffffffu;
    const bool idle = g0 == 0.f && h0 == 0.f;      // an unscored row (whose logits may be anything) or no upstream: zeros
    // The vectors' form: d = c x - lse log2(e), two elements an instruction, 2^d (-(g + h H) - h ln2 d).  Logits below `low`, from where
    // 2^d is 0, are lifted to it, so that d stays finite; where the type cannot hold that value (scales far below one), or c or the bracket
    // (d is above -1444) would leave FP32, one by one.
    const float c = a.scale * LOG2E, base = -lse * LOG2E, slope = -h * LN2, level = -(g + hh), low = (lse + LEAST) / a.scale;
    const bool fast = !(low < (std::is_same<T, __half>::value ? -65000.f : -1e38f)) && !(c > LARGEST) && !(fabsf(level) + 1001.f * fabsf(h) > LARGEST);      // a NaN row goes either way
    // one element, with the arithmetic that it has in a vector: results do not depend on the alignment of the rows
    auto one = [&](uint32_t i, T x) {
        if (idle) return 0.f;
        if (!fast) return gradient(to_f32(x), a.scale, lse, g0, h0, entropy, i == hot);
        alignas(4) const T pair[2] = {x, x};
        float xa, xb;
        lifted<T>(pair, low, xa, xb);
        const float d = fmaf(xa, c, base), f = fmaf(slope, d, level) * ex2(d);
        return i == hot ? f + g : f;
    };
    const RowView<T> view(row, a.vocab);
    if (((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15u) != 0) {
        // the rows are aligned differently: single elements, neighbouring threads on neighbouring elements
        const uint32_t span = THREADS * UNROLL * PER, first = seg * span;
        for (uint32_t i = first + threadIdx.x; i < a.vocab && i - first < span; i += THREADS) from_f32(one(i, row[i]), out[i]);
        return;
    }
    const uint32_t first = seg * THREADS * UNROLL + threadIdx.x;
    const Vec<T>* in = view.vec();
    Vec<T>* o = reinterpret_cast<Vec<T>*>(out + view.head);
    Vec<T> got[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) if (first + u * THREADS < view.vectors) got[u] = load_streaming(in + first + u * THREADS);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const uint32_t v = first + u * THREADS;
        if (v >= view.vectors) break;
        const uint32_t at = view.head + v * PER;
        Vec<T> d;
        if (fast && !idle) {
            float f[PER];
#pragma unroll
            for (int j = 0; j < PER; j += 2) {
                float xa, xb, da = base, db = base;
                lifted<T>(&got[u].v[j], low, xa, xb);
                fma2(da, db, xa, xb, c, c);
                f[j] = level; f[j + 1] = level;
                fma2(f[j], f[j + 1], slope, slope, da, db);
                mul2(f[j], f[j + 1], ex2(da), ex2(db));
            }
            if (hot - at < (uint32_t)PER) {
#pragma unroll
                for (int j = 0; j < PER; ++j) if (at + j == hot) f[j] += g;
            }
            d = narrowed<T>(f);
        } else {
#pragma unroll
            for (int j = 0; j < PER; ++j) from_f32(one(at + j, got[u].v[j]), d.v[j]);
        }
        store_streaming(o + v, d);
    }
    if (seg == 0) {      // the elements around the vectors
        const uint32_t loose = a.vocab - view.vectors * PER;
        if (threadIdx.x < loose) {
            const uint32_t i = threadIdx.x < view.head ? threadIdx.x : view.vectors * PER + threadIdx.x;
            from_f32(one(i, row[i]), out[i]);
        }
    }
}

bool is_float(uint32_t dtype) { return dtype == RB_F32 || dtype == RB_BF16 || dtype == RB_F16; }

template <typename T, int THREADS, bool TOP>
void launch_scores(rb_ctx* ctx, const ScoreArgs& a) {
    static rb::OncePerDevice once;
    const cudaError_t counted = once.run(ctx, [](int& blocks) { return cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, token_scores_kernel<T, THREADS, TOP>, THREADS, 0); });
    const int resident = counted == cudaSuccess && once.value[ctx->device] > 0 ? once.value[ctx->device] : 1;
    const uint64_t slots = (uint64_t)ctx->sm_count * resident, bytes = (uint64_t)a.vocab * sizeof(T);
    // A row is one block's work where the rows fill the GPU or are short; few long rows are split over clusters.  us at 1 / 2 / 4 / 8 blocks
    // a row, BF16: 4 x 128000 with 20 alternatives 11.8 / 10.3 / 8.9 / 9.1, without 8.4 / 6.4 / 4.8 / 4.0; 4 x 32000 with 20 6.3 / 7.2 / 8.1 / 9.4
    // (the join of the lists costs what the split saves).  With alternatives the curves cross late and flat, later for more rows: 20 at 100 KB 8.3 / 8.3 / 8.0 for 4
    // rows, 9.4 / 11.3 / 10.8 for 64; at 160 KB 9.2 / 9.4 / 9.0 and 11.6 / 13.5 / 14.1; at 200 KB 11.2 / 10.3 / 9.1 and 14.4 / 15.9 / 14.4.
    uint32_t log_parts = 0;
    if (bytes >= (TOP ? 160u : 96u) * 1024)
        while (log_parts < (TOP ? 2 : 3) && a.rows << (log_parts + 1) <= 3ull * ctx->sm_count) ++log_parts;
    const uint32_t parts = 1u << log_parts;
    const uint64_t clusters = a.rows < slots / parts ? a.rows : slots / parts;
    // Blocks that take several rows keep the placement of an empty GPU, which spreads the longer lists over the SMs (2048 rows of 128000
    // BF16: 90 us, overlapped 107).
    rb::launch_behind(ctx, token_scores_kernel<T, THREADS, TOP>, clusters * parts, THREADS, 0, parts, a.rows <= clusters, a, log_parts);
}

template <typename T>
void launch_scores(rb_ctx* ctx, const ScoreArgs& a) {
    // Blocks start together and so reach the search for the alternatives together, with DRAM idle meanwhile: with many rows, twice the rows
    // at a time in half the threads each meet it half as often.
    // us at 128 / 256 threads: 8000 rows of 4000 BF16, 5 alternatives 48 / 89, without 28 / 46; 2048 of 32000 FP32, 5: 48.6 / 51.3, 60: 65.8 /
    // 61.9; 2048 of 128000 BF16, 5: 102 / 107, without 94 / 91; 500 of 32003 FP32, 5: 20 / 16.
    const bool many = a.rows > 4ull * ctx->sm_count, shorter = (uint64_t)a.vocab * sizeof(T) <= 64 * 1024;
    if (a.k == 0) {
        if (many && shorter) launch_scores<T, 128, false>(ctx, a);
        else launch_scores<T, 256, false>(ctx, a);
    } else if (many && (shorter || a.k <= 32)) launch_scores<T, 128, true>(ctx, a);
    else launch_scores<T, 256, true>(ctx, a);
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
    // `low`: what lies below it has probability 0 beside anything above low / 2, and c low does not overflow
    const double c = (double)scale * 1.4426950408889634074;
    const bool half = logits->dtype == RB_F16;
    const double low = half ? -65504.0 : -std::fmin(1e30, 1e36 / c);
    const bool careful = c < (half ? 0.01 : 1e-15) || c > (half ? 1e30 : 1e15);
    ScoreArgs a{in.logits.ptr, in.logits.ld, in.ids, ids->dtype == RB_I64, ignore_index, scale, (float)c, (float)low, (float)(0.5 * low * c), careful, (float*)out[0], (float*)out[1], (float*)out[2], (float*)out[3], (int32_t*)out[4],
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
    if (logits->dtype == RB_F32) launch_behind(ctx, token_scores_grad_kernel<float>, grid, THREADS, 0, 0, true, a);
    else if (logits->dtype == RB_BF16) launch_behind(ctx, token_scores_grad_kernel<bf>, grid, THREADS, 0, 0, true, a);
    else launch_behind(ctx, token_scores_grad_kernel<__half>, grid, THREADS, 0, 0, true, a);
    return after_launch(ctx, what);
}

}  // extern "C"
