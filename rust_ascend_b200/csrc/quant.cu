// Rows held in 8 bits: RMSNorm (with the residual's addition) and row quantisation (plain, or behind SiLU * up) with an I8 result
// and one FP32 scale a row, and the way back.
//
// scale = max(max|y| / 127, 2^-126), q = rint(y / scale).  For the norm y = s r w with one r = 1/sqrt(mean(s^2) + eps) for the
// whole row, so max|y| = r max|s w| and y / scale = (s w) (127 / max|s w|): the quantised values do not need r at all, and one
// reduction (the sum of squares beside the maximum) is enough where a norm followed by a quantisation has two.
//
// These kernels are HBM-bound.  A group of warps owns a row and keeps it in shared memory between the reduction and the store; what
// does not fit is read again, which hits L2.
#include "common.cuh"

#include <type_traits>

namespace {

using bf = __nv_bfloat16;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ bf from_f32<bf>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// VEC neighbouring elements: VEC * sizeof(T) is a power of two up to 32 bytes, and addresses are aligned to it or to 16.
template <typename T, int VEC> struct __align__(VEC * sizeof(T) > 16 ? 16 : VEC * sizeof(T)) Pack { T v[VEC]; };

// Two FP32 operations in one instruction, each rounded as the single one is.
__device__ __forceinline__ void mul2(float& a, float& b, float x, float y) {
    asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tmul.rn.f32x2 p, p, q;\n\tmov.b64 {%0, %1}, p;\n\t}" : "+f"(a), "+f"(b) : "f"(x), "f"(y));
}
__device__ __forceinline__ void add2(float& a, float& b, float x, float y) {
    asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tadd.rn.f32x2 p, p, q;\n\tmov.b64 {%0, %1}, p;\n\t}" : "+f"(a), "+f"(b) : "f"(x), "f"(y));
}
// (c, d) += (a * x, b * y)
__device__ __forceinline__ void fma2(float& c, float& d, float a, float b, float x, float y) {
    asm("{\n\t.reg .b64 p, q, r;\n\tmov.b64 p, {%2, %3};\n\tmov.b64 q, {%4, %5};\n\tmov.b64 r, {%0, %1};\n\tfma.rn.f32x2 r, p, q, r;\n\tmov.b64 {%0, %1}, r;\n\t}"
        : "+f"(c), "+f"(d) : "f"(a), "f"(b), "f"(x), "f"(y));
}
// max(m, |a|, |b|), NaN if any of them is.
__device__ __forceinline__ float max_abs(float m, float a, float b) { float d; asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(m), "f"(a), "f"(b)); return d; }

// Elements widened to FP32; BF16 pairs by moving the bits.
template <typename T, int VEC>
__device__ __forceinline__ void widen(const Pack<T, VEC>& p, float (&v)[VEC]) {
    if constexpr (VEC == 1 || sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = to_f32(p.v[j]);
    } else {
        uint32_t w[VEC / 2];
        memcpy(w, &p, sizeof(w));
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) {
            if constexpr (std::is_same<T, bf>::value) { v[2 * j] = __uint_as_float(w[j] << 16); v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u); }
            else { const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j])); v[2 * j] = f.x; v[2 * j + 1] = f.y; }
        }
    }
}
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> narrow(const float (&v)[VEC]) {
    Pack<T, VEC> p;
    if constexpr (VEC == 1 || sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) p.v[j] = from_f32<T>(v[j]);
    } else {
        uint32_t w[VEC / 2];
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) {
            if constexpr (std::is_same<T, bf>::value) { const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]); w[j] = *reinterpret_cast<const uint32_t*>(&h); }
            else { const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]); w[j] = *reinterpret_cast<const uint32_t*>(&h); }
        }
        memcpy(&p, w, sizeof(w));
    }
    return p;
}
// a + b in the storage type.  The exact sum rounded once equals the FP32 sum rounded again: FP32 holds the sum of two 16-bit values
// exactly unless their exponents are so far apart that the small one cannot reach the border between two results.
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> sum_of(const Pack<T, VEC>& a, const Pack<T, VEC>& b) {
    Pack<T, VEC> p;
    if constexpr (sizeof(T) == 4 || VEC == 1) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) p.v[j] = from_f32<T>(__fadd_rn(to_f32(a.v[j]), to_f32(b.v[j])));
    } else {
        uint32_t x[VEC / 2], y[VEC / 2];
        memcpy(x, &a, sizeof(x)); memcpy(y, &b, sizeof(y));
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) {
            if constexpr (std::is_same<T, bf>::value) { const __nv_bfloat162 h = __hadd2_rn(*reinterpret_cast<__nv_bfloat162*>(&x[j]), *reinterpret_cast<__nv_bfloat162*>(&y[j])); x[j] = *reinterpret_cast<const uint32_t*>(&h); }
            else { const __half2 h = __hadd2_rn(*reinterpret_cast<__half2*>(&x[j]), *reinterpret_cast<__half2*>(&y[j])); x[j] = *reinterpret_cast<const uint32_t*>(&h); }
        }
        memcpy(&p, x, sizeof(x));
    }
    return p;
}
// rint(v * c) as bytes: adding 1.5 * 2^23 leaves the integer in the low bits of the sum, rounded once (|v * c| <= 128).
template <int VEC>
__device__ __forceinline__ Pack<int8_t, VEC> to_bytes(const float (&v)[VEC], float c) {
    constexpr float MAGIC = 12582912.0f;
    Pack<int8_t, VEC> p;
    if constexpr (VEC % 2 != 0) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) p.v[j] = (int8_t)__float_as_uint(__fmaf_rn(v[j], c, MAGIC));
    } else {
        uint32_t u[VEC];
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
            float lo = MAGIC, hi = MAGIC;
            fma2(lo, hi, v[j], v[j + 1], c, c);
            u[j] = __float_as_uint(lo); u[j + 1] = __float_as_uint(hi);
        }
        uint16_t h[VEC / 2];
        uint32_t w[(VEC + 3) / 4];
        if constexpr (VEC % 4 == 0) {
#pragma unroll
            for (int j = 0; j < VEC; j += 4) w[j / 4] = __byte_perm(__byte_perm(u[j], u[j + 1], 0x0040), __byte_perm(u[j + 2], u[j + 3], 0x0040), 0x5410);
            memcpy(&p, w, VEC);
        } else {
#pragma unroll
            for (int j = 0; j < VEC; j += 2) h[j / 2] = (uint16_t)__byte_perm(u[j], u[j + 1], 0x0040);
            memcpy(&p, h, VEC);
        }
    }
    return p;
}

enum Mode { PLAIN = 0, GATED = 1, NORM = 2, ADD_NORM = 3 };

struct QuantArgs {
    const void* x; uint64_t ldx;
    const void* other; uint64_t ldo;     // GATED: up; ADD_NORM: delta
    const void* w; void* x_out; int8_t* q; float* scales;
    uint64_t rows; uint32_t width;
    uint32_t warps;                      // warps that share a row
    uint32_t held;                       // vectors of a row that fit its shared memory
    uint32_t row_bytes;                  // shared memory of a row
    float eps;
};

// SiLU(x) u = x u / (1 + 2^(-x log2 e)): one exponential and one reciprocal.  The reciprocal flushes results below 2^-126 (from x = -87.3 on
// down, which large u make visible), so it is taken of a quarter of the denominator and its product with a quarter may be denormal (4096 x 14336
// BF16: 56.2 us, 53.9 without; products left four times as large and undone with the row's factor: 55.7).  From x = -88.8 on down the
// exponential is infinite and the result -0; an infinite or NaN x gives NaN or infinity, which marks the row.
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float rcp(float x) { float y; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
template <int VEC>
__device__ __forceinline__ void silu_mul(float (&x)[VEC], const float (&u)[VEC]) {
    constexpr float LOG2E = 1.44269504088896340736f, QUARTER = 0.25f;
    if constexpr (VEC % 2 != 0) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[j] = __fmul_rn(__fmul_rn(x[j], __fmul_rn(rcp(__fmaf_rn(ex2(x[j] * -LOG2E), QUARTER, QUARTER)), QUARTER)), u[j]);
    } else {
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
            float e = x[j], f = x[j + 1];
            mul2(e, f, -LOG2E, -LOG2E);
            float d = QUARTER, g = QUARTER;
            fma2(d, g, ex2(e), ex2(f), QUARTER, QUARTER);
            d = rcp(d); g = rcp(g);
            mul2(d, g, QUARTER, QUARTER);
            mul2(x[j], x[j + 1], d, g);
            mul2(x[j], x[j + 1], u[j], u[j + 1]);
        }
    }
}
template <int VEC>
__device__ __forceinline__ void times(float (&x)[VEC], const float (&w)[VEC]) {
    if constexpr (VEC % 2 != 0) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[j] = __fmul_rn(x[j], w[j]);
    } else {
#pragma unroll
        for (int j = 0; j < VEC; j += 2) mul2(x[j], x[j + 1], w[j], w[j + 1]);
    }
}

// A row between its two passes, in shared memory that only the thread which wrote it reads: the FP32 products where SiLU went
// into them, the storage type's own values otherwise (the sum of a residual is rounded to it, so nothing is lost).
// 32-byte vectors are kept as two planes of 16 bytes, so that neighbouring lanes stay on neighbouring banks.
template <typename H, int VEC> struct Held {
    static constexpr int PIECE = VEC * sizeof(H) > 16 ? 16 / sizeof(H) : VEC, PIECES = VEC / PIECE;
    typedef Pack<H, PIECE> Piece;
    static __device__ __forceinline__ void put(void* base, uint32_t held, uint32_t i, const Pack<H, VEC>& p) {
#pragma unroll
        for (int c = 0; c < PIECES; ++c) {
            Piece part;
#pragma unroll
            for (int j = 0; j < PIECE; ++j) part.v[j] = p.v[c * PIECE + j];
            static_cast<Piece*>(base)[c * held + i] = part;
        }
    }
    static __device__ __forceinline__ Pack<H, VEC> get(const void* base, uint32_t held, uint32_t i) {
        Pack<H, VEC> p;
#pragma unroll
        for (int c = 0; c < PIECES; ++c) {
            const Piece part = static_cast<const Piece*>(base)[c * held + i];
#pragma unroll
            for (int j = 0; j < PIECE; ++j) p.v[c * PIECE + j] = part.v[j];
        }
        return p;
    }
};

// What a row's values are multiplied by before they are rounded, from its largest magnitude (as bits) and, for the norm, its sum of
// squares; `first` stores the scale.  `raise`: the values are raised by 2^96 (exactly) first, where the factor would leave FP32's range.
struct Factor { float c; bool bad, raise; };
template <bool NORMS>
__device__ __forceinline__ Factor factor_of(const QuantArgs& a, uint64_t row, uint32_t bits, float sum, bool first) {
    const bool bad = bits >= 0x7f800000u || (NORMS && sum != sum);
    const float most = __uint_as_float(bits);
    const float least = 1.17549435e-38f;           // 2^-126
    const bool raise = most < 1e-16f;
    float c = __fdiv_rn(127.0f, most);
    // rows so small (or a norm so large) that the scale may end at 2^-126
    const bool small = raise || (NORMS && sum > 3.4028235e38f);
    if (first || small) {
        const float r = NORMS ? __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(sum, (float)a.width), a.eps))) : 1.0f;
        const float wanted = __fdiv_rn(__fmul_rn(r, most), 127.0f);
        const bool tiny = wanted < least;
        if (first) a.scales[row] = bad ? __int_as_float(0x7fc00000) : (tiny ? least : wanted);
        if (small) {
            c = tiny ? __fmul_rn(r, 1073741824.0f) : __fdiv_rn(127.0f, __fmul_rn(most, 7.9228163e28f));       // r 2^126, or 127 / max, over 2^96
            if (!raise) c = __fmul_rn(c, 7.9228163e28f);
        }
    }
    return {c, bad, raise};
}

// `warps` whole warps share a row: the whole block, or one warp where that is enough (a block then holds eight rows, which do not
// wait for each other).  Everything that the threads of a row compute alike is kept to one division: the root and the scale are the
// first thread's business.
template <typename T, typename TW, int MODE, int VEC, int UNROLL>
__global__ void __launch_bounds__(512, MODE == PLAIN ? 3 : 2) quant_rows_kernel(const QuantArgs a) {
    constexpr bool NORMS = MODE == NORM || MODE == ADD_NORM, TWO = MODE == GATED || MODE == ADD_NORM;
    typedef typename std::conditional<MODE == GATED, float, T>::type H;
    typedef Held<H, VEC> Hold;
    typedef Pack<T, VEC> In;
    typedef Pack<TW, VEC> Weight;
    typedef Pack<int8_t, VEC> Bytes;
    extern __shared__ __align__(16) uint8_t s_rows[];
    __shared__ float s_sum[16], s_most[16];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t group = warp / a.warps, groups = (blockDim.x >> 5) / a.warps, first_warp = group * a.warps;
    const uint32_t threads = a.warps * 32, tid = threadIdx.x - first_warp * 32;
    const uint32_t vectors = a.width / VEC;            // VEC divides the width
    void* mine = s_rows + (size_t)group * a.row_bytes;
    const Weight* weight = static_cast<const Weight*>(a.w);
    rb::predecessor_done();
    for (uint64_t row = (uint64_t)blockIdx.x * groups + group; row < a.rows; row += (uint64_t)gridDim.x * groups) {
        const In* x = reinterpret_cast<const In*>(static_cast<const T*>(a.x) + row * a.ldx);
        const In* o = reinterpret_cast<const In*>(static_cast<const T*>(a.other) + row * a.ldo);
        In* xo = reinterpret_cast<In*>(static_cast<T*>(a.x_out) + row * a.width);
        Bytes* q = reinterpret_cast<Bytes*>(a.q + row * a.width);
        float sum0 = 0.f, sum1 = 0.f, most = 0.f;
        auto chunk = [&](uint32_t base, auto whole) {
            In in[UNROLL], in2[TWO ? UNROLL : 1];
            Weight wt[NORMS ? UNROLL : 1];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const uint32_t i = base + u * threads;
                const uint32_t at = decltype(whole)::value || i < vectors ? i : base;      // behind the row: the thread's first vector of the round once more
                if (NORMS) wt[NORMS ? u : 0] = weight[at];
                in[u] = x[at];
                if (TWO) in2[TWO ? u : 0] = o[at];
            }
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                // No branch on it: that would move the loads down to where they are used, one DRAM latency after the other (8000 x 5000 FP32: 58 us
                // instead of 37).  What is done twice gives the same again, except for the sum.
                const bool live = decltype(whole)::value || base + u * threads < vectors;
                const uint32_t i = live ? base + u * threads : base;
                float v[VEC];
                [[maybe_unused]] float w[VEC];
                if constexpr (MODE == ADD_NORM) { in[u] = sum_of<T, VEC>(in[u], in2[u]); xo[i] = in[u]; }
                widen<T, VEC>(in[u], v);
                if constexpr (MODE == GATED) { widen<T, VEC>(in2[u], w); silu_mul<VEC>(v, w); if (i < a.held) Hold::put(mine, a.held, i, narrow<float, VEC>(v)); }
                else if (i < a.held) Hold::put(mine, a.held, i, in[u]);
                if constexpr (NORMS) {
                    const float old0 = sum0, old1 = sum1;
                    if constexpr (VEC % 2 != 0) sum0 = __fmaf_rn(v[0], v[0], sum0);
                    else {
#pragma unroll
                        for (int j = 0; j < VEC; j += 2) fma2(sum0, sum1, v[j], v[j + 1], v[j], v[j + 1]);
                    }
                    if (!live) { sum0 = old0; sum1 = old1; }
                    widen<TW, VEC>(wt[u], w);
                    times<VEC>(v, w);
                }
                if constexpr (VEC % 2 != 0) most = max_abs(most, v[0], 0.f);
                else {
#pragma unroll
                    for (int j = 0; j < VEC; j += 2) most = max_abs(most, v[j], v[j + 1]);
                }
            }
        };
        uint32_t base = tid;
        // The norm's full rounds without the selections, for whole warps (base | 31 is the last lane): a warp that went both ways would wait for
        // DRAM twice.
        if constexpr (NORMS) {
            for (; (base | 31) + (UNROLL - 1) * threads < vectors; base += UNROLL * threads) chunk(base, std::true_type());
            if (base < vectors) chunk(base, std::false_type());
        } else for (; base < vectors; base += UNROLL * threads) chunk(base, std::false_type());

        constexpr int AHEAD = NORMS && sizeof(Weight) > 16 ? 2 : 4;
        // magnitudes compare as integers, and in that order NaN lies above infinity
        uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
        float sum = sum0 + sum1;
        if (NORMS) {
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        }
        if (a.warps > 1) {
            // a row's partial results: written, read after the first barrier, and not overwritten before the second
            if (lane == 0) { s_sum[warp] = sum; s_most[warp] = __uint_as_float(bits); }
            __syncthreads();
            bits = __reduce_max_sync(0xffffffffu, __float_as_uint(s_most[lane < a.warps ? lane : 0]));
            if (NORMS) {
                sum = 0.f;
#pragma unroll 4
                for (uint32_t i = 0; i < a.warps; ++i) sum += s_sum[i];
            }
            if (gridDim.x < a.rows) __syncthreads();
        }
        const Factor f = factor_of<NORMS>(a, row, bits, sum, tid == 0);
        const float c = f.c;
        const bool bad = f.bad, raise = f.raise;
        auto finish = [&](uint32_t i, const Weight& by, auto plain) {
            float v[VEC];
            [[maybe_unused]] float w[VEC];
            if (i < a.held) widen<H, VEC>(Hold::get(mine, a.held, i), v);
            else {
                widen<T, VEC>(MODE == ADD_NORM ? xo[i] : x[i], v);
                if constexpr (MODE == GATED) { widen<T, VEC>(o[i], w); silu_mul<VEC>(v, w); }
            }
            if constexpr (NORMS) { widen<TW, VEC>(by, w); times<VEC>(v, w); }
            if (!decltype(plain)::value) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] = bad ? 0.f : (raise ? __fmul_rn(v[j], 7.9228163e28f) : v[j]);
            }
            q[i] = to_bytes<VEC>(v, !decltype(plain)::value && bad ? 0.f : c);
        };
        if (!bad && !raise) {
            // the weights of a few vectors in front of those vectors' stores, which a load may not pass (8192 x 4096: one by one 54 us instead of 37)
            uint32_t i = tid;
            for (; i + (AHEAD - 1) * threads < vectors; i += AHEAD * threads) {
                Weight by[AHEAD];
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) if (NORMS) by[u] = weight[i + u * threads];
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) finish(i + u * threads, by[u], std::true_type());
            }
            for (; i < vectors; i += threads) { Weight by; if (NORMS) by = weight[i]; finish(i, by, std::true_type()); }
        } else {
#pragma unroll 1
            for (uint32_t i = tid; i < vectors; i += threads) { Weight by; if (NORMS) by = weight[i]; finish(i, by, std::false_type()); }
        }
    }
}

// Plain rows that start anywhere (an odd width; 4000 x 14335 BF16: 38 us, aligned 30): vectors from the row's first 16-byte boundary on, the elements around them one by
// one, and single bytes out.  The row lies in shared memory with its vectors aligned, so element e is at e + VEC - head, and is read
// back by other threads than wrote it: lanes on neighbouring elements.
template <typename T>
__global__ void __launch_bounds__(512, 3) quant_shifted_kernel(const QuantArgs a) {
    constexpr int VEC = 16 / sizeof(T), UNROLL = 4;
    typedef Pack<T, VEC> In;
    extern __shared__ __align__(16) uint8_t s_rows[];
    __shared__ float s_most[16];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, threads = blockDim.x, tid = threadIdx.x;
    T* held = reinterpret_cast<T*>(s_rows);
    rb::predecessor_done();
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + row * a.ldx;
        const uint32_t to_boundary = (uint32_t)((16u - (reinterpret_cast<uintptr_t>(x) & 15u)) & 15u) / (uint32_t)sizeof(T);
        const uint32_t head = to_boundary < a.width ? to_boundary : a.width, vectors = (a.width - head) / VEC, shift = VEC - head;
        const In* in = reinterpret_cast<const In*>(x + head);
        In* out = reinterpret_cast<In*>(held) + 1;
        float most = 0.f;
        for (uint32_t base = tid; base < vectors; base += UNROLL * threads) {
            In p[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) { const uint32_t i = base + u * threads; p[u] = in[i < vectors ? i : vectors - 1]; }
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const uint32_t i = base + u * threads;
                if (i < vectors) out[i] = p[u];
                float v[VEC];
                widen<T, VEC>(p[u], v);
#pragma unroll
                for (int j = 0; j < VEC; j += 2) most = max_abs(most, v[j], v[j + 1]);
            }
        }
        const uint32_t loose = a.width - vectors * VEC;
        if (tid < loose) {
            const uint32_t e = tid < head ? tid : vectors * VEC + tid;
            const T v = x[e];
            held[e + shift] = v;
            most = max_abs(most, to_f32(v), 0.f);
        }
        uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
        if (lane == 0) s_most[warp] = __uint_as_float(bits);
        __syncthreads();
        bits = __reduce_max_sync(0xffffffffu, __float_as_uint(s_most[lane < threads / 32 ? lane : 0]));
        const Factor f = factor_of<false>(a, row, bits, 0.f, tid == 0);
        int8_t* q = a.q + row * a.width;
        if (!f.bad && !f.raise) {
#pragma unroll 4
            for (uint32_t e = tid; e < a.width; e += threads) { const float v[1] = {to_f32(held[e + shift])}; q[e] = to_bytes<1>(v, f.c).v[0]; }
        } else {
            for (uint32_t e = tid; e < a.width; e += threads) {
                const float v[1] = {f.bad ? 0.f : __fmul_rn(to_f32(held[e + shift]), 7.9228163e28f)};
                q[e] = to_bytes<1>(v, f.bad ? 0.f : f.c).v[0];
            }
        }
        if (gridDim.x < a.rows) __syncthreads();       // the row in shared memory has been read
    }
}

constexpr uint32_t SHIFTED_VECTORS = 4;      // 1777 x 5003 FP32: 10.9 us at four vectors a thread; at eight 3 % more, at twelve 22 % (single elements throughout: 16.0)
constexpr uint32_t ROW_SMEM = 96 * 1024;     // shared memory a row may take: at least two rows an SM

template <typename T, typename TW, int MODE, int VEC, int UNROLL>
int32_t launch(rb_ctx* ctx, QuantArgs a, const char* what) {
    typedef typename std::conditional<MODE == GATED, float, T>::type H;
    static rb::OncePerDevice once;
    const cudaError_t configured = once.run(ctx, [](int&) { return cudaFuncSetAttribute(quant_rows_kernel<T, TW, MODE, VEC, UNROLL>, cudaFuncAttributeMaxDynamicSharedMemorySize, ROW_SMEM); });
    if (configured != cudaSuccess) return rb::fail(RB_STATUS, "%s: cudaFuncSetAttribute failed with CUDA status %d (%s)", what, (int)configured, cudaGetErrorString(configured));
    const uint32_t vectors = a.width / VEC;
    // Many rows: a few vectors a thread, so that what all threads of a row do alike weighs little and several rows share an SM (one's
    // loads run under another's reduction).  8192 x 4096 BF16 with residual: 37.1 us at four vectors a thread, 42.2 at two, 70 at one.
    // SiLU over 4096 x 14336 BF16: 53.9 us at eight, 57.3 at four.  Few rows: latency, so one vector a thread where that fits.
    const uint32_t wanted = a.rows <= (uint64_t)ctx->sm_count ? 1 : (VEC == 1 ? 20 : (MODE == GATED ? 8 : 4));
    uint32_t warps = (vectors + wanted * 32 - 1) / (wanted * 32);
    if (warps == 2 && vectors <= wanted * 40) warps = 1;      // a little more than a warp's share: rows of one warp come eight a block (8000 x 516 BF16: 6.1 us, 8.9)
    if (warps > 16) warps = 16;
    a.warps = warps;
    const uint32_t groups = warps == 1 ? 8 : 1;
    const uint32_t vector_bytes = VEC * sizeof(H), most_held = ROW_SMEM / groups / vector_bytes;
    a.held = vectors < most_held ? vectors : most_held;
    a.row_bytes = (a.held * vector_bytes + 15) & ~15u;      // within ROW_SMEM / groups, a multiple of 16 and of every vector_bytes
    const uint64_t blocks = (a.rows + groups - 1) / groups, cap = 1u << 30;
    rb::launch_behind(ctx, quant_rows_kernel<T, TW, MODE, VEC, UNROLL>, blocks < cap ? blocks : cap, groups * warps * 32, a.row_bytes * groups, 0, true, a);
    return rb::after_launch(ctx, what);
}

template <typename T>
int32_t launch_shifted(rb_ctx* ctx, const QuantArgs& a, const char* what) {
    static rb::OncePerDevice once;
    const cudaError_t configured = once.run(ctx, [](int&) { return cudaFuncSetAttribute(quant_shifted_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, ROW_SMEM); });
    if (configured != cudaSuccess) return rb::fail(RB_STATUS, "%s: cudaFuncSetAttribute failed with CUDA status %d (%s)", what, (int)configured, cudaGetErrorString(configured));
    const uint32_t wanted = SHIFTED_VECTORS, vectors = a.width / (16 / sizeof(T)) + 1;
    uint32_t warps = (vectors + wanted * 32 - 1) / (wanted * 32);
    if (warps > 16) warps = 16;
    const uint64_t cap = 1u << 30;
    rb::launch_behind(ctx, quant_shifted_kernel<T>, a.rows < cap ? a.rows : cap, warps * 32, (a.width * sizeof(T) + 32 + 15) & ~15u, 0, true, a);
    return rb::after_launch(ctx, what);
}

// The widest vectors on which every row of every operand starts: 16 bytes, 8 bytes, or single elements.  Plain rows that do not start on 16
// bytes are read as shifted ones, unless they are short (us shifted / 8 bytes or single ones: 8000 x 5004 BF16 26 / 34, 8000 x 301 8.7 / 5.5).
template <typename T, typename TW, int MODE>
int32_t dispatch(rb_ctx* ctx, const QuantArgs& a, const char* what) {
    constexpr int FULL = 16 / sizeof(T), HALF = FULL / 2;
    auto fits = [&](int vec) {
        auto on = [](const void* p, uint64_t ld, size_t es, size_t bytes) { return p == nullptr || ((uintptr_t)p % bytes == 0 && ld * es % bytes == 0); };
        const size_t b = vec * sizeof(T), wb = vec * sizeof(TW) > 16 ? 16 : vec * sizeof(TW);
        return a.width % vec == 0 && on(a.x, a.ldx, sizeof(T), b) && on(a.other, a.ldo, sizeof(T), b) && on(a.w, 0, sizeof(TW), wb) &&
               on(a.x_out, a.width, sizeof(T), b) && on(a.q, a.width, 1, vec);
    };
    if (fits(FULL)) return launch<T, TW, MODE, FULL, MODE == ADD_NORM ? 2 : 4>(ctx, a, what);
    if (MODE == PLAIN && a.width >= 700 && a.width * sizeof(T) + 48 <= ROW_SMEM) return launch_shifted<T>(ctx, a, what);
    if (fits(HALF)) return launch<T, TW, MODE, HALF, 4>(ctx, a, what);
    return launch<T, TW, MODE, 1, 4>(ctx, a, what);
}

// Division by a number that is known on the host: n / d = (umulhi(n, m) + n) / 2^s for d < 2^31, with m = floor(2^32 (2^s - d) / d) + 1
// and s = ceil(log2 d) (Granlund and Montgomery, 1994), the sum taken in 33 bits by halving.
struct Divisor { uint32_t d, m, s; };
__host__ Divisor divisor(uint32_t d) {
    uint32_t s = 0;
    while ((uint64_t(1) << s) < d) ++s;
    return {d, (uint32_t)(((uint64_t(1) << 32) * ((uint64_t(1) << s) - d)) / d + 1), s};
}
__device__ __forceinline__ uint32_t divide(uint32_t n, const Divisor& v) {
    const uint32_t t = __umulhi(n, v.m);
    return v.s == 0 ? n : (t + ((n - t) >> 1)) >> (v.s - 1);
}
__device__ __forceinline__ uint64_t divide(uint64_t n, const Divisor& v) { return n / v.d; }

// y = q * scale on flat vectors of 16 bytes of y (q and y are contiguous, so they stay aligned whatever the width); the row of a
// vector's first element comes from one division, a row's end inside the vector steps to the next scale.
// A vector that is read once: first to leave the caches.
template <typename P> __device__ __forceinline__ P streamed(const P* at) {
    P p;
    if constexpr (sizeof(P) == 8) { const uint2 t = __ldcs(reinterpret_cast<const uint2*>(at)); memcpy(&p, &t, 8); }
    else { const uint32_t t = __ldcs(reinterpret_cast<const uint32_t*>(at)); memcpy(&p, &t, 4); }
    return p;
}

// 8192 x 4096 to BF16: 16.9 us = 6.0 TB/s.
template <typename T, typename Index>
__global__ void __launch_bounds__(256, 8) dequant_kernel(const int8_t* q, const float* scales, T* y, uint64_t total, uint32_t width, const Divisor by_width) {
    constexpr int PER = 16 / sizeof(T), UNROLL = 32 / PER;         // 32 elements a thread
    typedef Pack<int8_t, PER> Bytes;
    const Index vectors = (Index)(total / PER), base = (Index)blockIdx.x * 256 * UNROLL + threadIdx.x;
    Bytes b[UNROLL];
    float scale[UNROLL];
    rb::predecessor_done();
    // every load in front of the stores, which they may not pass
    if (base + (UNROLL - 1) * 256 < vectors) {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) b[u] = streamed(reinterpret_cast<const Bytes*>(q) + base + u * 256);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) scale[u] = scales[divide((base + u * 256) * PER, by_width)];
    } else {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) if (base + u * 256 < vectors) { b[u] = streamed(reinterpret_cast<const Bytes*>(q) + base + u * 256); scale[u] = scales[divide((base + u * 256) * PER, by_width)]; }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const Index v = base + u * 256;
        if (v >= vectors) break;
        const Index row = divide(v * PER, by_width);
        uint32_t col = (uint32_t)(v * PER - row * (Index)width);
        const float s = scale[u];
        float f[PER], by[PER];
        uint32_t word[PER / 4];
        memcpy(word, &b[u], PER);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            // byte + 128 as the low bits of 2^23, so that the difference is the signed byte, exactly
            f[j] = __uint_as_float(__byte_perm(word[j / 4] ^ 0x80808080u, 0x4b000000u, 0x7650 | (j % 4)));
            by[j] = s;
        }
        if (col + PER > width) {
            Index r = row;
#pragma unroll
            for (int j = 1; j < PER; ++j) { if (++col == width) { col = 0; ++r; } by[j] = scales[r]; }
        }
#pragma unroll
        for (int j = 0; j < PER; j += 2) add2(f[j], f[j + 1], -8388736.0f, -8388736.0f);
        times<PER>(f, by);
        const Pack<T, PER> o = narrow<T, PER>(f);
        uint4 t; memcpy(&t, &o, 16);
        __stcs(reinterpret_cast<uint4*>(y) + v, t);
    }
    const uint64_t tail = (uint64_t)vectors * PER + threadIdx.x;
    if (blockIdx.x == 0 && threadIdx.x < PER && tail < total) y[tail] = from_f32<T>(__fmul_rn((float)q[tail], scales[tail / width]));
}

template <typename T>
void launch_dequant(rb_ctx* ctx, const int8_t* q, const float* scales, void* y, uint64_t total, uint32_t width) {
    const uint64_t blocks = (total + 8191) / 8192;
    const unsigned grid = (unsigned)(blocks ? blocks : 1);
    if (total <= 0xf0000000ull) rb::launch_behind(ctx, dequant_kernel<T, uint32_t>, grid, 256, 0, 0, true, q, scales, (T*)y, total, width, divisor(width));
    else rb::launch_behind(ctx, dequant_kernel<T, uint64_t>, grid, 256, 0, 0, true, q, scales, (T*)y, total, width, divisor(width));
}

bool is_float(uint32_t dtype) { return dtype == RB_F32 || dtype == RB_BF16 || dtype == RB_F16; }

// q (I8, the input's shape) and scales (FP32, one value per row) of a call.
int32_t check_result(rb_ctx* ctx, const rb_tensor* shape_of, uint64_t rows, const rb_tensor* q, const rb_tensor* scales, const char* what, void** pq, void** ps) {
    RB_TRY(rb::resolve(ctx, q, what, pq)); RB_TRY(rb::resolve(ctx, scales, what, ps));
    if (q->dtype != RB_I8 || !rb::same_shape(q, shape_of)) return rb::fail(RB_INVALID_TENSOR, "%s: the quantised tensor must be I8 of the input's shape", what);
    if (scales->dtype != RB_F32 || rb::elements(scales) != rows) return rb::fail(RB_INVALID_TENSOR, "%s: scales must be FP32 with one value per row", what);
    return RB_OK;
}

}  // namespace

using namespace rb;

extern "C" {

int32_t rb_rms_norm_quant(rb_ctx* ctx, const rb_tensor* x, const rb_tensor* delta, const rb_tensor* weight, double epsilon,
                          const rb_tensor* x_out, const rb_tensor* q, const rb_tensor* scales) {
    const char* what = "8-bit RMSNorm";
    RB_TRY(check_ctx(ctx));
    void *px, *pd, *pw, *pxo, *pq, *ps;
    RB_TRY(resolve(ctx, x, what, &px)); RB_TRY(resolve(ctx, delta, what, &pd, true)); RB_TRY(resolve(ctx, weight, what, &pw)); RB_TRY(resolve(ctx, x_out, what, &pxo, true));
    const float eps = (float)epsilon;
    if (!(eps > 0.0f) || !(eps <= 3.402823466e38f)) return fail(RB_INVALID_TENSOR, "RMSNorm epsilon must be positive and representable in FP32");
    uint64_t rows, width; rows_width(x, &rows, &width);
    if (width == 0 || width > 0x7fffffffull) return fail(RB_INVALID_TENSOR, "%s requires a positive last dimension within INT32_MAX", what);
    if (!is_float(x->dtype) || (weight->dtype != x->dtype && weight->dtype != RB_F32)) return fail(RB_INVALID_TENSOR, "%s: x must be F32, BF16 or F16 and the weight of x's type or F32", what);
    if (elements(weight) != width) return fail(RB_INVALID_TENSOR, "%s: the weight must hold one value per column", what);
    if ((delta == nullptr) != (x_out == nullptr)) return fail(RB_INVALID_TENSOR, "%s: delta and x_out come together", what);
    if (delta && (!same_shape(x, delta) || !same_shape(x, x_out) || delta->dtype != x->dtype || x_out->dtype != x->dtype))
        return fail(RB_INVALID_TENSOR, "%s: delta and x_out must have x's shape and type", what);
    RB_TRY(check_result(ctx, x, rows, q, scales, what, &pq, &ps));
    const uint64_t n = rows * width, xb = n * dtype_size(x->dtype), wb = width * dtype_size(weight->dtype), sb = rows * 4;
    struct Span { const void* p; uint64_t bytes; };
    const Span in[] = {{px, xb}, {pd, pd ? xb : 0}, {pw, wb}}, out[] = {{pxo, pxo ? xb : 0}, {pq, n}, {ps, sb}};
    for (int i = 0; i < 3; ++i) {
        for (int j = 0; j < 3; ++j) if (!(i == 0 && j == 0 && pxo == px)) RB_TRY(no_overlap(out[i].p, out[i].bytes, in[j].p, in[j].bytes, what));   // x_out may be x itself
        for (int j = 0; j < i; ++j) RB_TRY(no_overlap(out[i].p, out[i].bytes, out[j].p, out[j].bytes, what));
    }
    if (rows == 0) return empty_call(ctx);
    DeviceGuard device(ctx);
    QuantArgs a{px, width, pd, width, pw, pxo, (int8_t*)pq, (float*)ps, rows, (uint32_t)width, 0, 0, 0, eps};
#define RB_NORM(T, TW) return delta ? dispatch<T, TW, ADD_NORM>(ctx, a, what) : dispatch<T, TW, NORM>(ctx, a, what)
    if (x->dtype == RB_F32) RB_NORM(float, float);
    if (x->dtype == RB_BF16 && weight->dtype == RB_BF16) RB_NORM(bf, bf);
    if (x->dtype == RB_BF16) RB_NORM(bf, float);
    if (weight->dtype == RB_F16) RB_NORM(__half, __half);
    RB_NORM(__half, float);
#undef RB_NORM
}

int32_t rb_quantize_rows(rb_ctx* ctx, const rb_tensor* x, const rb_tensor* up, const rb_tensor* q, const rb_tensor* scales) {
    const char* what = "row quantisation";
    RB_TRY(check_ctx(ctx));
    Rows rx, ru; void *pq, *ps;
    RB_TRY(resolve_rows(ctx, x, what, &rx));
    if (!is_float(x->dtype)) return fail(RB_INVALID_TENSOR, "%s: x must be F32, BF16 or F16", what);
    if (rx.width == 0 || rx.width > 0x7fffffffull) return fail(RB_INVALID_TENSOR, "%s requires a positive last dimension within INT32_MAX", what);
    if (up) {
        RB_TRY(resolve_rows(ctx, up, what, &ru));
        if (!same_shape(x, up) || up->dtype != x->dtype) return fail(RB_INVALID_TENSOR, "%s: gate and up must have one shape and type", what);
    }
    RB_TRY(check_result(ctx, x, rx.rows, q, scales, what, &pq, &ps));
    const uint64_t n = rx.rows * rx.width, sb = rx.rows * 4;
    RB_TRY(no_overlap(pq, n, rx.ptr, rx.extent_bytes, what)); RB_TRY(no_overlap(ps, sb, rx.ptr, rx.extent_bytes, what)); RB_TRY(no_overlap(ps, sb, pq, n, what));
    if (up) { RB_TRY(no_overlap(pq, n, ru.ptr, ru.extent_bytes, what)); RB_TRY(no_overlap(ps, sb, ru.ptr, ru.extent_bytes, what)); }
    if (rx.rows == 0) return empty_call(ctx);
    DeviceGuard device(ctx);
    QuantArgs a{rx.ptr, rx.ld, ru.ptr, ru.ld, nullptr, nullptr, (int8_t*)pq, (float*)ps, rx.rows, (uint32_t)rx.width, 0, 0, 0, 0.f};
    if (x->dtype == RB_F32) return up ? dispatch<float, float, GATED>(ctx, a, what) : dispatch<float, float, PLAIN>(ctx, a, what);
    if (x->dtype == RB_BF16) return up ? dispatch<bf, bf, GATED>(ctx, a, what) : dispatch<bf, bf, PLAIN>(ctx, a, what);
    return up ? dispatch<__half, __half, GATED>(ctx, a, what) : dispatch<__half, __half, PLAIN>(ctx, a, what);
}

int32_t rb_dequantize_rows(rb_ctx* ctx, const rb_tensor* q, const rb_tensor* scales, const rb_tensor* y) {
    const char* what = "row dequantisation";
    RB_TRY(check_ctx(ctx));
    void *pq, *ps, *py;
    RB_TRY(resolve(ctx, y, what, &py));
    uint64_t rows, width; rows_width(y, &rows, &width);
    if (!is_float(y->dtype)) return fail(RB_INVALID_TENSOR, "%s: y must be F32, BF16 or F16", what);
    if (width == 0 || width > 0x7fffffffull) return fail(RB_INVALID_TENSOR, "%s requires a positive last dimension within INT32_MAX", what);
    RB_TRY(check_result(ctx, y, rows, q, scales, what, &pq, &ps));
    const uint64_t n = rows * width, yb = n * dtype_size(y->dtype);
    if (n / 8192 > 0x7ffffff0ull) return fail(RB_INVALID_TENSOR, "%s: too many values for one launch", what);
    RB_TRY(no_overlap(py, yb, pq, n, what)); RB_TRY(no_overlap(py, yb, ps, rows * 4, what));
    if (rows == 0) return empty_call(ctx);
    DeviceGuard device(ctx);
    if (y->dtype == RB_F32) launch_dequant<float>(ctx, (const int8_t*)pq, (const float*)ps, py, n, (uint32_t)width);
    else if (y->dtype == RB_BF16) launch_dequant<bf>(ctx, (const int8_t*)pq, (const float*)ps, py, n, (uint32_t)width);
    else launch_dequant<__half>(ctx, (const int8_t*)pq, (const float*)ps, py, n, (uint32_t)width);
    return after_launch(ctx, what);
}

}  // extern "C"
