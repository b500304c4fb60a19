// Rows held in 8 bits: RMSNorm (with the residual's addition) and row quantisation (plain, or behind SiLU * up) with an I8 result
// and one FP32 scale a row, and the way back.
//
// scale = max(max|y| / 127, 2^-126), q = rint(y / scale).  For the norm y = s r w with one r = 1/sqrt(mean(s^2) + eps) for the
// whole row, so max|y| = r max|s w| and y / scale = (s w) (127 / max|s w|): the quantised values do not need r at all, and one
// reduction (the sum of squares beside the maximum) is enough where a norm followed by a quantisation has two.
//
// These kernels are HBM-bound.  One group of warps owns a row and keeps it in registers between the reduction and the store
// (ITEMS vectors a thread); what a group cannot hold is read again, which hits L2.
#include "common.cuh"

namespace {

using bf = __nv_bfloat16;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ bf from_f32<bf>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// BYTES-wide loads and stores of VEC elements; VEC * sizeof(T) is 1, 2, 4, 8, 16 or 32 bytes and the address is aligned to
// min(that, 16).
template <typename T, int VEC> struct __align__(VEC * sizeof(T) > 16 ? 16 : VEC * sizeof(T)) Pack { T v[VEC]; };

template <typename T, int VEC>
__device__ __forceinline__ void load(const T* p, float (&v)[VEC]) {
    const Pack<T, VEC> t = *reinterpret_cast<const Pack<T, VEC>*>(p);
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = to_f32(t.v[j]);
}
template <typename T, int VEC>
__device__ __forceinline__ void store(T* p, const float (&v)[VEC]) {
    Pack<T, VEC> t;
#pragma unroll
    for (int j = 0; j < VEC; ++j) t.v[j] = from_f32<T>(v[j]);
    *reinterpret_cast<Pack<T, VEC>*>(p) = t;
}
// rint(v * c) as bytes: adding 1.5 * 2^23 leaves the integer in the low bits of the sum, rounded once (|v * c| <= 128).
template <int VEC>
__device__ __forceinline__ void store_i8(int8_t* p, const float (&v)[VEC], float c, bool bad) {
    Pack<int8_t, VEC> t;
#pragma unroll
    for (int j = 0; j < VEC; ++j) t.v[j] = bad ? (int8_t)0 : (int8_t)__float_as_uint(__fmaf_rn(v[j], c, 12582912.0f));
    *reinterpret_cast<Pack<int8_t, VEC>*>(p) = t;
}

enum Mode { PLAIN = 0, GATED = 1, NORM = 2, ADD_NORM = 3 };

struct QuantArgs {
    const void* x; uint64_t ldx;
    const void* other; uint64_t ldo;     // GATED: up; ADD_NORM: delta
    const void* w; void* x_out; int8_t* q; float* scales;
    uint64_t rows; uint32_t width; uint32_t warps;   // warps that share a row
    float eps;
};

// SiLU with one exponential and one reciprocal: x / (1 + exp(-x)).  For x below -88 the exponential overflows and the quotient is
// the -0 that the limit has; an infinite or NaN x gives NaN or infinity, which marks the row.
__device__ __forceinline__ float silu(float x) { return __fdividef(x, 1.0f + __expf(-x)); }

// Folds one vector into the two row statistics and leaves in v what the quantisation multiplies by one factor: y itself, or s * w.
template <int MODE, int VEC>
__device__ __forceinline__ void fold(float (&v)[VEC], const float (&w)[VEC], float& sum, uint32_t& most) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        if (MODE == NORM || MODE == ADD_NORM) { sum = __fmaf_rn(v[j], v[j], sum); v[j] = __fmul_rn(v[j], w[j]); }
        // magnitudes compare as integers, and in that order NaN lies above infinity, so neither is lost
        const uint32_t bits = __float_as_uint(v[j]) & 0x7fffffffu;
        most = most > bits ? most : bits;
    }
}

// `warps` whole warps share a row; a block holds blockDim.x / (32 warps) rows at a time, each with its own named
// barrier, so rows of one block do not wait for each other.
template <typename T, typename TW, int MODE, int VEC, int ITEMS>
__global__ void __launch_bounds__(1024) quant_rows_kernel(const QuantArgs a) {
    __shared__ float s_sum[32];
    __shared__ uint32_t s_most[32];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t group = warp / a.warps, groups = (blockDim.x >> 5) / a.warps, first_warp = group * a.warps;
    const uint32_t threads = a.warps * 32, tid = threadIdx.x - first_warp * 32;
    const uint32_t vectors = a.width / VEC;            // VEC divides the width
    constexpr bool NORMS = MODE == NORM || MODE == ADD_NORM;
    const T* other = static_cast<const T*>(a.other);
    const TW* weight = static_cast<const TW*>(a.w);
    for (uint64_t row = (uint64_t)blockIdx.x * groups + group; row < a.rows; row += (uint64_t)gridDim.x * groups) {
        const T* x = static_cast<const T*>(a.x) + row * a.ldx;
        const T* o = other + row * a.ldo;
        T* xo = static_cast<T*>(a.x_out) + row * a.width;
        float v[ITEMS][VEC];
        float sum = 0.f;
        uint32_t most = 0;
        // y, or s * w, of vector i; the sum of a residual is stored the first time it is formed and read back after that
        auto fetch = [&](uint32_t i, float (&y)[VEC], float& acc, uint32_t& top, bool again) {
            float second[VEC];
            if (MODE == ADD_NORM && again) load<T, VEC>(xo + (size_t)i * VEC, y);
            else load<T, VEC>(x + (size_t)i * VEC, y);
            if (MODE == GATED || (MODE == ADD_NORM && !again)) load<T, VEC>(o + (size_t)i * VEC, second);
            float w[VEC];
            if (NORMS) load<TW, VEC>(weight + (size_t)i * VEC, w);
            if (MODE == GATED) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) y[j] = __fmul_rn(silu(y[j]), second[j]);
            }
            if (MODE == ADD_NORM && !again) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) y[j] = to_f32(from_f32<T>(__fadd_rn(y[j], second[j])));
                store<T, VEC>(xo + (size_t)i * VEC, y);
            }
            fold<MODE, VEC>(y, w, acc, top);
        };
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            const uint32_t i = k * threads + tid;
            if (i < vectors) fetch(i, v[k], sum, most, false);
        }
        for (uint32_t i = ITEMS * threads + tid; i < vectors; i += threads) { float y[VEC]; fetch(i, y, sum, most, false); }

        most = __reduce_max_sync(0xffffffffu, most);
        if (NORMS) {
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        }
        if (a.warps > 1) {
            // a row's partial results: written, read after the first barrier, and not overwritten before the second
            if (lane == 0) { s_sum[warp] = sum; s_most[warp] = most; }
            asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(threads) : "memory");
            const uint32_t from = first_warp + (lane < a.warps ? lane : 0);
            most = __reduce_max_sync(0xffffffffu, s_most[from]);
            if (NORMS) {
                sum = lane < a.warps ? s_sum[from] : 0.f;
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            }
            asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(threads) : "memory");
        }
        const bool bad = most >= 0x7f800000u || (NORMS && sum != sum);
        const float a_max = __uint_as_float(most);
        const float r = NORMS ? __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(sum, (float)a.width), a.eps))) : 1.0f;
        const float wanted = __fdiv_rn(__fmul_rn(r, a_max), 127.0f);
        const float least = 1.17549435e-38f;           // 2^-126
        const bool tiny = wanted < least;
        // The factor of a very small row would leave FP32's range: there the values are raised by 2^96 (exactly) first.
        const bool small = a_max < 1e-30f;
        const float c = tiny ? __fmul_rn(r, small ? 1073741824.0f : 8.5070592e37f)                    // r / 2^-126, over 2^96 where raised
                             : __fdiv_rn(127.0f, small ? __fmul_rn(a_max, 7.9228163e28f) : a_max);
        auto raise = [&](float (&y)[VEC]) {
            if (!small) return;
#pragma unroll
            for (int j = 0; j < VEC; ++j) y[j] = __fmul_rn(y[j], 7.9228163e28f);
        };
        if (tid == 0) a.scales[row] = bad ? __int_as_float(0x7fc00000) : (tiny ? least : wanted);
        int8_t* q = a.q + row * a.width;
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            const uint32_t i = k * threads + tid;
            if (i < vectors) { raise(v[k]); store_i8<VEC>(q + (size_t)i * VEC, v[k], c, bad); }
        }
        for (uint32_t i = ITEMS * threads + tid; i < vectors; i += threads) {
            float y[VEC], unused = 0.f; uint32_t none = 0;
            fetch(i, y, unused, none, true);
            raise(y);
            store_i8<VEC>(q + (size_t)i * VEC, y, c, bad);
        }
    }
}

template <typename T, typename TW, int MODE, int VEC, int ITEMS>
int32_t launch(rb_ctx* ctx, QuantArgs a, const char* what) {
    const uint32_t vectors = a.width / VEC;
    uint32_t warps = (vectors + ITEMS * 32 - 1) / (ITEMS * 32);
    if (warps < 1) warps = 1;
    if (warps > 32) warps = 32;
    a.warps = warps;
    const uint32_t groups = warps >= 8 ? 1 : 8 / warps;            // blocks of about 256 threads for narrow rows; at most 8 groups: barriers 1..8
    const uint64_t blocks = (a.rows + groups - 1) / groups, cap = (uint64_t)ctx->sm_count * 32;
    quant_rows_kernel<T, TW, MODE, VEC, ITEMS><<<(unsigned)(blocks < cap ? blocks : cap), groups * warps * 32, 0, ctx->stream>>>(a);
    return rb::after_launch(ctx, what);
}

// 16-byte vectors where every row of every operand starts on one; single elements otherwise.
template <typename T, typename TW, int MODE>
int32_t dispatch(rb_ctx* ctx, const QuantArgs& a, const char* what) {
    constexpr int VEC = 16 / sizeof(T);
    auto fits = [](const void* p, uint64_t ld, size_t es, size_t bytes) { return p == nullptr || ((uintptr_t)p % bytes == 0 && ld * es % bytes == 0); };
    const bool wide = a.width % VEC == 0 && fits(a.x, a.ldx, sizeof(T), 16) && fits(a.other, a.ldo, sizeof(T), 16) && fits(a.w, 0, sizeof(TW), 16) &&
                      fits(a.x_out, a.width, sizeof(T), 16) && fits(a.q, a.width, 1, VEC);
    if (wide) return launch<T, TW, MODE, VEC, 2>(ctx, a, what);
    return launch<T, TW, MODE, 1, 8>(ctx, a, what);
}

// y = q * scale on flat 16-element vectors (q and y are contiguous, so vectors stay aligned whatever the width); the row of a
// vector's first element comes from one division, a row's end inside the vector steps to the next scale.
template <typename T>
__global__ void __launch_bounds__(256) dequant_kernel(const int8_t* q, const float* scales, T* y, uint64_t total, uint32_t width) {
    const uint64_t vectors = total / 16, stride = (uint64_t)gridDim.x * blockDim.x;
    for (uint64_t v = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; v < vectors; v += stride) {
        const uint64_t at = v * 16;
        uint64_t row = total <= 0xffffffffull ? (uint64_t)((uint32_t)at / width) : at / width;
        uint32_t col = (uint32_t)(at - row * width);
        const uint4 b = __ldcs(reinterpret_cast<const uint4*>(q + at));
        float s = __ldg(scales + row);
        const uint32_t word[4] = {b.x, b.y, b.z, b.w};
        float o[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            // byte + 128 as the low bits of 2^23, so that the difference is the signed byte, exactly
            const float f = __uint_as_float(__byte_perm(word[j / 4] ^ 0x80808080u, 0x4b000000u, 0x7650 | (j % 4))) - 8388736.0f;
            o[j] = __fmul_rn(f, s);
            if (j < 15 && ++col == width) { col = 0; ++row; s = __ldg(scales + row); }
        }
        constexpr int PER = 16 / sizeof(T);
#pragma unroll
        for (int j = 0; j < 16; j += PER) {
            float part[PER];
#pragma unroll
            for (int i = 0; i < PER; ++i) part[i] = o[j + i];
            store<T, PER>(y + at + j, part);
        }
    }
    const uint64_t tail = vectors * 16 + threadIdx.x;
    if (blockIdx.x == 0 && threadIdx.x < 16 && tail < total) y[tail] = from_f32<T>(__fmul_rn((float)q[tail], scales[tail / width]));
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
    QuantArgs a{px, width, pd, width, pw, pxo, (int8_t*)pq, (float*)ps, rows, (uint32_t)width, 0, eps};
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
    QuantArgs a{rx.ptr, rx.ld, ru.ptr, ru.ld, nullptr, nullptr, (int8_t*)pq, (float*)ps, rx.rows, (uint32_t)rx.width, 0, 0.f};
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
    RB_TRY(no_overlap(py, yb, pq, n, what)); RB_TRY(no_overlap(py, yb, ps, rows * 4, what));
    if (rows == 0) return empty_call(ctx);
    DeviceGuard device(ctx);
    const uint64_t blocks = (n / 16 + 255) / 256, cap = (uint64_t)ctx->sm_count * 16;
    const unsigned grid = (unsigned)(blocks < 1 ? 1 : (blocks < cap ? blocks : cap));
    const int8_t* in = (const int8_t*)pq; const float* s = (const float*)ps;
    if (y->dtype == RB_F32) dequant_kernel<float><<<grid, 256, 0, ctx->stream>>>(in, s, (float*)py, n, (uint32_t)width);
    else if (y->dtype == RB_BF16) dequant_kernel<bf><<<grid, 256, 0, ctx->stream>>>(in, s, (bf*)py, n, (uint32_t)width);
    else dequant_kernel<__half><<<grid, 256, 0, ctx->stream>>>(in, s, (__half*)py, n, (uint32_t)width);
    return after_launch(ctx, what);
}

}  // extern "C"
