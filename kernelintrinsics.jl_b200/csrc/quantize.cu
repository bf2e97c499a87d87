// quantize.cu -- ki_quantize_rows: rows of Float32 / Float16 / BFloat16 to int8 with one scale per row.
//
//   scale[r] = max_c |x[r, c]| * (1 / 127),   q[r, c] = rint(x[r, c] / scale[r]), ties to even, in [-127, 127]
//
// The product (with 1 / 127 as a Float32) and the quotient are IEEE Float32, so the int8 values are
// defined bit for bit.  A row of zeros (or one
// whose scale underflows to zero) gives zeros; a NaN or an infinity makes the row's scale NaN or
// infinite and q zero where x / scale is NaN or zero, so that a product with the row shows NaN.
//
// Bound: HBM (one read of x, one write of q): 8192 x 4096 bf16 18.0 us, 5.6 TB/s.  The maximum is taken over the bit patterns of |x| as unsigned integers
// (two 16-bit elements at once): their order is the order of the values, with NaN above infinity, so a NaN is kept.
// Division of every element would cost more instructions than the row's bytes allow, so q is read off
// x * (1 / scale) + 1.5 * 2^23, whose last bits are the product rounded to an integer.  That product is within 8e-6 of the
// quotient, and the quotient's own rounding is 4e-6 at most (|q| <= 127.5), so only where it lies within 3e-5 of a
// half-way point could the two round apart; there, and for scales that are zero, subnormal or not finite, the
// division is done.
//
// A row stays in registers between the two passes: TPR threads hold VPT vectors each.  Rows longer
// than that are read twice (the second time from L2).
#include <type_traits>

#include "ki/layer.cuh"

namespace {

// Threads per block: one row, or four rows of one warp each (a row that shares its barrier with another row's threads
// waits for them: 8192 x 4096 bf16 23.4 us with 256 threads per row, 21.4 with two rows of 128, 18.2 with one).
constexpr int block_threads(int tpr) { return tpr > 32 ? tpr : 128; }

__device__ __forceinline__ int8_t divided(float x, float scale) {
    if (scale == 0.0f) return 0;
    return (int8_t)min(max(__float2int_rn(__fdiv_rn(x, scale)), -127), 127);  // NaN: 0
}

// The larger of m and |x| in either half; NaN stays.
template <class T>
__device__ __forceinline__ uint32_t max_abs2(uint32_t m, uint32_t x) {
    uint32_t r;
    if constexpr (std::is_same<T, __half>::value)
        asm("{\n\t.reg .b32 a;\n\tabs.f16x2 a, %2;\n\tmax.NaN.f16x2 %0, %1, a;\n\t}" : "=r"(r) : "r"(m), "r"(x));
    else
        asm("{\n\t.reg .b32 a;\n\tabs.bf16x2 a, %2;\n\tmax.NaN.bf16x2 %0, %1, a;\n\t}" : "=r"(r) : "r"(m), "r"(x));
    return r;
}

// The largest |x| so far and of a vector, as bits: of a Float32, or of two 16-bit elements in either half.
template <class T, int EV>
__device__ __forceinline__ uint32_t abs_bits(const ki::Vec<T, EV>& v, uint32_t m) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int e = 0; e < EV; ++e) m = max(m, __float_as_uint(v.e[e]) & 0x7fffffffu);
    } else if constexpr (EV == 1) {
        m = max(m, (uint32_t)(*reinterpret_cast<const uint16_t*>(&v) & 0x7fffu));
    } else {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
        for (int e = 0; e < EV / 2; ++e) m = max_abs2<T>(m, w[e]);
    }
    return m;
}
// Their value as Float32 bits, whose order is the same.
template <class T, int EV>
__device__ __forceinline__ uint32_t top_bits(uint32_t m) {
    if constexpr (sizeof(T) == 4) return m;
    const uint16_t h = (uint16_t)max(m & 0xffffu, m >> 16);
    return __float_as_uint(ki::to_f32(*reinterpret_cast<const T*>(&h)));
}

template <class T, int EV>
__device__ __forceinline__ ki::Vec<int8_t, EV> quantized(const ki::Vec<T, EV>& x, float scale, float inv, bool plain) {
    ki::Vec<int8_t, EV> q;
    float far = 1.0f;  // the largest distance from an integer
    if (plain) {
        constexpr int P = (EV + 1) / 2, one = EV > 1 ? 1 : 0;
        const ki::f32x2 i = ki::pair(inv), magic = ki::pair(12582912.0f), minus = ki::pair(-12582912.0f);
        uint32_t t[2 * P];
        far = 0.0f;
#pragma unroll
        for (int e = 0; e < P; ++e) {
            const ki::f32x2 v = ki::pair(ki::to_f32(x.e[2 * e]), ki::to_f32(x.e[2 * e + one]));
            const ki::f32x2 r = ki::fma2(v, i, magic);
            float a, b;
            ki::unpair(a, b, r);
            t[2 * e] = __float_as_uint(a), t[2 * e + 1] = __float_as_uint(b);
            ki::unpair(a, b, ki::add2(r, minus));
            ki::unpair(a, b, ki::fma2(v, i, ki::pair(-a, -b)));
            far = fmaxf(far, fmaxf(fabsf(a), fabsf(b)));
        }
#pragma unroll
        for (int e = 0; e < EV; ++e) q.e[e] = (int8_t)t[e];
    }
    if (far > 0.5f - 3e-5f) {
#pragma unroll
        for (int e = 0; e < EV; ++e) q.e[e] = divided(ki::to_f32(x.e[e]), scale);
    }
    return q;
}

// One row per group of TPR threads; EV elements per access.
template <class T, int EV, int VPT, int TPR>
__global__ void __launch_bounds__(block_threads(TPR))
    quantize_kernel(const T* __restrict__ x, size_t rows, size_t cols, size_t ld, int8_t* __restrict__ q, size_t ldq,
                    float* __restrict__ scale, bool q_aligned) {
    constexpr int kBlock = block_threads(TPR);
    constexpr int kRows = kBlock / TPR;
    constexpr int kRowWarps = TPR / 32;
    using V = ki::Vec<T, EV>;
    __shared__ uint32_t part[kBlock / 32];
    const int t = threadIdx.x % TPR;
    const size_t r = (size_t)blockIdx.x * kRows + threadIdx.x / TPR;
    const bool live = r < rows;
    const int nvec = (int)(cols / EV);
    const T* row = x + (live ? r : 0) * ld;
    const bool fits = nvec <= VPT * TPR;

    V v[VPT];
    uint32_t m = 0;
    if (live) {
        if (fits) {
#pragma unroll
            for (int i = 0; i < VPT; ++i)
                if (i * TPR + t < nvec) v[i] = ki::load_vec<T, EV>(row + (size_t)(i * TPR + t) * EV);
#pragma unroll
            for (int i = 0; i < VPT; ++i)
                if (i * TPR + t < nvec) m = abs_bits<T, EV>(v[i], m);
        } else {
#pragma unroll 4
            for (int i = t; i < nvec; i += TPR) m = abs_bits<T, EV>(ki::load_vec<T, EV>(row + (size_t)i * EV), m);
        }
        m = top_bits<T, EV>(m);
        for (size_t c = (size_t)nvec * EV + t; c < cols; c += TPR) m = max(m, __float_as_uint(ki::to_f32(row[c])) & 0x7fffffffu);
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (TPR > 32) {
        const int w = threadIdx.x >> 5;
        if ((threadIdx.x & 31) == 0) part[w] = m;
        __syncthreads();
        const int w0 = (threadIdx.x / TPR) * kRowWarps;
#pragma unroll
        for (int i = 0; i < kRowWarps; ++i) m = max(m, part[w0 + i]);
    }
    if (!live) return;
    const float s = __uint_as_float(m) * (1.0f / 127.0f);
    const bool plain = s >= 1.17549435e-38f && s < __uint_as_float(0x7f800000u);  // normal and finite, so 1 / s is too
    const float inv = __fdiv_rn(1.0f, s);
    if (t == 0) scale[r] = s;
    int8_t* out = q + r * ldq;
    auto put = [&](int i, const V& a) {
        const ki::Vec<int8_t, EV> b = quantized<T, EV>(a, s, inv, plain);
        if (q_aligned) {
            ki::store_vec<int8_t, EV>(out + (size_t)i * EV, b);
        } else {
#pragma unroll
            for (int e = 0; e < EV; ++e) out[(size_t)i * EV + e] = b.e[e];
        }
    };
    if (fits) {
#pragma unroll
        for (int i = 0; i < VPT; ++i)
            if (i * TPR + t < nvec) put(i * TPR + t, v[i]);
    } else {
        for (int i = t; i < nvec; i += TPR) put(i, ki::load_vec<T, EV>(row + (size_t)i * EV));
    }
    for (size_t c = (size_t)nvec * EV + t; c < cols; c += TPR) out[c] = divided(ki::to_f32(row[c]), s);
}

struct QuantArgs {
    const void* x;
    size_t rows, cols, ld;
    int8_t* q;
    size_t ldq;
    float* scale;
    cudaStream_t s;
};

template <class T, int EV, int VPT, int TPR>
int launch(ki_ctx* ctx, const QuantArgs& a) {
    constexpr int kBlock = block_threads(TPR);
    const size_t per = kBlock / TPR;
    const size_t blocks = (a.rows + per - 1) / per;
    if (blocks > 0x7fffffffu) return ki::set_error(ctx, KI_ERR_ARG, "quantize_rows: too many rows");
    quantize_kernel<T, EV, VPT, TPR><<<(unsigned)blocks, kBlock, 0, a.s>>>(
        static_cast<const T*>(a.x), a.rows, a.cols, a.ld, a.q, a.ldq, a.scale, ki::rows_aligned(a.q, a.ldq, 1, EV));
    return ki::check_launch(ctx, "quantize_kernel launch");
}

template <class T, int EV>
int launch_any(ki_ctx* ctx, const QuantArgs& a) {
    const size_t nvec = a.cols / EV;
    if (nvec <= 32) return launch<T, EV, 1, 32>(ctx, a);
    if (nvec <= 128) return launch<T, EV, 4, 32>(ctx, a);
    if (nvec <= 256) return launch<T, EV, 4, 64>(ctx, a);
    if (nvec <= 512) return launch<T, EV, 4, 128>(ctx, a);
    if (nvec <= 1024) return launch<T, EV, 4, 256>(ctx, a);
    if (nvec <= 2048) return launch<T, EV, 4, 512>(ctx, a);
    return launch<T, EV, 8, 512>(ctx, a);
}

}  // namespace

extern "C" int ki_quantize_rows(ki_ctx* ctx, int dtype, const void* d_x, size_t rows, size_t cols, size_t ld, int8_t* d_q,
                                size_t ldq, float* d_scale, void* stream) {
    KI_CHECK_CTX(ctx);
    const size_t es = ki::float_size(dtype);
    if (!es) return ki::set_error(ctx, KI_ERR_ARG, "quantize_rows: dtype must be KI_F32, KI_F16 or KI_BF16");
    if (rows == 0) return KI_OK;
    if (!d_scale || (cols > 0 && (!d_x || !d_q))) return ki::set_error(ctx, KI_ERR_ARG, "quantize_rows: null pointer");
    // an int index may pass a row's end by four strides of 512 threads
    if (cols > 0x7ffff000u) return ki::set_error(ctx, KI_ERR_ARG, "quantize_rows: too many columns");
    if (rows > 1 && (ld < cols || ldq < cols))
        return ki::set_error(ctx, KI_ERR_ARG, "quantize_rows: leading dimension smaller than cols");
    if (!ki::aligned(d_x, es) || !ki::aligned(d_scale, 4))
        return ki::set_error(ctx, KI_ERR_ARG, "quantize_rows: pointer not aligned to its element");
    const ki::Span x = ki::span(d_x, rows, ld, cols, es), q = ki::span(d_q, rows, ldq, cols, 1),
                   sc = ki::span(d_scale, rows, 1, 1, 4);
    if (ki::overlap(x, q) || ki::overlap(x, sc) || ki::overlap(q, sc))
        return ki::set_error(ctx, KI_ERR_ARG, "quantize_rows: ranges overlap");
    KI_GUARD(ctx);
    const QuantArgs a{d_x, rows, cols, ld, d_q, ldq, d_scale, ki::as_stream(stream)};
    return ki::with_float_type(dtype, [&](auto t) {
        using T = decltype(t);
        // 16-byte accesses where every row starts on one, else element by element
        if (ki::aligned(d_x, 16) && (rows == 1 || (ld * es) % 16 == 0)) return launch_any<T, 16 / (int)sizeof(T)>(ctx, a);
        return launch_any<T, 1>(ctx, a);
    });
}
