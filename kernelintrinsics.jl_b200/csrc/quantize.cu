// quantize.cu -- ki_quantize_rows: rows of Float32 / Float16 / BFloat16 to int8 with one scale per row.
//
//   scale[r] = max_c |x[r, c]| * (1 / 127),   q[r, c] = rint(x[r, c] / scale[r]), ties to even, in [-127, 127]
//
// The product (with 1 / 127 as a Float32) and the quotient are IEEE Float32, so the int8 values are
// defined bit for bit.  A row of zeros (or one
// whose scale underflows to zero) gives zeros; a NaN or an infinity makes the row's scale NaN or
// infinite and q zero where x / scale is NaN or zero, so that a product with the row shows NaN.
//
// The maximum is taken over the bit patterns of |x| as unsigned integers: their order is the order of
// the values, with NaN above infinity, so a NaN is kept.  Division of every element would cost more
// instructions than the row's bytes allow, so q comes from x * (1 / scale): that product is within
// 2e-5 of the quotient (|q| <= 127.5, two roundings of 2^-24 each), and only where it lies within 3e-5
// of a half-way point, where the two could round apart, is the division done.
//
// A row stays in registers between the two passes: TPR threads hold VPT vectors each.  Rows longer
// than that are read twice (the second time from L2).
#include "ki/layer.cuh"

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float quantum(float x, float scale, float inv) {
    const float p = x * inv;
    float q = rintf(p);
    if (!(fabsf(0.5f - fabsf(p - q)) >= 3e-5f)) q = rintf(__fdiv_rn(x, scale));  // also where p is not finite
    return q;
}

__device__ __forceinline__ int8_t to_i8(float q) { return (int8_t)min(max(__float2int_rn(q), -127), 127); }  // NaN: 0

template <class T, int EV>
__device__ __forceinline__ uint32_t abs_bits(const ki::Vec<T, EV>& v, uint32_t m) {
#pragma unroll
    for (int e = 0; e < EV; ++e) m = max(m, __float_as_uint(ki::to_f32(v.e[e])) & 0x7fffffffu);
    return m;
}

// One row per group of TPR threads; EV elements per access.
template <class T, int EV, int VPT, int TPR>
__global__ void __launch_bounds__(TPR > kThreads ? TPR : kThreads)
    quantize_kernel(const T* __restrict__ x, size_t rows, size_t cols, size_t ld, int8_t* __restrict__ q, size_t ldq,
                    float* __restrict__ scale, bool q_aligned) {
    constexpr int kBlock = TPR > kThreads ? TPR : kThreads;
    constexpr int kRows = kBlock / TPR;
    constexpr int kRowWarps = TPR / 32;
    using V = ki::Vec<T, EV>;
    __shared__ uint32_t part[kBlock / 32];
    const int t = threadIdx.x % TPR;
    const size_t r = (size_t)blockIdx.x * kRows + threadIdx.x / TPR;
    const bool live = r < rows;
    const size_t nvec = cols / EV;
    const T* row = x + (live ? r : 0) * ld;
    const bool fits = nvec <= (size_t)VPT * TPR;

    V v[VPT];
    uint32_t m = 0;
    if (live) {
        if (fits) {
#pragma unroll
            for (int i = 0; i < VPT; ++i)
                if ((size_t)(i * TPR + t) < nvec) v[i] = ki::load_vec<T, EV>(row + (size_t)(i * TPR + t) * EV);
#pragma unroll
            for (int i = 0; i < VPT; ++i)
                if ((size_t)(i * TPR + t) < nvec) m = abs_bits<T, EV>(v[i], m);
        } else {
            for (size_t i = t; i < nvec; i += TPR) m = abs_bits<T, EV>(ki::load_vec<T, EV>(row + i * EV), m);
        }
        for (size_t c = nvec * EV + t; c < cols; c += TPR) m = max(m, __float_as_uint(ki::to_f32(row[c])) & 0x7fffffffu);
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
    const bool zero = s == 0.0f;
    const float inv = zero ? 0.0f : __fdiv_rn(1.0f, s);
    if (t == 0) scale[r] = s;
    int8_t* out = q + r * ldq;
    auto put = [&](size_t i, const V& a) {
        ki::Vec<int8_t, EV> b;
#pragma unroll
        for (int e = 0; e < EV; ++e) b.e[e] = zero ? (int8_t)0 : to_i8(quantum(ki::to_f32(a.e[e]), s, inv));
        if (q_aligned) {
            ki::store_vec<int8_t, EV>(out + i * EV, b);
        } else {
#pragma unroll
            for (int e = 0; e < EV; ++e) out[i * EV + e] = b.e[e];
        }
    };
    if (fits) {
#pragma unroll
        for (int i = 0; i < VPT; ++i)
            if ((size_t)(i * TPR + t) < nvec) put(i * TPR + t, v[i]);
    } else {
        for (size_t i = t; i < nvec; i += TPR) put(i, ki::load_vec<T, EV>(row + i * EV));
    }
    for (size_t c = nvec * EV + t; c < cols; c += TPR)
        out[c] = zero ? (int8_t)0 : to_i8(quantum(ki::to_f32(row[c]), s, inv));
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
    constexpr int kBlock = TPR > kThreads ? TPR : kThreads;
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
    if (nvec <= 128) return launch<T, EV, 2, 64>(ctx, a);
    if (nvec <= 512) return launch<T, EV, 2, 256>(ctx, a);
    if (nvec <= 1024) return launch<T, EV, 4, 256>(ctx, a);
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
