// ki/layer.cuh -- what the operators of a model's layer share (quantize.cu, causal_conv.cu,
// selective_scan.cu, gemm_i8.cu): Float32 / Float16 / BFloat16 elements, the activations, packed
// sequences with their state slots, and checks of arguments.
//
// Elements are read in their type, every sum, state and scale is Float32 (the int8 product: Int32),
// and a result is rounded once, to nearest even, when it is stored.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "ki/intrinsics.cuh"

namespace ki {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two values to neighbouring elements of a word (16-bit types), lo in the lower half.
template <class T>
__device__ __forceinline__ uint32_t narrow2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t narrow2<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t narrow2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// V consecutive elements moved with one access of sizeof(T) * V bytes (at most 16).
template <class T, int V>
struct alignas(sizeof(T) * V) Vec {
    T e[V];
};
template <class T, int V>
__device__ __forceinline__ Vec<T, V> load_vec(const T* p) {
    return *reinterpret_cast<const Vec<T, V>*>(p);
}
template <class T, int V>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, V>& v) {
    *reinterpret_cast<Vec<T, V>*>(p) = v;
}

constexpr float kLog2e = 1.4426950408889634f;

// 2^x with one instruction (2 ulp); results below 2^-126 are zero, and so are reciprocals of numbers above 2^126: a gate
// of less than 1.2e-38 (z below -87.3) is zero, as a step or decay of that size is, in Float32 too.
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// x * sigmoid(x); -inf gives NaN as the formula does.
__device__ __forceinline__ float silu(float x) { return x * rcp_fast(1.0f + exp2_fast(-kLog2e * x)); }

// x log2(e), finite wherever x is: a step of zero then leaves a state as it is however large the magnitude of A (0 * inf would be NaN).
__device__ __forceinline__ float times_log2e(float x) {
    const float y = x * kLog2e, top = 3.402823466e38f;
    return fabsf(x) <= top ? fminf(fmaxf(y, -top), top) : y;
}

// Two Float32 in one register pair; one instruction works on both.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pair(float lo, float hi) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ f32x2 pair(float v) { return pair(v, v); }
__device__ __forceinline__ void unpair(float& lo, float& hi, f32x2 v) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// max(x, 0); NaN stays.
__device__ __forceinline__ float relu(float x) {
    float y;
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(y) : "f"(x));
    return y;
}
// log(1 + e^x) = max(x, 0) + log1p(e), e = e^-|x| <= 1.  The exponent's product with log2(e) is kept to twice
// Float32's precision; log1p(e) / e is a polynomial of degree 8, fitted on [0, 1] for the smallest relative error (3e-8).
// With Float32 arithmetic and the fast exponential at most 3.2e-7 off, relative (16 million points of [-87, 100]); zero
// below -87.3.  No branches, so neighbouring values overlap.
__device__ __forceinline__ float softplus(float x) {
    const float n = fmaxf(-fabsf(x), -200.0f);
    const float minus = n * -kLog2e;
    const float lo = fmaf(n, 1.92596299e-8f, fmaf(n, kLog2e, minus));
    float e = exp2_fast(-minus);
    e = fmaf(e, lo * 0.693147182f, e);
    float p = fmaf(e, 0.005232684314250946f, -0.029505198821425438f);
    p = fmaf(e, p, 0.07822588831186295f);
    p = fmaf(e, p, -0.13663239777088165f);
    p = fmaf(e, p, 0.19106003642082214f);
    p = fmaf(e, p, -0.2484298199415207f);
    p = fmaf(e, p, 0.3331909775733948f);
    p = fmaf(e, p, -0.4999949336051941f);
    p = fmaf(e, p, 0.9999999403953552f);
    return fmaf(e, p, relu(x));
}

// ---- packed sequences ---------------------------------------------------------------------------
// Sequence i holds tokens [offsets[i], offsets[i+1]) of the packed rows; without offsets there is one
// sequence of all rows.  Offsets are read on the device, so they are clamped to the rows there are
// and never trusted.
constexpr size_t kMaxSequences = 0x7ffff000u;  // an int index may pass the last one by a block's threads

struct Sequences {
    const int32_t* offsets;
    const int32_t* slots;    // state slot of each sequence; negative: the sequence is padding; null: slot i
    const uint8_t* initial;  // nonzero: the sequence continues from its slot; null: every sequence does
    int count;
    int tokens;
    int64_t nslots;
    uint32_t* status;

    __device__ __forceinline__ int begin(int i) const {
        return offsets ? min(max(offsets[i], 0), tokens) : (i == 0 ? 0 : tokens);
    }
    // Slot of sequence i, or -1 where it has none (padding, or a number that no slot has, which is latched).
    __device__ __forceinline__ int64_t slot(int i) const {
        const int64_t s = slots ? (int64_t)slots[i] : (int64_t)i;
        if (s >= nslots) {
            atomicOr(status, (uint32_t)KI_DEV_BAD_INDEX);
            return -1;
        }
        return s;
    }
    __device__ __forceinline__ bool continues(int i) const { return initial ? initial[i] != 0 : true; }
    // Latches offsets that decrease or leave the rows (run by one block).
    __device__ __forceinline__ void check(int tid, int threads) const {
        if (!offsets) return;
        bool bad = false;
        for (int i = tid; i <= count; i += threads) {
            const int o = offsets[i];
            bad |= o < 0 || o > tokens || (i > 0 && offsets[i - 1] > o);
        }
        if (bad) atomicOr(status, (uint32_t)KI_DEV_BAD_INDEX);
    }
};

// ---- host side ------------------------------------------------------------------------------------
// Bytes [lo, hi) of a strided array: the first byte of its first row to the last of its last.
struct Span {
    uintptr_t lo = 0, hi = 0;
};
inline Span span(const void* p, size_t rows, size_t ld, size_t cols, size_t elem) {
    Span s;
    if (!p || rows == 0 || cols == 0) return s;
    s.lo = (uintptr_t)p;
    s.hi = s.lo + ((rows - 1) * ld + cols) * elem;
    return s;
}
inline bool overlap(const Span& a, const Span& b) { return a.lo < b.hi && b.lo < a.hi; }

inline size_t float_size(int dtype) { return dtype == KI_F32 ? 4 : dtype == KI_F16 || dtype == KI_BF16 ? 2 : 0; }

// Whether every row of an array starts on a multiple of `bytes`.
inline bool rows_aligned(const void* p, size_t ld, size_t elem, size_t bytes) {
    return aligned(p, bytes) && (ld * elem) % bytes == 0;
}

// Calls f with a value of the element type of dtype (KI_F32, KI_F16 or KI_BF16).
template <class F>
inline int with_float_type(int dtype, F f) {
    switch (dtype) {
        case KI_F32: return f(float());
        case KI_F16: return f(__half());
        default: return f(__nv_bfloat16());
    }
}

}  // namespace ki
