// selective_scan.cu -- ki_selective_scan / ki_selective_scan_step: the recurrence of a selective state
// space layer over packed sequences and for single tokens.
//
//   s_t = delta[t, d] (+ delta_bias[d]), softplus(s_t) where asked for
//   h_t[n] = exp(s_t A[d, n]) h_{t-1}[n] + s_t u[t, d] B[t, g, n]
//   y[t, d] = sum_n C[t, g, n] h_t[n] + D[d] u[t, d],  times z sigmoid(z) where there is a gate
//
// with g = d / (channels / groups); h is Float32 and starts from the sequence's slot or from zero.
//
// Bound: one exponential per token, channel and state (16 a clock and SM) at 16 states; the tokens'
// bytes take a third of that time.  So every (d, n) pair has a lane slot of its own: LPC lanes share a
// channel and each holds K states, the block walks the sequence in chunks of kChunk tokens, and the sums over
// n are folded across the lanes LPC tokens at a time, which takes one shuffle per token and state pair.
#include "ki/layer.cuh"

namespace {

constexpr int kThreads = 256;

struct ScanArgs {
    const void* u;
    size_t ldu;
    const void* delta;
    size_t ldd;
    const float* A;
    const void* B;
    size_t ldb;
    const void* C;
    size_t ldc;
    const float* D;
    const void* z;
    size_t ldz;
    const float* delta_bias;
    float* state;
    size_t state_ld;
    void* y;
    size_t ldy;
    int channels, states, groups;
    bool soft;
    ki::Sequences seq;
};

// Folds p[0..L) over the L lanes that share a channel: lane l ends up with the sum of p[l].
template <int L>
__device__ __forceinline__ float fold_lanes(float (&p)[L], int lane) {
#pragma unroll
    for (int h = L / 2; h >= 1; h /= 2) {
        const bool up = lane & h;
#pragma unroll
        for (int i = 0; i < h; ++i) {
            const float send = up ? p[i] : p[i + h];
            const float keep = up ? p[i + h] : p[i];
            p[i] = keep + __shfl_xor_sync(0xffffffffu, send, h);
        }
    }
    return p[0];
}

template <class T, int LPC, int K>
__global__ void __launch_bounds__(kThreads) scan_kernel(const ScanArgs a, int tiles) {
    constexpr int DT = kThreads / LPC;         // channels per block
    constexpr int NP = LPC * K;                // states, padded
    constexpr int TC = NP <= 64 ? 64 : 16;     // tokens per chunk
    __shared__ float2 s_step[TC][DT];          // (s_t, s_t u_t)
    __shared__ float2 s_bc[TC][NP];
    __shared__ float s_y[TC][DT + 1];
    const ki::Sequences& q = a.seq;
    if (blockIdx.x == 0) q.check(threadIdx.x, kThreads);
    const int seq = blockIdx.x / (tiles * a.groups);
    const int rest = blockIdx.x % (tiles * a.groups);
    const int g = rest / tiles;
    const int per = a.channels / a.groups;
    const int in0 = (rest % tiles) * DT;  // first channel within the group
    const int width = min(DT, per - in0);
    const int d0 = g * per + in0;
    const int b = q.begin(seq), e = max(b, q.begin(seq + 1));
    float* st = nullptr;
    if (a.state) {
        const int64_t slot = q.slot(seq);
        if (slot < 0) return;  // padding: its rows and state stay as they are
        st = a.state + (size_t)slot * a.state_ld;
    }
    const int lane = threadIdx.x % LPC, dl = threadIdx.x / LPC;
    const int n0 = lane * K;
    const bool live = dl < width;
    float A[K], h[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const bool on = live && n0 + k < a.states;
        const size_t at = (size_t)(d0 + dl) * a.states + n0 + k;
        A[k] = on ? a.A[at] * ki::kLog2e : 0.0f;
        h[k] = on && st && q.continues(seq) ? st[at] : 0.0f;
    }
    const T* u = static_cast<const T*>(a.u);
    const T* delta = static_cast<const T*>(a.delta);
    const T* B = static_cast<const T*>(a.B) + (size_t)g * a.states;
    const T* C = static_cast<const T*>(a.C) + (size_t)g * a.states;
    for (int t0 = b; t0 < e; t0 += TC) {
        const int tn = min(TC, e - t0);
        for (int i = threadIdx.x; i < tn * DT; i += kThreads) {
            const int t = i / DT, d = i % DT;
            float2 v = make_float2(0.0f, 0.0f);
            if (d < width) {
                float s = ki::to_f32(delta[(size_t)(t0 + t) * a.ldd + d0 + d]);
                if (a.delta_bias) s += a.delta_bias[d0 + d];
                if (a.soft) s = ki::softplus(s);
                v = make_float2(s, s * ki::to_f32(u[(size_t)(t0 + t) * a.ldu + d0 + d]));
            }
            s_step[t][d] = v;
        }
        for (int i = threadIdx.x; i < tn * NP; i += kThreads) {
            const int t = i / NP, n = i % NP;
            float2 v = make_float2(0.0f, 0.0f);
            if (n < a.states)
                v = make_float2(ki::to_f32(B[(size_t)(t0 + t) * a.ldb + n]), ki::to_f32(C[(size_t)(t0 + t) * a.ldc + n]));
            s_bc[t][n] = v;
        }
        __syncthreads();
        for (int t = 0; t < tn; t += LPC) {
            float p[LPC];
#pragma unroll
            for (int i = 0; i < LPC; ++i) {
                p[i] = 0.0f;
                if (t + i < tn) {
                    const float2 x = s_step[t + i][dl];
#pragma unroll
                    for (int k = 0; k < K; ++k) {
                        const float2 bc = s_bc[t + i][n0 + k];
                        h[k] = fmaf(ki::exp2_fast(x.x * A[k]), h[k], x.y * bc.x);
                        p[i] = fmaf(bc.y, h[k], p[i]);
                    }
                }
            }
            const float sum = fold_lanes<LPC>(p, lane);
            if (t + lane < tn) s_y[t + lane][dl] = sum;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < tn * DT; i += kThreads) {
            const int t = i / DT, d = i % DT;
            if (d < width) {
                float y = s_y[t][d];
                if (a.D) y = fmaf(a.D[d0 + d], ki::to_f32(u[(size_t)(t0 + t) * a.ldu + d0 + d]), y);
                if (a.z) y *= ki::silu(ki::to_f32(static_cast<const T*>(a.z)[(size_t)(t0 + t) * a.ldz + d0 + d]));
                static_cast<T*>(a.y)[(size_t)(t0 + t) * a.ldy + d0 + d] = ki::from_f32<T>(y);
            }
        }
    }
    if (st && live) {
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (n0 + k < a.states) st[(size_t)(d0 + dl) * a.states + n0 + k] = h[k];
    }
}

// One token per row: row r continues slot slots[r].  LPC lanes share a channel.
template <class T, int LPC>
__global__ void __launch_bounds__(kThreads) scan_step_kernel(const ScanArgs a, int tiles) {
    constexpr int DT = kThreads / LPC;
    const int r = blockIdx.x / tiles;
    const int d = (int)(blockIdx.x % tiles) * DT + (int)threadIdx.x / LPC;
    const int lane = threadIdx.x % LPC;
    const int64_t slot = a.seq.slot(r);
    if (slot < 0) return;
    const bool live = d < a.channels;
    float p = 0.0f, u = 0.0f;
    if (live) {
        const int g = d / (a.channels / a.groups);
        u = ki::to_f32(static_cast<const T*>(a.u)[(size_t)r * a.ldu + d]);
        float s = ki::to_f32(static_cast<const T*>(a.delta)[(size_t)r * a.ldd + d]);
        if (a.delta_bias) s += a.delta_bias[d];
        if (a.soft) s = ki::softplus(s);
        const float su = s * u;
        float* st = a.state + (size_t)slot * a.state_ld + (size_t)d * a.states;
        const float* A = a.A + (size_t)d * a.states;
        const T* B = static_cast<const T*>(a.B) + (size_t)r * a.ldb + (size_t)g * a.states;
        const T* C = static_cast<const T*>(a.C) + (size_t)r * a.ldc + (size_t)g * a.states;
        for (int n = lane; n < a.states; n += LPC) {
            const float h = fmaf(ki::exp2_fast(s * (A[n] * ki::kLog2e)), st[n], su * ki::to_f32(B[n]));
            st[n] = h;
            p = fmaf(ki::to_f32(C[n]), h, p);
        }
    }
#pragma unroll
    for (int h = LPC / 2; h >= 1; h /= 2) p += __shfl_xor_sync(0xffffffffu, p, h);
    if (live && lane == 0) {
        if (a.D) p = fmaf(a.D[d], u, p);
        if (a.z) p *= ki::silu(ki::to_f32(static_cast<const T*>(a.z)[(size_t)r * a.ldz + d]));
        static_cast<T*>(a.y)[(size_t)r * a.ldy + d] = ki::from_f32<T>(p);
    }
}

template <class T, int LPC, int K>
int launch(ki_ctx* ctx, const ScanArgs& a, cudaStream_t s) {
    constexpr int DT = kThreads / LPC;
    const long long tiles = (a.channels / a.groups + DT - 1) / DT;
    const long long blocks = tiles * a.groups * a.seq.count;
    if (blocks > 0x7fffffffll) return ki::set_error(ctx, KI_ERR_ARG, "selective_scan: too many sequences");
    scan_kernel<T, LPC, K><<<(unsigned)blocks, kThreads, 0, s>>>(a, (int)tiles);
    return ki::check_launch(ctx, "selective_scan launch");
}

template <class T>
int launch_scan(ki_ctx* ctx, const ScanArgs& a, cudaStream_t s) {
    if (a.states <= 16) return launch<T, 16, 1>(ctx, a, s);
    if (a.states <= 32) return launch<T, 16, 2>(ctx, a, s);
    if (a.states <= 64) return launch<T, 16, 4>(ctx, a, s);
    if (a.states <= 128) return launch<T, 16, 8>(ctx, a, s);
    return launch<T, 16, 16>(ctx, a, s);
}

template <class T>
int launch_step(ki_ctx* ctx, const ScanArgs& a, cudaStream_t s) {
    constexpr int LPC = 8, DT = kThreads / LPC;
    const long long tiles = (a.channels + DT - 1) / DT;
    if (tiles * a.seq.count > 0x7fffffffll) return ki::set_error(ctx, KI_ERR_ARG, "selective_scan_step: too many rows");
    scan_step_kernel<T, LPC><<<(unsigned)(tiles * a.seq.count), kThreads, 0, s>>>(a, (int)tiles);
    return ki::check_launch(ctx, "selective_scan_step launch");
}

int scan(ki_ctx* ctx, const char* what, int dtype, ScanArgs& a, size_t rows, size_t channels, size_t states, size_t groups,
         bool step, void* stream) {
    const size_t es = ki::float_size(dtype);
    if (!es) return ki::set_error(ctx, KI_ERR_ARG, "%s: dtype must be KI_F32, KI_F16 or KI_BF16", what);
    if (states < 1 || states > 256) return ki::set_error(ctx, KI_ERR_ARG, "%s: states must be 1 to 256", what);
    if (groups < 1 || channels % groups) return ki::set_error(ctx, KI_ERR_ARG, "%s: channels must be a multiple of groups", what);
    if (rows > 0x7fffff00u || channels > 0x7fffffu || a.seq.count < 0)
        return ki::set_error(ctx, KI_ERR_ARG, "%s: too large", what);
    if (channels == 0 || a.seq.count == 0) return KI_OK;
    if (!a.A || (rows > 0 && (!a.u || !a.delta || !a.B || !a.C || !a.y)))
        return ki::set_error(ctx, KI_ERR_ARG, "%s: null pointer", what);
    const size_t bc = groups * states;
    if (rows > 1 && (a.ldu < channels || a.ldd < channels || a.ldy < channels || a.ldb < bc || a.ldc < bc ||
                     (a.z && a.ldz < channels)))
        return ki::set_error(ctx, KI_ERR_ARG, "%s: leading dimension smaller than a row", what);
    if (!a.state && (a.seq.slots || a.seq.initial))
        return ki::set_error(ctx, KI_ERR_ARG, "%s: slots or initial without a state", what);
    const size_t held = channels * states;
    if (a.state) {
        if (a.seq.nslots > 1 && a.state_ld < held)
            return ki::set_error(ctx, KI_ERR_ARG, "%s: slots of the state closer than channels * states", what);
        if (!a.seq.slots && a.seq.nslots < a.seq.count)
            return ki::set_error(ctx, KI_ERR_ARG, "%s: fewer state slots than sequences", what);
    }
    if (!ki::aligned(a.u, es) || !ki::aligned(a.delta, es) || !ki::aligned(a.B, es) || !ki::aligned(a.C, es) ||
        !ki::aligned(a.z, es) || !ki::aligned(a.y, es) || !ki::aligned(a.A, 4) || !ki::aligned(a.D, 4) ||
        !ki::aligned(a.delta_bias, 4) || !ki::aligned(a.state, 4) || !ki::aligned(a.seq.offsets, 4) ||
        !ki::aligned(a.seq.slots, 4))
        return ki::set_error(ctx, KI_ERR_ARG, "%s: pointer not aligned to its element", what);
    const size_t nseq = (size_t)a.seq.count;
    const ki::Span y = ki::span(a.y, rows, a.ldy, channels, es),
                   st = ki::span(a.state, (size_t)a.seq.nslots, a.state_ld, held, 4);
    const ki::Span in[] = {ki::span(a.u, rows, a.ldu, channels, es), ki::span(a.delta, rows, a.ldd, channels, es),
                           ki::span(a.z, rows, a.ldz, channels, es), ki::span(a.B, rows, a.ldb, bc, es),
                           ki::span(a.C, rows, a.ldc, bc, es),       ki::span(a.A, channels, states, states, 4),
                           ki::span(a.D, 1, channels, channels, 4),  ki::span(a.delta_bias, 1, channels, channels, 4),
                           ki::span(a.seq.offsets, 1, 1, nseq + 1, 4), ki::span(a.seq.slots, 1, 1, nseq, 4),
                           ki::span(a.seq.initial, 1, 1, nseq, 1)};
    bool bad = ki::overlap(y, st);
    for (const ki::Span& i : in) bad |= ki::overlap(y, i) || ki::overlap(st, i);
    if (bad) return ki::set_error(ctx, KI_ERR_ARG, "%s: an output overlaps another range", what);
    KI_GUARD(ctx);
    a.channels = (int)channels;
    a.states = (int)states;
    a.groups = (int)groups;
    a.seq.tokens = (int)rows;
    a.seq.status = ctx->d_status;
    return ki::with_float_type(dtype, [&](auto t) {
        using T = decltype(t);
        return step ? launch_step<T>(ctx, a, ki::as_stream(stream)) : launch_scan<T>(ctx, a, ki::as_stream(stream));
    });
}

}  // namespace

extern "C" int ki_selective_scan(ki_ctx* ctx, int dtype, const void* d_u, size_t ldu, const void* d_delta, size_t ldd,
                                 const float* d_A, const void* d_B, size_t ldb, const void* d_C, size_t ldc,
                                 const float* d_D, const void* d_z, size_t ldz, const float* d_delta_bias, int softplus,
                                 float* d_state, size_t state_ld, size_t slots, const int32_t* d_slots,
                                 const uint8_t* d_initial, const int32_t* d_offsets, size_t seqs, void* d_y, size_t ldy,
                                 size_t tokens, size_t channels, size_t states, size_t groups, void* stream) {
    KI_CHECK_CTX(ctx);
    if (seqs > 0x7ffffffeu || slots > 0x7fffffffffu)
        return ki::set_error(ctx, KI_ERR_ARG, "selective_scan: too many sequences or slots");
    if (!d_offsets && seqs != 1) return ki::set_error(ctx, KI_ERR_ARG, "selective_scan: several sequences need offsets");
    ScanArgs a{d_u, ldu, d_delta, ldd, d_A, d_B, ldb, d_C, ldc, d_D, d_z, ldz, d_delta_bias, d_state, state_ld, d_y, ldy,
               0, 0, 0, softplus != 0, {d_offsets, d_slots, d_initial, (int)seqs, 0, (int64_t)slots, nullptr}};
    return scan(ctx, "selective_scan", dtype, a, tokens, channels, states, groups, false, stream);
}

extern "C" int ki_selective_scan_step(ki_ctx* ctx, int dtype, const void* d_u, size_t ldu, const void* d_delta, size_t ldd,
                                      const float* d_A, const void* d_B, size_t ldb, const void* d_C, size_t ldc,
                                      const float* d_D, const void* d_z, size_t ldz, const float* d_delta_bias,
                                      int softplus, float* d_state, size_t state_ld, size_t slots, const int32_t* d_slots,
                                      void* d_y, size_t ldy, size_t rows, size_t channels, size_t states, size_t groups,
                                      void* stream) {
    KI_CHECK_CTX(ctx);
    if (rows > 0x7ffffffeu || slots > 0x7fffffffffu)
        return ki::set_error(ctx, KI_ERR_ARG, "selective_scan_step: too many rows or slots");
    if (!d_state) return ki::set_error(ctx, KI_ERR_ARG, "selective_scan_step: null pointer");
    ScanArgs a{d_u, ldu, d_delta, ldd, d_A, d_B, ldb, d_C, ldc, d_D, d_z, ldz, d_delta_bias, d_state, state_ld, d_y, ldy,
               0, 0, 0, softplus != 0, {nullptr, d_slots, nullptr, (int)rows, 0, (int64_t)slots, nullptr}};
    return scan(ctx, "selective_scan_step", dtype, a, rows, channels, states, groups, true, stream);
}
