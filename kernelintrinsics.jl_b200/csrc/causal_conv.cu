// causal_conv.cu -- ki_causal_conv / ki_causal_conv_step: the short depthwise convolution before a
// selective scan, over packed sequences and for single tokens.
//
//   y[t, d] = act(bias[d] + sum_{j < W} w[d, j] * x[t - (W-1) + j, d])
//
// with positions before a sequence's first token taken from its state (its last W-1 inputs) or zero;
// the state after a sequence is the last W-1 inputs of (state, tokens).
//
// Bound: HBM (one read and one write of the tokens).  A thread owns neighbouring channels (8 bytes of a row) and walks
// a run of tokens with the inputs it needs in registers, so a token is read once per run plus W-1 rows at the run's start.
// Rows ahead are on their way to shared memory (cp.async, each thread its own bytes).  At 8192 x 4096 bf16, W = 4:
// 28.6 us, 4.7 TB/s (54 us with 16-byte loads to registers, scalar loads of the taps and a window that moved along).
//
// A sequence's state is read by its first W-1 tokens and replaced by its last ones.  So that no other
// block reads a state that has been replaced, the first W-1 tokens of a sequence belong to the run that
// holds its first token, even where they lie in the next run, and the same threads write the new state
// when they are done with them.
#include "ki/layer.cuh"

namespace {

constexpr int kThreads = 128;
constexpr int kBytes = 8;    // of a row per thread and access, where the rows allow it
constexpr int kGroups = 4;   // ring slots of a group of rows each, a power of two

struct ConvArgs {
    const void* x;
    size_t ldx;
    const void* w;
    const void* bias;
    void* state;
    size_t state_ld;  // elements between slots
    void* y;
    size_t ldy;
    int channels;
    int run;  // tokens per run
    bool silu;
    bool vec_w;  // d_w allows 16-byte accesses
    ki::Sequences seq;
};

// V channels of one row as Float32 pairs (a single channel: the second half is not used).
template <int V>
struct Row {
    static constexpr int P = (V + 1) / 2;
    ki::f32x2 p[P];
    template <class T>
    __device__ __forceinline__ void widen(const ki::Vec<T, V>& v) {
#pragma unroll
        for (int i = 0; i < P; ++i) p[i] = ki::pair(ki::to_f32(v.e[2 * i]), V > 1 ? ki::to_f32(v.e[2 * i + (V > 1)]) : 0.0f);
    }
    template <class T>
    __device__ __forceinline__ ki::Vec<T, V> narrow() const {
        ki::Vec<T, V> v;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            float lo, hi;
            ki::unpair(lo, hi, p[i]);
            v.e[2 * i] = ki::from_f32<T>(lo);
            if (V > 1) v.e[2 * i + (V > 1)] = ki::from_f32<T>(hi);
        }
        return v;
    }
    __device__ __forceinline__ void silu() {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            float lo, hi;
            ki::unpair(lo, hi, ki::mul2(p[i], ki::pair(-ki::kLog2e)));
            ki::unpair(lo, hi, ki::add2(ki::pair(ki::exp2_fast(lo), ki::exp2_fast(hi)), ki::pair(1.0f)));
            p[i] = ki::mul2(p[i], ki::pair(ki::rcp_fast(lo), ki::rcp_fast(hi)));
        }
    }
};

template <class T, int V, int W>
struct Taps {
    Row<V> w[W], bias;
    __device__ __forceinline__ Taps(const ConvArgs& a, int c0) {
        // the taps of neighbouring channels lie together: as few accesses as their bytes allow
        constexpr int BYTES = V * W * (int)sizeof(T);
        constexpr int A = V == 1 ? (int)sizeof(T) : BYTES % 16 == 0 ? 16 : BYTES % 8 == 0 ? 8 : (int)sizeof(T);
        constexpr int N = A / (int)sizeof(T);
        T all[V * W];
        const T* pw = static_cast<const T*>(a.w) + (size_t)c0 * W;
        if (a.vec_w) {
#pragma unroll
            for (int i = 0; i < V * W; i += N) {
                const ki::Vec<T, N> v = ki::load_vec<T, N>(pw + i);
#pragma unroll
                for (int e = 0; e < N; ++e) all[i + e] = v.e[e];
            }
        } else {
#pragma unroll
            for (int i = 0; i < V * W; ++i) all[i] = pw[i];
        }
        ki::Vec<T, V> v;
#pragma unroll
        for (int j = 0; j < W; ++j) {
#pragma unroll
            for (int c = 0; c < V; ++c) v.e[c] = all[c * W + j];
            w[j].widen(v);
        }
#pragma unroll
        for (int c = 0; c < V; ++c) v.e[c] = a.bias ? static_cast<const T*>(a.bias)[c0 + c] : ki::from_f32<T>(0.0f);
        bias.widen(v);
    }
    // One output from its W inputs, oldest first.
    template <class F>
    __device__ __forceinline__ ki::Vec<T, V> output(F input, bool silu) const {
        Row<V> s = bias;
#pragma unroll
        for (int j = 0; j < W; ++j) {
            const Row<V>& x = input(j);
#pragma unroll
            for (int i = 0; i < Row<V>::P; ++i) s.p[i] = ki::fma2(w[j].p[i], x.p[i], s.p[i]);
        }
        if (silu) s.silu();
        return s.template narrow<T>();
    }
};

// Rows per group: the W-1 inputs before a group are all in the group before it.
constexpr int group_rows(int width) { return width <= 5 ? 4 : 8; }

// Tokens [lo, hi) of a sequence that starts at token b; `st`: its state's rows, or null for zeros.
//
// The inputs come through a ring of groups of rows in shared memory, each thread its own bytes, so that nothing has to
// be waited for but a thread's own copies, and many rows are in flight without registers.  Two groups' values are held,
// and take turns, so that no value is moved.
template <class T, int V, int W>
__device__ __forceinline__ void conv_tokens(const ConvArgs& a, const Taps<T, V, W>& k, int c0, int b, int lo, int hi,
                                            const T* st, ki::Vec<T, V>* ring) {
    constexpr int U = group_rows(W);
    constexpr int BYTES = (int)sizeof(T) * V;
    constexpr bool kRing = BYTES >= 4;
    if (lo >= hi) return;
    const T* x = static_cast<const T*>(a.x) + c0;
    T* y = static_cast<T*>(a.y) + c0 + (size_t)lo * a.ldy;
    const T* ahead = x + (size_t)lo * a.ldx;  // the next row to be fetched
    int left = hi - lo;                       // rows to be fetched
    int put = 0, got = 0;                     // ring slots of the next group to be fetched and to be used
    auto fetch = [&]() {
        if constexpr (kRing) {
            ki::Vec<T, V>* to = ring + put * (U * kThreads);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (u < left)
                    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(
                                     (uint32_t)__cvta_generic_to_shared(to + u * kThreads)),
                                 "l"(ahead + u * a.ldx), "n"(BYTES < 4 ? 4 : BYTES)
                                 : "memory");
            asm volatile("cp.async.commit_group;" ::: "memory");
            put = (put + 1) & (kGroups - 1);
            ahead += U * a.ldx;
            left -= U;
        }
    };
    auto get = [&](Row<V>(&in)[U], int n) {  // the next group, of which n rows exist
        if constexpr (kRing) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kGroups - 2) : "memory");
            const ki::Vec<T, V>* from = ring + got * (U * kThreads);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (u < n) in[u].widen(from[u * kThreads]);
            got = (got + 1) & (kGroups - 1);
            fetch();
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (u < n) in[u].widen(ki::load_vec<T, V>(ahead + u * a.ldx));
            ahead += U * a.ldx;
        }
    };
    auto emit = [&](const Row<V>(&before)[U], const Row<V>(&in)[U], int n) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u < n) {
                auto input = [&](int j) -> const Row<V>& {
                    const int i = u + j - (W - 1);
                    return i >= 0 ? in[i < 0 ? 0 : i] : before[i < 0 ? U + i : 0];
                };
                ki::store_vec<T, V>(y + u * a.ldy, k.output(input, a.silu));
            }
        }
        y += U * a.ldy;
    };
#pragma unroll
    for (int i = 0; i < kGroups - 1; ++i) fetch();
    Row<V> even[U], odd[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
        ki::Vec<T, V> v;
#pragma unroll
        for (int c = 0; c < V; ++c) v.e[c] = ki::from_f32<T>(0.0f);
        const int t = lo - U + j;
        if (j >= U - (W - 1)) {
            if (t >= b)
                v = ki::load_vec<T, V>(x + (size_t)t * a.ldx);
            else if (st)
                v = ki::load_vec<T, V>(st + (size_t)(W - 1 + t - b) * a.channels);
        }
        odd[j].widen(v);
    }
    int n = hi - lo;
    for (; n >= 2 * U; n -= 2 * U) {
        get(even, U);
        emit(odd, even, U);
        get(odd, U);
        emit(even, odd, U);
    }
    if (n > 0) {
        get(even, n);
        emit(odd, even, n);
        if (n > U) {
            get(odd, n - U);
            emit(even, odd, n - U);
        }
    }
    if constexpr (kRing) asm volatile("cp.async.wait_all;" ::: "memory");
}

template <class T, int V, int W>
__global__ void __launch_bounds__(kThreads) conv_kernel(const ConvArgs a, int tiles) {
    const int tile = blockIdx.x % tiles, run = blockIdx.x / tiles;
    const ki::Sequences& q = a.seq;
    const int t0 = (int)min((long long)run * a.run, (long long)q.tokens);
    const int t1 = (int)min((long long)t0 + a.run, (long long)q.tokens);
    const bool last = t1 == q.tokens;
    if (blockIdx.x == 0) q.check(threadIdx.x, kThreads);
    // the first sequence that starts at t0 or later
    int first = 0;
    if (q.offsets && t0 > 0) {
        for (int i0 = 0; i0 < q.count; i0 += kThreads) {
            const int i = i0 + (int)threadIdx.x;
            first += __syncthreads_count(i < q.count && q.begin(i) < t0);
        }
    } else if (t0 > 0) {
        first = 1;
    }
    const int c0 = (tile * kThreads + (int)threadIdx.x) * V;
    if (c0 >= a.channels) return;
    const Taps<T, V, W> k(a, c0);
    __shared__ ki::Vec<T, V> rows[sizeof(T) * V >= 4 ? kGroups * group_rows(W) * kThreads : 1];
    ki::Vec<T, V>* ring = rows + (sizeof(T) * V >= 4 ? threadIdx.x : 0);
    if (first > 0) {  // the sequence that an earlier run began; its first W-1 tokens are done there
        const int b = q.begin(first - 1), e = min(q.begin(first), t1);
        const int lo = max(t0, b + W - 1);
        if (lo < e && (!a.state || q.slot(first - 1) >= 0)) conv_tokens<T, V, W>(a, k, c0, b, lo, e, nullptr, ring);
    }
    for (int s = first; s < q.count; ++s) {
        const int b = q.begin(s);
        if (b >= t1 && !last) break;
        const int e = max(b, q.begin(s + 1));
        T* st = nullptr;
        if (a.state) {
            const int64_t slot = q.slot(s);
            if (slot < 0) continue;  // padding: its rows and state stay as they are
            st = static_cast<T*>(a.state) + (size_t)slot * a.state_ld + c0;
        }
        const bool keep = st && q.continues(s);
        conv_tokens<T, V, W>(a, k, c0, b, b, min(e, max(t1, b + W - 1)), keep ? st : nullptr, ring);
        if (st) {
            const T* x = static_cast<const T*>(a.x) + c0;
#pragma unroll
            for (int j = 0; j < W - 1; ++j) {  // row j takes a later row of the old state, so rising order is safe
                const int t = e - (W - 1) + j;
                ki::Vec<T, V> v;
                if (t >= b) {
                    v = ki::load_vec<T, V>(x + (size_t)t * a.ldx);
                } else if (keep) {
                    v = ki::load_vec<T, V>(st + (size_t)(W - 1 + t - b) * a.channels);
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i) v.e[i] = ki::from_f32<T>(0.0f);
                }
                ki::store_vec<T, V>(st + (size_t)j * a.channels, v);
            }
        }
    }
}

// One token per row: row r continues slot slots[r].
template <class T, int V, int W>
__global__ void __launch_bounds__(kThreads) conv_step_kernel(const ConvArgs a, int tiles) {
    const int r = blockIdx.x / tiles;
    const int c0 = ((int)(blockIdx.x % tiles) * kThreads + (int)threadIdx.x) * V;
    if (c0 >= a.channels) return;
    const int64_t slot = a.seq.slot(r);
    if (slot < 0) return;
    T* st = static_cast<T*>(a.state) + (size_t)slot * a.state_ld + c0;
    ki::Vec<T, V> in[W];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) in[j] = ki::load_vec<T, V>(st + (size_t)j * a.channels);
    in[W - 1] = ki::load_vec<T, V>(static_cast<const T*>(a.x) + (size_t)r * a.ldx + c0);
    const Taps<T, V, W> k(a, c0);
    Row<V> row;
    ki::store_vec<T, V>(static_cast<T*>(a.y) + (size_t)r * a.ldy + c0, k.output(
                                                                           [&](int j) -> const Row<V>& {
                                                                               row.widen(in[j]);
                                                                               return row;
                                                                           },
                                                                           a.silu));
#pragma unroll
    for (int j = 0; j < W - 1; ++j) ki::store_vec<T, V>(st + (size_t)j * a.channels, in[j + 1]);
}

template <class T, int V, int W>
int launch(ki_ctx* ctx, ConvArgs& a, bool step, cudaStream_t s) {
    const long long tiles = (a.channels + (long long)kThreads * V - 1) / ((long long)kThreads * V);
    long long rows = a.seq.count;
    if (!step) {
        // runs as long as 64 tokens (8192 x 4096 bf16: 28.6 us; 32: 28.6, 128: 30.3), shorter where that leaves SMs idle
        a.run = 64;
        while (a.run > 8 && tiles * ((a.seq.tokens + a.run - 1) / a.run) < 4ll * ctx->sm_count) a.run /= 2;
        rows = a.seq.tokens ? (a.seq.tokens + a.run - 1) / a.run : 1;
    }
    if (tiles * rows > 0x7fffffffll) return ki::set_error(ctx, KI_ERR_ARG, "causal_conv: too many rows");
    if (step)
        conv_step_kernel<T, V, W><<<(unsigned)(tiles * rows), kThreads, 0, s>>>(a, (int)tiles);
    else
        conv_kernel<T, V, W><<<(unsigned)(tiles * rows), kThreads, 0, s>>>(a, (int)tiles);
    return ki::check_launch(ctx, "causal_conv launch");
}

template <class T, int V>
int launch_width(ki_ctx* ctx, ConvArgs& a, int width, bool step, cudaStream_t s) {
    switch (width) {
        case 2: return launch<T, V, 2>(ctx, a, step, s);
        case 3: return launch<T, V, 3>(ctx, a, step, s);
        case 4: return launch<T, V, 4>(ctx, a, step, s);
        case 5: return launch<T, V, 5>(ctx, a, step, s);
        case 6: return launch<T, V, 6>(ctx, a, step, s);
        case 7: return launch<T, V, 7>(ctx, a, step, s);
        default: return launch<T, V, 8>(ctx, a, step, s);
    }
}

int conv(ki_ctx* ctx, const char* what, int dtype, ConvArgs& a, size_t rows, size_t channels, int width, bool step,
         void* stream) {
    const size_t es = ki::float_size(dtype);
    if (!es) return ki::set_error(ctx, KI_ERR_ARG, "%s: dtype must be KI_F32, KI_F16 or KI_BF16", what);
    if (width < 2 || width > 8) return ki::set_error(ctx, KI_ERR_ARG, "%s: width must be 2 to 8", what);
    if (rows > 0x7fffff00u || channels > 0x3fffffffu) return ki::set_error(ctx, KI_ERR_ARG, "%s: too large", what);
    if (channels == 0 || a.seq.count == 0) return KI_OK;
    if (!a.w || (rows > 0 && (!a.x || !a.y))) return ki::set_error(ctx, KI_ERR_ARG, "%s: null pointer", what);
    if (rows > 1 && (a.ldx < channels || a.ldy < channels))
        return ki::set_error(ctx, KI_ERR_ARG, "%s: leading dimension smaller than channels", what);
    if (!a.state && (a.seq.slots || a.seq.initial))
        return ki::set_error(ctx, KI_ERR_ARG, "%s: slots or initial without a state", what);
    const size_t held = (size_t)(width - 1) * channels;
    if (a.state) {
        if (a.seq.nslots > 1 && a.state_ld < held)
            return ki::set_error(ctx, KI_ERR_ARG, "%s: slots of the state closer than (width - 1) * channels", what);
        if (!a.seq.slots && a.seq.nslots < a.seq.count)
            return ki::set_error(ctx, KI_ERR_ARG, "%s: fewer state slots than sequences", what);
    }
    if (!ki::aligned(a.x, es) || !ki::aligned(a.w, es) || !ki::aligned(a.bias, es) || !ki::aligned(a.state, es) ||
        !ki::aligned(a.y, es) || !ki::aligned(a.seq.offsets, 4) || !ki::aligned(a.seq.slots, 4))
        return ki::set_error(ctx, KI_ERR_ARG, "%s: pointer not aligned to its element", what);
    const size_t nseq = (size_t)a.seq.count;
    const ki::Span y = ki::span(a.y, rows, a.ldy, channels, es),
                   st = ki::span(a.state, (size_t)a.seq.nslots, a.state_ld, held, es);
    const ki::Span in[] = {ki::span(a.x, rows, a.ldx, channels, es), ki::span(a.w, channels, width, width, es),
                           ki::span(a.bias, 1, channels, channels, es), ki::span(a.seq.offsets, 1, 1, nseq + 1, 4),
                           ki::span(a.seq.slots, 1, 1, nseq, 4), ki::span(a.seq.initial, 1, 1, nseq, 1)};
    bool bad = ki::overlap(y, st);
    for (const ki::Span& i : in) bad |= ki::overlap(y, i) || ki::overlap(st, i);
    if (bad) return ki::set_error(ctx, KI_ERR_ARG, "%s: an output overlaps another range", what);
    KI_GUARD(ctx);
    a.channels = (int)channels;
    a.vec_w = ki::aligned(a.w, 16);
    a.seq.tokens = (int)rows;
    a.seq.status = ctx->d_status;
    return ki::with_float_type(dtype, [&](auto t) {
        using T = decltype(t);
        constexpr int V = kBytes / (int)sizeof(T);
        // whole accesses where every row of every array allows them, else channel by channel
        const bool vec = channels % V == 0 && ki::rows_aligned(a.x, rows > 1 ? a.ldx : 0, es, kBytes) &&
                         ki::rows_aligned(a.y, rows > 1 ? a.ldy : 0, es, kBytes) &&
                         ki::rows_aligned(a.state, a.seq.nslots > 1 ? a.state_ld : 0, es, kBytes);
        return vec ? launch_width<T, V>(ctx, a, width, step, ki::as_stream(stream))
                   : launch_width<T, 1>(ctx, a, width, step, ki::as_stream(stream));
    });
}

}  // namespace

extern "C" int ki_causal_conv(ki_ctx* ctx, int dtype, const void* d_x, size_t ldx, const void* d_w, const void* d_bias,
                              void* d_state, size_t state_ld, size_t slots, const int32_t* d_slots,
                              const uint8_t* d_initial, const int32_t* d_offsets, size_t seqs, void* d_y, size_t ldy,
                              size_t tokens, size_t channels, int width, int silu, void* stream) {
    KI_CHECK_CTX(ctx);
    if (seqs > ki::kMaxSequences || slots > 0x7fffffffffffu)
        return ki::set_error(ctx, KI_ERR_ARG, "causal_conv: too many sequences or slots");
    if (!d_offsets && seqs != 1) return ki::set_error(ctx, KI_ERR_ARG, "causal_conv: several sequences need offsets");
    ConvArgs a{d_x, ldx, d_w, d_bias, d_state, state_ld, d_y, ldy, 0, 0, silu != 0, false,
               {d_offsets, d_slots, d_initial, (int)seqs, 0, (int64_t)slots, nullptr}};
    return conv(ctx, "causal_conv", dtype, a, tokens, channels, width, false, stream);
}

extern "C" int ki_causal_conv_step(ki_ctx* ctx, int dtype, const void* d_x, size_t ldx, const void* d_w,
                                   const void* d_bias, void* d_state, size_t state_ld, size_t slots,
                                   const int32_t* d_slots, void* d_y, size_t ldy, size_t rows, size_t channels, int width,
                                   int silu, void* stream) {
    KI_CHECK_CTX(ctx);
    if (rows > ki::kMaxSequences || slots > 0x7fffffffffffu)
        return ki::set_error(ctx, KI_ERR_ARG, "causal_conv_step: too many rows or slots");
    if (!d_state) return ki::set_error(ctx, KI_ERR_ARG, "causal_conv_step: null pointer");
    ConvArgs a{d_x, ldx, d_w, d_bias, d_state, state_ld, d_y, ldy, 0, 0, silu != 0, false,
               {nullptr, d_slots, nullptr, (int)rows, 0, (int64_t)slots, nullptr}};
    return conv(ctx, "causal_conv_step", dtype, a, rows, channels, width, true, stream);
}
