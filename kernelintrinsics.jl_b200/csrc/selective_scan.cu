// selective_scan.cu -- ki_selective_scan / ki_selective_scan_step: the recurrence of a selective state
// space layer over packed sequences and for single tokens.
//
//   s_t = delta[t, d] (+ delta_bias[d]), softplus(s_t) where asked for
//   h_t[n] = exp(s_t A[d, n]) h_{t-1}[n] + s_t u[t, d] B[t, g, n]
//   y[t, d] = sum_n C[t, g, n] h_t[n] + D[d] u[t, d],  times z sigmoid(z) where there is a gate
//
// with g = d / (channels / groups); h is Float32 and starts from the sequence's slot or from zero.
//
// Bound: one exponential per token, channel and state (16 a clock and SM) at 16 states, and the instructions around it;
// the tokens' bytes take a third of that time.  The (channel, state) pairs are all the parallelism that one sequence has:
// LPC lanes share a channel and hold K states each, and 128 such lanes walk the sequence in chunks of 32 tokens.  As many
// helper threads bring the next chunk to shared memory as the lanes want it (steps through softplus, B and C side by
// side) and finish the chunk before (sums over the lanes, D, gate, store), so that the lanes do nothing but the recurrence
// and the two never wait for global memory.  At 8192 x 4096 x 16 bf16: 316 us (1240 us with one kind of thread, and the
// sums folded by shuffles); the exponentials alone take 137 us.  Two warps per scheduler issue an instruction in 59 % of
// the cycles there.  Tried without gain: loading and storing threads apart, two tokens per instruction instead of two
// states, 64-token chunks, steps stored twice (shared-memory bandwidth: 82 -> 89 us at 2048 tokens), scalar arithmetic.
#include "ki/layer.cuh"

namespace {

constexpr int kStepThreads = 128;

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
    bool sort;          // the longest sequences first
    bool vec;           // rows of u, delta, z and y are aligned for accesses of a thread's channels
    bool vec_b, vec_c;  // rows of B and C are aligned for accesses of a thread's states
    ki::Sequences seq;
};

constexpr int kTime = 32;      // tokens per chunk
constexpr int kUnroll = 8;
constexpr int kLanes = 128;    // threads per block that compute
constexpr int kHelpers = 128;  // and that load and store
constexpr int kShare = kHelpers / kTime;  // helper threads that share a token

__device__ __forceinline__ void prefetch(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// N elements of a row, kept as they lie in memory until they are used, so that nothing waits for a load that runs
// ahead.  `vec`: the row is aligned for whole accesses; n: how many elements exist.
template <class T, int N>
struct Raw {
    static constexpr int BYTES = N * (int)sizeof(T);
    static constexpr int NW = BYTES < 4 ? 1 : BYTES / 4;
    uint32_t w[NW];

    __device__ __forceinline__ void load(const T* p, bool vec, int n) {
        if (vec && n >= N) {
            if constexpr (BYTES >= 16) {
#pragma unroll
                for (int i = 0; i < NW; i += 4) {
                    const uint4 v = reinterpret_cast<const uint4*>(p)[i / 4];
                    w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
                }
            } else if constexpr (BYTES == 8) {
                const uint2 v = *reinterpret_cast<const uint2*>(p);
                w[0] = v.x, w[1] = v.y;
            } else if constexpr (BYTES == 4) {
                w[0] = *reinterpret_cast<const uint32_t*>(p);
            } else {
                w[0] = *reinterpret_cast<const uint16_t*>(p);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NW; ++i) w[i] = 0;
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i < n) set(i, p[i]);
        }
    }
    __device__ __forceinline__ void store(T* p, bool vec, int n) const {
        if (vec && n >= N) {
            if constexpr (BYTES >= 16) {
#pragma unroll
                for (int i = 0; i < NW; i += 4)
                    reinterpret_cast<uint4*>(p)[i / 4] = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
            } else if constexpr (BYTES == 8) {
                *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
            } else if constexpr (BYTES == 4) {
                *reinterpret_cast<uint32_t*>(p) = w[0];
            } else {
                *reinterpret_cast<uint16_t*>(p) = (uint16_t)w[0];
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i < n) p[i] = get(i);
        }
    }
    __device__ __forceinline__ T get(int i) const {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(w[i]);
        } else {
            const uint16_t h = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
            return *reinterpret_cast<const T*>(&h);
        }
    }
    __device__ __forceinline__ void set(const float (&v)[N]) {
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            if constexpr (sizeof(T) == 4)
                w[i] = __float_as_uint(v[i]);
            else
                w[i] = ki::narrow2<T>(v[2 * i], N > 1 ? v[2 * i + (N > 1)] : 0.0f);
        }
    }
    __device__ __forceinline__ uint32_t half(int i) const { return (w[i / 2] >> (16 * (i & 1))) & 0xffffu; }
    __device__ __forceinline__ void set(int i, T v) {  // into words that were zero there
        if constexpr (sizeof(T) == 4)
            w[i] = __float_as_uint(v);
        else
            w[i / 2] |= (uint32_t)*reinterpret_cast<const uint16_t*>(&v) << (16 * (i & 1));
    }
};

template <class T, int LPC, int K>
struct Tile {
    static constexpr int DT = kLanes / LPC;         // channels per block
    static constexpr int VC = DT / kShare;         // channels per helper thread
    static constexpr int NP = LPC * K;             // states, padded
    static constexpr int NB = NP / kShare;          // states of B and C per helper thread
    static constexpr int GW = 2 * K * (int)sizeof(T) / 4;  // words of a lane's states: K of B, then K of C, as loaded
    static constexpr int ROW = DT + 2;             // of steps, padded so that neighbouring tokens' banks differ
    struct Stage {
        float4 part[kTime * kLanes / 4];  // each lane's sum over its states, swizzled
        uint32_t bc[kTime * LPC * GW];
        float2 step[kTime * ROW];        // (s, s u) of a token and channel
    };
    // 16 bytes number `slot` of a token's sums.  The helper threads of a token and of the next ones read the same
    // banks at once; the exclusive-or puts eight neighbouring threads on all of them.
    static __device__ __forceinline__ int part_at(int t, int slot) {
        return t * (kLanes / 4) + (slot ^ (slot / (kLanes / 4 / kShare) + kShare * (t & (8 / kShare - 1))));
    }
};

// Two neighbouring 16-bit values of a word.
template <class T>
__device__ __forceinline__ ki::f32x2 widen2(uint32_t w);
template <>
__device__ __forceinline__ ki::f32x2 widen2<__nv_bfloat16>(uint32_t w) {
    return ki::pair(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ ki::f32x2 widen2<__half>(uint32_t w) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return ki::pair(f.x, f.y);
}

// Compute threads.  A token passes three stages that run on three tokens at once, so that the exponentials of one
// (16 a clock and SM) and the multiply-adds of another share the time: its values are loaded, then its decays and
// what it adds are computed, then the states and the sum over them.
//
// Some lanes may hold states that do not exist.  Their A, B and C are zero, but an infinite step or s u makes them NaN
// (inf * 0), so the sum leaves them out: a lane's sum where only whole lanes are empty, else state by state (2048 tokens, bf16:
// 4096 channels of 24 states 128.7 us, of 13 states 97.6 against 96.5 with the padding summed, 512 of 100 193 against 185).
enum Pad { kNoPad, kPadLanes, kPadStates };
template <class T, int LPC, int K, Pad PAD>
struct Lane {
    using L = Tile<T, LPC, K>;
    static constexpr int GW = L::GW;
    static constexpr int P = K == 1 ? 1 : K / 2;  // pairs of states (one state: only the first half is used)
    ki::f32x2 A[P], h[P];
    int held;  // the lane's states that exist, 0 to K

    struct In {
        float2 x;
        uint32_t w[GW];
    };
    struct Mid {
        ki::f32x2 a[P], add[P], c[P];
    };
    static __device__ __forceinline__ In load(const float2* step, const uint32_t* bc, int t) {
        In in;
        in.x = step[t * L::ROW];
        constexpr int W = GW < 4 ? GW : 4;
#pragma unroll
        for (int i = 0; i < GW; i += W) {
            const ki::Vec<uint32_t, W> v = ki::load_vec<uint32_t, W>(bc + t * (LPC * GW) + i);
#pragma unroll
            for (int j = 0; j < W; ++j) in.w[i + j] = v.e[j];
        }
        return in;
    }
    __device__ __forceinline__ Mid decays(const In& in) const {
        Mid m;
        if constexpr (K == 1) {
            float b, c;
            if constexpr (sizeof(T) == 4)
                b = __uint_as_float(in.w[0]), c = __uint_as_float(in.w[1]);
            else
                ki::unpair(b, c, widen2<T>(in.w[0]));
            float a0, a1;
            ki::unpair(a0, a1, A[0]);
            m.a[0] = ki::pair(ki::exp2_fast(in.x.x * a0), 0.0f);
            m.add[0] = ki::pair(in.x.y * b, 0.0f);
            m.c[0] = ki::pair(c, 0.0f);
        } else {
            const ki::f32x2 s = ki::pair(in.x.x), su = ki::pair(in.x.y);
#pragma unroll
            for (int k = 0; k < K; k += 2) {
                ki::f32x2 b;
                if constexpr (sizeof(T) == 4) {
                    b = ki::pair(__uint_as_float(in.w[k]), __uint_as_float(in.w[k + 1]));
                    m.c[k / 2] = ki::pair(__uint_as_float(in.w[K + k]), __uint_as_float(in.w[K + k + 1]));
                } else {
                    b = widen2<T>(in.w[k / 2]);
                    m.c[k / 2] = widen2<T>(in.w[(K + k) / 2]);
                }
                float e0, e1;
                ki::unpair(e0, e1, ki::mul2(s, A[k / 2]));
                m.a[k / 2] = ki::pair(ki::exp2_fast(e0), ki::exp2_fast(e1));
                m.add[k / 2] = ki::mul2(su, b);
            }
        }
        return m;
    }
    __device__ __forceinline__ float apply(const Mid& m) {
        float lo, hi;
        if constexpr (K == 1) {
            float a, add, c;
            ki::unpair(a, hi, m.a[0]);
            ki::unpair(add, hi, m.add[0]);
            ki::unpair(c, hi, m.c[0]);
            ki::unpair(lo, hi, h[0]);
            lo = fmaf(a, lo, add);
            h[0] = ki::pair(lo, 0.0f);
            return PAD != kNoPad && held == 0 ? 0.0f : c * lo;
        } else {
            ki::f32x2 sum = 0;
#pragma unroll
            for (int k = 0; k < P; ++k) {
                h[k] = ki::fma2(m.a[k], h[k], m.add[k]);
                ki::f32x2 v = h[k];
                if constexpr (PAD == kPadStates) {
                    ki::unpair(lo, hi, v);
                    v = ki::pair(2 * k < held ? lo : 0.0f, 2 * k + 1 < held ? hi : 0.0f);
                }
                sum = k == 0 ? ki::mul2(m.c[k], v) : ki::fma2(m.c[k], v, sum);
            }
            ki::unpair(lo, hi, sum);
            return PAD == kPadLanes && held == 0 ? 0.0f : lo + hi;
        }
    }
    // Tokens 0 to tn of a chunk.  The arrays do not overlap: loads of later tokens pass the stores of earlier ones.
    // Loads ahead wrap around at the chunk's end; what they bring is not used.
    __device__ __forceinline__ void chunk(const float2* __restrict__ step, const uint32_t* __restrict__ bc,
                                          float* __restrict__ part, int tn, int tid) {
        auto at = [&](int t) { return L::part_at(t, tid >> 2) * 4 + (tid & 3); };
        if (tn >= kTime) {
            Mid m = decays(load(step, bc, 0));
            In in = load(step, bc, 1);
#pragma unroll 1
            for (int t0 = 0; t0 < kTime; t0 += kUnroll) {
#pragma unroll
                for (int t = 0; t < kUnroll; ++t) {
                    const In in2 = load(step, bc, t + 2 < kUnroll ? t0 + t + 2 : (t0 + t + 2) & (kTime - 1));
                    const Mid m2 = decays(in);
                    part[at(t0 + t)] = apply(m);
                    m = m2;
                    in = in2;
                }
            }
        } else {
            for (int t = 0; t < tn; ++t) part[at(t)] = apply(decays(load(step, bc, t)));
        }
    }
};

// The sequence that is rank-th by length, the longest first (equal ones in order): with more blocks than SMs, a long
// sequence that starts last would run alone at the end.  At most kSort sequences, one for each thread; run by the whole
// block.  (More sequences are taken in order: a longer sort in every block was not tried.)
constexpr int kSort = kLanes + kHelpers;
__device__ __forceinline__ int longest(const ki::Sequences& q, int rank, int* lengths) {
    __shared__ int found;
    const int i = threadIdx.x;
    const int mine = i < q.count ? max(0, q.begin(i + 1) - q.begin(i)) : 0;
    lengths[i] = mine;
    __syncthreads();
    int before = 0;
    for (int j = 0; j < q.count; ++j) before += lengths[j] > mine || (lengths[j] == mine && j < i);
    if (i < q.count && before == rank) found = i;
    __syncthreads();
    return found;
}

template <class T, int LPC, int K, Pad PAD>
__global__ void __launch_bounds__(kLanes + kHelpers, Tile<T, LPC, K>::NP <= 64 ? 2 : 1)
    scan_kernel(const ScanArgs a, int tiles) {
    using L = Tile<T, LPC, K>;
    constexpr int DT = L::DT, VC = L::VC, NB = L::NB;
    extern __shared__ __align__(16) uint8_t smem[];
    typename L::Stage* stage = reinterpret_cast<typename L::Stage*>(smem);
    const ki::Sequences& q = a.seq;
    if (blockIdx.x == 0) q.check(threadIdx.x, kLanes + kHelpers);
    int seq = blockIdx.x / (tiles * a.groups);
    const int rest = blockIdx.x % (tiles * a.groups);
    if (a.sort) seq = longest(q, seq, reinterpret_cast<int*>(smem));
    const int g = rest / tiles;
    const int per = a.channels / a.groups;
    const int in0 = (rest % tiles) * DT;  // first channel within the group
    const int width = min(DT, per - in0);
    const int d0 = g * per + in0;
    const int b0 = q.begin(seq), len = max(0, q.begin(seq + 1) - b0);
    float* st = nullptr;
    if (a.state) {
        const int64_t slot = q.slot(seq);
        if (slot < 0) return;  // padding: its rows and state stay as they are
        st = a.state + (size_t)slot * a.state_ld;
    }
    const int chunks = (len + kTime - 1) / kTime;

    if (threadIdx.x < kLanes) {
        const int dl = threadIdx.x / LPC, ln = threadIdx.x % LPC;
        const bool keep = st && q.continues(seq);
        Lane<T, LPC, K, PAD> lane;
        lane.held = min(max(a.states - ln * K, 0), K);
        float A[2 * lane.P] = {}, h[2 * lane.P] = {};
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const bool on = dl < width && ln * K + k < a.states;
            const size_t at = (size_t)(d0 + dl) * a.states + ln * K + k;
            A[k] = on ? ki::times_log2e(a.A[at]) : 0.0f;
            h[k] = on && keep ? st[at] : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < lane.P; ++k) {
            asm volatile("mov.b64 %0, {%1, %2};" : "=l"(lane.A[k]) : "f"(A[2 * k]), "f"(A[2 * k + 1]));
            lane.h[k] = ki::pair(h[2 * k], h[2 * k + 1]);
        }
        __syncthreads();
        for (int i = 0; i < chunks; ++i) {
            typename L::Stage& s = stage[i & 1];
            lane.chunk(s.step + dl, s.bc + ln * L::GW, reinterpret_cast<float*>(s.part), len - i * kTime, threadIdx.x);
            __syncthreads();
        }
        if (st) {
#pragma unroll
            for (int k = 0; k < lane.P; ++k) ki::unpair(h[2 * k], h[2 * k + 1], lane.h[k]);
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (dl < width && ln * K + k < a.states) st[(size_t)(d0 + dl) * a.states + ln * K + k] = h[k];
        }
        return;
    }

    // Helper threads: VC channels, and a share of B and C, of one token of each chunk.
    const int tid = threadIdx.x - kLanes, t = tid / kShare, sh = tid % kShare;
    const int c0 = sh * VC, n = min(max(width - c0, 0), VC);
    const T* u = static_cast<const T*>(a.u) + d0 + c0;
    const T* delta = static_cast<const T*>(a.delta) + d0 + c0;
    const T* z = a.z ? static_cast<const T*>(a.z) + d0 + c0 : nullptr;
    T* y = static_cast<T*>(a.y) + d0 + c0;
    const T* B = static_cast<const T*>(a.B) + (size_t)g * a.states + sh * NB;
    const T* C = static_cast<const T*>(a.C) + (size_t)g * a.states + sh * NB;
    const int states = min(max(a.states - sh * NB, 0), NB);
    float bias[VC], skip[VC];
#pragma unroll
    for (int j = 0; j < VC; ++j) {
        bias[j] = a.delta_bias && j < n ? a.delta_bias[d0 + c0 + j] : 0.0f;
        skip[j] = a.D && j < n ? a.D[d0 + c0 + j] : 0.0f;
    }
    constexpr bool kAhead = NB <= 8;  // few enough states to be loaded a chunk ahead
    constexpr int NC = kAhead ? NB : K;
    struct Loads {
        Raw<T, VC> delta, u;
        Raw<T, NC> b, c;
    } next = {}, now = {};         // the chunk after the next one (in flight), the next one
    Raw<T, VC> u1 = {}, u0, znext = {}, z0;  // u of the chunk being computed and of the one before it; z of those

    auto load = [&](int i) {
        const int at = i * kTime + t;
        if (at >= len) return;
        const size_t row = (size_t)b0 + at;
        next.delta.load(delta + row * a.ldd, a.vec, n);
        next.u.load(u + row * a.ldu, a.vec, n);
        if constexpr (kAhead) {
            next.b.load(B + row * a.ldb, a.vec_b, states);
            next.c.load(C + row * a.ldc, a.vec_c, states);
        }
        if (n > 0 && at + 2 * kTime < len) {  // DRAM's part of the latency is taken two chunks earlier still
            const size_t far = row + 2 * kTime;
            prefetch(delta + far * a.ldd);
            prefetch(u + far * a.ldu);
            if (z) prefetch(z + far * a.ldz);
        }
    };
    auto load_z = [&](int i) {
        if (z && i * kTime + t < len) znext.load(z + ((size_t)b0 + (size_t)i * kTime + t) * a.ldz, a.vec, n);
    };
    auto take = [&]() {
        u0 = u1;
        u1 = now.u;
        now = next;
        z0 = znext;
    };
    auto fill = [&](int i) {  // the loaded chunk, as the compute threads want it
        if (i * kTime + t >= len) return;
        typename L::Stage& s = stage[i & 1];
        float2* step = s.step + t * L::ROW + c0;
#pragma unroll
        for (int j = 0; j < VC; j += 2) {
            constexpr int one = VC > 1 ? 1 : 0;
            float x0 = ki::to_f32(now.delta.get(j)) + bias[j], x1 = ki::to_f32(now.delta.get(j + one)) + bias[j + one];
            if (a.soft) x0 = ki::softplus(x0), x1 = ki::softplus(x1);
            const float v0 = x0 * ki::to_f32(now.u.get(j)), v1 = x1 * ki::to_f32(now.u.get(j + one));
            step[j] = make_float2(x0, v0);
            if (one) step[j + one] = make_float2(x1, v1);
        }
        const size_t row = (size_t)b0 + (size_t)i * kTime + t;
#pragma unroll
        for (int j = 0; j < NB; j += K) {  // a compute lane's states
            if constexpr (!kAhead) {
                now.b.load(B + row * a.ldb + j, a.vec_b, states - j);
                now.c.load(C + row * a.ldc + j, a.vec_c, states - j);
            }
            const int at = kAhead ? j : 0;
            uint32_t w[L::GW];
            if constexpr (K * sizeof(T) >= 4) {
#pragma unroll
                for (int k = 0; k < L::GW / 2; ++k) {
                    w[k] = now.b.w[at * (int)sizeof(T) / 4 + k];
                    w[L::GW / 2 + k] = now.c.w[at * (int)sizeof(T) / 4 + k];
                }
            } else {
                w[0] = now.b.half(at) | now.c.half(at) << 16;
            }
            constexpr int W = L::GW < 4 ? L::GW : 4;
            uint32_t* to = s.bc + (t * LPC + (sh * NB + j) / K) * L::GW;
#pragma unroll
            for (int k = 0; k < L::GW; k += W) {
                ki::Vec<uint32_t, W> v;
#pragma unroll
                for (int e = 0; e < W; ++e) v.e[e] = w[k + e];
                ki::store_vec(to + k, v);
            }
        }
    };
    auto finish = [&](int i) {  // outputs of a computed chunk
        if (i * kTime + t >= len || n == 0) return;
        const size_t row = (size_t)b0 + (size_t)i * kTime + t;
        typename L::Stage& s = stage[i & 1];
        float v[VC];
#pragma unroll
        for (int j = 0; j < VC; ++j) {
            v[j] = 0.0f;
#pragma unroll
            for (int k = 0; k < LPC / 4; ++k) {
                const float4 p = s.part[L::part_at(t, (c0 + j) * (LPC / 4) + k)];
                v[j] += (p.x + p.y) + (p.z + p.w);
            }
            if (a.D) v[j] = fmaf(skip[j], ki::to_f32(u0.get(j)), v[j]);
            if (z) v[j] *= ki::silu(ki::to_f32(z0.get(j)));
        }
        Raw<T, VC> out;
        out.set(v);
        out.store(y + row * a.ldy, a.vec, n);
    };

    load(0);
    take();
    load(1);
    fill(0);
    __syncthreads();
    for (int i = 0; i < chunks; ++i) {
        take();
        load(i + 2);
        load_z(i);
        if (i > 0) finish(i - 1);
        fill(i + 1);
        __syncthreads();
    }
    take();
    if (chunks > 0) finish(chunks - 1);
}

// One token per row: row r continues slot slots[r].  Bound: the states' bytes (one read and one write; 128 x 4096 x 16:
// 18.3 us, 3.9 TB/s; one row at a time 26.5, two 20.5), so LPC lanes
// share a channel with K states each (16 bytes and more per access) and take R rows at once: A is read once for them and
// their states' loads are in flight together.  What is done once per row and channel (the step, the gate) is done
// by lane r of the group for row r.
template <class T, int LPC, int K, int R>
__global__ void __launch_bounds__(kStepThreads) scan_step_kernel(const ScanArgs a, int tiles) {
    static_assert(LPC >= R, "a lane per row");
    constexpr int DT = kStepThreads / LPC;
    const int r0 = (int)(blockIdx.x / tiles) * R;
    const int d = (int)(blockIdx.x % tiles) * DT + (int)threadIdx.x / LPC;
    const int lane = threadIdx.x % LPC, n0 = lane * K;
    const bool live = d < a.channels;
    const int n = live ? min(max(a.states - n0, 0), K) : 0;
    const int g = live ? d / (a.channels / a.groups) : 0;

    int64_t slot[R];
#pragma unroll
    for (int r = 0; r < R; ++r) slot[r] = r0 + r < a.seq.count ? a.seq.slot(r0 + r) : -1;
    Raw<float, K> h[R];
    Raw<T, K> b[R], c[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (slot[r] < 0) continue;
        h[r].load(a.state + (size_t)slot[r] * a.state_ld + (size_t)d * a.states + n0, a.vec, n);
        b[r].load(static_cast<const T*>(a.B) + (size_t)(r0 + r) * a.ldb + (size_t)g * a.states + n0, a.vec_b, n);
        c[r].load(static_cast<const T*>(a.C) + (size_t)(r0 + r) * a.ldc + (size_t)g * a.states + n0, a.vec_c, n);
    }
    Raw<float, K> A;
    A.load(a.A + (size_t)d * a.states + n0, a.vec, n);
    float s = 0.0f, u = 0.0f, z = 0.0f;  // of row r0 + lane
    const int row = r0 + lane;
    const bool mine = lane < R && row < a.seq.count && live;
    if (mine) {
        u = ki::to_f32(static_cast<const T*>(a.u)[(size_t)row * a.ldu + d]);
        s = ki::to_f32(static_cast<const T*>(a.delta)[(size_t)row * a.ldd + d]);
        if (a.z) z = ki::to_f32(static_cast<const T*>(a.z)[(size_t)row * a.ldz + d]);
        if (a.delta_bias) s += a.delta_bias[d];
        if (a.soft) s = ki::softplus(s);
    }
    const float s2 = ki::times_log2e(s);
    float y = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float sr = __shfl_sync(0xffffffffu, s2, r, LPC);
        const float su = __shfl_sync(0xffffffffu, s * u, r, LPC);
        float p = 0.0f;
        if (slot[r] >= 0 && live) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const float v = fmaf(ki::exp2_fast(sr * A.get(k)), h[r].get(k), su * ki::to_f32(b[r].get(k)));
                h[r].w[k] = __float_as_uint(v);
                if (k < n) p = fmaf(ki::to_f32(c[r].get(k)), v, p);
            }
            h[r].store(a.state + (size_t)slot[r] * a.state_ld + (size_t)d * a.states + n0, a.vec, n);
        }
#pragma unroll
        for (int x = LPC / 2; x >= 1; x /= 2) p += __shfl_xor_sync(0xffffffffu, p, x);
        if (lane == r) y = p;
    }
    if (mine && a.seq.slot(row) >= 0) {
        if (a.D) y = fmaf(a.D[d], u, y);
        if (a.z) y *= ki::silu(z);
        static_cast<T*>(a.y)[(size_t)row * a.ldy + d] = ki::from_f32<T>(y);
    }
}

template <class T, int LPC, int K, Pad PAD>
int launch_padded(ki_ctx* ctx, ScanArgs& a, cudaStream_t s) {
    using L = Tile<T, LPC, K>;
    const int per = a.channels / a.groups;
    const long long tiles = (per + L::DT - 1) / L::DT;
    const long long blocks = tiles * a.groups * a.seq.count;
    if (blocks > 0x7fffffffll) return ki::set_error(ctx, KI_ERR_ARG, "selective_scan: too many sequences");
    const size_t es = sizeof(T), w = L::VC * es > 16 ? 16 : L::VC * es;
    const bool one = a.seq.tokens <= 1;
    a.vec = ki::rows_aligned(a.u, one ? 0 : a.ldu, es, w) && ki::rows_aligned(a.delta, one ? 0 : a.ldd, es, w) &&
            ki::rows_aligned(a.z, one || !a.z ? 0 : a.ldz, es, w) && ki::rows_aligned(a.y, one ? 0 : a.ldy, es, w) &&
            (a.groups == 1 || per * es % w == 0);
    const size_t wb = (L::NB <= 8 ? L::NB : K) * es, wv = wb > 16 ? 16 : wb;
    const bool whole = a.groups == 1 || a.states * es % wv == 0;
    a.vec_b = whole && ki::rows_aligned(a.B, one ? 0 : a.ldb, es, wv);
    a.vec_c = whole && ki::rows_aligned(a.C, one ? 0 : a.ldc, es, wv);
    constexpr int smem = 2 * sizeof(typename L::Stage);
    a.sort = a.seq.count > 1 && a.seq.count <= kSort && blocks > ctx->sm_count;
    auto kern = scan_kernel<T, LPC, K, PAD>;
    KI_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    kern<<<(unsigned)blocks, kLanes + kHelpers, smem, s>>>(a, (int)tiles);
    return ki::check_launch(ctx, "selective_scan launch");
}

template <class T, int LPC, int K>
int launch(ki_ctx* ctx, ScanArgs& a, cudaStream_t s) {
    if (a.states == LPC * K) return launch_padded<T, LPC, K, kNoPad>(ctx, a, s);
    if (K == 1 || a.states % K == 0) return launch_padded<T, LPC, K, kPadLanes>(ctx, a, s);
    return launch_padded<T, LPC, K, K == 1 ? kPadLanes : kPadStates>(ctx, a, s);
}

template <class T>
int launch_scan(ki_ctx* ctx, ScanArgs& a, cudaStream_t s) {
    // Blocks if every lane held four states.  A lane with fewer takes less time for a token (D = 256, 2048 tokens, N = 16:
    // 77 us with four states, 54 with two, 43 with one), but more of the SM's issue slots in all, so fewer states pay
    // while every block has an SM of its own (D = 4096: 79, 85, 128 us).
    const int per = a.channels / a.groups, sms = ctx->sm_count;
    auto blocks = [&](int channels) { return (long long)a.seq.count * a.groups * ((per + channels - 1) / channels); };
    if (a.states <= 8) return blocks(16) <= sms ? launch<T, 8, 1>(ctx, a, s) : launch<T, 4, 2>(ctx, a, s);
    if (a.states <= 16) {
        if (blocks(8) <= sms) return launch<T, 16, 1>(ctx, a, s);
        return blocks(16) <= sms ? launch<T, 8, 2>(ctx, a, s) : launch<T, 4, 4>(ctx, a, s);
    }
    if (a.states <= 32) return blocks(8) <= sms ? launch<T, 16, 2>(ctx, a, s) : launch<T, 8, 4>(ctx, a, s);
    if (a.states <= 64) return launch<T, 16, 4>(ctx, a, s);
    if (a.states <= 128) return launch<T, 16, 8>(ctx, a, s);
    return launch<T, 32, 8>(ctx, a, s);
}

template <class T, int LPC, int K, int R>
int launch_rows(ki_ctx* ctx, ScanArgs& a, cudaStream_t s) {
    constexpr int DT = kStepThreads / LPC;
    const long long tiles = (a.channels + DT - 1) / DT;
    const long long blocks = tiles * ((a.seq.count + R - 1) / R);
    if (blocks > 0x7fffffffll) return ki::set_error(ctx, KI_ERR_ARG, "selective_scan_step: too many rows");
    const size_t es = sizeof(T), w = K * es > 16 ? 16 : K * es;
    const bool one = a.seq.count <= 1;
    a.vec = a.states % 4 == 0 && ki::aligned(a.A, 16) && ki::rows_aligned(a.state, a.seq.nslots > 1 ? a.state_ld : 0, 4, 16);
    a.vec_b = (a.groups == 1 || a.states * es % w == 0) && ki::rows_aligned(a.B, one ? 0 : a.ldb, es, w);
    a.vec_c = (a.groups == 1 || a.states * es % w == 0) && ki::rows_aligned(a.C, one ? 0 : a.ldc, es, w);
    scan_step_kernel<T, LPC, K, R><<<(unsigned)blocks, kStepThreads, 0, s>>>(a, (int)tiles);
    return ki::check_launch(ctx, "selective_scan_step launch");
}

template <class T, int LPC, int K>
int launch_step_lanes(ki_ctx* ctx, ScanArgs& a, cudaStream_t s) {
    // several rows per block where that still leaves two blocks for every SM
    constexpr int DT = kStepThreads / LPC;
    const long long tiles = (a.channels + DT - 1) / DT;
    if (LPC >= 4 && tiles * ((a.seq.count + 3) / 4) >= 2ll * ctx->sm_count) return launch_rows<T, LPC, K, LPC >= 4 ? 4 : 1>(ctx, a, s);
    return launch_rows<T, LPC, K, 1>(ctx, a, s);
}

template <class T>
int launch_step(ki_ctx* ctx, ScanArgs& a, cudaStream_t s) {
    if (a.states <= 8) return launch_step_lanes<T, 4, 2>(ctx, a, s);
    if (a.states <= 16) return launch_step_lanes<T, 4, 4>(ctx, a, s);
    if (a.states <= 32) return launch_step_lanes<T, 8, 4>(ctx, a, s);
    if (a.states <= 64) return launch_step_lanes<T, 16, 4>(ctx, a, s);
    if (a.states <= 128) return launch_step_lanes<T, 32, 4>(ctx, a, s);
    return launch_step_lanes<T, 32, 8>(ctx, a, s);
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
    if (seqs > ki::kMaxSequences || slots > 0x7fffffffffu)
        return ki::set_error(ctx, KI_ERR_ARG, "selective_scan: too many sequences or slots");
    if (!d_offsets && seqs != 1) return ki::set_error(ctx, KI_ERR_ARG, "selective_scan: several sequences need offsets");
    ScanArgs a{d_u, ldu, d_delta, ldd, d_A, d_B, ldb, d_C, ldc, d_D, d_z, ldz, d_delta_bias, d_state, state_ld, d_y, ldy,
               0, 0, 0, softplus != 0, false, false, false, false, {d_offsets, d_slots, d_initial, (int)seqs, 0, (int64_t)slots, nullptr}};
    return scan(ctx, "selective_scan", dtype, a, tokens, channels, states, groups, false, stream);
}

extern "C" int ki_selective_scan_step(ki_ctx* ctx, int dtype, const void* d_u, size_t ldu, const void* d_delta, size_t ldd,
                                      const float* d_A, const void* d_B, size_t ldb, const void* d_C, size_t ldc,
                                      const float* d_D, const void* d_z, size_t ldz, const float* d_delta_bias,
                                      int softplus, float* d_state, size_t state_ld, size_t slots, const int32_t* d_slots,
                                      void* d_y, size_t ldy, size_t rows, size_t channels, size_t states, size_t groups,
                                      void* stream) {
    KI_CHECK_CTX(ctx);
    if (rows > ki::kMaxSequences || slots > 0x7fffffffffu)
        return ki::set_error(ctx, KI_ERR_ARG, "selective_scan_step: too many rows or slots");
    if (!d_state) return ki::set_error(ctx, KI_ERR_ARG, "selective_scan_step: null pointer");
    ScanArgs a{d_u, ldu, d_delta, ldd, d_A, d_B, ldb, d_C, ldc, d_D, d_z, ldz, d_delta_bias, d_state, state_ld, d_y, ldy,
               0, 0, 0, softplus != 0, false, false, false, false, {nullptr, d_slots, nullptr, (int)rows, 0, (int64_t)slots, nullptr}};
    return scan(ctx, "selective_scan_step", dtype, a, rows, channels, states, groups, true, stream);
}
