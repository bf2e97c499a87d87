// gemm_i8.cu -- ki_gemm_i8: the product of int8 tokens and int8 weights on the tensor cores
// (tcgen05 kind::i8, Int32 accumulators in TMEM), with a scale for each token and each channel.
//
//   C[m, n] = float(sum_k A[m, k] W[n, k]) * scale_a[m] * scale_w[n] (+ bias[n])
//
// A: tokens x inner, W: channels x inner, both row-major (so both operands are K-major), C: tokens x
// channels in Float32, Float16 or BFloat16.  The Int32 sums are exact (inner <= 131071, where 128 * 128
// * inner still fits), so the result does not depend on the order of the sums or on how they are split.
//
// The weights are the MMA's M side: lanes of TMEM are channels and columns are tokens.  A warp's store of one column
// is then 32 neighbouring channels of one token, whatever the sizes and strides of C, and a few tokens cost a few
// columns instead of a mostly empty tile of 128 rows.  Two kernels:
//
// gemm_i8_kernel, one tile of 128 channels x BN tokens per CTA:
//   warp 0     loads K blocks of 128 into a ring of stages (TMA, 128-byte swizzle);
//   warp 1     allocates TMEM and issues the MMAs (M 128, N BN, K 32) from one thread;
//   warps 2-5  (2-9 from BN = 64) epilogue: TMEM -> registers -> scales -> C.
// With few tiles the K blocks of a tile are split over the CTAs of a cluster; each CTA then leaves its
// Int32 sums in its own shared memory and adds up and stores a share of the tile's columns, read from
// every CTA of the cluster.  Rows that are not 16-byte aligned are loaded by warps 2-17 (2-19 from BN = 160) with plain loads.
//
// gemm_i8_pair_kernel, persistent CTA pairs on tiles of 256 channels x 256 tokens (cta_group::2): each CTA loads
// 128 rows of either operand, each SM's TMEM holds two accumulators of its 128 channels x 256 tokens, so that the
// epilogue of a tile runs beside the next tile's MMAs.
//
// Bounds and times (M x N x K, bf16 out; one B200): 8192 x 8192 x 4096 183-190 us, 2.9-3.0 P operations/s (tensor pipe 72 %
// busy at 4096^3; the epilogue beside it: 236 us with four epilogue warps and scales from shuffles).  512 x 4096 x 4096 13.9 us.
// 48 x 8192 x 4096 11.8 us and 1 x 4096 x 4096 6.4 us: the weight's bytes (5.3 and 2.6 us) and the latency of a launch, of the
// first loads and of the join.  1111 x 4099 x 2057, rows at any byte: 52.5 us, bound by the loading warps (the
// integer pipe is 54 % busy with shifting the loaded words into place).
//
// Every mbarrier wait is bounded, as in gemm_e4m3.cu.
#include "ki/layer.cuh"
#include "ki/lookback.cuh"
#include "ki/tcgen05.cuh"

namespace {

constexpr int BM = 128, BK = 128;
constexpr int W_BYTES = BM * BK;
constexpr int MAX_SPLIT = 8;

// D = S32 (2), A = S8 (1), B = S8 (1), both K-major
constexpr uint32_t idesc(int bn) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(bn >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
}

template <int BN, bool TMA>
struct Shape {
    static constexpr int X_BYTES = BN * BK;
    static constexpr int STAGE_BYTES = W_BYTES + X_BYTES;
    // two CTAs per SM, but one with a deeper ring for the widest tiles (and where threads load the rows: their registers)
    static constexpr int STAGES = BN <= 16 ? 6 : BN <= 32 ? 5 : BN <= 64 ? 4 : BN <= 128 ? 6 : 5;
    static constexpr int SUM_BYTES = BM * BN * 4;  // a split's Int32 sums, over the ring
    static constexpr int RING_BYTES = STAGES * STAGE_BYTES > SUM_BYTES ? STAGES * STAGE_BYTES : SUM_BYTES;
    static constexpr int SA_COLS = BN < 32 ? 32 : BN;  // the tokens' scales, behind the barriers
    static constexpr int SMEM_BYTES = 1024 + RING_BYTES + 256 + 4 * SA_COLS;
    static constexpr int TMEM_COLS = BN < 32 ? 32 : BN <= 128 ? BN : 256;
    static constexpr int EPI_WARPS = BN < 64 ? 4 : 8;  // four per 32 TMEM lanes, or eight with half of the columns each
    static constexpr int EPI_COLS = BN < 64 ? TMEM_COLS : (BN / 2 + 31) / 32 * 32;
    static constexpr int LOADERS = BN <= 128 ? 16 : (BM + BN) / 16;  // warps that load rows which TMA cannot, 16 each
    static constexpr int THREADS = 64 + 32 * (TMA ? EPI_WARPS : LOADERS);
};

struct GemmArgs {
    const int8_t* a;
    size_t lda;
    const int8_t* w;
    size_t ldw;
    const float* sa;
    const float* sw;
    const float* bias;
    void* c;
    size_t ldc;
    int m, n, k;
    int mtiles, ntiles;
    uint32_t* status;
    uint64_t timeout_ns;
};

__device__ __forceinline__ void mma_i8(uint32_t d_tmem, uint64_t wdesc, uint64_t xdesc, uint32_t id, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(wdesc), "l"(xdesc), "r"(id), "r"(accumulate)
        : "memory");
}

// 16 rows of a matrix, a K block at a time, loaded by one warp from rows that start at any byte.  Eight lanes share a
// row and load its 16-byte words, as they lie aligned in memory, four rows at once.  A lane's 16 bytes of the block are
// then its word and the next one, shifted by the row's misalignment; the word behind the last lane's is the first of the
// next block, which is loaded by then.  Only words that hold a byte of a row are read; what lies behind the rows' end is
// zero, and rows that do not exist hold anything finite, since their outputs are not stored.
struct Rows {
    static constexpr int N = 16, G = N / 4;
    const int8_t* x;  // this lane's word of its first row (aligned to 16 bytes), K block 0
    size_t step;      // bytes from a row to the fourth after it
    int rows;         // rows of this lane's that exist: its own, and every fourth after it
    int k;            // bytes of a row that exist, counted from x's row's start
    int lane;
    uint32_t off[G];  // misalignment of this lane's rows
    struct Words {
        uint4 v[G];
    };
    __device__ __forceinline__ Rows(const int8_t* base, size_t ld, int row0, int end, int k_, int lane_) : k(k_), lane(lane_) {
        const int r = lane >> 3;
        const int8_t* p = base + (size_t)(row0 + r) * ld;
        x = p + 16 * (lane & 7);
        step = 4 * ld;
        rows = (end - row0 - r + 3) / 4;
#pragma unroll
        for (int g = 0; g < G; ++g) off[g] = (uint32_t)(uintptr_t)(p + g * step) & 15;  // the same in every K block
    }
    // The words of the block that starts with byte k0 of the rows (k0 may lie behind their end, and k is positive).
    __device__ __forceinline__ void load(Words& w, int k0) const {
#pragma unroll
        for (int g = 0; g < G; ++g) {
            w.v[g] = make_uint4(0, 0, 0, 0);
            if (g < rows && 16 * (lane & 7) < (int)off[g] + k - k0)
                w.v[g] = __ldg(reinterpret_cast<const uint4*>(x + g * step + k0 - off[g]));
        }
    }
    // To shared memory at dst, as a TMA tile with the 128-byte swizzle: row r at 128 r, its 16-byte pieces exchanged by
    // r mod 8.
    __device__ __forceinline__ void store(const Words& w, const Words& next, uint32_t dst, int k0) const {
        const int j = lane & 7, from = (lane & ~7) | ((j + 1) & 7);
#pragma unroll
        for (int g = 0; g < G; ++g) {
            uint32_t a[8] = {w.v[g].x, w.v[g].y, w.v[g].z, w.v[g].w};
            const uint32_t n[4] = {next.v[g].x, next.v[g].y, next.v[g].z, next.v[g].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) a[4 + i] = __shfl_sync(0xffffffffu, j == 0 ? n[i] : a[i], from);
            // left by whole words, then by bytes
            const bool one = off[g] & 4, two = off[g] & 8;
#pragma unroll
            for (int i = 0; i < 7; ++i) a[i] = one ? a[i + 1] : a[i];
#pragma unroll
            for (int i = 0; i < 5; ++i) a[i] = two ? a[i + 2] : a[i];
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = __funnelshift_r(a[i], a[i + 1], 8 * (off[g] & 3));
            if (k - k0 < BK) {  // bytes behind the end
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int left = min(max(k - k0 - 16 * j - 4 * i, 0), 4);
                    a[i] &= left == 4 ? 0xffffffffu : (1u << (8 * left)) - 1u;
                }
            }
            const int r = (lane >> 3) + 4 * g;
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + (uint32_t)(r * 128 + ((j ^ (r & 7)) << 4))),
                         "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3])
                         : "memory");
        }
    }
};

template <class O>
__device__ __forceinline__ O scaled(int32_t v, float sa, float sw, float bias) {
    return ki::from_f32<O>(fmaf((float)v * sa, sw, bias));
}

// 32 tokens' sums of a channel: scaled and stored to column c of their rows, as many as there are.
template <class O>
__device__ __forceinline__ void store_columns(O* c, size_t ldc, const uint32_t (&v)[32], const float* sa, float sw,
                                              float bias, int count) {
    if (count >= 32) {
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
            const float4 s = *reinterpret_cast<const float4*>(sa + j);
            c[0] = scaled<O>((int)v[j], s.x, sw, bias);
            c[ldc] = scaled<O>((int)v[j + 1], s.y, sw, bias);
            c[2 * ldc] = scaled<O>((int)v[j + 2], s.z, sw, bias);
            c[3 * ldc] = scaled<O>((int)v[j + 3], s.w, sw, bias);
            c += 4 * ldc;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if (j < count) c[(size_t)j * ldc] = scaled<O>((int)v[j], sa[j], sw, bias);
    }
}

template <int BN, class O, bool TMA>
__global__ void __launch_bounds__(Shape<BN, TMA>::THREADS, 1)
    gemm_i8_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW, const GemmArgs g,
                   int split) {
    using S = Shape<BN, TMA>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t raw = ki::smem_addr(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    const uint32_t ring = base, bars = base + S::RING_BYTES;
    const uint32_t full0 = bars, empty0 = bars + 8 * S::STAGES, tfull = bars + 16 * S::STAGES;
    uint8_t* gbase = smem_raw + (base - raw);
    volatile int* abort = reinterpret_cast<volatile int*>(gbase + S::RING_BYTES + 128);
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(gbase + S::RING_BYTES + 136);
    float* scales = reinterpret_cast<float*>(gbase + S::RING_BYTES + 256);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int part = blockIdx.x % split, tile = blockIdx.x / split;
    const int n0 = (tile % g.ntiles) * BM, m0 = (tile / g.ntiles) * BN, end = min(g.m, m0 + BN);
    const int blocks = (g.k + BK - 1) / BK;
    const int kb0 = (int)((long long)blocks * part / split), kb1 = (int)((long long)blocks * (part + 1) / split);

    for (int i = threadIdx.x; i < S::SA_COLS; i += blockDim.x) scales[i] = m0 + i < end ? g.sa[m0 + i] : 0.0f;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::STAGES; ++s) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(full0 + 8 * s), "r"(TMA ? 1 : S::LOADERS));
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(empty0 + 8 * s));
        }
        asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(tfull));
        *abort = 0;
        ki::fence_mbar_init();
        if (TMA) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&tmA) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&tmW) : "memory");
        }
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(ki::smem_addr(tmem_holder)),
                     "r"(S::TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_holder;

    if (TMA && warp == 0) {
        if (lane == 0) {
            int s = 0;
            uint32_t ph = 1;
            int last_kb = kb0;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!wait_bar(empty0 + 8 * s, ph, abort, g.status, g.timeout_ns)) break;
                const uint32_t sw = ring + s * S::STAGE_BYTES;
                mbar_expect_tx(full0 + 8 * s, S::STAGE_BYTES);
                tma_load_2d(sw, &tmW, kb * BK, n0, full0 + 8 * s);
                tma_load_2d(sw + W_BYTES, &tmA, kb * BK, m0, full0 + 8 * s);
                last_kb = kb + 1;
                if (++s == S::STAGES) {
                    s = 0;
                    ph ^= 1;
                }
            }
            if (*abort) {  // loads may still be in flight: wait (bounded) until each stage's last one landed
                for (int i = kb0 > last_kb - S::STAGES ? kb0 : last_kb - S::STAGES; i < last_kb; ++i)
                    wait_drain(full0 + 8 * ((i - kb0) % S::STAGES), ((i - kb0) / S::STAGES) & 1, g.status, g.timeout_ns);
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            int s = 0;
            uint32_t ph = 0;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!wait_bar(full0 + 8 * s, ph, abort, g.status, g.timeout_ns)) break;
                tc_fence_after();
                const uint32_t sw = ring + s * S::STAGE_BYTES;
                const uint64_t wdesc = make_desc(sw, 16, 1024), xdesc = make_desc(sw + W_BYTES, 16, 1024);
#pragma unroll
                for (int k = 0; k < BK / 32; ++k)
                    mma_i8(tmem, wdesc + (uint64_t)(2 * k), xdesc + (uint64_t)(2 * k), idesc(BN), kb != kb0 || k != 0);
                mma_commit(empty0 + 8 * s);
                if (++s == S::STAGES) {
                    s = 0;
                    ph ^= 1;
                }
            }
            // every MMA issued has finished before the sums are read and TMEM and the ring are released
            mma_commit(tfull);
            wait_drain(tfull, 0, g.status, g.timeout_ns);
        }
    } else if (!TMA && warp >= 2) {
        // W's 128 rows, then A's BN, 16 to a warp
        static_assert(BM + BN <= Rows::N * S::LOADERS && BN % Rows::N == 0, "16 rows per warp");
        const int r0 = Rows::N * (warp - 2);
        const bool some = r0 < BM + BN && kb0 < kb1, isw = r0 < BM;  // without an inner dimension there is nothing to read
        const Rows rows(isw ? g.w : g.a, isw ? g.ldw : g.lda, isw ? n0 + r0 : m0 + r0 - BM, isw ? g.n : end,
                        g.k, lane);
        int s = 0;
        uint32_t ph = 1;
        auto put = [&](const Rows::Words& v, const Rows::Words& behind, int kb) {
            int ok = 0;
            if (lane == 0) ok = wait_bar(empty0 + 8 * s, ph, abort, g.status, g.timeout_ns) ? 1 : 0;
            if (!__shfl_sync(0xffffffffu, ok, 0)) return false;
            if (some) rows.store(v, behind, ring + s * S::STAGE_BYTES + r0 * BK, kb * BK);
            ki::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(full0 + 8 * s);
            if (++s == S::STAGES) {
                s = 0;
                ph ^= 1;
            }
            return true;
        };
        // three blocks in turn: one is stored, the next has to be there, the one after it is in flight
        Rows::Words w0, w1, w2;
        auto load = [&](Rows::Words& w, int kb) {
            if (some) rows.load(w, kb * BK);
        };
        load(w0, kb0);
        load(w1, kb0 + 1);
        for (int kb = kb0; kb < kb1; kb += 3) {
            load(w2, kb + 2);
            if (!put(w0, w1, kb) || kb + 1 >= kb1) break;
            load(w0, kb + 3);
            if (!put(w1, w2, kb + 1) || kb + 2 >= kb1) break;
            load(w1, kb + 4);
            if (!put(w2, w0, kb + 2)) break;
        }
    }
    __syncwarp();

    if (warp >= 2 && warp < 2 + S::EPI_WARPS) {
        int ok = 0;
        if (lane == 0) ok = wait_bar(tfull, 0, abort, g.status, g.timeout_ns) ? 1 : 0;
        ok = __shfl_sync(0xffffffffu, ok, 0);
        tc_fence_after();
        const int row = (warp & 3) * 32;                              // TMEM lanes that this warp may read
        const int first = (warp - 2) / 4 * S::EPI_COLS;               // and its columns
        const int n = n0 + row + lane;
        const bool on = n < g.n;
        const float sw = on ? g.sw[n] : 0.0f, bias = on && g.bias ? g.bias[n] : 0.0f;
        if (ok) {
#pragma unroll 1
            for (int c0 = first; c0 < first + S::EPI_COLS; c0 += 32) {
                if (m0 + c0 >= end) break;
                uint32_t v[32];
                if (kb1 > kb0) {
                    KI_TMEM_LD_X32(tmem + ((uint32_t)row << 16) + (uint32_t)c0, v);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = 0;
                }
                if (split == 1) {
                    if (on)
                        store_columns(static_cast<O*>(g.c) + (size_t)(m0 + c0) * g.ldc + n, g.ldc, v, scales + c0, sw, bias,
                                      end - m0 - c0);
                } else {
#pragma unroll
                    for (int j = 0; j < (BN < 32 ? BN : 32); ++j)
                        asm volatile("st.shared.b32 [%0], %1;" ::"r"(ring + (uint32_t)(((c0 + j) * BM + row + lane) * 4)),
                                     "r"(v[j])
                                     : "memory");
                }
            }
        }
    }
    if (split > 1) {
        __syncwarp();
        cluster_sync_all();  // every part's sums are in its shared memory
        if (!*abort) {
            // this CTA's share of the columns; a thread takes four neighbouring channels of one
            const int n = n0 + 4 * lane, live = min(max(g.n - n, 0), 4);
            const int columns = end - m0;
            float sw[4], bias[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sw[e] = e < live ? g.sw[n + e] : 0.0f;
                bias[e] = e < live && g.bias ? g.bias[n + e] : 0.0f;
            }
            for (int j = part + split * warp; j < columns; j += split * (int)(blockDim.x / 32)) {
                const uint32_t at = ring + (uint32_t)((j * BM + 4 * lane) * 4);
                int4 v[MAX_SPLIT];
#pragma unroll
                for (int p = 0; p < MAX_SPLIT; ++p) {
                    v[p] = make_int4(0, 0, 0, 0);
                    if (p < split)
                        asm volatile("ld.shared::cluster.v4.b32 {%0, %1, %2, %3}, [%4];"
                                     : "=r"(v[p].x), "=r"(v[p].y), "=r"(v[p].z), "=r"(v[p].w)
                                     : "r"(map_rank(at, (uint32_t)p)));
                }
                int sum[4] = {0, 0, 0, 0};
#pragma unroll
                for (int p = 0; p < MAX_SPLIT; ++p) sum[0] += v[p].x, sum[1] += v[p].y, sum[2] += v[p].z, sum[3] += v[p].w;
                const float sa = scales[j];
                O* c = static_cast<O*>(g.c) + (size_t)(m0 + j) * g.ldc + n;
                ki::Vec<O, 4> o;
#pragma unroll
                for (int e = 0; e < 4; ++e) o.e[e] = scaled<O>(sum[e], sa, sw[e], bias[e]);
                if (live == 4 && (reinterpret_cast<uintptr_t>(c) % sizeof(o)) == 0) {
                    ki::store_vec(c, o);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (e < live) c[e] = o.e[e];
                }
            }
        }
        __syncwarp();
        cluster_sync_all();  // no CTA leaves while another may still read its shared memory
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::TMEM_COLS) : "memory");
    }
}

// ---------------------------------------------------------------------------------------------
// CTA pairs: rank r of a pair loads the channels [n0 + 128 r, +128) of W and the tokens [m0 + 128 r, +128) of A of each
// K block (no multicast: every CTA loads only its own half); both CTAs' loads complete on rank 0's full barrier, and
// rank 0's MMA thread issues M=256 N=256 K=32 MMAs that read both CTAs' shared memory at the same offsets.  The commits
// arrive on the empty and accumulator-full barriers of both CTAs, both CTAs' epilogue warps on rank 0's
// accumulator-empty barrier.
// ---------------------------------------------------------------------------------------------
constexpr int TILE2 = 256, STAGES2 = 6, ACCS2 = 2;
constexpr int X2_BYTES = 128 * BK, STAGE2_BYTES = W_BYTES + X2_BYTES;
constexpr int RING2_BYTES = STAGES2 * STAGE2_BYTES;
constexpr int SA2_BYTES = ACCS2 * TILE2 * 4;  // the tokens' scales of the tile in either accumulator
constexpr int SMEM2_BYTES = 1024 + RING2_BYTES + 256 + SA2_BYTES;
constexpr uint32_t IDESC2 = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(TILE2 >> 3) << 17) | ((uint32_t)(TILE2 >> 4) << 24);
constexpr int EPI2_WARPS = 8;  // two per TMEM lane quadrant, half of the columns each
constexpr int THREADS2 = 32 * (2 + EPI2_WARPS);

__device__ __forceinline__ void mma_i8_pair(uint32_t d_tmem, uint64_t wdesc, uint64_t xdesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(wdesc), "l"(xdesc), "r"(IDESC2), "r"(accumulate)
        : "memory");
}

// Output tile t -> (token block, channel block): groups of 16 token blocks are walked channel block by channel block,
// so that the rows of A and W in flight stay in L2.
__device__ __forceinline__ void tile2_coords(int t, int mtiles, int ntiles, int& mb, int& nb) {
    const int group = t / (16 * ntiles), first = group * 16, size = min(16, mtiles - first);
    const int in = t - group * 16 * ntiles;
    mb = first + in % size;
    nb = in / size;
}

template <class O>
__global__ void __launch_bounds__(THREADS2, 1)
    gemm_i8_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW, const GemmArgs g) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t raw = ki::smem_addr(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;  // identical in both CTAs: same kernel, same layout
    const uint32_t ring = base, bars = base + RING2_BYTES;
    const uint32_t full0 = bars, empty0 = bars + 8 * STAGES2, tfull0 = bars + 16 * STAGES2;
    const uint32_t tempty0 = tfull0 + 8 * ACCS2, drain = tempty0 + 8 * ACCS2;
    uint8_t* gbase = smem_raw + (base - raw);
    volatile int* abort = reinterpret_cast<volatile int*>(gbase + RING2_BYTES + 192);
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(gbase + RING2_BYTES + 200);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const bool leader = rank == 0;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES2; ++s) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(full0 + 8 * s));
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(empty0 + 8 * s));
        }
        for (int b = 0; b < ACCS2; ++b) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(tfull0 + 8 * b));
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(tempty0 + 8 * b), "r"(2 * EPI2_WARPS));
        }
        asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(drain));
        *abort = 0;
        ki::fence_mbar_init();
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tmA) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tmW) : "memory");
    }
    if (warp == 1) {  // the same warp in both CTAs allocates the pair's TMEM together
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(ki::smem_addr(tmem_holder)),
                     "r"(ACCS2 * TILE2)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // both CTAs' barriers are initialised before any copy or arrive crosses over
    tc_fence_after();
    const uint32_t tmem = *tmem_holder;
    const int tiles = g.mtiles * g.ntiles, blocks = (g.k + BK - 1) / BK;
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

    if (warp == 0) {
        if (lane == 0) {
            const uint32_t full_lead0 = map_rank(full0, 0);
            int s = 0;
            uint32_t ph = 1;  // a fresh barrier's preceding phase counts as complete
            uint32_t issued_ph[STAGES2];
            bool issued[STAGES2];
            for (int k = 0; k < STAGES2; ++k) issued[k] = false;
            for (int tile = pair; tile < tiles && !*abort; tile += pairs) {
                int mb, nb;
                tile2_coords(tile, g.mtiles, g.ntiles, mb, nb);
                const int m0 = mb * TILE2 + 128 * (int)rank, n0 = nb * TILE2 + 128 * (int)rank;
                for (int kb = 0; kb < blocks; ++kb) {
                    if (!wait_bar(empty0 + 8 * s, ph, abort, g.status, g.timeout_ns)) break;
                    const uint32_t sw = ring + s * STAGE2_BYTES;
                    if (leader) mbar_expect_tx(full0 + 8 * s, 2 * STAGE2_BYTES);  // both CTAs' bytes
                    tma_load_2d_pair(sw, &tmW, kb * BK, n0, full_lead0 + 8 * s);
                    tma_load_2d_pair(sw + W_BYTES, &tmA, kb * BK, m0, full_lead0 + 8 * s);
                    issued[s] = true;
                    issued_ph[s] = ph ^ 1;  // the full-barrier phase this issue completes
                    if (++s == STAGES2) {
                        s = 0;
                        ph ^= 1;
                    }
                }
            }
            if (*abort) {
                if (leader) {  // loads may still be in flight into both CTAs: wait (bounded) for them
                    for (int k = 0; k < STAGES2; ++k)
                        if (issued[k]) wait_drain(full0 + 8 * k, issued_ph[k], g.status, g.timeout_ns);
                } else {  // this CTA cannot observe rank 0's barrier: give its last loads time to land
                    const uint64_t t0 = ki::globaltimer_ns();
                    while (ki::globaltimer_ns() - t0 < 200000ull) {
                    }
                }
            }
        }
    } else if (warp == 1) {
        if (leader && lane == 0) {
            const uint32_t empty_peer0 = map_rank(empty0, 1), tfull_peer0 = map_rank(tfull0, 1);
            int s = 0, acc = 0;
            uint32_t ph_full = 0, ph_empty = 1;
            for (int tile = pair; tile < tiles && !*abort; tile += pairs) {
                if (!wait_bar(tempty0 + 8 * acc, ph_empty, abort, g.status, g.timeout_ns)) break;
                tc_fence_after();
                const uint32_t d = tmem + (uint32_t)(acc * TILE2);
                bool ok = true;
                for (int kb = 0; kb < blocks; ++kb) {
                    if (!wait_bar(full0 + 8 * s, ph_full, abort, g.status, g.timeout_ns)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t sw = ring + s * STAGE2_BYTES;
                    const uint64_t wdesc = make_desc(sw, 16, 1024), xdesc = make_desc(sw + W_BYTES, 16, 1024);
#pragma unroll
                    for (int k = 0; k < BK / 32; ++k)
                        mma_i8_pair(d, wdesc + (uint64_t)(2 * k), xdesc + (uint64_t)(2 * k), (kb | k) != 0);
                    mma_commit_pair(empty0 + 8 * s);       // this CTA's stage is free again
                    mma_commit_pair(empty_peer0 + 8 * s);  // and the peer's
                    if (++s == STAGES2) {
                        s = 0;
                        ph_full ^= 1;
                    }
                }
                if (!ok) break;
                mma_commit_pair(tfull0 + 8 * acc);
                mma_commit_pair(tfull_peer0 + 8 * acc);
                if (++acc == ACCS2) {
                    acc = 0;
                    ph_empty ^= 1;
                }
            }
            mma_commit_pair(drain);  // every MMA issued has finished before TMEM and the rings go
            wait_drain(drain, 0, g.status, g.timeout_ns);
        }
    } else {
        const int row = (warp & 3) * 32;  // TMEM lanes that this warp may read
        const int half = (warp - 2) / 4 * (TILE2 / 2);  // and its columns
        const uint32_t tempty_lead0 = map_rank(tempty0, 0);
        float* scales = reinterpret_cast<float*>(gbase + RING2_BYTES + 256);
        int acc = 0;
        uint32_t ph = 0;
        for (int tile = pair; tile < tiles; tile += pairs) {
            int mb, nb;
            tile2_coords(tile, g.mtiles, g.ntiles, mb, nb);
            const int m0 = mb * TILE2, n = nb * TILE2 + 128 * (int)rank + row + lane;
            const bool on = n < g.n;
            const float sw = on ? g.sw[n] : 0.0f, bias = on && g.bias ? g.bias[n] : 0.0f;
            // a buffer is written again two tiles later, behind the next tile's barrier, when all have read it
            float* sa = scales + acc * TILE2;
            const int mine = (int)threadIdx.x - 64;
            sa[mine] = m0 + mine < g.m ? g.sa[m0 + mine] : 0.0f;
            asm volatile("bar.sync 1, %0;" ::"r"(32 * EPI2_WARPS) : "memory");
            int ok = 0;
            if (lane == 0) ok = wait_bar(tfull0 + 8 * acc, ph, abort, g.status, g.timeout_ns) ? 1 : 0;
            ok = __shfl_sync(0xffffffffu, ok, 0);
            if (ok) {
                tc_fence_after();
#pragma unroll 1
                for (int c0 = half; c0 < half + TILE2 / 2; c0 += 32) {
                    uint32_t v[32];
                    KI_TMEM_LD_X32(tmem + ((uint32_t)row << 16) + (uint32_t)(acc * TILE2 + c0), v);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    if (c0 == half + TILE2 / 2 - 32) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_cluster(tempty_lead0 + 8 * acc);
                    }
                    if (on)
                        store_columns(static_cast<O*>(g.c) + (size_t)(m0 + c0) * g.ldc + n, g.ldc, v, sa + c0, sw, bias,
                                      g.m - m0 - c0);
                }
            }
            if (++acc == ACCS2) {
                acc = 0;
                ph ^= 1;
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // neither CTA leaves while the other may still read its shared memory or TMEM
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(ACCS2 * TILE2) : "memory");
    }
}

// Tensor maps of both operands with boxes of rows_a and rows_w rows x 128 bytes.
int encode_operands(ki_ctx* ctx, const GemmArgs& g, CUtensorMap* tA, CUtensorMap* tW, int rows_a, int rows_w) {
    auto enc = get_encode();
    if (!enc) return ki::set_error(ctx, KI_ERR_CUDA, "gemm_i8: cuTensorMapEncodeTiled unavailable");
    // a single row has no stride of its own
    const uint64_t one = (uint64_t)(g.k + 15) / 16 * 16, lda = g.m > 1 ? g.lda : one, ldw = g.n > 1 ? g.ldw : one;
    if (!encode_2d(enc, tA, CU_TENSOR_MAP_DATA_TYPE_UINT8, g.a, (uint64_t)g.k, (uint64_t)g.m, lda, BK, rows_a,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B) ||
        !encode_2d(enc, tW, CU_TENSOR_MAP_DATA_TYPE_UINT8, g.w, (uint64_t)g.k, (uint64_t)g.n, ldw, BK, rows_w,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B))
        return ki::set_error(ctx, KI_ERR_ARG, "gemm_i8: tensor map encoding failed");
    return KI_OK;
}

template <class O>
int launch_pairs(ki_ctx* ctx, GemmArgs& g, cudaStream_t s) {
    CUtensorMap tA, tW;
    const int st = encode_operands(ctx, g, &tA, &tW, 128, 128);
    if (st != KI_OK) return st;
    auto kern = gemm_i8_pair_kernel<O>;
    KI_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM2_BYTES));
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.blockDim = dim3(THREADS2);
    cfg.dynamicSmemBytes = SMEM2_BYTES;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (ctx->gemm_i8_pairs == 0) {
        int nc = 0;
        cfg.gridDim = dim3(2 * (ctx->sm_count / 2));
        if (cudaOccupancyMaxActiveClusters(&nc, kern, &cfg) != cudaSuccess || nc < 1) {
            cudaGetLastError();
            nc = ctx->sm_count / 2;
        }
        ctx->gemm_i8_pairs = nc;
    }
    g.ntiles = (g.n + TILE2 - 1) / TILE2;
    g.mtiles = (g.m + TILE2 - 1) / TILE2;
    const long long tiles = (long long)g.ntiles * g.mtiles;
    if (tiles > 0x3fffffffll) return ki::set_error(ctx, KI_ERR_ARG, "gemm_i8: too many tiles");
    cfg.gridDim = dim3(2 * (unsigned)(tiles < ctx->gemm_i8_pairs ? tiles : ctx->gemm_i8_pairs));
    KI_CUDA(ctx, cudaLaunchKernelEx(&cfg, kern, tA, tW, g));
    return ki::check_launch(ctx, "gemm_i8_pair_kernel launch");
}

// Clusters of MAX_SPLIT CTAs that run at once when each CTA takes an SM.
int clusters_of_eight(ki_ctx* ctx) {
    if (ctx->gemm_i8_eights == 0) {
        using S = Shape<128, true>;
        auto kern = gemm_i8_kernel<128, float, true>;
        int nc = 0;
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = MAX_SPLIT;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.gridDim = dim3(MAX_SPLIT * (ctx->sm_count / MAX_SPLIT));
        cfg.blockDim = dim3(S::THREADS);
        cfg.dynamicSmemBytes = S::SMEM_BYTES;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM_BYTES) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&nc, kern, &cfg) != cudaSuccess || nc < 1) {
            cudaGetLastError();
            nc = ctx->sm_count / 16;
        }
        ctx->gemm_i8_eights = nc;
    }
    return ctx->gemm_i8_eights;
}

template <int BN, class O, bool TMA>
int launch(ki_ctx* ctx, GemmArgs& g, cudaStream_t s) {
    using S = Shape<BN, TMA>;
    CUtensorMap tA = {}, tW = {};
    if (TMA) {
        const int st = encode_operands(ctx, g, &tA, &tW, BN, BM);
        if (st != KI_OK) return st;
    }
    g.ntiles = (g.n + BM - 1) / BM;
    g.mtiles = (g.m + BN - 1) / BN;
    const long long tiles = (long long)g.ntiles * g.mtiles;
    if (tiles * MAX_SPLIT > 0x7fffffffll) return ki::set_error(ctx, KI_ERR_ARG, "gemm_i8: too many tiles");
    const int blocks = (g.k + BK - 1) / BK;
    // Eight parts where the clusters of eight run at once: two CTAs of up to 32 tokens fit an SM unless threads load the rows; wider
    // ones take an SM each, and a sixteenth cluster waits for the first fifteen (bf16 out, 15 and 16 tiles of 128 channels:
    // 128 x 4096 inner 9.6 and 16.7 us in eight parts, 9.8 and 9.9 in four; 1 x 4097 inner 11.1 and 19.7, 15.6 and 15.7).
    // Tiles of 64 fit twice, but in four parts 16 of them take no longer (48 x 4096 inner 9.3 and 8.8 us; 10 tiles 6.7 and 7.6).
    const int most = (TMA && BN <= 32) || tiles <= clusters_of_eight(ctx) ? MAX_SPLIT : 4;
    int split = 1;
    while (split < most && 2 * split * tiles <= ctx->sm_count && 2 * split <= blocks) split *= 2;
    auto kern = gemm_i8_kernel<BN, O, TMA>;
    KI_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM_BYTES));
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = split;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(tiles * split));
    cfg.blockDim = dim3(S::THREADS);
    cfg.dynamicSmemBytes = S::SMEM_BYTES;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    KI_CUDA(ctx, cudaLaunchKernelEx(&cfg, kern, tA, tW, g, split));
    return ki::check_launch(ctx, "gemm_i8_kernel launch");
}

template <int BN, class O>
int launch_tma(ki_ctx* ctx, GemmArgs& g, bool tma, cudaStream_t s) {
    return tma ? launch<BN, O, true>(ctx, g, s) : launch<BN, O, false>(ctx, g, s);
}

}  // namespace

extern "C" int ki_gemm_i8(ki_ctx* ctx, const int8_t* d_A, size_t lda, const int8_t* d_W, size_t ldw, const float* d_scale_a,
                          const float* d_scale_w, const float* d_bias, int out_dtype, void* d_C, size_t ldc, size_t M,
                          size_t N, size_t K, void* stream) {
    KI_CHECK_CTX(ctx);
    const size_t es = ki::float_size(out_dtype);
    if (!es) return ki::set_error(ctx, KI_ERR_ARG, "gemm_i8: output dtype must be KI_F32, KI_F16 or KI_BF16");
    if (K > 131071) return ki::set_error(ctx, KI_ERR_ARG, "gemm_i8: K above 131071 could overflow the Int32 sums");
    if (M > 0x7fffff00u || N > 0x7fffff00u) return ki::set_error(ctx, KI_ERR_ARG, "gemm_i8: too large");
    if (M == 0 || N == 0) return KI_OK;
    if (!d_C || !d_scale_a || !d_scale_w || (K > 0 && (!d_A || !d_W)))
        return ki::set_error(ctx, KI_ERR_ARG, "gemm_i8: null pointer");
    if ((M > 1 && (lda < K || ldc < N)) || (N > 1 && ldw < K))
        return ki::set_error(ctx, KI_ERR_ARG, "gemm_i8: leading dimension smaller than a row");
    if (!ki::aligned(d_C, es) || !ki::aligned(d_scale_a, 4) || !ki::aligned(d_scale_w, 4) || !ki::aligned(d_bias, 4))
        return ki::set_error(ctx, KI_ERR_ARG, "gemm_i8: pointer not aligned to its element");
    const ki::Span c = ki::span(d_C, M, ldc, N, es);
    const ki::Span in[] = {ki::span(d_A, M, lda, K, 1), ki::span(d_W, N, ldw, K, 1), ki::span(d_scale_a, 1, M, M, 4),
                           ki::span(d_scale_w, 1, N, N, 4), ki::span(d_bias, 1, N, N, 4)};
    for (const ki::Span& i : in)
        if (ki::overlap(c, i)) return ki::set_error(ctx, KI_ERR_ARG, "gemm_i8: the output overlaps an input");
    KI_GUARD(ctx);
    GemmArgs g{d_A, lda, d_W, ldw, d_scale_a, d_scale_w, d_bias, d_C, ldc, (int)M, (int)N, (int)K, 0, 0, ctx->d_status,
               ctx->wait_timeout_ns};
    // TMA wants 16-byte aligned rows; others are loaded by threads
    const bool tma = K > 0 && ki::rows_aligned(d_A, M > 1 ? lda : 0, 1, 16) && ki::rows_aligned(d_W, N > 1 ? ldw : 0, 1, 16);
    cudaStream_t s = ki::as_stream(stream);
    return ki::with_float_type(out_dtype, [&](auto t) {
        using O = decltype(t);
        // Pairs where the tiles of 128 x 128 would take more than one round: 768 x 4096 x 4096 17.0 us in pairs, 25.8 in
        // two rounds of single tiles; 512 x 4096 x 4096 16.6 and 13.9 us in one round.
        const long long tiles = (long long)((N + BM - 1) / BM) * (long long)((M + 127) / 128);
        if (tma && M > 64 && tiles > ctx->sm_count) return launch_pairs<O>(ctx, g, s);
        if (M <= 16) return launch_tma<16, O>(ctx, g, tma, s);
        if (M <= 32) return launch_tma<32, O>(ctx, g, tma, s);
        if (M <= 64) return launch_tma<64, O>(ctx, g, tma, s);
        // Rows that threads load: tiles of 160 tokens where that saves enough rounds.  A round of them takes a third
        // longer (18 loading warps are five on a scheduler, not four; at K = 2057 26.7 and 20 us): 640 x 4099 x 2057 26.8 us in one
        // round, 41.8 in two of 128 tokens; 1111 x 4099 x 2057 52.5 in two, 59.7 in three.
        const long long wide = (long long)((N + BM - 1) / BM) * (long long)((M + 159) / 160);
        auto rounds = [&](long long all) { return (all + ctx->sm_count - 1) / ctx->sm_count; };
        if (!tma && 4 * rounds(wide) < 3 * rounds(tiles)) return launch<160, O, false>(ctx, g, s);
        return launch_tma<128, O>(ctx, g, tma, s);
    });
}
