// gemm_i8.cu -- ki_gemm_i8: the product of int8 tokens and int8 weights on the tensor cores
// (tcgen05 kind::i8, Int32 accumulators in TMEM), with a scale for each token and each channel.
//
//   C[m, n] = float(sum_k A[m, k] W[n, k]) * scale_a[m] * scale_w[n] (+ bias[n])
//
// A: tokens x inner, W: channels x inner, both row-major (so both operands are K-major), C: tokens x
// channels in Float32, Float16 or BFloat16.  The Int32 sums are exact (inner <= 131071, where 128 * 128
// * inner still fits), so the result does not depend on the order of the sums or on how they are split.
//
// The weights are the MMA's M side: a CTA holds 128 channels x BN tokens, lanes of TMEM are channels and
// columns are tokens.  A warp's store of one column is then 32 neighbouring channels of one token, and a
// few tokens (BN = 16) cost a few columns instead of a mostly empty tile of 128 rows.
//   warp 0     loads K blocks of 128 into a ring of stages (TMA, 128-byte swizzle); rows that are not
//              16-byte aligned are loaded by warps 2-5 with plain loads instead (load_rows);
//   warp 1     allocates TMEM and issues the MMAs (M 128, N BN, K 32) from one thread;
//   warps 2-5  epilogue: TMEM -> registers -> scales -> C.
// With few tiles the K blocks of a tile are split over the CTAs of a cluster; each CTA then leaves its
// Int32 sums in its own shared memory and adds up and stores a share of the tile's columns, read from
// every CTA of the cluster.
//
// Every mbarrier wait is bounded, as in gemm_e4m3.cu.
#include "ki/layer.cuh"
#include "ki/lookback.cuh"
#include "ki/tcgen05.cuh"

namespace {

constexpr int BM = 128, BK = 128;
constexpr int THREADS = 192;
constexpr int W_BYTES = BM * BK;
constexpr int MAX_SPLIT = 8;

// D = S32 (2), A = S8 (1), B = S8 (1), both K-major
constexpr uint32_t idesc(int bn) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(bn >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
}

template <int BN>
struct Shape {
    static constexpr int X_BYTES = BN * BK;
    static constexpr int STAGE_BYTES = W_BYTES + X_BYTES;
    static constexpr int STAGES = BN <= 64 ? 5 : 4;
    static constexpr int SUM_BYTES = BM * BN * 4;  // a split's Int32 sums, over the ring
    static constexpr int RING_BYTES = STAGES * STAGE_BYTES > SUM_BYTES ? STAGES * STAGE_BYTES : SUM_BYTES;
    static constexpr int SMEM_BYTES = 1024 + RING_BYTES + 256;
    static constexpr int TMEM_COLS = BN < 32 ? 32 : BN;
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

// 16 bytes from p, of which the first nb (0 to 16) exist and the others read as zero; any alignment.
// Only 4-byte words that hold one of those bytes are read.
__device__ __forceinline__ uint4 load16(const int8_t* p, int nb) {
    uint32_t w[5];
    const uintptr_t at = (uintptr_t)p;
    const uint32_t off = (uint32_t)(at & 3);
    const uint32_t* q = reinterpret_cast<const uint32_t*>(at - off);
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = nb > 0 && 4 * i < (int)off + nb ? __ldg(q + i) : 0u;
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        o[i] = __funnelshift_r(w[i], w[i + 1], 8 * off);
        const int v = min(max(nb - 4 * i, 0), 4);
        o[i] &= v == 4 ? 0xffffffffu : (1u << (8 * v)) - 1u;
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
}

// `count` rows of a K block to shared memory in the layout that the 128-byte swizzle gives a TMA tile:
// row r at 128 r, its 16-byte pieces exchanged by r mod 8.  Run by 128 threads.
__device__ __forceinline__ void load_rows(uint32_t dst, const int8_t* x, size_t ld, int row0, int rows, int k0, int k,
                                          int count, int tid) {
    for (int i = tid; i < count * 8; i += 128) {
        const int r = i >> 3, j = i & 7;
        const int kk = k0 + 16 * j;
        const int nb = row0 + r < rows ? min(max(k - kk, 0), 16) : 0;
        const uint4 v = load16(x + (nb > 0 ? (size_t)(row0 + r) * ld + kk : 0), nb);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + (uint32_t)(r * 128 + ((j ^ (r & 7)) << 4))),
                     "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                     : "memory");
    }
}

template <class O>
__device__ __forceinline__ O scaled(int32_t v, float sa, float sw, float bias) {
    return ki::from_f32<O>(fmaf((float)v * sa, sw, bias));
}

template <int BN, class O, bool TMA>
__global__ void __launch_bounds__(THREADS)
    gemm_i8_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW, const GemmArgs g,
                   int split) {
    using S = Shape<BN>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t raw = ki::smem_addr(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    const uint32_t ring = base, bars = base + S::RING_BYTES;
    const uint32_t full0 = bars, empty0 = bars + 8 * S::STAGES, tfull = bars + 16 * S::STAGES;
    uint8_t* gbase = smem_raw + (base - raw);
    volatile int* abort = reinterpret_cast<volatile int*>(gbase + S::RING_BYTES + 128);
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(gbase + S::RING_BYTES + 136);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int part = blockIdx.x % split, tile = blockIdx.x / split;
    const int n0 = (tile % g.ntiles) * BM, m0 = (tile / g.ntiles) * BN;
    const int blocks = (g.k + BK - 1) / BK;
    const int kb0 = (int)((long long)blocks * part / split), kb1 = (int)((long long)blocks * (part + 1) / split);

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::STAGES; ++s) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(full0 + 8 * s), "r"(TMA ? 1 : 128));
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
        const int tid = threadIdx.x - 64;
        int s = 0;
        uint32_t ph = 1;
        for (int kb = kb0; kb < kb1; ++kb) {
            int ok = 0;
            if (lane == 0) ok = wait_bar(empty0 + 8 * s, ph, abort, g.status, g.timeout_ns) ? 1 : 0;
            if (!__shfl_sync(0xffffffffu, ok, 0)) break;
            const uint32_t sw = ring + s * S::STAGE_BYTES;
            load_rows(sw, g.w, g.ldw, n0, g.n, kb * BK, g.k, BM, tid);
            load_rows(sw + W_BYTES, g.a, g.lda, m0, g.m, kb * BK, g.k, BN, tid);
            ki::fence_proxy_async_smem();
            mbar_arrive(full0 + 8 * s);
            if (++s == S::STAGES) {
                s = 0;
                ph ^= 1;
            }
        }
    }
    __syncwarp();

    if (warp >= 2) {
        int ok = 0;
        if (lane == 0) ok = wait_bar(tfull, 0, abort, g.status, g.timeout_ns) ? 1 : 0;
        ok = __shfl_sync(0xffffffffu, ok, 0);
        tc_fence_after();
        const int row = (warp & 3) * 32;  // TMEM lanes that this warp may read
        const int n = n0 + row + lane;
        const bool on = n < g.n;
        const float sw = on ? g.sw[n] : 0.0f, bias = on && g.bias ? g.bias[n] : 0.0f;
        O* c = static_cast<O*>(g.c) + n;
        constexpr int STEP = BN < 32 ? BN : 32;
        if (ok) {
#pragma unroll 1
            for (int c0 = 0; c0 < BN; c0 += STEP) {
                if (split == 1 && m0 + c0 >= g.m) break;
                uint32_t v[32];
                if (kb1 > kb0) {
                    KI_TMEM_LD_X32(tmem + ((uint32_t)row << 16) + (uint32_t)c0, v);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = 0;
                }
                if (split == 1) {
                    const float mine = m0 + c0 + lane < g.m ? g.sa[m0 + c0 + lane] : 0.0f;
#pragma unroll
                    for (int j = 0; j < STEP; ++j) {
                        const float sa = __shfl_sync(0xffffffffu, mine, j);
                        if (on && m0 + c0 + j < g.m) c[(size_t)(m0 + c0 + j) * g.ldc] = scaled<O>((int)v[j], sa, sw, bias);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < STEP; ++j)
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
        if (warp >= 2 && !*abort) {
            const int row = (warp & 3) * 32;
            const int n = n0 + row + lane;
            if (n < g.n) {
                const float sw = g.sw[n], bias = g.bias ? g.bias[n] : 0.0f;
                O* c = static_cast<O*>(g.c) + n;
                for (int j = part; j < BN && m0 + j < g.m; j += split) {
                    int32_t sum = 0;
                    for (int p = 0; p < split; ++p) {
                        int32_t v;
                        asm volatile("ld.shared::cluster.b32 %0, [%1];"
                                     : "=r"(v)
                                     : "r"(map_rank(ring + (uint32_t)((j * BM + row + lane) * 4), (uint32_t)p))
                                     : "memory");
                        sum += v;
                    }
                    c[(size_t)(m0 + j) * g.ldc] = scaled<O>(sum, g.sa[m0 + j], sw, bias);
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

template <int BN, class O, bool TMA>
int launch(ki_ctx* ctx, GemmArgs& g, cudaStream_t s) {
    using S = Shape<BN>;
    CUtensorMap tA = {}, tW = {};
    if (TMA) {
        auto enc = get_encode();
        if (!enc) return ki::set_error(ctx, KI_ERR_CUDA, "gemm_i8: cuTensorMapEncodeTiled unavailable");
        // a single row has no stride of its own
        const uint64_t lda = g.m > 1 ? g.lda : (g.k + 15) / 16 * 16, ldw = g.n > 1 ? g.ldw : (g.k + 15) / 16 * 16;
        if (!encode_2d(enc, &tA, CU_TENSOR_MAP_DATA_TYPE_UINT8, g.a, (uint64_t)g.k, (uint64_t)g.m, lda, BK, BN,
                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B) ||
            !encode_2d(enc, &tW, CU_TENSOR_MAP_DATA_TYPE_UINT8, g.w, (uint64_t)g.k, (uint64_t)g.n, ldw, BK, BM,
                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B))
            return ki::set_error(ctx, KI_ERR_ARG, "gemm_i8: tensor map encoding failed");
    }
    g.ntiles = (g.n + BM - 1) / BM;
    g.mtiles = (g.m + BN - 1) / BN;
    const long long tiles = (long long)g.ntiles * g.mtiles;
    if (tiles * MAX_SPLIT > 0x7fffffffll) return ki::set_error(ctx, KI_ERR_ARG, "gemm_i8: too many tiles");
    const int blocks = (g.k + BK - 1) / BK;
    int split = 1;
    while (split < MAX_SPLIT && 2 * split * tiles <= ctx->sm_count && 2 * split <= blocks) split *= 2;
    auto kern = gemm_i8_kernel<BN, O, TMA>;
    KI_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM_BYTES));
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = split;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(tiles * split));
    cfg.blockDim = dim3(THREADS);
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
        if (M <= 16) return launch_tma<16, O>(ctx, g, tma, s);
        if (M <= 32) return launch_tma<32, O>(ctx, g, tma, s);
        if (M <= 64) return launch_tma<64, O>(ctx, g, tma, s);
        return launch_tma<128, O>(ctx, g, tma, s);
    });
}
