// Matrix product in 8-bit integers on the 5th-generation tensor cores: out[n, f] = (sum_k x[n, k] w[f, k]) xs[n] ws[f] (+ bias[f]), the sum
// exact in 32 bits (127^2 K < 2^31 for K up to 131,072), then three or four roundings in float and one to the output's type.
//
// Few tokens (`narrow`): bound by the weights' bytes.  Weight rows are the M side of tcgen05.mma (128 to a block), 16 to 128 tokens its N
// side; the blocks of a cluster divide k and add their tiles up through distributed shared memory - in any order, the sums are exact.
// Many tokens (`wide`): bound by the tensor cores, which take 8-bit operands at twice bfloat16's rate.  Tiles of 256 tokens x up to 256
// features on pairs of SMs (cta_group::2): a block then loads 256 rows of 128 bytes for 512 cycles of products, 64 bytes a cycle, which is
// what an SM takes in.  The pairs stay and walk over the tiles with two accumulators, so that one tile's epilogue runs beside the next one's
// products; where the tiles are few, the pairs of a cluster divide k instead.
#include "tcgen05_utils.cuh"

namespace {

constexpr int BM = 128, BK = 128, UMMA_K = 32;  // bytes: a stage's row is one 128-byte swizzle row

enum I8Error { kErrProducerWait = 61, kErrMmaWait = 62, kErrEpilogueWait = 63, kErrDrainWait = 64 };

// D = 32-bit integers, A = B = signed 8-bit integers, both K-major
__host__ __device__ constexpr uint32_t i8_desc(int m, int n) { return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }

// (spelled out, so that every tile rounds alike: an output's bits do not depend on which one it fell into)
__device__ __forceinline__ float scaled(int sum, float x_scale, float w_scale) { return __fmul_rn(__int2float_rn(sum), __fmul_rn(x_scale, w_scale)); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// ---- few tokens ------------------------------------------------------------------------------------------------------------
namespace narrow {
constexpr int kThreads = 192;

template <int BN>
struct Cfg {
    static constexpr int kStages = BN == 16 ? 6 : BN == 32 ? 5 : BN == 64 ? 4 : 6;
    static constexpr int kMinBlocks = BN <= 64 ? 2 : 1;
    static constexpr int kABytes = BM * BK, kBBytes = BN * BK, kStageBytes = kABytes + kBBytes;
    static constexpr int kTmemCols = BN < 32 ? 32 : BN;
    static constexpr size_t kSmemBytes = (size_t)kStages * kStageBytes + 1024 /* alignment slack */ + 256 /* barriers */;
    static_assert(BN * BM * 4 <= kStages * kStageBytes, "the accumulator is staged where the ring was");
};

__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&r)[16]) { tmem_ld16(taddr, r); }
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&r)[32]) { tmem_ld32(taddr, r); }

// Warps: 0 loads, 1 issues, 2-5 read the accumulator; then all of them finish the tile.  `early`: the kernel before this one did not
// write w, whose first tiles are then asked for before this kernel waits for it.
template <int BN, typename OutT>
__global__ void __launch_bounds__(kThreads, Cfg<BN>::kMinBlocks)
gemm_i8_narrow_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const float* __restrict__ xs,
                      const float* __restrict__ ws, const float* __restrict__ bias, OutT* __restrict__ out, long long ldo, int M, int N, int k_blocks,
                      int splits, int early, int* __restrict__ error_flag) {
    using C = Cfg<BN>;
    extern __shared__ unsigned char smem_dyn[];
    __shared__ float xs_s[BN];
    __shared__ int failed;
    const uint32_t base = (smem_u32(smem_dyn) + 1023u) & ~1023u;
    const uint32_t bar_base = base + C::kStages * C::kStageBytes;
    auto full_bar = [&](int s) { return bar_base + 8u * s; };
    auto empty_bar = [&](int s) { return bar_base + 8u * (C::kStages + s); };
    const uint32_t accum_bar = bar_base + 8u * (2 * C::kStages);
    const uint32_t holder = accum_bar + 8u;
    int* stage = reinterpret_cast<int*>(smem_dyn + (base - smem_u32(smem_dyn)));  // [BN][BM]

    ns_pdl_launch_dependents();
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int n0 = blockIdx.x * BM, tok0 = blockIdx.y * BN, split = blockIdx.z;
    const int per = k_blocks / splits, rem = k_blocks % splits;
    const int kb_begin = split * per + min(split, rem), kb_count = per + (split < rem ? 1 : 0);
    if (threadIdx.x == 0) {
        failed = 0;
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        mbar_init(accum_bar, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
    }
    if (warp == 1) tmem_alloc(holder, C::kTmemCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    uint32_t tmem_base;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem_base) : "r"(holder));
    tmem_base = __shfl_sync(0xffffffffu, tmem_base, 0);

    if (warp == 0) {
        const int first = min(kb_count, C::kStages);
        int issued = 0;
        bool ok = true;
        if (!early) ns_pdl_wait();
        if (elect_one()) {
            for (int i = 0; i < first; ++i) {
                mbar_expect_tx(full_bar(i), C::kStageBytes);
                tma_load_2d(base + i * C::kStageBytes, &map_w, (kb_begin + i) * BK, n0, full_bar(i));
            }
        }
        if (early) ns_pdl_wait();
        if (elect_one()) {
            for (int i = 0; i < first; ++i) tma_load_2d(base + i * C::kStageBytes + C::kABytes, &map_x, (kb_begin + i) * BK, tok0, full_bar(i));
        }
        issued = first;
        for (int i = first; i < kb_count; ++i) {
            const int s = i % C::kStages;
            if (!mbar_wait_warp(empty_bar(s), (uint32_t)(i / C::kStages - 1) & 1u)) {
                ok = false;
                if (lane == 0) atomicExch(error_flag, kErrProducerWait);
                break;
            }
            if (elect_one()) {
                mbar_expect_tx(full_bar(s), C::kStageBytes);
                const uint32_t a = base + s * C::kStageBytes;
                tma_load_2d(a, &map_w, (kb_begin + i) * BK, n0, full_bar(s));
                tma_load_2d(a + C::kABytes, &map_x, (kb_begin + i) * BK, tok0, full_bar(s));
            }
            ++issued;
        }
        if (!ok) {  // wait, bounded, for the copies that are still in flight before the block may exit
            if (lane == 0) failed = 1;
            for (int i = max(0, issued - C::kStages); i < issued; ++i)
                if (!mbar_wait_warp(full_bar(i % C::kStages), (uint32_t)(i / C::kStages) & 1u)) {
                    if (lane == 0) atomicExch(error_flag, kErrDrainWait);
                    break;
                }
        }
    } else if (warp == 1) {
        constexpr uint32_t idesc = i8_desc(BM, BN);
        for (int i = 0; i < kb_count; ++i) {
            const int s = i % C::kStages;
            if (!mbar_wait_warp(full_bar(s), (uint32_t)(i / C::kStages) & 1u)) {
                if (lane == 0) { failed = 1; atomicExch(error_flag, kErrMmaWait); }
                break;
            }
            tc_fence_after();
            const uint32_t a = base + s * C::kStageBytes, b = a + C::kABytes;
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < BK / UMMA_K; ++k)
                    umma_i8(tmem_base, smem_desc(a + k * UMMA_K), smem_desc(b + k * UMMA_K), idesc, (i > 0 || k > 0) ? 1u : 0u);
                umma_commit(empty_bar(s));
            }
        }
        if (elect_one()) umma_commit(accum_bar);
        ns_pdl_wait();
    } else {
        ns_pdl_wait();
        for (int t = threadIdx.x - 64; t < BN; t += 128) xs_s[t] = tok0 + t < M ? xs[tok0 + t] : 0.f;
        if (!mbar_wait_warp(accum_bar, 0)) {
            if (lane == 0) { failed = 1; atomicExch(error_flag, kErrEpilogueWait); }
        } else {
            tc_fence_after();
            const int q = warp & 3;  // the TMEM lane quarter this warp may read
            const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16);
            constexpr int CH = BN >= 32 ? 32 : 16;
#pragma unroll 1
            for (int c0 = 0; c0 < BN; c0 += CH) {
                if (tok0 + c0 >= M) break;  // uniform across the warp
                uint32_t r[CH];
                tmem_ld_cols(taddr + c0, r);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < CH; ++j) stage[(c0 + j) * BM + q * 32 + lane] = (int)r[j];
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, C::kTmemCols);
    }
    // Every block adds up one slice of the features from the shared memory of its cluster's blocks and writes it, four features a thread.
    if (splits > 1) cluster_sync();  // (blocks that gave up still take part)
    if (!failed) {
        const int groups = BM / splits / 4, toks = min(BN, M - tok0);
        for (int e = threadIdx.x; e < toks * groups; e += kThreads) {
            const int j = e / groups, fl = split * (BM / splits) + (e - j * groups) * 4, f = n0 + fl;
            if (f >= N) continue;
            int4 sum = make_int4(0, 0, 0, 0);
            for (int s = 0; s < splits; ++s) {
                const int* at = stage + j * BM + fl;
                int4 v;
                if (splits == 1) {
                    v = *reinterpret_cast<const int4*>(at);
                } else {
                    const float4 raw = ld_cluster_f32x4(smem_u32(at), (uint32_t)s);
                    v = make_int4(__float_as_int(raw.x), __float_as_int(raw.y), __float_as_int(raw.z), __float_as_int(raw.w));
                }
                sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
            }
            const float scale = xs_s[j];
            const int part[4] = {sum.x, sum.y, sum.z, sum.w};
            OutT* to = out + (size_t)(tok0 + j) * ldo + f;
            float y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool live = f + i < N;
                y[i] = scaled(part[i], scale, live ? __ldg(ws + f + i) : 0.f);
                if (bias && live) y[i] = __fadd_rn(y[i], __ldg(bias + f + i));
            }
            if (f + 4 <= N && (reinterpret_cast<uintptr_t>(to) & (4 * sizeof(OutT) - 1)) == 0) {
                if constexpr (sizeof(OutT) == 4) {
                    *reinterpret_cast<float4*>(to) = make_float4(y[0], y[1], y[2], y[3]);
                } else {
                    const __nv_bfloat162 lo = __floats2bfloat162_rn(y[0], y[1]), hi = __floats2bfloat162_rn(y[2], y[3]);
                    *reinterpret_cast<uint2*>(to) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (f + i < N) put(to + i, y[i]);
            }
        }
    }
    if (splits > 1) {
        __syncthreads();
        cluster_sync();  // nobody's shared memory goes while another block reads it
    }
}

template <int BN, typename OutT>
int launch(const void* x, long long ldx, const float* xs, const void* w, long long ldw, const float* ws, const float* bias, void* out, long long ldo,
           int M, int N, int K, int splits, int early, int* error_flag, cudaStream_t stream) {
    using C = Cfg<BN>;
    static std::atomic<unsigned long long> allowed{0};
    NS_CUDA(ns_allow_smem((const void*)gemm_i8_narrow_kernel<BN, OutT>, (int)C::kSmemBytes, allowed));
    CUtensorMap mw, mx;
    if (const int rc = ns_make_map<1>(&mw, w, N, K, ldw, BM, "ns_gemm_i8")) return rc;
    if (const int rc = ns_make_map<1>(&mx, x, M, K, ldx, BN, "ns_gemm_i8")) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((N + BM - 1) / BM, (M + BN - 1) / BN, splits);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = C::kSmemBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n_attr = 0;
    if (ns_take_pdl()) {
        attr[n_attr].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n_attr++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (splits > 1) {
        attr[n_attr].id = cudaLaunchAttributeClusterDimension;
        attr[n_attr].val.clusterDim.x = attr[n_attr].val.clusterDim.y = 1;
        attr[n_attr++].val.clusterDim.z = splits;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n_attr;
    (void)cudaLaunchKernelEx(&cfg, gemm_i8_narrow_kernel<BN, OutT>, mw, mx, xs, ws, bias, (OutT*)out, ldo, M, N, (K + BK - 1) / BK, splits, early, error_flag);
    NS_CHECK_LAUNCH("ns_gemm_i8");
    return NS_OK;
}
}  // namespace narrow

// ---- many tokens -------------------------------------------------------------------------------------------------------------
// A cluster is `splits` (1 or 2) pairs of blocks.  Of a pair, each block holds 128 tokens of A and of the accumulator, and half of the rows of B; the
// pair's first block (the leader) issues.  Warps: 0 loads (each block its own operands; the bytes count on the leader's barrier), 1 issues (the
// leader's), 2-9 the epilogue: four warps for each half of the columns.
namespace wide {
constexpr int kTok = 256, kFeat = 256, kStages = 6, kThreads = 64 + 256;
constexpr int kABytes = BM * BK, kStageBytes = 2 * BM * BK;
constexpr int kPitch = 80, kBarBytes = 256;             // bytes of a staged row: 64 of outputs, so that eight rows fall in different banks
constexpr int kSmem = kStages * kStageBytes + kBarBytes + 8 * 32 * kPitch + 1024;
static_assert(kSmem <= 232448 && BM * kFeat / 2 * 4 <= kStages * kStageBytes, "shared memory of a block");

__device__ __forceinline__ uint32_t at_rank(uint32_t local, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(rank));
    return r;
}
__device__ __forceinline__ void commit_pair(uint32_t bar, uint32_t leader) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"((uint16_t)(3u << leader)) : "memory");
}

// 32 columns of a warp's 32 rows: scaled, brought into rows through the warp's own shared memory, written in 16-byte pieces where they may be
template <typename OutT>
__device__ __forceinline__ void emit(const uint32_t (&r)[32], unsigned char* st, float row_scale, const float* __restrict__ ws, const float* __restrict__ bias,
                                     OutT* __restrict__ out, long long ldo, int row0, int col0, int M, int N, bool aligned) {
    constexpr int kPer = 16 / sizeof(OutT), kCols = 64 / sizeof(OutT);
    const int lane = threadIdx.x & 31;
    const float mine_ws = col0 + lane < N ? __ldg(ws + col0 + lane) : 0.f;
    const float mine_b = bias && col0 + lane < N ? __ldg(bias + col0 + lane) : 0.f;
#pragma unroll
    for (int c1 = 0; c1 < 32; c1 += kCols) {
        __syncwarp();  // the columns before these have been read
#pragma unroll
        for (int c = 0; c < kCols; c += kPer) {
            float y[kPer];
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                y[i] = scaled((int)r[c1 + c + i], row_scale, __shfl_sync(0xffffffffu, mine_ws, c1 + c + i));
                if (bias) y[i] = __fadd_rn(y[i], __shfl_sync(0xffffffffu, mine_b, c1 + c + i));
            }
            unsigned char* p = st + lane * kPitch + c * sizeof(OutT);
            if constexpr (sizeof(OutT) == 4) *reinterpret_cast<float4*>(p) = make_float4(y[0], y[1], y[2], y[3]);
            else st8(reinterpret_cast<__nv_bfloat16*>(p), y);
        }
        __syncwarp();
#pragma unroll
        for (int j0 = 0; j0 < 32; j0 += 8) {  // eight rows of four pieces
            const int j = j0 + (lane >> 2), c = (lane & 3) * kPer, col = col0 + c1 + c;
            if (row0 + j >= M) continue;
            const unsigned char* p = st + j * kPitch + c * sizeof(OutT);
            OutT* to = out + (size_t)(row0 + j) * ldo + col;
            if (aligned && col + kPer <= N) {
                *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(p);
            } else {
                for (int i = 0; i < kPer; ++i)
                    if (col + i < N) to[i] = reinterpret_cast<const OutT*>(p)[i];
            }
        }
    }
}

template <typename OutT>
__global__ void __launch_bounds__(kThreads, 1)
gemm_i8_wide_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const float* __restrict__ xs,
                    const float* __restrict__ ws, const float* __restrict__ bias, OutT* __restrict__ out, long long ldo, int M, int N, int k_blocks,
                    int tile_n, int splits, int aligned, int* __restrict__ error_flag) {
    extern __shared__ unsigned char smem_dyn[];
    const uint32_t base = (smem_u32(smem_dyn) + 1023u) & ~1023u;
    unsigned char* smem = smem_dyn + (base - smem_u32(smem_dyn));
    const uint32_t bar_base = base + kStages * kStageBytes;
    unsigned char* out_s = smem + kStages * kStageBytes + kBarBytes;
    auto full_bar = [&](int s) { return bar_base + 8u * s; };  // (the leader's count)
    auto empty_bar = [&](int s) { return bar_base + 8u * (kStages + s); };
    auto acc_full = [&](int b) { return bar_base + 8u * (2 * kStages + b); };
    auto acc_free = [&](int b) { return bar_base + 8u * (2 * kStages + 2 + b); };  // (the leader's counts)
    const uint32_t holder = bar_base + 8u * (2 * kStages + 4);
    __shared__ int failed;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank(), side = rank & 1u, leader = rank & ~1u;
    const int split = (int)rank >> 1;
    const int cluster = (int)blockIdx.x / (2 * splits), clusters = (int)gridDim.x / (2 * splits);

    ns_pdl_launch_dependents();
    if (threadIdx.x == 0) {
        failed = 0;
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full(b), 1);
            mbar_init(acc_free(b), 16);  // eight warps of each block
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
    }
    if (warp == 1) tmem_alloc_pair(holder, 512);
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // the barriers and the tensor memory of all blocks are there
    tc_fence_after();
    uint32_t tmem_base;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem_base) : "r"(holder));
    tmem_base = __shfl_sync(0xffffffffu, tmem_base, 0);
    ns_pdl_wait();

    const int tok_tiles = (M + kTok - 1) / kTok, tiles = tok_tiles * ((N + tile_n - 1) / tile_n);
    const int per = k_blocks / splits, rem = k_blocks % splits;
    const int kb_begin = split * per + min(split, rem), kb_count = per + (split < rem ? 1 : 0);
    const uint32_t b_bytes = (uint32_t)(tile_n / 2) * BK;
    // tile i: all tiles of tokens for one tile of features, then the next features (the weights are read once, the tokens stay in L2)
    auto tok_of = [&](int i) { return (i % tok_tiles) * kTok + (int)side * BM; };
    auto feat_of = [&](int i) { return (i / tok_tiles) * tile_n; };

    if (warp == 0) {
        int g = 0;
        bool ok = true;
        for (int i = cluster; ok && i < tiles; i += clusters) {
            const int tok = tok_of(i), feat = feat_of(i) + (int)side * (tile_n / 2);
            for (int kb = 0; kb < kb_count; ++kb, ++g) {
                const int s = g % kStages;
                if (g >= kStages && !mbar_wait_warp(empty_bar(s), (uint32_t)(g / kStages - 1) & 1u)) {
                    ok = false;
                    if (lane == 0) atomicExch(error_flag, kErrProducerWait);
                    break;
                }
                if (elect_one()) {
                    if (side == 0) mbar_expect_tx(full_bar(s), 2 * (kABytes + b_bytes));
                    const uint32_t a = base + s * kStageBytes, bar = at_rank(full_bar(s), leader);
                    tma_load_2d_pair(a, &map_x, (kb_begin + kb) * BK, tok, bar);
                    tma_load_2d_pair(a + kABytes, &map_w, (kb_begin + kb) * BK, feat, bar);
                }
            }
        }
        // Before a block leaves, the pair's copies have landed (the leader's barriers count them) and the leader's last commits have arrived at
        // the other block's barriers (at its own: warp 1 below).
        for (int i = max(0, g - kStages); i < g; ++i)
            if (!mbar_wait_warp(side == 0 ? full_bar(i % kStages) : empty_bar(i % kStages), (uint32_t)(i / kStages) & 1u)) {
                if (lane == 0) atomicExch(error_flag, kErrDrainWait);
                break;
            }
    } else if (warp == 1) {
        if (side == 0) {
            const uint32_t idesc = i8_desc(2 * BM, tile_n);
            int g = 0, n = 0;
            bool ok = true;
            for (int i = cluster; ok && i < tiles; i += clusters, ++n) {
                const int b = n & 1;
                if (n > 1 && !mbar_wait_warp(acc_free(b), (uint32_t)((n >> 1) - 1) & 1u)) {
                    if (lane == 0) atomicExch(error_flag, kErrMmaWait);
                    break;
                }
                tc_fence_after();
                for (int kb = 0; kb < kb_count; ++kb, ++g) {
                    const int s = g % kStages;
                    if (!mbar_wait_warp(full_bar(s), (uint32_t)(g / kStages) & 1u)) {
                        ok = false;
                        if (lane == 0) atomicExch(error_flag, kErrMmaWait);
                        break;
                    }
                    tc_fence_after();
                    const uint64_t a = smem_desc(base + s * kStageBytes), w = smem_desc(base + s * kStageBytes + kABytes);
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < BK / UMMA_K; ++k)
                            umma_i8_pair(tmem_base + b * kFeat, a + (uint64_t)(k * UMMA_K >> 4), w + (uint64_t)(k * UMMA_K >> 4), idesc, (kb > 0 || k > 0) ? 1u : 0u);
                        commit_pair(empty_bar(s), leader);
                    }
                }
                if (ok && elect_one()) commit_pair(acc_full(b), leader);
            }
            for (int i = max(0, g - kStages); i < g; ++i)  // nothing may still be multiplied when the blocks leave
                if (!mbar_wait_warp(empty_bar(i % kStages), (uint32_t)(i / kStages) & 1u)) {
                    if (lane == 0) atomicExch(error_flag, kErrDrainWait);
                    break;
                }
        }
    } else if (splits == 1) {
        const int q = warp & 3, half = (warp - 2) >> 2;  // q: the TMEM lane quarter this warp may read
        unsigned char* st = out_s + (warp - 2) * 32 * kPitch;
        const int row_in = q * 32, half_n = tile_n / 2;
        int n = 0;
        for (int i = cluster; i < tiles; i += clusters, ++n) {
            const int b = n & 1;
            if (!mbar_wait_warp(acc_full(b), (uint32_t)(n >> 1) & 1u)) {
                if (lane == 0) { failed = 1; atomicExch(error_flag, kErrEpilogueWait); }
                break;
            }
            tc_fence_after();
            const int row0 = tok_of(i) + row_in, col0 = feat_of(i);
            const uint32_t taddr = tmem_base + b * kFeat + ((uint32_t)row_in << 16);
            const float row_scale = row0 + lane < M ? __ldg(xs + row0 + lane) : 0.f;
            for (int c0 = half * half_n; c0 < (half + 1) * half_n; c0 += 32) {
                uint32_t r[32];
                tmem_ld32(taddr + c0, r);
                tmem_ld_wait();
                if (c0 + 32 >= (half + 1) * half_n) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(at_rank(acc_free(b), leader));
                }
                if (row0 < M && col0 + c0 < N) emit(r, st, row_scale, ws, bias, out, ldo, row0, col0 + c0, M, N, aligned);
            }
        }
    }
    if (splits > 1) {
        // Two pairs, one tile: each finishes half of its columns.  The columns that are the other pair's go to shared memory (the ring is free: the
        // tile is multiplied), its own stay in tensor memory until the other pair's part of them can be read.
        const int q = warp & 3, group = (warp - 2) >> 2, half_n = tile_n / 2;
        const int row_in = q * 32, row0 = tok_of(cluster) + row_in, col0 = feat_of(cluster);
        const uint32_t taddr = tmem_base + ((uint32_t)row_in << 16);
        uint32_t* part = reinterpret_cast<uint32_t*>(smem) + row_in + lane;  // [column][128 rows]: a warp's 32 rows lie side by side, here and from another block
        if (warp >= 2) {
            if (!mbar_wait_warp(acc_full(0), 0)) {
                if (lane == 0) { failed = 1; atomicExch(error_flag, kErrEpilogueWait); }
            } else {
                tc_fence_after();
                for (int c = group * 32; c < half_n; c += 64) {
                    uint32_t r[32];
                    tmem_ld32(taddr + (1 - split) * half_n + c, r);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 32; ++j) part[(c + j) * BM] = r[j];
                }
            }
        }
        __syncthreads();
        cluster_sync();
        if (warp >= 2 && !failed && row0 < M) {
            unsigned char* st = out_s + (warp - 2) * 32 * kPitch;
            const float row_scale = row0 + lane < M ? __ldg(xs + row0 + lane) : 0.f;
            for (int c = group * 32; c < half_n; c += 64) {
                const int col = col0 + split * half_n + c;
                if (col >= N) break;
                uint32_t r[32];
                tmem_ld32(taddr + split * half_n + c, r);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 32; ++j) r[j] += __float_as_uint(ld_cluster_f32(smem_u32(part + (c + j) * BM), rank ^ 2u));
                emit(r, st, row_scale, ws, bias, out, ldo, row0, col, M, N, aligned);
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // no block's shared or tensor memory is in use any more
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, 512);
    }
}

template <typename OutT>
int launch(const void* x, long long ldx, const float* xs, const void* w, long long ldw, const float* ws, const float* bias, void* out, long long ldo,
           int M, int N, int K, int tile_n, int splits, int sms, int* error_flag, cudaStream_t stream) {
    static std::atomic<unsigned long long> allowed{0};
    NS_CUDA(ns_allow_smem((const void*)gemm_i8_wide_kernel<OutT>, kSmem, allowed));
    CUtensorMap mx, mw;
    if (const int rc = ns_make_map<1>(&mx, x, M, K, ldx, BM, "ns_gemm_i8")) return rc;
    if (const int rc = ns_make_map<1>(&mw, w, N, K, ldw, tile_n / 2, "ns_gemm_i8")) return rc;
    const long long tiles = (long long)((M + kTok - 1) / kTok) * ((N + tile_n - 1) / tile_n);
    const long long most = splits > 1 ? tiles : tiles < sms / 2 ? tiles : sms / 2;
    if (tiles > 0x7fffffff / 16) NS_FAIL(NS_ERR_UNSUPPORTED, "ns_gemm_i8: too many tiles (%d x %d)", M, N);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(most * 2 * splits));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2 * splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ns_take_pdl() ? 2 : 1;
    const int aligned = (uintptr_t)out % 16 == 0 && ldo * (long long)sizeof(OutT) % 16 == 0;
    (void)cudaLaunchKernelEx(&cfg, gemm_i8_wide_kernel<OutT>, mx, mw, xs, ws, bias, (OutT*)out, ldo, M, N, (K + BK - 1) / BK, tile_n, splits, aligned, error_flag);
    NS_CHECK_LAUNCH("ns_gemm_i8");
    return NS_OK;
}
}  // namespace wide

}  // namespace

// x [M, ldx], w [N, ldw] 8-bit integers whose rows start on 16-byte boundaries; xs [M], ws [N] (and bias [N] or null) float; out [M, ldo].
// tile 16, 32, 64 or 128: that many tokens to a block, `splits` (1, 2, 4, 8, at most the blocks of 128 k) blocks to a tile; tile 256: 256 tokens and
// `features` (a multiple of 64 up to 256) to a pair, `splits` (1 or 2) pairs to a tile.  `early`: the kernel before this one in the stream did not write w.
NS_API int ns_gemm_i8(const void* x, long long ldx, const float* xs, const void* w, long long ldw, const float* ws, const float* bias, void* out,
                      long long ldo, int M, int N, int K, int dtype, int tile, int features, int splits, int early, int sms, int* error_flag, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return NS_OK;
    if (K < 1 || K > 131072) NS_FAIL(NS_ERR_UNSUPPORTED, "ns_gemm_i8: K=%d (1 to 131072)", K);
    if (ldx % 16 || ldw % 16 || ((uintptr_t)x | (uintptr_t)w) % 16) NS_FAIL(NS_ERR_UNSUPPORTED, "ns_gemm_i8: rows must start on 16-byte boundaries");
    if (dtype != NS_BF16 && dtype != NS_F32) NS_FAIL(NS_ERR_UNSUPPORTED, "ns_gemm_i8: float32 and bfloat16 outputs, not type %d", dtype);
    const int k_blocks = (K + BK - 1) / BK;
    if (!error_flag || splits < 1 || splits > (tile == 256 ? 2 : 8) || (splits & (splits - 1)) || splits > k_blocks ||
        (tile == 256 && (features < 64 || features > 256 || features % 64)))
        NS_FAIL(NS_ERR_ARGUMENT, "ns_gemm_i8: tiles of %d x %d, %d blocks to a tile with %d blocks of k", tile, features, splits, k_blocks);
    if (tile < 256 && (M + tile - 1) / tile > 65535) NS_FAIL(NS_ERR_UNSUPPORTED, "ns_gemm_i8: too many rows (%d)", M);
#define NS_I8_NARROW(BNN)                                                                                                                            \
    case BNN:                                                                                                                                        \
        return dtype == NS_F32 ? narrow::launch<BNN, float>(x, ldx, xs, w, ldw, ws, bias, out, ldo, M, N, K, splits, early, error_flag, stream)     \
                               : narrow::launch<BNN, __nv_bfloat16>(x, ldx, xs, w, ldw, ws, bias, out, ldo, M, N, K, splits, early, error_flag, stream);
    switch (tile) {
        NS_I8_NARROW(16) NS_I8_NARROW(32) NS_I8_NARROW(64) NS_I8_NARROW(128)
        case 256:
            return dtype == NS_F32 ? wide::launch<float>(x, ldx, xs, w, ldw, ws, bias, out, ldo, M, N, K, features, splits, sms, error_flag, stream)
                                   : wide::launch<__nv_bfloat16>(x, ldx, xs, w, ldw, ws, bias, out, ldo, M, N, K, features, splits, sms, error_flag, stream);
    }
#undef NS_I8_NARROW
    NS_FAIL(NS_ERR_ARGUMENT, "ns_gemm_i8: tiles of %d tokens", tile);
}

extern "C" int ns_quantize_rows(const void* x, long long ldx, void* q, long long ldq, float* scale, int rows, int K, int dtype, cudaStream_t stream);

// The product of x [M, ldx] in `x_dtype`, quantised by rows on the way: `scratch`, on a 16-byte boundary, holds M rows of K bytes rounded up to 16 and M floats.
NS_API int ns_linear_i8(const void* x, long long ldx, int x_dtype, void* scratch, const void* w, long long ldw, const float* ws, const float* bias, void* out,
                        long long ldo, int M, int N, int K, int dtype, int tile, int features, int splits, int sms, int* error_flag, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return NS_OK;
    if (K < 1 || K > 131072) NS_FAIL(NS_ERR_UNSUPPORTED, "ns_linear_i8: K=%d (1 to 131072)", K);
    const long long ldq = (K + 15) / 16 * 16;
    float* xs = reinterpret_cast<float*>(static_cast<char*>(scratch) + (size_t)M * ldq);
    if (const int rc = ns_quantize_rows(x, ldx, scratch, ldq, xs, M, K, x_dtype, stream)) return rc;
    return ns_gemm_i8(scratch, ldq, xs, w, ldw, ws, bias, out, ldo, M, N, K, dtype, tile, features, splits, 1, sms, error_flag, stream);
}
