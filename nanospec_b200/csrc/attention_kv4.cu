// Attention over the 4-bit cache (kv4.cuh) for every head size, page size and type: softmax(q k^T scale) v over the positions
// max(0, p - window + 1) .. p of a token at position p, in float from the cached values on.
//
// A block takes a token and two, four or eight query heads of a kv head; its eight warps, and those of up to seven more blocks of a cluster, take tiles of 32 keys in
// turn, each with a running maximum and sum of its own, and are joined at the end in a fixed order.  Scores: a lane holds a key; weighted values: a lane holds
// features, and asks for the codes of eight keys before it uses the first (one at a time, the latency of each bounds the kernel: 2,236 keys of 16 heads of 32 168 us).
//
// 64 requests on up to 2,000 keys, four heads to each of 8 kv heads of 128: 162 us, 256 where every block computed for eight heads; four portions of up to 64 tokens on
// up to 500: 145, 273.  No pipe is near its limit there: its fused multiply-adds, two a feature, key and head, would take some 18 us.  While an SM has work, which is 71 %
// of the time on these ragged lengths, its schedulers issue in 57 % of the cycles (logic pipe 37 % busy, multiply-adds 27 %); the registers leave them four warps each,
// which wait for the codes (long scoreboard 1.3 an instruction), for one another's results (wait 1.2) and for q in shared memory (short scoreboard 0.8).
#include "kv4.cuh"
#include "tcgen05_utils.cuh"

namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps, kAhead = 8;

// kChunks of 128 features, kHeads query heads.  Two blocks an SM, which costs eight heads a few spilled registers: 16 requests on up to 2,000 keys, eight heads to each of 4
// kv heads of 128: 64 us with one block, 49 with two.
template <typename T, int kChunks, int kHeads>
__global__ void __launch_bounds__(kThreads, kChunks == 1 ? 2 : 1)
attention_kv4_kernel(const T* __restrict__ q, long long ldq, const uint8_t* __restrict__ k_pages, const uint8_t* __restrict__ v_pages,
                     const int* __restrict__ block_table, int table_stride, const int* __restrict__ token_req, const int* __restrict__ positions,
                     const int* __restrict__ rows, T* __restrict__ out, long long ldo, int nq, int nkv, int D, int page_size, float scale, int window,
                     const float* __restrict__ sink, int splits) {
    ns_pdl_launch_dependents();
    ns_pdl_wait();
    __shared__ __align__(16) float qs[kHeads][128 * kChunks];
    __shared__ float ps[kWarps][32][kHeads];
    __shared__ float ms[kWarps][kHeads], ls[kWarps][kHeads], mb[kHeads], lb[kHeads];
    extern __shared__ __align__(16) float os_dyn[];
    float (*os)[kHeads][128 * kChunks] = reinterpret_cast<float (*)[kHeads][128 * kChunks]>(os_dyn);
    const int z = blockIdx.x / splits, split = blockIdx.x % splits, n = rows ? rows[z] : z;
    const int req = token_req[n];
    if (req < 0) return;  // (all blocks of the cluster)
    const int G = nq / nkv, tiles = (G + kHeads - 1) / kHeads;
    const int hk = blockIdx.y / tiles, h0 = hk * G + (blockIdx.y % tiles) * kHeads;
    const int heads = min(kHeads, hk * G + G - h0);
    const int pos = positions[n], first = window > 0 ? max(0, pos - window + 1) : 0;
    const int* bt = block_table + (size_t)req * table_stride;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int i = threadIdx.x; i < kHeads * D; i += kThreads) {
        const int h = i / D, f = i % D;
        qs[h][f] = h < heads ? ns_ld(q, (size_t)n * ldq + (size_t)(h0 + h) * D + f) * scale : 0.f;
    }
    __syncthreads();
    float m[kHeads], l[kHeads], o[kHeads][kChunks][4];
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
        m[h] = -INFINITY;
        l[h] = 0.f;
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[h][c][i] = 0.f;
    }
    for (int k0 = first + (split * kWarps + warp) * 32; k0 <= pos; k0 += splits * kThreads) {
        const int key = k0 + lane, count = min(32, pos + 1 - k0);
        const bool seen = key <= pos;
        size_t block = 0;
        int slot = 0;
        float s[kHeads];
#pragma unroll
        for (int h = 0; h < kHeads; ++h) s[h] = 0.f;
        if (seen) {
            slot = key % page_size;
            block = ((size_t)bt[key / page_size] * nkv + hk) * kv4_block_bytes(page_size, D);
            const uint32_t* codes = reinterpret_cast<const uint32_t*>(k_pages + block + (size_t)slot * (D / 2));
            const uint32_t* pairs = reinterpret_cast<const uint32_t*>(k_pages + block + (size_t)page_size * (D / 2) + (size_t)slot * (D / 8));
#pragma unroll 4
            for (int w = 0; w < D / 8; ++w) {
                uint32_t S2, B2, v[4];
                kv4_pair(pairs[w / 4], S2, B2);
                kv4_word(codes[w], S2, B2, v);
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    const float2 x = kv4_floats(v[p]);
#pragma unroll
                    for (int h = 0; h < kHeads; ++h) s[h] = fmaf(qs[h][8 * w + p], x.x, fmaf(qs[h][8 * w + 4 + p], x.y, s[h]));
                }
            }
        }
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
            const float top = ns_warp_max(seen ? s[h] : -INFINITY), now = fmaxf(m[h], top), use = now == -INFINITY ? 0.f : now;
            const float keep = expf(m[h] - use), p = seen ? expf(s[h] - use) : 0.f;
            m[h] = now;
            l[h] = l[h] * keep + p;
#pragma unroll
            for (int c = 0; c < kChunks; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[h][c][i] *= keep;
            ps[warp][lane][h] = p;
        }
        __syncwarp();
        for (int j0 = 0; j0 < count; j0 += kAhead) {
            uint32_t code[kAhead][kChunks], pair[kAhead][kChunks];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const size_t b = __shfl_sync(0xffffffffu, block, j0 + u);
                const int at = __shfl_sync(0xffffffffu, slot, j0 + u);
#pragma unroll
                for (int c = 0; c < kChunks; ++c) {
                    const int f = c * 128 + lane * 4;
                    const bool live = f < D && j0 + u < count;
                    code[u][c] = live ? *reinterpret_cast<const uint16_t*>(v_pages + b + (size_t)at * (D / 2) + f / 2) : 0u;
                    pair[u][c] = live ? *reinterpret_cast<const uint32_t*>(v_pages + b + (size_t)page_size * (D / 2) + ((size_t)at * (D / kGroup) + f / kGroup) * 4) : 0u;
                }
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                if (j0 + u >= count) break;
#pragma unroll
                for (int c = 0; c < kChunks; ++c) {
                    uint32_t S2, B2;
                    kv4_pair(pair[u][c], S2, B2);
                    // codes 0 and 1 beside each other, then 2 and 3
                    const float2 x = kv4_floats(kv4_fma((code[u][c] << 3) | (code[u][c] & 0xf0u) << 15, S2, B2));
                    const float2 y = kv4_floats(kv4_fma((code[u][c] >> 5) | (code[u][c] & 0xf000u) << 7, S2, B2));
#pragma unroll
                    for (int h = 0; h < kHeads; ++h) {
                        const float p = ps[warp][j0 + u][h];
                        o[h][c][0] = fmaf(p, x.x, o[h][c][0]);
                        o[h][c][1] = fmaf(p, x.y, o[h][c][1]);
                        o[h][c][2] = fmaf(p, y.x, o[h][c][2]);
                        o[h][c][3] = fmaf(p, y.y, o[h][c][3]);
                    }
                }
            }
        }
        __syncwarp();
    }
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
        l[h] = ns_warp_sum(l[h]);
        if (lane == 0) { ms[warp][h] = m[h]; ls[warp][h] = l[h]; }
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
            *reinterpret_cast<float4*>(&os[warp][h][c * 128 + lane * 4]) = make_float4(o[h][c][0], o[h][c][1], o[h][c][2], o[h][c][3]);
    }
    __syncthreads();
    // the block's warps: a warp's part is 2^(its maximum - theirs); one that saw no key adds nothing, one whose scores are all NaN makes the row NaN
    auto share = [](float m_part, float l_part, float top) { return m_part == -INFINITY ? 0.f * l_part : expf(m_part - top); };
    for (int i = threadIdx.x; i < heads * D; i += kThreads) {
        const int h = i / D, f = i % D;
        float top = -INFINITY, sum = 0.f, acc = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ms[w][h]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float part = share(ms[w][h], ls[w][h], top);
            sum += part * ls[w][h];
            acc += part * os[w][h][f];
        }
        os[0][h][f] = acc;  // (this thread alone reads the element)
        if (f == 0) { mb[h] = top; lb[h] = sum; }
    }
    __syncthreads();
    // the cluster's blocks: each writes a share of the outputs
    if (splits > 1) cluster_sync();
    for (int i = split * kThreads + threadIdx.x; i < heads * D; i += splits * kThreads) {
        const int h = i / D, f = i % D;
        auto from = [&](const float* p, int s) { return splits == 1 ? *p : ld_cluster_f32(smem_u32(p), (uint32_t)s); };
        float top = sink ? sink[h0 + h] : -INFINITY, acc = 0.f;
        for (int s = 0; s < splits; ++s) top = fmaxf(top, from(&mb[h], s));
        float sum = sink ? expf(sink[h0 + h] - top) : 0.f;
        for (int s = 0; s < splits; ++s) {
            const float l_part = from(&lb[h], s), part = share(from(&mb[h], s), l_part, top);
            sum += part * l_part;
            acc += part * from(&os[0][h][f], s);
        }
        ns_st(out, (size_t)n * ldo + (size_t)(h0 + h) * D + f, acc / sum);
    }
    if (splits > 1) {
        __syncthreads();
        cluster_sync();  // nobody's shared memory goes while another block reads it
    }
}

template <typename T>
int launch(const void* q, long long ldq, const void* k, const void* v, const int* table, int table_stride, const int* token_req, const int* positions,
           const int* rows, int n_rows, void* out, long long ldo, int nq, int nkv, int D, int page_size, float scale, int window, const float* sink,
           int splits, cudaStream_t stream) {
    const int G = nq / nkv;
    auto run = [&](auto* kernel, int chunks, int heads, std::atomic<unsigned long long>& allowed) -> int {
        const int bytes = kWarps * heads * 128 * chunks * 4;
        NS_CUDA(ns_allow_smem((const void*)kernel, bytes, allowed));
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(n_rows * splits, nkv * ((G + heads - 1) / heads));
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = bytes;
        cfg.stream = stream;
        cudaLaunchAttribute attr[2];
        int n_attr = 0;
        if (ns_take_pdl()) {
            attr[n_attr].id = cudaLaunchAttributeProgrammaticStreamSerialization;
            attr[n_attr++].val.programmaticStreamSerializationAllowed = 1;
        }
        if (splits > 1) {
            attr[n_attr].id = cudaLaunchAttributeClusterDimension;
            attr[n_attr].val.clusterDim.x = splits;
            attr[n_attr].val.clusterDim.y = attr[n_attr].val.clusterDim.z = 1;
            ++n_attr;
        }
        cfg.attrs = attr;
        cfg.numAttrs = n_attr;
        (void)cudaLaunchKernelEx(&cfg, kernel, (const T*)q, ldq, (const uint8_t*)k, (const uint8_t*)v, table, table_stride, token_req, positions, rows, (T*)out, ldo,
                                 nq, nkv, D, page_size, scale, window, sink, splits);
        NS_CHECK_LAUNCH("ns_attention_kv4");
        return NS_OK;
    };
#define NS_KV4_HEADS(H)                                                                                   \
    {                                                                                                      \
        static std::atomic<unsigned long long> one{0}, two{0};                                            \
        return D <= 128 ? run(attention_kv4_kernel<T, 1, H>, 1, H, one) : run(attention_kv4_kernel<T, 2, H>, 2, H, two); \
    }
    if (G <= 2) NS_KV4_HEADS(2)
    if (G <= 4) NS_KV4_HEADS(4)
    NS_KV4_HEADS(8)
#undef NS_KV4_HEADS
}

}  // namespace

// q [tokens, ldq], out [tokens, ldo]; rows [n_rows]: the tokens to take (null: all n_rows); sink [nq] or null; splits: blocks that share a token's keys (1, 2, 4, 8).
NS_API int ns_attention_kv4(const void* q, long long ldq, const void* k, const void* v, const int* table, int table_stride, const int* token_req,
                            const int* positions, const int* rows, int n_rows, void* out, long long ldo, int nq, int nkv, int D, int page_size, float scale,
                            int window, const float* sink, int splits, int dtype, cudaStream_t stream) {
    if (n_rows <= 0) return NS_OK;
    if (D < kGroup || D % kGroup || D > 256 || nkv < 1 || nq < 1 || nq % nkv || page_size < 1 || window < 0)
        NS_FAIL(NS_ERR_UNSUPPORTED, "ns_attention_kv4: %d heads of %d over %d, pages of %d, a window of %d", nq, D, nkv, page_size, window);
    if (nkv * ((nq / nkv + 7) / 8) > 65535) NS_FAIL(NS_ERR_UNSUPPORTED, "ns_attention_kv4: too many heads (%d)", nq);
    if (splits < 1 || splits > 8 || (splits & (splits - 1)) || (long long)n_rows * splits > 0x7fffffff) NS_FAIL(NS_ERR_ARGUMENT, "ns_attention_kv4: %d blocks to each of %d tokens", splits, n_rows);
    if (dtype == NS_BF16)
        return launch<__nv_bfloat16>(q, ldq, k, v, table, table_stride, token_req, positions, rows, n_rows, out, ldo, nq, nkv, D, page_size, scale, window, sink, splits, stream);
    if (dtype == NS_F32)
        return launch<float>(q, ldq, k, v, table, table_stride, token_req, positions, rows, n_rows, out, ldo, nq, nkv, D, page_size, scale, window, sink, splits, stream);
    NS_FAIL(NS_ERR_UNSUPPORTED, "ns_attention_kv4: float32 and bfloat16, not type %d", dtype);
}
