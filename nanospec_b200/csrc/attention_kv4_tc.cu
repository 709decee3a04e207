// Attention of single tokens, and of a few tokens of a request, over the 4-bit cache (kv4.cuh) in bfloat16 on the tensor cores (m16n8k16).
//
// A (query head, token) pair is a column, eight to an n-block: the cached keys and values are the left operands, so that a group of up to
// eight query heads fills the instruction, and the scores' and the outputs' columns are the same lanes'.
//   scores^T [keys x columns] = K [keys x features] q^T.  The contracted order is free as long as q has the same: a lane takes a quarter of a
//     key's features in one load, which lie in one or two groups, and pairs feature p with p + 4 of every word, as the codes lie.
//   out^T [features x columns] += V^T [features x keys] weights^T.  A lane takes an eighth of four keys' features; the codes of two keys are
//     brought side by side (two byte permutations for eight features), and the same shift, mask and fma make two values.  The weights turn from
//     the scores' layout into the right operand's by one 8 x 8 transposition of 16-bit numbers in registers.
// Rows of the score tile are dealt to keys (row_key) such that both sides' reads of shared memory spread over the banks.
//
// Every warp is on its own: it takes every (warps of the request's blocks)-th tile of 32 keys, brings it in 16-byte pieces into its own ring (bulk copies, a
// lane each for the codes and pairs of a page, took as long as the tile's arithmetic: their addresses are not a warp's but a lane's), and keeps its own maximum,
// sum and output; the block's warps are joined at its end in a fixed order.  A request that has several blocks leaves their parts in a workspace, which a second
// kernel joins in a fixed order too: blocks of one size then fill the SMs whatever the requests' lengths are (a cluster that joins its blocks over distributed shared
// memory ends at sixteen and leaves the SMs beyond its own idle: one request on 100,000 keys took 72 us so, 47 now).  The running maximum moves only when a score
// exceeds it by more than 2^8 (weights are then at most 256, far from any limit of float or bfloat16); the common tile costs a vote.
//
// The weights meet the values as bfloat16, as in the attention over a bfloat16 cache; sums, maximum and outputs are float.
//
// Where all SMs have as much to do, bound by their integer pipe, not by memory: 384 of a tile's about 690 instructions a warp (heads of 128) make values of codes, more than half of those in the logic
// pipe, which issues every second cycle and is busy for 60 % of 1,160 cycles a tile and scheduler; the rest is four warps a scheduler that wait for it or for
// one another's turn.  74 requests on 4,096 keys of 8 kv heads: 86 us (pages of 64 tokens; 94 of 16), 4.5 TB/s, the same where all requests read the same
// page.  On ragged lengths nothing is near a limit: 64 on up to 2,300 keys, 111 MB, 49 us (SMs 38 % busy, memory 30 %: the blocks of the longest requests outlast the
// others); two, on 100,001 and 33,428, 171 MB, 49 us with the join (49 and 47 %); 18 tiles of a few tokens on up to 3,000, 43 MB, 31 us (34 and 19 %: a block's five tiles a
// warp stand between a chain of dependent loads and the merging of its warps).
#include "kv4.cuh"
#include "mma_utils.cuh"
#include "tcgen05_utils.cuh"

namespace {

constexpr int kTile = 32, kStages = 2;
constexpr float kLog2e = 1.4426950408889634f, kSlack = 8.f;

__device__ __forceinline__ void copy16(void* to, const void* from) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(ns_smem_u32(to)), "l"(from) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <int N>
__device__ __forceinline__ void lds(uint32_t (&v)[N], const unsigned char* p) {
    if constexpr (N == 1) v[0] = *reinterpret_cast<const uint32_t*>(p);
    else if constexpr (N == 2) {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        v[0] = u.x; v[1] = u.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 u = *reinterpret_cast<const uint4*>(p + 4 * i);
            v[i] = u.x; v[i + 1] = u.y; v[i + 2] = u.z; v[i + 3] = u.w;
        }
    }
}

template <int D, int NB, int kWarps>
struct Shape {
    static constexpr int kThreads = 32 * kWarps, kResident = D > 128 ? 8 / kWarps : kWarps == 8 ? 2 : NB == 2 ? 3 : D == 64 ? 6 : 4;  // blocks an SM (185 requests on
    // 1,023 keys, heads of 64: four 52 us, six 49; of 128, whose registers would do for five, no gain)
    static constexpr int kCols = 8 * NB, kWords = D / 32, kVWords = D / 64, kBlocks = D / 16;  // words of a lane per key; m-blocks of features
    static constexpr int kCodes = kTile * D / 2, kPairs = kTile * D / 8, kStage = 2 * (kCodes + kPairs);
    static constexpr int kRing = kStages * kStage;
    static_assert(kRing >= kCols * D * 4, "a warp's output is staged where its ring was");
    static constexpr int kQBytes = NB * kWords * 512;  // q's operands, 16 bytes a lane
    static constexpr size_t kSmem = (size_t)kWarps * kRing + kQBytes;
};

// What a block, or all blocks of a (row, kv head), have in common.  tokens: `items` [n, 2] = (first row, tokens), rows `rows` [n] of one token each, or row z.
struct Place {
    int n0, count, req, pos0, hk, h0, heads, cols, end, start, tile0, tiles;
    __device__ __forceinline__ Place(int z, int y, const int* items, const int* rows, const int* token_req, const int* positions, int nq, int nkv, int head_tiles,
                                     int kCols, int window)
        : Place(items ? items[2 * z] : rows ? rows[z] : z, items ? items[2 * z + 1] : 1, y, token_req, positions, nq, nkv, head_tiles, kCols, window) {}
    __device__ __forceinline__ Place(int row, int tokens, int y, const int* token_req, const int* positions, int nq, int nkv, int head_tiles, int kCols, int window) {
        n0 = row, count = tokens;
        req = token_req[n0], pos0 = positions[n0];
        const int G = nq / nkv, ht = y % head_tiles, per = min(G, kCols);
        hk = y / head_tiles, h0 = hk * G + ht * per, heads = min(per, hk * G + G - h0);  // heads of a token here
        cols = count * heads;
        end = pos0 + count;  // keys below `end` are seen by some column
        start = window > 0 ? max(0, pos0 - window + 1) : 0;
        tile0 = start / kTile, tiles = (end + kTile - 1) / kTile - tile0;
    }
    __device__ __forceinline__ int parts(int most, int least) const { return max(1, min(most, (tiles + least - 1) / least)); }  // blocks, of `least` tiles or more each
};
// A warp's part of a column, or a block's: 2^(its maximum - the whole's); one that saw no key adds nothing, one whose scores are all NaN makes the column NaN.
__device__ __forceinline__ float share(float m_part, float l_part, float top) { return m_part == -INFINITY ? 0.f * l_part : ns_exp2(m_part - top); }

// kPages: pages of a tile, 1 or 2 (whole or half tiles in a page), or 0: by page_size
template <int D, int NB, int kWarps, int kPages>
__global__ void __launch_bounds__(32 * kWarps, Shape<D, NB, kWarps>::kResident)
attention_kv4_tc_kernel(const __nv_bfloat16* __restrict__ q, long long ldq, const uint8_t* __restrict__ k_pages, const uint8_t* __restrict__ v_pages,
                        const int* __restrict__ block_table, int table_stride, const int* __restrict__ token_req, const int* __restrict__ positions,
                        const int* __restrict__ rows, const int* __restrict__ items, __nv_bfloat16* __restrict__ out, long long ldo, int nq, int nkv,
                        int page_size, float scale, int window, const float* __restrict__ sink, int head_tiles, int splits, int page_shift, float* __restrict__ part,
                        const int4* __restrict__ jobs, int least) {
    using S = Shape<D, NB, kWarps>;
    constexpr int kThreads = S::kThreads;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float m_s[kWarps][S::kCols], l_s[kWarps][S::kCols], mb_s[S::kCols], lb_s[S::kCols];
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, t = lane & 3, r = lane >> 2;
    unsigned char* ring = smem + warp * S::kRing;
    uint4* q_s = reinterpret_cast<uint4*>(smem + (size_t)kWarps * S::kRing);

    ns_pdl_launch_dependents();
    ns_pdl_wait();

    const int unit = (int)blockIdx.x / (nkv * head_tiles), y = (int)blockIdx.x - unit * nkv * head_tiles;  // (a row's heads come together: the longest rows first)
    const int z = unit / splits;
    const int4 job = jobs ? jobs[unit] : make_int4(items ? items[2 * z] : rows ? rows[z] : z, items ? items[2 * z + 1] : 1, unit - z * splits, 0);  // row, tokens, part, of how many
    const Place at(job.x, job.y, y, token_req, positions, nq, nkv, head_tiles, S::kCols, window);
    if (at.req < 0) return;  // a row of padding
    const int n0 = at.n0, pos0 = at.pos0, hk = at.hk, h0 = at.h0, heads = at.heads, cols = at.cols, end = at.end, start = at.start, tile0 = at.tile0, tiles = at.tiles;
    const int* bt = block_table + (size_t)at.req * table_stride;
    const int blocks = jobs ? job.w : part ? at.parts(splits, least) : 1;
    if (job.z >= blocks) return;
    const int step = blocks * kWarps, first = job.z * kWarps + warp;

    // a tile: 16-byte pieces, codes and pairs of keys and of values, from the pages that it lies in (1, 2 or 4)
    const int page_log = kPages == 1 ? 5 : kPages == 2 ? 4 : 31 - __clz(min(kTile, page_size)), pages = kTile >> page_log;  // keys of a page in a tile
    const unsigned block_bytes = (unsigned)kv4_block_bytes(page_size, D);
    // Where the blocks of a tile begin, or -1 (the table is read a tile ahead: its latency would stand before every copy): each lane knows the one or two,
    // or lane i the i-th of more.
    constexpr int kKnown = kPages == 2 ? 2 : 1;
    struct Blocks { long long at[kKnown]; };
    auto blocks_of = [&](int i) {
        Blocks b;
#pragma unroll
        for (int u = 0; u < kKnown; ++u) {
            const int which = kPages ? u : lane, key = (tile0 + i) * kTile + (which << page_log);
            const bool live = i < tiles && which < pages && key < end && key + (1 << page_log) > start;
            b.at[u] = live ? (long long)((unsigned)(bt[page_shift >= 0 ? key >> page_shift : key / page_size] * nkv + hk) * (unsigned long long)block_bytes) : -1;
        }
        return b;
    };
    auto request = [&](int i, int turn, const Blocks& b) {  // tile `i` of this request's, the warp's turn-th, into stage turn % kStages
        unsigned char* to = ring + turn % kStages * S::kStage + lane * 16;
        const int key0 = (tile0 + i) * kTile, slot0 = kPages == 2 ? 0 : page_shift >= 0 ? key0 & (page_size - 1) : key0 % page_size;
        const uint8_t *kb = k_pages + slot0 * (D / 2) + lane * 16, *vb = v_pages + slot0 * (D / 2) + lane * 16;
        const int to_pairs = page_size * (D / 2) - slot0 * (D / 2 - D / 8);
        // (the block of a lane's piece, and how far the piece's page lies behind the tile's beginning)
        auto copy = [&](int o, int row, unsigned char* k_to, unsigned char* v_to, int skip, bool there) {  // o: the lane's byte among those of `row` bytes a token
            const int which = o / row >> page_log;
            long long from;
            if (kPages == 1) from = b.at[0];
            else if (kPages == 2) from = which ? b.at[kKnown - 1] : b.at[0];
            else from = __shfl_sync(0xffffffffu, b.at[0], which & 31);
            from += skip - (which << page_log) * row;
            if (there && (kPages == 1 || from >= skip - (which << page_log) * row)) {
                copy16(k_to, kb + from);
                copy16(v_to, vb + from);
            }
        };
#pragma unroll
        for (int c = 0; c < S::kCodes / 512; ++c) copy(c * 512 + lane * 16, D / 2, to + c * 512, to + S::kCodes + S::kPairs + c * 512, c * 512, true);
#pragma unroll
        for (int c = 0; c < (S::kPairs + 511) / 512; ++c)  // (every lane takes part in the exchange, those beyond the pairs copy nothing)
            copy(c * 512 + lane * 16, D / 8, to + S::kCodes + c * 512, to + 2 * S::kCodes + S::kPairs + c * 512, to_pairs + c * 512, c * 512 + lane * 16 < S::kPairs);
    };
    {
        Blocks block[kStages];
#pragma unroll
        for (int s = 0; s < kStages; ++s) block[s] = blocks_of(first + s * step);
#pragma unroll
        for (int s = 0; s < kStages; ++s) {
            if (first + s * step < tiles) request(first + s * step, s, block[s]);
            ns_cp_async_commit();
        }
    }

    // q as right operand: column r of each n-block, word w of the lane's quarter: pairs (p, p + 4)
    for (int i = warp; i < NB * S::kWords; i += kWarps) {
        const int nb = i / S::kWords, w = i - nb * S::kWords, c = nb * 8 + r;
        uint32_t v[4] = {0u, 0u, 0u, 0u};
        if (c < cols) {
            const __nv_bfloat16* x = q + (size_t)(n0 + c / heads) * ldq + (size_t)(h0 + c % heads) * D + 8 * (t * S::kWords + w);
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const __nv_bfloat162 two = __halves2bfloat162(x[p], x[p + 4]);
                v[p] = *reinterpret_cast<const uint32_t*>(&two);
            }
        }
        q_s[i * 32 + lane] = make_uint4(v[0], v[1], v[2], v[3]);
    }
    __syncthreads();
    uint32_t qf[NB == 1 ? S::kWords : 1][4];
    if constexpr (NB == 1) {
#pragma unroll
        for (int w = 0; w < S::kWords; ++w) {
            const uint4 u = q_s[w * 32 + lane];
            qf[w][0] = u.x; qf[w][1] = u.y; qf[w][2] = u.z; qf[w][3] = u.w;
        }
    }
    // the last key that each of this lane's columns sees (columns beyond the last: of the last)
    int limit[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int j = 0; j < 2; ++j) limit[nb][j] = pos0 + min(nb * 8 + 2 * t + j, cols - 1) / heads;

    float m_use[NB][2], slack[NB][2], l[NB][2], o[NB][S::kBlocks][4];  // the maximum, or 0 while no key was seen (slack: -infinity then)
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int j = 0; j < 2; ++j) { slack[nb][j] = -INFINITY; m_use[nb][j] = l[nb][j] = 0.f; }
#pragma unroll
        for (int b = 0; b < S::kBlocks; ++b)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[nb][b][j] = 0.f;
    }
    const float sl = scale * kLog2e;
    const int row_key = (r & 1) ? 4 + ((r >> 1) ^ 1) : r >> 1;  // key of row r (and, 8 further, of row r + 8)
    int turn = 0;
    for (int i = first; i < tiles; i += step, ++turn) {
        const int stage = turn % kStages;
        const Blocks next_block = blocks_of(i + kStages * step);
        ns_cp_async_wait<kStages - 1>();
        __syncwarp();  // ... of every lane
        const unsigned char *kc = ring + stage * S::kStage, *kp = kc + S::kCodes, *vc = kp + S::kPairs, *vp = vc + S::kCodes;
        const int key0 = (tile0 + i) * kTile;
        float s[NB][2][4];  // [half of the tile][(row r, columns 2t, 2t + 1), (row r + 8, ...)]
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int ka = half * 16 + row_key;
            uint32_t ca[S::kWords], cb[S::kWords];
            lds(ca, kc + ka * (D / 2) + t * (D / 8));
            lds(cb, kc + (ka + 8) * (D / 2) + t * (D / 8));
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[nb][half][j] = 0.f;
            uint32_t Sa = 0u, Ba = 0u, Sb = 0u, Bb = 0u;
#pragma unroll
            for (int w = 0; w < S::kWords; ++w) {
                if (w % 4 == 0) {  // (a lane's words begin at a group, or lie in one)
                    const int g = (t * S::kWords + w) / 4;
                    kv4_pair(*reinterpret_cast<const uint32_t*>(kp + ka * (D / 8) + 4 * g), Sa, Ba);
                    kv4_pair(*reinterpret_cast<const uint32_t*>(kp + (ka + 8) * (D / 8) + 4 * g), Sb, Bb);
                }
                uint32_t va[4], vb[4];
                kv4_word(ca[w], Sa, Ba, va);
                kv4_word(cb[w], Sb, Bb, vb);
                const uint32_t a0[4] = {va[0], vb[0], va[1], vb[1]}, a1[4] = {va[2], vb[2], va[3], vb[3]};
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    if constexpr (NB == 1) {
                        ns_mma_bf16(s[nb][half], a0, qf[w][0], qf[w][1]);
                        ns_mma_bf16(s[nb][half], a1, qf[w][2], qf[w][3]);
                    } else {
                        const uint4 u = q_s[(nb * S::kWords + w) * 32 + lane];
                        ns_mma_bf16(s[nb][half], a0, u.x, u.y);
                        ns_mma_bf16(s[nb][half], a1, u.z, u.w);
                    }
                }
            }
        }
        // scores in base 2, relative to the running maximum; keys that a column does not see
        const bool whole = key0 >= start && key0 + kTile <= end;                          // every key is there
        const bool plain = key0 + kTile - 1 <= pos0 && (window <= 0 || key0 > end - 1 - window);  // ... and seen by every column
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float v = s[nb][half][j] * sl - m_use[nb][j & 1];
                    s[nb][half][j] = v;
                }
        if (!plain) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int key = key0 + half * 16 + row_key + (j & 2 ? 8 : 0), last = limit[nb][j & 1];
                        if (key > last || (window > 0 && key <= last - window)) s[nb][half][j] = -INFINITY;
                    }
        }
        bool over = false;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                over |= fmaxf(fmaxf(s[nb][0][j], s[nb][0][j + 2]), fmaxf(s[nb][1][j], s[nb][1][j + 2])) > slack[nb][j];
        if (__any_sync(0xffffffffu, over)) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float top = fmaxf(fmaxf(s[nb][0][j], s[nb][0][j + 2]), fmaxf(s[nb][1][j], s[nb][1][j + 2]));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                    // (relative to the maximum so far: what lies below it does not move it)
                    const bool none = slack[nb][j] == -INFINITY;
                    const float by = none ? (top == -INFINITY ? 0.f : -top) : fminf(-top, 0.f), keep = none ? 1.f : ns_exp2(by);
                    if (top != -INFINITY) slack[nb][j] = kSlack;
                    m_use[nb][j] -= by;
#pragma unroll
                    for (int half = 0; half < 2; ++half) { s[nb][half][j] += by; s[nb][half][j + 2] += by; }
                    l[nb][j] *= keep;
#pragma unroll
                    for (int b = 0; b < S::kBlocks; ++b) { o[nb][b][j] *= keep; o[nb][b][j + 2] *= keep; }
                }
        }
        uint32_t pb[NB][2][2];  // the weights as right operand, [half][keys 2t, 2t + 1; 2t + 8, 2t + 9]
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const float p0 = ns_exp2(s[nb][half][0]), p1 = ns_exp2(s[nb][half][1]), p2 = ns_exp2(s[nb][half][2]), p3 = ns_exp2(s[nb][half][3]);
                l[nb][0] += p0 + p2;
                l[nb][1] += p1 + p3;
                pb[nb][half][0] = transpose8(ns_pack_bf16(p0, p1));
                pb[nb][half][1] = transpose8(ns_pack_bf16(p2, p3));
            }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            // keys of rows 2t, 2t + 1, 2t + 8, 2t + 9
            const int keys[4] = {half * 16 + t, half * 16 + 4 + (t ^ 1), half * 16 + 8 + t, half * 16 + 12 + (t ^ 1)};
            uint32_t c[4][S::kVWords], pair[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                lds(c[k], vc + keys[k] * (D / 2) + r * (D / 16));
                pair[k] = *reinterpret_cast<const uint32_t*>(vp + keys[k] * (D / 8) + 4 * (r * S::kVWords / 4));
            }
            if (!whole) {  // what is not there (or nobody's yet) counts as zeros: a weight of zero must not meet a NaN
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (key0 + keys[k] < start || key0 + keys[k] >= end) pair[k] = 0u;
            }
            const uint32_t S01 = __byte_perm(pair[0], pair[1], 0x5410), B01 = __byte_perm(pair[0], pair[1], 0x7632);
            const uint32_t S89 = __byte_perm(pair[2], pair[3], 0x5410), B89 = __byte_perm(pair[2], pair[3], 0x7632);
#pragma unroll
            for (int w = 0; w < S::kVWords; ++w) {
                // features 0-3 of two keys side by side, then 4-7
                uint32_t x01[4], y01[4], x89[4], y89[4];
                kv4_word(__byte_perm(c[0][w], c[1][w], 0x5410), S01, B01, x01);
                kv4_word(__byte_perm(c[0][w], c[1][w], 0x7632), S01, B01, y01);
                kv4_word(__byte_perm(c[2][w], c[3][w], 0x5410), S89, B89, x89);
                kv4_word(__byte_perm(c[2][w], c[3][w], 0x7632), S89, B89, y89);
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    const uint32_t a[4] = {x01[p], y01[p], x89[p], y89[p]};
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) ns_mma_bf16(o[nb][w * 4 + p], a, pb[nb][half][0], pb[nb][half][1]);
                }
            }
        }
        __syncwarp();  // every lane has read the tile
        if (i + kStages * step < tiles) request(i + kStages * step, turn, next_block);
        ns_cp_async_commit();
    }
    ns_cp_async_wait<0>();

    // ---- the block's warps -----------------------------------------------------------------------------------------------------------
    float* mine = reinterpret_cast<float*>(ring);  // [column][feature]
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            l[nb][j] += __shfl_xor_sync(0xffffffffu, l[nb][j], 4);
            l[nb][j] += __shfl_xor_sync(0xffffffffu, l[nb][j], 8);
            l[nb][j] += __shfl_xor_sync(0xffffffffu, l[nb][j], 16);
            if (r == 0) {
                m_s[warp][nb * 8 + 2 * t + j] = slack[nb][j] == -INFINITY ? -INFINITY : m_use[nb][j];
                l_s[warp][nb * 8 + 2 * t + j] = l[nb][j];
            }
        }
#pragma unroll
        for (int b = 0; b < S::kBlocks; ++b) {
            const int f = r * (D / 8) + (b / 4) * 8 + (b & 3), c = nb * 8 + 2 * t;
            mine[c * D + f] = o[nb][b][0];
            mine[(c + 1) * D + f] = o[nb][b][1];
            mine[c * D + f + 4] = o[nb][b][2];
            mine[(c + 1) * D + f + 4] = o[nb][b][3];
        }
    }
    __syncthreads();
    float* block_o = reinterpret_cast<float*>(smem);  // (warp 0's: every thread reads its own elements before it writes them)
    for (int e = threadIdx.x; e < cols * D; e += kThreads) {
        const int c = e / D;
        float top = -INFINITY, acc = 0.f, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, m_s[w][c]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = share(m_s[w][c], l_s[w][c], top);
            acc += f * reinterpret_cast<const float*>(smem + w * S::kRing)[e];
            sum += f * l_s[w][c];
        }
        block_o[e] = acc;
        if (e % D == 0) { mb_s[c] = top; lb_s[c] = sum; }
    }
    __syncthreads();
    if (part) {  // attention_kv4_join_kernel goes on from here
        float* to = part + (size_t)blockIdx.x * S::kCols * (D + 2);
        for (int c = threadIdx.x; c < cols; c += kThreads) { to[2 * c] = mb_s[c]; to[2 * c + 1] = lb_s[c]; }
        for (int e = threadIdx.x; e < cols * D / 4; e += kThreads) reinterpret_cast<float4*>(to + 2 * S::kCols)[e] = reinterpret_cast<const float4*>(block_o)[e];
        return;
    }
    for (int e = threadIdx.x; e < cols * D / 2; e += kThreads) {
        const int c = 2 * e / D, f = 2 * e - c * D, h = h0 + c % heads;
        const float sink2 = sink ? sink[h] * kLog2e : -INFINITY, top = fmaxf(sink2, mb_s[c]), w = share(mb_s[c], lb_s[c], top);
        const float sum = w * lb_s[c] + (sink ? ns_exp2(sink2 - top) : 0.f);
        __nv_bfloat16* to = out + (size_t)(n0 + c / heads) * ldo + (size_t)h * D + f;
        to[0] = __float2bfloat16_rn(w * block_o[2 * e] / sum);
        to[1] = __float2bfloat16_rn(w * block_o[2 * e + 1] / sum);
    }
}

// Joins the blocks of a (row, kv head): `team` warps a column (1, 2, 4 or 8, more where there are more parts), each of which forms the weights of all parts and
// adds up every team-th part, a lane D / 32 features; then the team's sums in their order.  (With a block of 256 threads to every column, 16 requests of up to 6
// tokens on 3,000 keys took 32.4 us in all, now 31.0.)
constexpr int kMostParts = 256, kJoinWarps = 8;
template <int D>
__global__ void __launch_bounds__(32 * kJoinWarps)
attention_kv4_join_kernel(const float* __restrict__ part, const int* __restrict__ token_req, const int* __restrict__ positions, const int* __restrict__ rows,
                          const int* __restrict__ items, __nv_bfloat16* __restrict__ out, long long ldo, int nq, int nkv, int kCols, int window,
                          const float* __restrict__ sink, int head_tiles, int splits, const int* __restrict__ spans, int least, int team) {
    constexpr int kPer = D / 32;
    __shared__ float w_s[kJoinWarps][kMostParts];
    __shared__ float o_s[kJoinWarps][D];
    ns_pdl_launch_dependents();
    ns_pdl_wait();
    const int per_row = nkv * head_tiles, z = (int)blockIdx.x / per_row, y = (int)blockIdx.x - z * per_row;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, member = warp & (team - 1), c = (int)blockIdx.y * (kJoinWarps / team) + warp / team;
    const Place at(z, y, items, rows, token_req, positions, nq, nkv, head_tiles, kCols, window);
    const int blocks = spans ? spans[2 * z + 1] : at.parts(splits, least);
    const size_t each = (size_t)per_row * kCols * (D + 2);  // from a part of the row to its next one
    const float* from = part + ((size_t)(spans ? spans[2 * z] : z * splits) * per_row + y) * kCols * (D + 2);
    const bool live = at.req >= 0 && c < at.cols;
    float acc[kPer], sum = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] = 0.f;
    if (live) {
        const float sink2 = sink ? sink[at.h0 + c % at.heads] * kLog2e : -INFINITY;
        float2 ml[kMostParts / 32];
        float top = sink2;
#pragma unroll
        for (int i = 0; i < kMostParts / 32; ++i) {
            ml[i] = make_float2(-INFINITY, 0.f);
            if (i * 32 + lane < blocks) ml[i] = *reinterpret_cast<const float2*>(from + (i * 32 + lane) * each + 2 * c);
            top = fmaxf(top, ml[i].x);
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
#pragma unroll
        for (int i = 0; i < kMostParts / 32; ++i) {
            if (i * 32 >= blocks) break;
            const float w = share(ml[i].x, ml[i].y, top);
            w_s[warp][i * 32 + lane] = w;
            sum += w * ml[i].y;
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (sink) sum += ns_exp2(sink2 - top);
        __syncwarp();
        const float* o = from + 2 * kCols + c * D + kPer * lane;
#pragma unroll 8
        for (int b = member; b < blocks; b += team) {
            const float w = w_s[warp][b];
            float v[kPer];
            if constexpr (kPer == 2) { const float2 u = *reinterpret_cast<const float2*>(o + b * each); v[0] = u.x; v[1] = u.y; }
            else {
#pragma unroll
                for (int i = 0; i < kPer; i += 4) {
                    const float4 u = *reinterpret_cast<const float4*>(o + b * each + i);
                    v[i] = u.x; v[i + 1] = u.y; v[i + 2] = u.z; v[i + 3] = u.w;
                }
            }
#pragma unroll
            for (int i = 0; i < kPer; ++i) acc[i] += w * v[i];
        }
    }
    if (team > 1) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) o_s[warp][kPer * lane + i] = acc[i];
        __syncthreads();
        if (member == 0)
            for (int w = 1; w < team; ++w)
#pragma unroll
                for (int i = 0; i < kPer; ++i) acc[i] += o_s[warp + w][kPer * lane + i];
    }
    if (live && member == 0) {
        __nv_bfloat16* to = out + (size_t)(at.n0 + c / at.heads) * ldo + (size_t)(at.h0 + c % at.heads) * D + kPer * lane;
#pragma unroll
        for (int i = 0; i < kPer; ++i) to[i] = __float2bfloat16_rn(acc[i] / sum);
    }
}

template <int D, int NB, int kWarps, int kPages>
int launch(const void* q, long long ldq, const void* k, const void* v, const int* table, int table_stride, const int* token_req, const int* positions,
           const int* rows, const int* items, int n, void* out, long long ldo, int nq, int nkv, int page_size, float scale, int window, const float* sink,
           int splits, float* part, const int* jobs, int n_jobs, int least, cudaStream_t stream) {
    using S = Shape<D, NB, kWarps>;
    static std::atomic<unsigned long long> allowed{0};
    auto* kernel = attention_kv4_tc_kernel<D, NB, kWarps, kPages>;
    NS_CUDA(ns_allow_smem((const void*)kernel, (int)S::kSmem, allowed));
    const int head_tiles = (nq / nkv + S::kCols - 1) / S::kCols;
    const long long per_row = (long long)nkv * head_tiles, grid = per_row * (jobs ? n_jobs : (long long)n * splits);
    if (grid > 0x7fffffff) NS_FAIL(NS_ERR_UNSUPPORTED, "ns_attention_kv4_tc: %d tokens, %d heads exceed the grid", n, nq);
    NS_LAUNCH(kernel, (unsigned)grid, S::kThreads, S::kSmem, stream, (const __nv_bfloat16*)q, ldq, (const uint8_t*)k, (const uint8_t*)v, table,
              table_stride, token_req, positions, rows, items, (__nv_bfloat16*)out, ldo, nq, nkv, page_size, scale, window, sink, head_tiles, splits,
              (page_size & (page_size - 1)) == 0 ? 31 - __builtin_clz(page_size) : -1, part, reinterpret_cast<const int4*>(jobs), least);
    NS_CHECK_LAUNCH("ns_attention_kv4_tc");
    if (part) {
        const int columns = items ? S::kCols : nq / nkv < S::kCols ? nq / nkv : S::kCols, team = splits <= 8 ? 1 : splits <= 16 ? 2 : splits <= 32 ? 4 : 8;
        NS_LAUNCH((attention_kv4_join_kernel<D>), dim3((unsigned)(per_row * n), (columns * team + kJoinWarps - 1) / kJoinWarps), 32 * kJoinWarps, 0, stream, part,
                  token_req, positions, rows, items, (__nv_bfloat16*)out, ldo, nq, nkv, S::kCols, window, sink, head_tiles, splits,
                  jobs ? jobs + 4 * n_jobs : nullptr, least, team);
        NS_CHECK_LAUNCH("ns_attention_kv4_tc");
    }
    return NS_OK;
}

}  // namespace

// bfloat16 q [tokens, ldq] and out [tokens, ldo]; heads of 64, 128 or 256; pages of 8, 16 or a multiple of 32 tokens.  Which tokens: `items` [n, 2] =
// (first row, tokens of one request, of which the heads that share a kv head fill at most 8 * n_blocks columns), or one token each: rows [n], or all n.
// A block to a (token or item, kv head), or, with `part`, several and a second kernel that joins them: `splits` (256 at most), of which those beyond one for each `least`
// tiles of 32 keys leave at once, or those of `jobs` [n_jobs, 4] = (first row, tokens, which part, of how many), each token's or item's in order and together, which
// [n, 2] = (first job, how many) follow.  `part`: nkv * tiles of heads * (n * splits or n_jobs) * 8 * n_blocks * (D + 2) floats.
NS_API int ns_attention_kv4_tc(const void* q, long long ldq, const void* k, const void* v, const int* table, int table_stride, const int* token_req,
                               const int* positions, const int* rows, const int* items, int n, void* out, long long ldo, int nq, int nkv, int D, int page_size,
                               float scale, int window, const float* sink, int n_blocks, int warps, int splits, float* part, const int* jobs, int n_jobs, int least, cudaStream_t stream) {
    if (n <= 0) return NS_OK;
    if (nkv < 1 || nq < 1 || nq % nkv || window < 0 || !(page_size == 8 || page_size == 16 || (page_size > 0 && page_size % 32 == 0)))
        NS_FAIL(NS_ERR_UNSUPPORTED, "ns_attention_kv4_tc: %d heads over %d, pages of %d, a window of %d", nq, nkv, page_size, window);
    if (splits < 1 || splits > (part ? kMostParts : 1) || (part && least < 1) || ((uintptr_t)part | (uintptr_t)jobs) % 16 || (jobs && (!part || n_jobs < 1)))
        NS_FAIL(NS_ERR_ARGUMENT, "ns_attention_kv4_tc: %d blocks to a request, of %d tiles or more", splits, least);
    if (((uintptr_t)k | (uintptr_t)v) % 16) NS_FAIL(NS_ERR_ARGUMENT, "ns_attention_kv4_tc: pages on 16-byte boundaries");
#define NS_KV4_CASE(DD, NBB, WW)                                                                                                                        \
    if (D == DD && n_blocks == NBB && warps == WW)                                                                                                     \
        return (page_size == 16 ? launch<DD, NBB, WW, 2> : page_size < 16 ? launch<DD, NBB, WW, 0> : launch<DD, NBB, WW, 1>)(q, ldq, k, v, table, table_stride, token_req, positions, rows, items, n, out, ldo, nq, nkv, page_size, scale,     \
                                   window, sink, splits, part, jobs, n_jobs, least, stream);
    NS_KV4_CASE(64, 1, 4) NS_KV4_CASE(64, 2, 4) NS_KV4_CASE(128, 1, 4) NS_KV4_CASE(128, 2, 4) NS_KV4_CASE(256, 1, 4) NS_KV4_CASE(256, 2, 4)
    NS_KV4_CASE(64, 1, 8) NS_KV4_CASE(64, 2, 8) NS_KV4_CASE(128, 1, 8) NS_KV4_CASE(128, 2, 8) NS_KV4_CASE(256, 1, 8) NS_KV4_CASE(256, 2, 8)
#undef NS_KV4_CASE
    NS_FAIL(NS_ERR_UNSUPPORTED, "ns_attention_kv4_tc: heads of %d, %d n-blocks, %d warps", D, n_blocks, warps);
}
