// Store into the 4-bit cache, with the rotation of q and k, and reading values back (the format: kv4.cuh).
//
// What the cache holds is the definition's to the last bit: k rotated exactly and rounded once to the activations' type, S and B rounded once, codes decided by
// exact remainders.  One rounding that fell on the other side of a border would move a feature by a whole code, or a group by its S.  Computed in double
// throughout, a prompt is bound by its instructions (3,739 tokens of 32 + 2 x 8 heads of 128, 81 MB: 53 us, as all times here of a launch alone, 6 of which an empty
// one takes too); so everything is first done in float, with a bound of its error, and again in double where a border between two roundings lies within the
// bound - one element in some thousands.  The same tokens now take 38.9 us, of which 12.4 are their bytes at the rate of a copy: instructions still bound it, the
// schedulers issue in two cycles of three.  float32 activations, which have no bits to spare in float, are rotated in double (71.7 us, 158 MB, 24.1 at the rate of
// a copy).  q, which is rounded to the activations' type and not quantised, is rotated in float in both.
#include "kv4.cuh"

namespace {

constexpr int kThreads = 256;

// a double to the nearest bfloat16, ties to even, in one rounding: to float towards zero with the last bit marking that something was
// dropped (float has more than two bits beyond bfloat16's), then to bfloat16
__device__ __forceinline__ __nv_bfloat16 nearest_bf16(double d) {
    const float f = __double2float_rz(d);
    return __float2bfloat16_rn((double)f == d ? f : __uint_as_float(__float_as_uint(f) | 1u));
}
// Whether a float that is off by no more than a few of its last bits may lie on the other side of the middle between two bfloat16 numbers.
__device__ __forceinline__ bool near_middle(float f) { return (__float_as_uint(f) & 0xffffu) - 0x7ff8u <= 16u; }

// The angle position * frequency less whole turns, as a sum of two floats.
__device__ __forceinline__ void turned_angle(int pos, float freq, float& hi, float& lo) {
    const double a = (double)pos * (double)freq, n = rint(a * 0.15915494309189535);
    const double r = fma(-n, 2.4492935982947064e-16, fma(-n, 6.283185307179586, a));
    hi = (float)r;
    lo = (float)(r - (double)hi);
}
// Its cosine and sine to about three half steps: of the larger float, turned on by the smaller one.
__device__ __forceinline__ void cos_sin(int pos, float freq, float& c, float& s) {
    float hi, lo, c0, s0;
    turned_angle(pos, freq, hi, lo);
    sincosf(hi, &s0, &c0);
    c = fmaf(-s0, lo, c0);
    s = fmaf(c0, lo, s0);
}

__device__ __forceinline__ void ld4(const float* p, float (&v)[4]) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
}
__device__ __forceinline__ void ld4(const __nv_bfloat16* p, float (&v)[4]) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x)), b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
}

constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: added to it, a small number is rounded to an integer, which the last bits hold

constexpr float kHugeS = 8.507059173023462e37f;  // 2^126: from here on x - B, up to 1.95 S, may lie beyond float's range

// the code of x in a group: the integer nearest to 16 (x - B) / S - 16, ties to even, within 0 .. 15
__device__ __noinline__ uint32_t code_of(float x, float S, float B, float inv) {
    if (S >= kHugeS) {  // a quarter of everything: exact but for an x that counts in a tie only, by its sign
        if (fabsf(x) >= 1.f) x *= 0.25f;
        S *= 0.25f;
        B *= 0.25f;
        inv *= 4.f;
    }
    // d + rest = x - B without error
    const float d = __fsub_rn(x, B), back = __fsub_rn(d, x);
    const float rest = __fadd_rn(__fsub_rn(x, __fsub_rn(d, back)), __fsub_rn(-B, back));
    const float step = S * 0.0625f, half = 0.5f * step;
    float k = rintf(d * inv);
    const float e = fmaf(-k, step, d);  // exact where the code is not clamped: d is at most 33 steps
    const bool odd = ((int)k) & 1;
    if (e > half || (e == half && (rest > 0.f || (rest == 0.f && odd)))) k += 1.f;
    else if (e < -half || (e == -half && (rest < 0.f || (rest == 0.f && odd)))) k -= 1.f;
    return (uint32_t)fminf(fmaxf(k - 16.f, 0.f), 15.f);
}

struct Group { __nv_bfloat16 S, B; };

__device__ __noinline__ Group exact_group(float lo, float hi) {
    const double spread = ((double)hi - (double)lo) * 16.0 / 15.0;
    Group g;
    g.S = spread < 7.888609052210118e-31 /* 2^-100 */ ? __float2bfloat16_rn(0.f) : nearest_bf16(spread);
    g.B = nearest_bf16((double)lo - (double)__bfloat162float(g.S));
    return g;
}

// smallest and largest of a group, which lies over 8 neighbouring lanes
__device__ __forceinline__ void bounds(const float*, float& lo, float& hi) {
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
}
__device__ __forceinline__ void bounds(const __nv_bfloat16*, float& lo, float& hi) {  // (bfloat16 numbers, both in one register)
    __nv_bfloat162 b = __floats2bfloat162_rn(lo, -hi);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) b = __hmin2(b, __shfl_xor_sync(0xffffffffu, b, o));
    lo = __low2float(b);
    hi = -__high2float(b);
}

// S and B of a group, four features in each of 8 neighbouring lanes; S is NaN where the group, or what its largest code would stand for, is not finite
template <typename T>
__device__ __forceinline__ Group group_of(const T* type, const float (&x)[4], bool live) {
    float lo = fminf(fminf(x[0], x[1]), fminf(x[2], x[3])), hi = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    // (x - x is NaN for infinities and NaN, whose presence the minimum and maximum would hide)
    const bool mine = live && !((x[0] - x[0]) + (x[1] - x[1]) + (x[2] - x[2]) + (x[3] - x[3]) == 0.f);
    const bool bad = (__ballot_sync(0xffffffffu, mine) >> (threadIdx.x & 24u)) & 0xffu;
    bounds(type, lo, hi);
    const float spread = (hi - lo) * (16.f / 15.f);  // off by three half steps
    Group g;
    g.S = __float2bfloat16_rn(spread);
    const float S = __bfloat162float(g.S), base = __fsub_rn(lo, S), back = __fsub_rn(base, lo);
    g.B = __float2bfloat16_rn(base);
    // (the difference of two bfloat16 numbers is mostly exact, and often just in the middle)
    const bool inexact = __fadd_rn(__fsub_rn(lo, __fsub_rn(base, back)), __fsub_rn(-S, back)) != 0.f;
    if (near_middle(spread) || (inexact && near_middle(base)) || spread < 1.5777218e-30f /* 2^-99 */) g = exact_group(lo, hi);
    // (what the largest code stands for is not finite either where S or B is not)
    const float top = __bfloat162float(__hfma(g.S, __float2bfloat16_rn(1.9375f), g.B));
    if (bad || !(top - top == 0.f)) g.S = g.B = __ushort_as_bfloat16(0x7fff);
    return g;
}

// Whether d = x - B, half way between two codes, may not be all of x - B: never between bfloat16 numbers, but where x is next to nothing beside B.
__device__ __forceinline__ bool more_than(const float*, float, float) { return true; }
__device__ __forceinline__ bool more_than(const __nv_bfloat16*, float x, float step) { return x != 0.f && fabsf(x) < step; }

// four neighbouring codes and, from one lane of the group, its pair (codes of 0 where S is not a positive number)
template <typename T>
__device__ __forceinline__ void put_group(const T* type, const float (&x)[4], Group g, uint8_t* codes, uint8_t* pair, bool first) {
    const float S = __bfloat162float(g.S), B = __bfloat162float(g.B);
    uint32_t c = 0u;
    if (S > 0.f) {
        const float inv = __fdividef(16.f, S), step = S * 0.0625f, half = 0.5f * step;
        uint32_t t[4];
        bool again = S >= kHugeS;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float d = __fsub_rn(x[i], B);
            float sum = __fmaf_rn(d, inv, kMagic);
            const float e = __fmaf_rn(__fsub_rn(kMagic, sum), step, d);
            again |= fabsf(e) > half;
            if (fabsf(e) == half) {  // half way: to the even one
                if (__float_as_uint(sum) & 1u) sum += copysignf(1.f, e);
                again |= more_than(type, x[i], step);
            }
            t[i] = __float_as_uint(fminf(fmaxf(sum, kMagic + 16.f), kMagic + 31.f)) & 15u;  // 16 .. 31: code + 16
        }
        if (again) {
            const float near = __fdiv_rn(16.f, S);
#pragma unroll
            for (int i = 0; i < 4; ++i) t[i] = code_of(x[i], S, B, near);
        }
        c = t[0] | t[1] << 4 | t[2] << 8 | t[3] << 12;
    }
    *reinterpret_cast<uint16_t*>(codes) = (uint16_t)c;
    if (first) *reinterpret_cast<__nv_bfloat162*>(pair) = __halves2bfloat162(g.S, g.B);
}

// A feature of k rotated, rounded to the type once: a c - b s for the first of its pair (`low`, b the other one), a c + b s for the second.
__device__ __noinline__ float exact_rotation(float a, float b, int pos, const float* freq, bool low) {
    double s, c;
    sincos((double)pos * (double)*freq, &s, &c);
    return __bfloat162float(nearest_bf16(fma((double)a, c, (double)b * (low ? -s : s))));
}
__device__ __forceinline__ float rotated(const float*, float a, float b, double c, double s, int, const float*, bool low) {
    return __double2float_rn(fma((double)a, c, (double)b * (low ? -s : s)));
}
__device__ __forceinline__ float rotated(const __nv_bfloat16*, float a, float b, float c, float s, int pos, const float* freq, bool low) {
    const float r = fmaf(a, c, b * (low ? -s : s));
    // cosine and sine are off by less than 1.25 * 2^-23, the product, the sum and the bounds themselves by half a step each: 1.4 * 2^-22 in all
    const float off = (fabsf(a) + fabsf(b)) * 4.7683716e-7f;  // 2^-21
    const __nv_bfloat162 both = __floats2bfloat162_rn(r - off, r + off);
    const uint32_t u = *reinterpret_cast<const uint32_t*>(&both);
    return (u & 0xffffu) == u >> 16 ? __low2float(both) : exact_rotation(a, b, pos, freq, low);
}
__device__ __forceinline__ void angles(int pos, float freq, float& c, float& s) { cos_sin(pos, freq, c, s); }
__device__ __forceinline__ void angles(int pos, float freq, double& c, double& s) { sincos((double)pos * (double)freq, &s, &c); }

// what a token's cosines and sines are held in
template <typename T> struct Angle { using type = float; };
template <> struct Angle<float> { using type = double; };

// One block (or `gridDim.y` blocks, which share its heads) per token.  For keys and values a lane holds four neighbouring features of every 128, eight lanes a group.
// kD: the size of a head, where it is a usual one (3,739 tokens of 32 + 2 x 8 heads of 128: 44.0 us without, 39.9), or 0.  bfloat16 in 48 registers, which spills a
// little, holds five blocks an SM rather than four (37.9 to 38.9).
template <typename T, int kChunks, int kD>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 && kChunks == 1 ? 5 : 1)
kv4_store_kernel(const T* __restrict__ qkv, long long ld, T* __restrict__ q_out, long long ldq, const int* __restrict__ positions,
                 const int* __restrict__ token_req, const int* __restrict__ block_table, int table_stride, const float* __restrict__ inv_freq,
                 int pairs, uint8_t* __restrict__ k_pages, uint8_t* __restrict__ v_pages, int page_size, int nq, int nkv, int any_D) {
    const int D = kD ? kD : any_D;
    using A = typename Angle<T>::type;
    __shared__ __align__(16) A cs[256];  // cosines of the token's angles, then their sines
    __shared__ long long block_s;        // where the token's page begins
    __shared__ int slot_s;
    ns_pdl_wait();
    ns_pdl_launch_dependents();
    const int n = blockIdx.x, half = D / 2, req = token_req[n], pos = positions[n];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = kThreads / 32 * gridDim.y, first = blockIdx.y * (kThreads / 32) + warp;
    const T* row = qkv + (size_t)n * ld;
    // What this thread takes first is asked for before the angles are worked out.
    // q: eight pairs of a head to a thread (both features of a pair: q may be rotated in place); nothing to do without a rotation whose output stays in place
    const int per_head = half / 8, q_units = pairs > 0 || q_out != qkv ? nq * per_head : 0;
    int q_unit = blockIdx.y * kThreads + threadIdx.x;
    float a[8], b[8];
    auto load_q = [&] {
        const int h = q_unit / per_head;
        const T* x = row + (size_t)h * D + (q_unit - h * per_head) * 8;
        ld8(x, a);
        ld8(x + half, b);
    };
    if (q_unit < q_units) load_q();
    // keys and values: a warp to each kv head's
    float mine[kChunks][4], other[kChunks][4], v[kChunks][4];
    auto load_kv = [&](int u) {
        const T* kx = row + (size_t)(nq + u) * D;
#pragma unroll
        for (int ch = 0; ch < kChunks; ++ch) {
            const int f = ch * 128 + lane * 4;
            if (f >= D) break;
            ld4(kx + f, mine[ch]);
            ld4(kx + (f < half ? f + half : f - half), other[ch]);
            ld4(kx + (size_t)nkv * D + f, v[ch]);
        }
    };
    if (first < nkv) load_kv(first);
    if (req < 0) return;  // a padding row
    if (threadIdx.x == kThreads - 1) {
        const int page = block_table[(size_t)req * table_stride + pos / page_size];
        block_s = (long long)page * nkv * (long long)kv4_block_bytes(page_size, D);
        slot_s = pos % page_size;
    }
    for (int j = threadIdx.x; j < half; j += kThreads) {
        A s = 0, c = 1;
        if (j < pairs) angles(pos, inv_freq[j], c, s);
        cs[j] = c;
        cs[half + j] = s;
    }
    __syncthreads();
    for (; q_unit < q_units; q_unit += gridDim.y * kThreads) {
        if (q_unit >= (int)gridDim.y * kThreads) load_q();
        const int h = q_unit / per_head, f = (q_unit - h * per_head) * 8;
        T* y = q_out + (size_t)n * ldq + (size_t)h * D + f;
        float oa[8], ob[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float c = (float)cs[f + k], s = (float)cs[half + f + k];
            const bool turned = f + k < pairs;  // (what is not rotated does not meet its partner, which may not be finite)
            oa[k] = turned ? __fmaf_rn(a[k], c, -__fmul_rn(b[k], s)) : a[k];
            ob[k] = turned ? __fmaf_rn(b[k], c, __fmul_rn(a[k], s)) : b[k];
        }
        st8(y, oa);
        st8(y + half, ob);
    }
    const int slot = slot_s, pair_at = page_size * half + slot * (D / 8);
    for (int u = first; u < nkv; u += warps) {
        if (u != first) load_kv(u);
        float k[kChunks][4];
        Group gk[kChunks], gv[kChunks];
        bool bad = false;  // the token's key or value is not finite
#pragma unroll
        for (int ch = 0; ch < kChunks; ++ch) {
            const int f = ch * 128 + lane * 4, j = f < half ? f : f - half;
            const bool live = f < D;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                k[ch][i] = !live ? 0.f : j + i < pairs ? rotated(qkv, mine[ch][i], other[ch][i], cs[j + i], cs[half + j + i], pos, inv_freq + j + i, f < half) : mine[ch][i];
                if (!live) v[ch][i] = 0.f;
            }
            gk[ch] = group_of(qkv, k[ch], live);
            gv[ch] = group_of(qkv, v[ch], live);
            bad |= live && (__hisnan(gk[ch].S) || __hisnan(gv[ch].S));
        }
        bad = __any_sync(0xffffffffu, bad);
        const size_t block = (size_t)block_s + (size_t)u * kv4_block_bytes(page_size, D);
#pragma unroll
        for (int ch = 0; ch < kChunks; ++ch) {
            const int f = ch * 128 + lane * 4;
            if (f >= D) break;
            const size_t codes = block + slot * half + f / 2, pair = block + pair_at + f / kGroup * 4;
            const Group nan = {__ushort_as_bfloat16(0x7fff), __ushort_as_bfloat16(0x7fff)}, zero = {__ushort_as_bfloat16(0), __ushort_as_bfloat16(0)};
            put_group(qkv, k[ch], bad ? nan : gk[ch], k_pages + codes, k_pages + pair, (lane & 7) == 0);
            put_group(qkv, v[ch], __hisnan(gv[ch].S) ? zero : gv[ch], v_pages + codes, v_pages + pair, (lane & 7) == 0);
        }
    }
}

// One value of a word (eight features) per thread: k and v of (token, kv head); zeros where the table holds no page of the pool for the position.
__global__ void __launch_bounds__(kThreads)
kv4_read_kernel(const uint8_t* __restrict__ k_pages, const uint8_t* __restrict__ v_pages, const int* __restrict__ positions,
                const int* __restrict__ token_req, const int* __restrict__ block_table, int table_stride, int table_rows, int table_columns, int n_pages,
                __nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out, int n_tokens, int page_size, int nkv, int D) {
    ns_pdl_launch_dependents();
    ns_pdl_wait();
    const int words = D / 8, per_token = nkv * words;
    // a block takes tokens in turn (their number, and not that of all words, holds in 32 bits)
    const int side = max(1, kThreads / per_token), lanes = kThreads / side;  // tokens at a time, threads of each
    const int part = threadIdx.x / lanes;
    if (part >= side) return;
    for (long long n = (long long)blockIdx.x * side + part; n < n_tokens; n += (long long)gridDim.x * side)
    for (int u = threadIdx.x - part * lanes; u < per_token; u += lanes) {
        const long long i = n * per_token + u;
        const int h = u / words, w = u - h * words;
        const int req = token_req[n], pos = positions[n];
        const bool listed = req >= 0 && req < table_rows && pos >= 0 && pos / page_size < table_columns;
        const int page = listed ? block_table[(size_t)req * table_stride + pos / page_size] : -1;
        uint4 k = make_uint4(0u, 0u, 0u, 0u), v = k;
        if (page >= 0 && page < n_pages) {
            const int slot = pos % page_size;
            const size_t block = ((size_t)page * nkv + h) * kv4_block_bytes(page_size, D);
            const size_t codes = block + ((size_t)slot * words + w) * 4;
            const size_t pair = block + (size_t)page_size * (D / 2) + ((size_t)slot * (D / kGroup) + w / 4) * 4;
            k = kv4_in_order(*reinterpret_cast<const uint32_t*>(k_pages + codes), *reinterpret_cast<const uint32_t*>(k_pages + pair));
            v = kv4_in_order(*reinterpret_cast<const uint32_t*>(v_pages + codes), *reinterpret_cast<const uint32_t*>(v_pages + pair));
        }
        *reinterpret_cast<uint4*>(k_out + i * 8) = k;
        *reinterpret_cast<uint4*>(v_out + i * 8) = v;
    }
}

int check_geometry(const char* who, int D, int nkv, int page_size) {
    if (D < kGroup || D % kGroup || D > 256 || nkv < 1 || page_size < 1)
        NS_FAIL(NS_ERR_UNSUPPORTED, "%s: heads of %d (multiples of 32 up to 256), %d kv heads, pages of %d", who, D, nkv, page_size);
    return NS_OK;
}

}  // namespace

// qkv [n_tokens, ld] in the activations' type; q rotated into q_out [n_tokens, ldq] (which may be qkv itself), k and v into the cache.  `pairs`:
// features j and j + D / 2 with j < pairs are rotated by positions[n] * inv_freq[j] (0: none).
NS_API int ns_kv4_store(const void* qkv, long long ld, void* q_out, long long ldq, const int* positions, const int* token_req, const int* block_table,
                        int table_stride, const float* inv_freq, int pairs, void* k_pages, void* v_pages, int page_size, int nq, int nkv, int D,
                        int n_tokens, int sms, int dtype, cudaStream_t stream) {
    if (n_tokens <= 0) return NS_OK;
    int rc = check_geometry("ns_kv4_store", D, nkv, page_size);
    if (rc) return rc;
    const int size = dtype == NS_BF16 ? 2 : 4;
    if (nq < 1 || pairs < 0 || pairs > D / 2 || ld * size % 16 || ldq * size % 16 || ((uintptr_t)qkv | (uintptr_t)q_out) % 16 || ((uintptr_t)k_pages | (uintptr_t)v_pages) % 4)
        NS_FAIL(NS_ERR_ARGUMENT, "ns_kv4_store: rows on 16-byte boundaries, at most %d rotated pairs (%d)", D / 2, pairs);
    // a token's heads over several blocks while there are fewer tokens than SMs
    const int most = (nq + nkv + kThreads / 32 - 1) / (kThreads / 32);
    int parts = (2 * sms + n_tokens - 1) / n_tokens;
    parts = parts < 1 ? 1 : parts > most ? most : parts;
    dim3 grid(n_tokens, parts);
#define NS_KV4_STORE(T, CHUNKS, DD)                                                                                                   \
    NS_LAUNCH((kv4_store_kernel<T, CHUNKS, DD>), grid, kThreads, 0, stream, (const T*)qkv, ld, (T*)q_out, ldq, positions, token_req,    \
              block_table, table_stride, inv_freq, pairs, (uint8_t*)k_pages, (uint8_t*)v_pages, page_size, nq, nkv, D)
    if (dtype == NS_BF16 && D == 128) NS_KV4_STORE(__nv_bfloat16, 1, 128);
    else if (dtype == NS_BF16 && D == 64) NS_KV4_STORE(__nv_bfloat16, 1, 64);
    else if (dtype == NS_BF16 && D < 128) NS_KV4_STORE(__nv_bfloat16, 1, 0);
    else if (dtype == NS_BF16) NS_KV4_STORE(__nv_bfloat16, 2, 0);
    else if (dtype == NS_F32 && D <= 128) NS_KV4_STORE(float, 1, 0);
    else if (dtype == NS_F32) NS_KV4_STORE(float, 2, 0);
    else NS_FAIL(NS_ERR_UNSUPPORTED, "ns_kv4_store: float32 and bfloat16, not type %d", dtype);
#undef NS_KV4_STORE
    NS_CHECK_LAUNCH("ns_kv4_store");
    return NS_OK;
}

// k_out, v_out [n_tokens, nkv, D]: what the cache (`n_pages` pages) holds at positions[n] of request token_req[n]; zeros where that is negative, or where the table
// [table_rows, table_columns] does not say in which page: a page given back, a position that nobody has.
NS_API int ns_kv4_read(const void* k_pages, const void* v_pages, const int* positions, const int* token_req, const int* block_table, int table_stride,
                       int table_rows, int table_columns, int n_pages, void* k_out, void* v_out, int n_tokens, int page_size, int nkv, int D, int sms, cudaStream_t stream) {
    if (n_tokens <= 0) return NS_OK;
    int rc = check_geometry("ns_kv4_read", D, nkv, page_size);
    if (rc) return rc;
    const int per_token = nkv * (D / 8), side = per_token < kThreads ? kThreads / per_token : 1, blocks = (n_tokens + side - 1) / side;
    const int grid = blocks < 16 * sms ? blocks : 16 * sms;
    NS_LAUNCH(kv4_read_kernel, grid, kThreads, 0, stream, (const uint8_t*)k_pages, (const uint8_t*)v_pages, positions, token_req, block_table, table_stride,
              table_rows, table_columns, n_pages, (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, n_tokens, page_size, nkv, D);
    NS_CHECK_LAUNCH("ns_kv4_read");
    return NS_OK;
}

// ---- whole portions in bfloat16 -----------------------------------------------------------------------------------------------------
// 64 tokens of a request and a kv head to a block: what their bytes stand for, as pages of 64 tokens of a bfloat16 cache, [item, head, token, D].  Tokens that the
// request does not hold (any more) are zeros.  Bound by memory: 5 D / 4 bytes read and 4 D written for a token.
namespace {
constexpr int kUnfoldTokens = 64;

__global__ void __launch_bounds__(kThreads)
kv4_unfold_kernel(const uint8_t* __restrict__ k_pages, const uint8_t* __restrict__ v_pages, const int* __restrict__ block_table, int table_stride,
                  const int* __restrict__ items, const int* __restrict__ kv_len, __nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out,
                  int page_size, int nkv, int head0, int D) {
    ns_pdl_wait();
    ns_pdl_launch_dependents();
    __shared__ long long base[kUnfoldTokens];  // where a token's block begins; -1: not held
    __shared__ int slots[kUnfoldTokens];
    const int req = items[2 * blockIdx.x], pos0 = items[2 * blockIdx.x + 1] * kUnfoldTokens, words = D / 8;
    const int h = blockIdx.y, held = kv_len[req];
    if (threadIdx.x < kUnfoldTokens) {
        const int pos = pos0 + threadIdx.x;
        long long at = -1;
        const int page = pos < held ? block_table[(size_t)req * table_stride + pos / page_size] : -1;
        if (page >= 0) at = (long long)(((size_t)page * nkv + head0 + h) * kv4_block_bytes(page_size, D));
        base[threadIdx.x] = at;
        slots[threadIdx.x] = pos % page_size;
    }
    __syncthreads();
    const unsigned by_words = (65536u + words - 1u) / words;
    const size_t out0 = ((size_t)blockIdx.x * gridDim.y + h) * kUnfoldTokens * D;
    for (int i = threadIdx.x; i < kUnfoldTokens * words; i += kThreads) {
        const int token = (int)((unsigned)i * by_words >> 16), w = i - token * words;  // i / words: exact below 2^16 / words
        const long long at = base[token];
        uint4 k = make_uint4(0u, 0u, 0u, 0u), v = k;
        if (at >= 0) {
            const int slot = slots[token];
            const size_t codes = (size_t)at + ((size_t)slot * words + w) * 4, pair = (size_t)at + (size_t)page_size * (D / 2) + ((size_t)slot * (D / kGroup) + w / 4) * 4;
            k = kv4_in_order(*reinterpret_cast<const uint32_t*>(k_pages + codes), *reinterpret_cast<const uint32_t*>(k_pages + pair));
            v = kv4_in_order(*reinterpret_cast<const uint32_t*>(v_pages + codes), *reinterpret_cast<const uint32_t*>(v_pages + pair));
        }
        *reinterpret_cast<uint4*>(k_out + out0 + (size_t)i * 8) = k;
        *reinterpret_cast<uint4*>(v_out + out0 + (size_t)i * 8) = v;
    }
}
}  // namespace

// items [n, 2] = (request, block of 64 positions); k_out, v_out [n, heads, 64, D]: kv heads head0 .. head0 + heads - 1 of nkv.
NS_API int ns_kv4_unfold(const void* k_pages, const void* v_pages, const int* block_table, int table_stride, const int* items, int n, const int* kv_len,
                         void* k_out, void* v_out, int page_size, int nkv, int head0, int heads, int D, cudaStream_t stream) {
    if (n <= 0 || heads <= 0) return NS_OK;
    int rc = check_geometry("ns_kv4_unfold", D, nkv, page_size);
    if (rc) return rc;
    if (head0 < 0 || head0 + heads > nkv || heads > 65535) NS_FAIL(NS_ERR_ARGUMENT, "ns_kv4_unfold: heads %d to %d of %d", head0, head0 + heads, nkv);
    NS_LAUNCH(kv4_unfold_kernel, dim3(n, heads), kThreads, 0, stream, (const uint8_t*)k_pages, (const uint8_t*)v_pages, block_table, table_stride, items, kv_len,
              (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, page_size, nkv, head0, D);
    NS_CHECK_LAUNCH("ns_kv4_unfold");
    return NS_OK;
}
