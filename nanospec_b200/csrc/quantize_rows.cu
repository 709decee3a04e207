// Rows in 8-bit integers with a float scale each: s = max |x| / 127 rounded to float, q = x / s to the nearest integer, ties to even.
//
// The quotient that is rounded is the exact one: a first guess (x times the reciprocal, added to 1.5 * 2^23, whose last bits are then the integer) is off by
// one at most, and the remainder x - q s, which one fused multiply-add gives without error (its bits are no finer than half of s's last and it is at most
// about s / 2), says whether the guess stays.  It nearly always does: a piece of eight elements is looked at once more only when a remainder reaches s / 2.
// The maximum is taken over the bit patterns of |x|, in whose order infinities and NaN come last.
//
// A row is read once (its pieces stay in registers where the block holds them) and written once in a byte per element; one block a row, since a row's maximum
// stands before its first quotient.  4,096 x 4,096 bfloat16 take 16.4 us (7.7 at the rate of a copy), float32 18.5 (12.8), from rows off 16-byte boundaries, which
// are read an element at a time, 20.5 both.  Neither instructions nor memory are at their limit (SMs 54 % busy, memory 27 %; 512 x 14,336: 24 and 13 %): a block first
// waits for its row, then for its maximum, then computes, and the few blocks of an SM overlap these in part.  Instructions count all the same: with a test
// of each element's remainder in place of each piece's, on numbers unpacked for the maximum too, the same rows took 32.
#include "common.cuh"

namespace {

constexpr int kHeld = 4;  // pieces of 8 elements that a thread keeps: a block of 512 holds rows of up to 16,384

constexpr float kMagic = 12582912.f;  // 1.5 * 2^23

__device__ __noinline__ int nearest(float x, float s, float inv) {
    float r = rintf(x * inv);
    const float e = fmaf(-r, s, x), half = 0.5f * s;
    const bool odd = ((int)r) & 1;
    if (e > half || (e == half && odd)) r += 1.f;
    else if (e < -half || (e == -half && odd)) r -= 1.f;
    return (int)r;
}

// A piece of eight elements as it lies in memory, the largest |x| of it, and its elements as floats.
template <typename T> struct Piece;
template <> struct Piece<float> {
    float v[8];
    __device__ __forceinline__ void load(const float* p) { ld8(p, v); }
    __device__ __forceinline__ void set(int i, float x) { v[i] = x; }
    __device__ __forceinline__ uint32_t top() const {
        uint32_t m = 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
        return m;
    }
    __device__ __forceinline__ void floats(float (&x)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = v[i];
    }
};
template <> struct Piece<__nv_bfloat16> {
    uint32_t u[4];
    __device__ __forceinline__ void load(const __nv_bfloat16* p) {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        u[0] = a.x; u[1] = a.y; u[2] = a.z; u[3] = a.w;
    }
    __device__ __forceinline__ void set(int i, __nv_bfloat16 x) {
        const uint32_t b = __bfloat16_as_ushort(x);
        u[i >> 1] = i & 1 ? (u[i >> 1] & 0xffffu) | b << 16 : (u[i >> 1] & 0xffff0000u) | b;
    }
    __device__ __forceinline__ uint32_t top() const {  // (two at a time: the order of the bits is that of the numbers)
        const uint32_t m = __vmaxu2(__vmaxu2(u[0] & 0x7fff7fffu, u[1] & 0x7fff7fffu), __vmaxu2(u[2] & 0x7fff7fffu, u[3] & 0x7fff7fffu));
        return max(m << 16, m & 0xffff0000u);
    }
    __device__ __forceinline__ void floats(float (&x)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(u[i] << 16); x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
    }
};
template <typename T>
__device__ __forceinline__ void load_piece(Piece<T>& p, const T* row, int k, int K, bool wide) {
    if (wide && k + 8 <= K) {
        p.load(row + k);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p.set(i, k + i < K ? row[k + i] : T(0.f));
    }
}

__device__ __forceinline__ void store_piece(int8_t* out, int k, int K, const float (&v)[8], float s, float inv) {
    uint32_t w[2] = {0u, 0u};
    if (inv != 0.f) {
        const float half = 0.5f * s;
        uint32_t t[8];
        bool again = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float sum = __fmaf_rn(v[i], inv, kMagic), r = __fsub_rn(sum, kMagic);
            again |= fabsf(__fmaf_rn(-r, s, v[i])) >= half;
            t[i] = __float_as_uint(sum);
        }
        if (again) {
#pragma unroll
            for (int i = 0; i < 8; ++i) t[i] = (uint32_t)nearest(v[i], s, inv);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
            w[i] = __byte_perm(__byte_perm(t[4 * i], t[4 * i + 1], 0x0040), __byte_perm(t[4 * i + 2], t[4 * i + 3], 0x0040), 0x5410);
    }
    if (k + 8 <= K) {
        *reinterpret_cast<uint2*>(out + k) = make_uint2(w[0], w[1]);
    } else {
        for (int i = 0; k + i < K; ++i) out[k + i] = (int8_t)(w[i >> 2] >> (8 * (i & 3)));
    }
}

template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads)
quantize_rows_kernel(const T* __restrict__ x, long long ldx, int8_t* __restrict__ q, long long ldq, float* __restrict__ scale, int K, int wide) {
    ns_pdl_wait();
    ns_pdl_launch_dependents();  // in this order: the product asks for its weights without a wait of its own, and a kernel before this one may have written them
    __shared__ uint32_t tops[kThreads / 32];
    const T* row = x + (size_t)blockIdx.x * ldx;
    Piece<T> held[kHeld];
    uint32_t top = 0u;
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
        const int k = (u * kThreads + threadIdx.x) * 8;
        if (k >= K) break;
        load_piece(held[u], row, k, K, wide);
    }
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
        if ((u * kThreads + threadIdx.x) * 8 >= K) break;
        top = max(top, held[u].top());
    }
    for (int k = (kHeld * kThreads + threadIdx.x) * 8; k < K; k += kThreads * 8) {  // what is beyond the block's registers is read again below
        Piece<T> p;
        load_piece(p, row, k, K, wide);
        top = max(top, p.top());
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) top = max(top, tops[w]);
    float s = __fdiv_rn(__uint_as_float(top), 127.f), inv = 0.f;
    if (top >= 0x7f800000u) s = __uint_as_float(0x7fffffffu);  // an infinity or a NaN: the row has no scale
    else if (s < 7.52316385e-37f) s = 0.f;                     // 2^-120: a row of zeros
    else inv = __frcp_rn(s);
    if (threadIdx.x == 0) scale[blockIdx.x] = s;
    int8_t* out = q + (size_t)blockIdx.x * ldq;
    float v[8];
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
        const int k = (u * kThreads + threadIdx.x) * 8;
        if (k >= K) break;
        held[u].floats(v);
        store_piece(out, k, K, v, s, inv);
    }
    for (int k = (kHeld * kThreads + threadIdx.x) * 8; k < K; k += kThreads * 8) {
        Piece<T> p;
        load_piece(p, row, k, K, wide);
        p.floats(v);
        store_piece(out, k, K, v, s, inv);
    }
}

}  // namespace

// q [rows, ldq] (8-bit integers, rows on 8-byte boundaries) and scale [rows] of x [rows, ldx].  A row that holds an infinity or a NaN gets
// NaN for its scale and zeros; one whose scale would be below 2^-120 gets zeros and 0.
NS_API int ns_quantize_rows(const void* x, long long ldx, void* q, long long ldq, float* scale, int rows, int K, int dtype, cudaStream_t stream) {
    if (rows <= 0) return NS_OK;
    if (K < 1 || ldq % 8 || (uintptr_t)q % 8) NS_FAIL(NS_ERR_ARGUMENT, "ns_quantize_rows: %d columns, output rows %lld apart (multiples of 8 on an 8-byte boundary)", K, ldq);
    const int size = dtype == NS_BF16 ? 2 : 4;
    const int wide = (uintptr_t)x % 16 == 0 && ldx * size % 16 == 0;
    // Short rows leave most threads of a large block idle; long ones pass through a small one twice.  Launches in a row on bfloat16, 256 threads against the
    // rule's: 4,096 x 1,024 9.1 us, 6.8; 4,096 x 2,048 11.2, 9.6; 512 x 14,336 15.7, 10.7 (of which 3.4 are its bytes at the rate of a copy).
#define NS_QUANTIZE(T, THREADS) NS_LAUNCH((quantize_rows_kernel<T, THREADS>), rows, THREADS, 0, stream, (const T*)x, ldx, (int8_t*)q, ldq, scale, K, wide)
    if (dtype == NS_BF16) {
        if (K <= 2048) NS_QUANTIZE(__nv_bfloat16, 128);
        else if (K <= 8192) NS_QUANTIZE(__nv_bfloat16, 256);
        else NS_QUANTIZE(__nv_bfloat16, 512);
    } else if (dtype == NS_F32) {
        if (K <= 2048) NS_QUANTIZE(float, 128);
        else if (K <= 8192) NS_QUANTIZE(float, 256);
        else NS_QUANTIZE(float, 512);
    } else {
        NS_FAIL(NS_ERR_UNSUPPORTED, "ns_quantize_rows: float32 and bfloat16, not type %d", dtype);
    }
#undef NS_QUANTIZE
    NS_CHECK_LAUNCH("ns_quantize_rows");
    return NS_OK;
}
