// Matrix product in 8-bit integers: out[n, f] = (sum_k x[n, k] w[f, k]) xs[n] ws[f] (+ bias[f]), the sum exact in 32 bits
// (127^2 K < 2^31 for K up to 131,072), then three roundings in float and one to the output's type.
#include "common.cuh"

namespace {

constexpr int BM = 64, BN = 64, BK = 64, kThreads = 256;

template <typename OutT>
__global__ void __launch_bounds__(kThreads)
gemm_i8_kernel(const int8_t* __restrict__ x, long long ldx, const float* __restrict__ xs, const int8_t* __restrict__ w, long long ldw,
               const float* __restrict__ ws, const float* __restrict__ bias, OutT* __restrict__ out, long long ldo, int M, int N, int K) {
    ns_pdl_launch_dependents();
    ns_pdl_wait();
    __shared__ __align__(16) int8_t a[BM][BK + 16], b[BN][BK + 16];
    const int m0 = blockIdx.y * BM, n0 = blockIdx.x * BN;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    int acc[4][4] = {};
    auto piece = [&](const int8_t* row, bool live, int k) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (live && k + 16 <= K) return *reinterpret_cast<const uint4*>(row + k);
        if (live)
            for (int i = 0; k + i < K; ++i) reinterpret_cast<int8_t*>(&v)[i] = row[k + i];
        return v;
    };
    for (int k0 = 0; k0 < K; k0 += BK) {
        const int r = threadIdx.x >> 2, c = (threadIdx.x & 3) * 16;
        *reinterpret_cast<uint4*>(&a[r][c]) = piece(x + (size_t)(m0 + r) * ldx, m0 + r < M, k0 + c);
        *reinterpret_cast<uint4*>(&b[r][c]) = piece(w + (size_t)(n0 + r) * ldw, n0 + r < N, k0 + c);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < BK; k += 4) {
            int av[4], bv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                av[i] = *reinterpret_cast<const int*>(&a[ty + 16 * i][k]);
                bv[i] = *reinterpret_cast<const int*>(&b[tx + 16 * i][k]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(av[i], bv[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
            if (m < M && n < N) {
                float v = __int2float_rn(acc[i][j]) * (xs[m] * ws[n]);
                if (bias) v += bias[n];
                ns_st(out, (size_t)m * ldo + n, v);
            }
        }
}

}  // namespace

// x [M, ldx], w [N, ldw] 8-bit integers whose rows start on 16-byte boundaries; xs [M], ws [N] (and bias [N] or null) float; out [M, ldo].
NS_API int ns_gemm_i8(const void* x, long long ldx, const float* xs, const void* w, long long ldw, const float* ws, const float* bias, void* out,
                      long long ldo, int M, int N, int K, int dtype, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return NS_OK;
    if (K < 1 || K > 131072) NS_FAIL(NS_ERR_UNSUPPORTED, "ns_gemm_i8: K=%d (1 to 131072)", K);
    if (ldx % 16 || ldw % 16 || ((uintptr_t)x | (uintptr_t)w) % 16) NS_FAIL(NS_ERR_UNSUPPORTED, "ns_gemm_i8: rows must start on 16-byte boundaries");
    dim3 grid((N + BN - 1) / BN, (M + BM - 1) / BM);
    if (grid.y > 65535) NS_FAIL(NS_ERR_UNSUPPORTED, "ns_gemm_i8: too many rows (%d)", M);
    if (dtype == NS_BF16)
        NS_LAUNCH((gemm_i8_kernel<__nv_bfloat16>), grid, kThreads, 0, stream, (const int8_t*)x, ldx, xs, (const int8_t*)w, ldw, ws, bias, (__nv_bfloat16*)out, ldo, M, N, K);
    else if (dtype == NS_F32)
        NS_LAUNCH((gemm_i8_kernel<float>), grid, kThreads, 0, stream, (const int8_t*)x, ldx, xs, (const int8_t*)w, ldw, ws, bias, (float*)out, ldo, M, N, K);
    else
        NS_FAIL(NS_ERR_UNSUPPORTED, "ns_gemm_i8: float32 and bfloat16 outputs, not type %d", dtype);
    NS_CHECK_LAUNCH("ns_gemm_i8");
    return NS_OK;
}
