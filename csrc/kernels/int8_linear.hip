// K24: dense layer on 8-bit integers (gfx950): a scale for each row of the input and for each output channel.
//
//   top_m = max_k |x[m][k]|,  xq[m][k] = rne(x[m][k] * (127 * (1 / top_m))),  sx_m = top_m / 127      (fp32, a rounding each)
//   y[m][n] = (sum_k xq[m][k] q[n][k]) * (sx_m * s[n]) + bias[n]
//
// The sum is exact in int32 for K <= 133 144 (127^2 K < 2^31) whatever its order; rows below 1e-30 count as zero (127 / top
// would overflow), a row with an infinity or a NaN gives NaN (its scale is NaN).
#include "common.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float ld_in(const float* p) { return *p; }
__device__ __forceinline__ float ld_in(const bf16_t* p) { return bf2f(*p); }

// one row a workgroup: codes [M][Kp] (zeros from K on) and the scales
template <typename T>
__global__ void __launch_bounds__(256) int8_rows_kernel(const T* __restrict__ x, long long ldx, int K, int Kp, signed char* __restrict__ q,
                                                       float* __restrict__ scale) {
    __shared__ float red[4];
    __shared__ int redb[4];
    const long long m = blockIdx.x;
    const T* row = x + m * ldx;
    float top = 0.f;
    int bad = 0;
    for (int k = threadIdx.x; k < K; k += 256) {
        const float v = fabsf(ld_in(row + k));
        bad |= !(v < __builtin_inff());
        top = fmaxf(top, v);
    }
    top = wave_max(top);
    bad = __any(bad);
    if ((threadIdx.x & 63) == 0) { red[threadIdx.x >> 6] = top; redb[threadIdx.x >> 6] = bad; }
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    bad = redb[0] | redb[1] | redb[2] | redb[3];
    const bool zero = bad || top < 1e-30f;
    const float inv = zero ? 0.f : 127.f * (1.f / top);
    if (threadIdx.x == 0) scale[m] = bad ? __builtin_nanf("") : (zero ? 0.f : top / 127.f);
    signed char* out = q + m * Kp;
    for (int k = threadIdx.x; k < Kp; k += 256) out[k] = k < K && !zero ? (signed char)(int)rintf(ld_in(row + k) * inv) : (signed char)0;
}

// 64 x 64 tile of y, 4 waves of 32 x 32; both operands row-major and k-contiguous
template <typename T>
__global__ void __launch_bounds__(256) int8_gemm_kernel(const signed char* __restrict__ xq, const float* __restrict__ sx, const signed char* __restrict__ q,
                                                       long long ldq, const float* __restrict__ s, const float* __restrict__ bias,
                                                       T* __restrict__ y, long long ldy, int M, int N, int K, int Kp, int tiles_n) {
    constexpr int LD = 80;
    __shared__ __attribute__((aligned(16))) signed char As[64 * LD], Bs[64 * LD];
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, wm = wid >> 1, wn = wid & 1;
    const int tm = blockIdx.x / tiles_n, tn = blockIdx.x - tm * tiles_n, m0 = tm * 64, n0 = tn * 64;
    const int row = tid >> 2, ch = (tid & 3) * 16;
    i32x4 acc[2][2] = {};
    for (int k0 = 0; k0 < Kp; k0 += 64) {
        i32x4 va = {}, vb = {};
        if (m0 + row < M) va = *reinterpret_cast<const i32x4*>(xq + (long long)(m0 + row) * Kp + k0 + ch);
        if (n0 + row < N && k0 + ch < K) vb = *reinterpret_cast<const i32x4*>(q + (n0 + row) * ldq + k0 + ch);
        __syncthreads();
        *reinterpret_cast<i32x4*>(As + row * LD + ch) = va;
        *reinterpret_cast<i32x4*>(Bs + row * LD + ch) = vb;
        __syncthreads();
        i32x4 fa[2], fb[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            fa[i] = *reinterpret_cast<const i32x4*>(As + (wm * 32 + i * 16 + (lane & 15)) * LD + (lane >> 4) * 16);
            fb[i] = *reinterpret_cast<const i32x4*>(Bs + (wn * 32 + i * 16 + (lane & 15)) * LD + (lane >> 4) * 16);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fa[i], fb[j], acc[i][j], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int m = m0 + wm * 32 + i * 16 + (lane >> 4) * 4 + e, n = n0 + wn * 32 + j * 16 + (lane & 15);
                if (m >= M || n >= N) continue;
                const float v = (float)acc[i][j][e] * (sx[m] * s[n]) + (bias ? bias[n] : 0.f);
                if constexpr (sizeof(T) == 4) y[m * ldy + n] = v; else y[m * ldy + n] = f2bf(v);
            }
}

}  // namespace

// codes and scales of the rows of x [M][K] (row stride ldx elements); q [M][Kp], zeros from K on
extern "C" int ddl_int8_rows(const void* x, int x_bf16, long long ldx, long long M, int K, int Kp, void* q, void* scale, hipStream_t stream) {
    if (M == 0) return DDL_OK;
    if (!x || !q || !scale || M < 0 || M > 0x7fffffffLL || K <= 0 || Kp < K || ldx < 0) return DDL_EINVAL;
    if (x_bf16) DDL_KLAUNCH(int8_rows_kernel<bf16_t>, dim3((unsigned)M), dim3(256), 0, stream, (const bf16_t*)x, ldx, K, Kp, (signed char*)q, (float*)scale);
    else DDL_KLAUNCH(int8_rows_kernel<float>, dim3((unsigned)M), dim3(256), 0, stream, (const float*)x, ldx, K, Kp, (signed char*)q, (float*)scale);
    return ddl_launch_status();
}

extern "C" int ddl_int8_max_k() { return 133144; }

// bytes of workspace of ddl_int8_linear
extern "C" long long ddl_int8_linear_workspace(long long M, int N, int K) {
    const long long Kp = (K + 63LL) / 64 * 64;
    return (M * Kp + 255) / 256 * 256 + M * 4;
}

// y [M][N] (bf16 or fp32 like x) = x [M][K] times q [N][K]^T with scales; rows of q start at multiples of 16 bytes and may be
// read up to the next multiple of 16 behind K; q_bytes: what may be read from q on
extern "C" int ddl_int8_linear(const void* x, int x_bf16, long long ldx, const void* q, long long ldq, long long q_bytes, const void* s, const void* bias,
                               void* y, long long ldy, long long M, int N, int K, void* ws, long long ws_bytes, hipStream_t stream) {
    if (M == 0 || N == 0) return DDL_OK;
    if (!x || !q || !s || !y || !ws || M < 0 || N < 0 || K <= 0 || K > ddl_int8_max_k() || ldx < 0 || ldq < K || ldy < N) return DDL_EINVAL;
    if (M > 0x7fffffffLL - 256 || N > 0x7fffffff - 256) return DDL_EINVAL;
    if (!ddl_aligned16(q) || ldq % 16 || (reinterpret_cast<uintptr_t>(ws) & 255)) return DDL_EALIGN;
    if (q_bytes < (N - 1LL) * ldq + (K + 15) / 16 * 16 || ws_bytes < ddl_int8_linear_workspace(M, N, K)) return DDL_EINVAL;
    const int Kp = (K + 63) / 64 * 64;
    signed char* xq = (signed char*)ws;
    float* sx = (float*)((char*)ws + (M * Kp + 255) / 256 * 256);
    const int rc = ddl_int8_rows(x, x_bf16, ldx, M, K, Kp, xq, sx, stream);
    if (rc != DDL_OK) return rc;
    const long long tn = (N + 63) / 64, tiles = (M + 63) / 64 * tn;
    if (tiles > 0x7fffffffLL) return DDL_EINVAL;
    const dim3 grid((unsigned)tiles), block(256);
    if (x_bf16)
        DDL_KLAUNCH(int8_gemm_kernel<bf16_t>, grid, block, 0, stream, xq, sx, (const signed char*)q, ldq, (const float*)s, (const float*)bias, (bf16_t*)y, ldy,
                    (int)M, N, K, Kp, (int)tn);
    else
        DDL_KLAUNCH(int8_gemm_kernel<float>, grid, block, 0, stream, xq, sx, (const signed char*)q, ldq, (const float*)s, (const float*)bias, (float*)y, ldy,
                    (int)M, N, K, Kp, (int)tn);
    return ddl_launch_status();
}
