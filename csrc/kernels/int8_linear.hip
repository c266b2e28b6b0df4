// K24: dense layer on 8-bit integers (gfx950): a scale for each row of the input and for each output channel.
//
//   top_m = max_k |x[m][k]|,  xq[m][k] = rne(x[m][k] * (127 * (1 / top_m))),  sx_m = top_m / 127      (fp32, a rounding each)
//   y[m][n] = (sum_k xq[m][k] q[n][k]) * (sx_m * s[n]) + bias[n]
//
// The sum is exact in int32 for K <= 133 144 (127^2 K < 2^31) whatever its order; rows below 1e-30 count as zero (127 / top
// would overflow), a row with an infinity or a NaN gives NaN (its scale is NaN).
//
// Up to 16 rows: one launch that is bound by reading the weights once (int8_skinny_kernel).  More: the rows are quantised first
// (int8_rows_kernel, bound by memory), then multiplied tile by tile (int8_gemm_kernel, bound by the matrix pipe).
#include "common.h"
#include "tile_mul.h"
#include <math.h>

namespace {

template <typename T>
__device__ __forceinline__ void ld8(const T* p, float (&v)[8]) {
    if constexpr (sizeof(T) == 2) {
        const bf16x8 b = *reinterpret_cast<const bf16x8*>(p);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = bf2f(b[j]);
    } else {
        load8f(p, v);
    }
}
__device__ __forceinline__ float ld1(const float* p) { return *p; }
__device__ __forceinline__ float ld1(const bf16_t* p) { return bf2f(*p); }
__device__ __forceinline__ void st1(float* p, float v) { *p = v; }
__device__ __forceinline__ void st1(bf16_t* p, float v) { *p = f2bf(v); }
__device__ __forceinline__ unsigned code_of(float v, float inv) { return (unsigned)(int)rintf(v * inv) & 255u; }

// 8 values of a row from k on, zeros from K on; vec: the row starts at a multiple of 16 bytes
template <typename T>
__device__ __forceinline__ void ld_row(const T* __restrict__ row, int k, int K, bool vec, float (&v)[8]) {
    if (vec && k + 8 <= K) {
        ld8(row + k, v);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = k + j < K ? ld1(row + k + j) : 0.f;
    }
}

// One wave (W = 1) or a workgroup of W: the codes of a row (K values, zeros up to Kp, a multiple of 16) to q, which starts at a
// multiple of 16 bytes; returns its scale.  The first 2048 W values are read at once and stay in registers between the two passes.
template <int W, typename T>
__device__ __forceinline__ float quantize_row(const T* __restrict__ row, int K, int Kp, bool vec, signed char* q) {
    const int lane = W == 1 ? threadIdx.x & 63 : threadIdx.x;
    constexpr int HOLD = 4;
    float held[HOLD][8], top = 0.f;
    int bad = 0;
#pragma unroll
    for (int h = 0; h < HOLD; ++h) ld_row(row, (h * 64 * W + lane) * 8, K, vec, held[h]);
    auto see = [&](const float (&v)[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float a = fabsf(v[j]);
            bad |= !(a < __builtin_inff());
            top = fmaxf(top, a);
        }
    };
#pragma unroll
    for (int h = 0; h < HOLD; ++h) see(held[h]);
#pragma unroll 2
    for (int k = (HOLD * 64 * W + lane) * 8; k < K; k += 512 * W) {
        float v[8];
        ld_row(row, k, K, vec, v);
        see(v);
    }
    top = wave_max(top);
    bad = __any(bad);
    if constexpr (W > 1) {
        __shared__ float tops[W];
        __shared__ int bads[W];
        __syncthreads();                     // (a row before this one)
        if ((threadIdx.x & 63) == 0) {
            tops[threadIdx.x >> 6] = top;
            bads[threadIdx.x >> 6] = bad;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) {
            top = fmaxf(top, tops[w]);
            bad |= bads[w];
        }
    }
    const bool zero = bad || top < 1e-30f;
    const float inv = zero ? 0.f : 127.f * (1.f / top);
    auto put = [&](int k, const float (&v)[8]) {
        if (k >= Kp) return;
        u32x2 o;
#pragma unroll
        for (int p = 0; p < 2; ++p)
            o[p] = zero ? 0u : code_of(v[4 * p], inv) | code_of(v[4 * p + 1], inv) << 8 | code_of(v[4 * p + 2], inv) << 16 | code_of(v[4 * p + 3], inv) << 24;
        *reinterpret_cast<u32x2*>(q + k) = o;
    };
#pragma unroll
    for (int h = 0; h < HOLD; ++h) put((h * 64 * W + lane) * 8, held[h]);
#pragma unroll 2
    for (int k = (HOLD * 64 * W + lane) * 8; k < Kp; k += 512 * W) {
        float v[8];
        ld_row(row, k, K, vec, v);
        put(k, v);
    }
    return bad ? __builtin_nanf("") : (zero ? 0.f : top / 127.f);
}

// Codes [M][Kp], scales; a row a wave (W = 1) or a workgroup of W waves.  Also clears what int8_gemm_kernel counts with.
// 12 544 rows of 4096 bf16 values (154 MB): 29 us (values of a row held in registers between its largest and its codes; read a second
// time: 94)
template <int W, typename T>
__global__ void __launch_bounds__(256) int8_rows_kernel(const T* __restrict__ x, long long ldx, int M, int K, int Kp, int vec, signed char* __restrict__ q,
                                                       float* __restrict__ scale, unsigned* __restrict__ counters, int ncount) {
    if (blockIdx.x == 0 && (int)threadIdx.x < ncount) counters[threadIdx.x] = 0u;
    const int m = W == 1 ? blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
    if (m >= M) return;
    const float s = quantize_row<W>(x + m * ldx, K, Kp, vec, q + (long long)m * Kp);
    if ((threadIdx.x & (64 * W - 1)) == 0) scale[m] = s;
}

// B x B tile of y (or a part of its sum): F = output channels, S = rows of x.  12 544 x 4096 x 4096: 250 to 290 us (tiles of 128, bound by the
// matrix pipe: 1450 to 1680 TOPS); 256 x 1000 x 2047: 8.6 us (64 tiles of 64, two groups of waves each, bound by the latency of 16 stages).
template <typename T, int B, int W0, int W1, int NST, int KS>
__global__ void __launch_bounds__(KS * W0 * W1 * 64, 2) int8_gemm_kernel(const signed char* __restrict__ xq, const float* __restrict__ sx,
                                                                   const signed char* __restrict__ q, long long ldq,
                                                                   const float* __restrict__ s, const float* __restrict__ bias, T* __restrict__ y, long long ldy,
                                                                   int M, int N, int K, int Kp, int tm, int tn, int split, int* __restrict__ slabs,
                                                                   unsigned* __restrict__ counters) {
    typedef TileMul<MulI8, B, B, W0, W1, NST, false, KS> Mu;
    __shared__ __attribute__((aligned(16))) unsigned char smem[Mu::LDS];
    // an XCD (workgroup number modulo 8) has a run of tiles, in bands of 8 rows, a band column by column
    const int all = tm * tn * split, per = (all + 7) >> 3, item = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || item >= all) return;
    const int idx = item / split, part = item - idx * split, each = (Kp / 128 + split - 1) / split, k0 = part * each;
    const int stages = Kp / 128 - k0 < each ? Kp / 128 - k0 : each;
    const int band = idx / (8 * tn), rem = idx - band * 8 * tn, h = tm - band * 8 < 8 ? tm - band * 8 : 8;
    const int ni = rem / h, mi = band * 8 + rem - ni * h, m0 = mi * B, n0 = ni * B;
    Mu mu;
    // (the codes' rows may be read up to the next multiple of 16 bytes behind K, the workspace's are whole stages)
    mu.run(smem, q + n0 * ldq + k0 * 128, (unsigned)ldq, N - n0, xq + (long long)m0 * Kp + k0 * 128, Kp, M - m0, stages,
           k0 + stages == Kp / 128 ? ((K + 15) & ~15) - (Kp - 128) : 128);
    if constexpr (B == 64) {
        if (split > 1 && !join_parts<int, Mu>(mu, smem, slabs + (long long)idx * split * (B * B), counters + idx, part, split)) return;
    }
#pragma unroll
    for (int pass = 0; pass < Mu::PASSES; ++pass) {
        if (Mu::PASSES > 1 && pass > 0) __syncthreads();
        if (B > 64 || split == 1) mu.to_lds(smem, pass);
        __syncthreads();
        // a lane an element: a wave's loads of s and bias and its stores are side by side, whatever N is (8 elements a lane, 16-byte
        // stores: 12 544 x 4096 x 64 122 us, so 97; where rows begin anywhere, 770 x 6171 x 26 28.8, so 20.4; 12 544 x 4096 x 4096 291, so 279)
#pragma unroll 1
        for (int k = threadIdx.x; k < Mu::ROWS * B; k += Mu::THREADS) {
            const int r = k / B, c = k % B, m = m0 + Mu::tile_row(r, pass), n = n0 + c;
            if (m >= M || n >= N) continue;
            const int v = __float_as_int(Mu::at1(reinterpret_cast<const float*>(smem), r, c));
            st1(y + m * ldy + n, (float)v * (sx[m] * s[n]) + (bias ? bias[n] : 0.f));
        }
    }
}

// Up to 16 rows.  A workgroup of 8 waves takes tiles of 16 output channels (tile w, w + grid, ..); a wave 128-byte pieces of their
// rows, every 8th, straight from memory into the matrix pipe's operand (16 channels x 64 values), three pieces ahead; the rows of x
// are quantised into LDS meanwhile, once a workgroup.  The waves' integer sums are added in LDS.
// Bound by latency, then by reading the codes: 1 x 1000 x 2048 5.4 us, 7 x 21 841 x 2048 (45 MB) 12 to 14 us.
template <typename T>
__global__ void __launch_bounds__(512) int8_skinny_kernel(const T* __restrict__ x, long long ldx, int vec, const signed char* __restrict__ q, long long ldq,
                                                         const float* __restrict__ s, const float* __restrict__ bias, T* __restrict__ y, long long ldy,
                                                         int M, int N, int K, int tiles) {
    extern __shared__ __attribute__((aligned(16))) signed char xs[];       // [M][Kp + 16]
    __shared__ __attribute__((aligned(16))) i32x4 red[2][8][64];
    __shared__ float sx[16];
    const int Kp = (K + 127) & ~127, LD = Kp + 16, pieces = Kp >> 7, P = (pieces + 7) >> 3;
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), fr = lane & 15, fq = lane >> 4;
    const int total = ((tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x) * P;
    struct Pair { i32x4 a, b; };
    auto load = [&](int it) {
        Pair p = {};
        const int n = ((int)blockIdx.x + it / P * (int)gridDim.x) * 16 + fr, k = (wid + 8 * (it % P)) * 128 + fq * 16;
        if (it < total && n < N) {
            const signed char* at = q + n * ldq + k;
            if (k < K) p.a = *reinterpret_cast<const i32x4*>(at);
            if (k + 64 < K) p.b = *reinterpret_cast<const i32x4*>(at + 64);
        }
        return p;
    };
    Pair buf[4];
#pragma unroll
    for (int u = 0; u < 3; ++u) buf[u] = load(u);
    if (M <= 4 && K > 2048) {                  // long rows, fewer than waves: 1 x 1000 x 25 088 36 -> 17 us
        for (int m = 0; m < M; ++m) {
            const float t = quantize_row<8>(x + m * ldx, K, Kp, vec, xs + m * LD);
            if (threadIdx.x == 0) sx[m] = t;
        }
    } else {
        for (int m = wid; m < M; m += 8) {
            const float t = quantize_row<1>(x + m * ldx, K, Kp, vec, xs + m * LD);
            if (lane == 0) sx[m] = t;
        }
    }
    __syncthreads();
    const signed char* row = xs + (fr < M ? fr : 0) * LD + fq * 16;        // (columns from M on repeat row 0 and are not stored)
    i32x4 acc = {0, 0, 0, 0};
    int done = 0;                                                          // tiles finished
    for (int base = 0; base < total; base += 4) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int it = base + u;
            if (it >= total) break;
            buf[(u + 3) & 3] = load(it + 3);
            const int k = (wid + 8 * (it % P)) * 128;
            if (k < Kp) {
                acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(buf[u].a, *reinterpret_cast<const i32x4*>(row + k), acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(buf[u].b, *reinterpret_cast<const i32x4*>(row + k + 64), acc, 0, 0, 0);
            }
            if (it % P != P - 1) continue;
            i32x4(&mine)[8][64] = red[done & 1];
            mine[wid][lane] = acc;
            acc = i32x4{0, 0, 0, 0};
            __syncthreads();
            // channel 4 (lane / 16) + e of row lane % 16 lies at [lane][e]; the buffer of two tiles ago is free behind this barrier
            if (threadIdx.x < 256) {
                const int c = threadIdx.x & 15, m = threadIdx.x >> 4, n = ((int)blockIdx.x + done * (int)gridDim.x) * 16 + c;
                if (m < M && n < N) {
                    const int l = (c >> 2) * 16 + m, e = c & 3;
                    int sum = 0;
#pragma unroll
                    for (int w = 0; w < 8; ++w) sum += mine[w][l][e];
                    st1(y + m * ldy + n, (float)sum * (sx[m] * s[n]) + (bias ? bias[n] : 0.f));
                }
            }
            ++done;
        }
    }
}

constexpr int SKINNY = 16, SKINNY_LDS = 40 * 1024;
bool skinny(long long M, int K) { return M <= SKINNY && M * ((K + 127LL) / 128 * 128 + 16) <= SKINNY_LDS; }
bool rows_vec(const void* x, int bf16, long long ldx) { return ddl_aligned16(x) && ldx % (bf16 ? 8 : 4) == 0; }

// (a launch's threads are counted in 32 bits: 2^23 rows at a time)
template <typename T>
void launch_rows(const T* x, long long ldx, long long M, int K, int Kp, int vec, signed char* q, float* scale, unsigned* counters, int ncount, hipStream_t stream) {
    constexpr long long AT_ONCE = 1LL << 23;
    for (long long m = 0; m < M; m += AT_ONCE) {
        const int rows = (int)(M - m < AT_ONCE ? M - m : AT_ONCE);
        // (rows that a wave does not hold: 12 544 of 4096 values 31 -> 29 us, 16 of 25 088 in the whole product 66 -> 43)
        if (K > 2048)
            DDL_KLAUNCH((int8_rows_kernel<4, T>), dim3(rows), dim3(256), 0, stream, x + m * ldx, ldx, rows, K, Kp, vec, q + m * Kp, scale + m, counters,
                        m == 0 ? ncount : 0);
        else
            DDL_KLAUNCH((int8_rows_kernel<1, T>), dim3((rows + 3) / 4), dim3(256), 0, stream, x + m * ldx, ldx, rows, K, Kp, vec, q + m * Kp, scale + m, counters,
                        m == 0 ? ncount : 0);
    }
}

long long codes_bytes(long long M, int Kp) { return (M * Kp + 255) / 256 * 256 + (M * 4 + 255) / 256 * 256; }
// Parts of the sums of tiles of 64 (1: none).  A workgroup alone on its CU takes 0.15 us per 128 columns, the join 4 us and 0.3 us a
// part: sqrt(stages / 2) parts from 96 stages on, while each part has a CU.  64 x 4096 x 25 088 49 -> 38 us, 256 x 1000 x 25 088 50 -> 35,
// 1 x 1000 x 100 000 147 -> 58; 64 stages, 7 x 4096 x 8192: 17.7 -> 19.6.
int split_of(long long M, int N, int K) {
    const long long t64 = ((M + 63) / 64) * ((N + 63LL) / 64), stages = (K + 127) / 128;
    if (stages < 96 || t64 > 128) return 1;
    const double most = fmin(256.0 / (double)t64, fmin(32.0, sqrt(0.5 * (double)stages)));
    const long long each = (stages + (int)most - 1) / (int)most;
    return (int)((stages + each - 1) / each);
}

template <typename T>
int run(const T* x, long long ldx, const signed char* q, long long ldq, const float* s, const float* bias, T* y, long long ldy, int M, int N, int K,
        char* ws, hipStream_t stream) {
    const int vec = rows_vec(x, sizeof(T) == 2, ldx), Kp = (K + 127) / 128 * 128;
    if (skinny(M, K)) {
        const int tiles = (N + 15) / 16, grid = tiles < 512 ? tiles : 512;
        DDL_KLAUNCH(int8_skinny_kernel<T>, dim3(grid), dim3(512), (size_t)M * (Kp + 16), stream, x, ldx, vec, q, ldq, s, bias, y, ldy, M, N, K, tiles);
        return ddl_launch_status();
    }
    signed char* xq = (signed char*)ws;
    float* sx = (float*)(ws + ((long long)M * Kp + 255) / 256 * 256);
    // 128 x 128 tiles, two a CU, unless they are fewer than the CUs; two groups of waves a tile where even 64 x 64 are.  (256 x 256 in 8 waves is no faster where it fills whole rounds,
    // 4096^3 in 100 / 101 us, and 12 544 x 4096 x 4096 takes 4 rounds for 3.06: 333 / 304 us.  256 x 128: 328; 4 waves of 128 x 128:
    // 396, copies between register halves.)
    const long long t128 = ((M + 127LL) / 128) * ((N + 127) / 128), t64 = ((M + 63LL) / 64) * ((N + 63) / 64);
    if (t128 > 0xffffffLL - 8) return DDL_EINVAL;
    const int split = split_of(M, N, K);
    int* slabs = (int*)(ws + codes_bytes(M, Kp));
    unsigned* counters = (unsigned*)(slabs + t64 * split * 64 * 64);
    launch_rows(x, ldx, M, K, Kp, vec, xq, sx, counters, split > 1 ? (int)t64 : 0, stream);
#define GEMM(B, W0, W1, NST, KS, t) DDL_KLAUNCH((int8_gemm_kernel<T, B, W0, W1, NST, KS>), dim3((unsigned)((t + 7) / 8 * 8)), dim3(KS * W0 * W1 * 64), 0, stream, xq, sx, q, \
                                            ldq, s, bias, y, ldy, M, N, K, Kp, (M + B - 1) / B, (N + B - 1) / B, split, slabs, counters)
    if (t128 >= 256) GEMM(128, 2, 2, 2, 1, t128);
    else if (t64 <= 256 && Kp > 128) GEMM(64, 2, 2, 3, 2, t64 * split);
    else GEMM(64, 2, 2, 3, 1, t64);
#undef GEMM
    return ddl_launch_status();
}

}  // namespace

// codes and scales of the rows of x [M][K] (row stride ldx elements); q [M][Kp], zeros from K on, Kp a multiple of 16, q aligned
extern "C" int ddl_int8_rows(const void* x, int x_bf16, long long ldx, long long M, int K, int Kp, void* q, void* scale, hipStream_t stream) {
    if (M == 0) return DDL_OK;
    if (!x || !q || !scale || M < 0 || M > 0x7fffff00LL || K <= 0 || Kp < K || Kp % 16 || ldx < 0) return DDL_EINVAL;
    if (!ddl_aligned16(q)) return DDL_EALIGN;
    const int vec = rows_vec(x, x_bf16, ldx);
    if (x_bf16) launch_rows((const bf16_t*)x, ldx, M, K, Kp, vec, (signed char*)q, (float*)scale, nullptr, 0, stream);
    else launch_rows((const float*)x, ldx, M, K, Kp, vec, (signed char*)q, (float*)scale, nullptr, 0, stream);
    return ddl_launch_status();
}

extern "C" int ddl_int8_max_k() { return 133144; }

// bytes of workspace of ddl_int8_linear
extern "C" long long ddl_int8_linear_workspace(long long M, int N, int K) {
    if (skinny(M, K)) return 0;
    const long long Kp = (K + 127LL) / 128 * 128;
    const int split = split_of(M, N, K);
    return codes_bytes(M, (int)Kp) + (split > 1 ? ((M + 63) / 64) * ((N + 63LL) / 64) * (split * 64LL * 64 * 4 + 4) : 0);
}

// y [M][N] (bf16 or fp32 like x) = x [M][K] times q [N][K]^T with scales; rows of q start at multiples of 16 bytes and may be
// read up to the next multiple of 16 behind K; q_bytes: what may be read from q on
extern "C" int ddl_int8_linear(const void* x, int x_bf16, long long ldx, const void* q, long long ldq, long long q_bytes, const void* s, const void* bias,
                               void* y, long long ldy, long long M, int N, int K, void* ws, long long ws_bytes, hipStream_t stream) {
    if (M == 0 || N == 0) return DDL_OK;
    if (!x || !q || !s || !y || M < 0 || N < 0 || K <= 0 || K > ddl_int8_max_k() || ldx < 0 || ldq < K || ldy < N) return DDL_EINVAL;
    // (a tile's byte offsets have 31 bits)
    if (M > 0x7fffff00LL || N > 0x7fffff00 || ldq >= (1 << 22)) return DDL_EINVAL;
    if (!ddl_aligned16(q) || ldq % 16 || !ddl_aligned16(y) || (reinterpret_cast<uintptr_t>(ws) & 255)) return DDL_EALIGN;
    if (q_bytes < (N - 1LL) * ldq + (K + 15) / 16 * 16) return DDL_EINVAL;
    const long long need = ddl_int8_linear_workspace(M, N, K);
    if (need > 0 && (!ws || ws_bytes < need)) return DDL_EINVAL;
    if (x_bf16)
        return run((const bf16_t*)x, ldx, (const signed char*)q, ldq, (const float*)s, (const float*)bias, (bf16_t*)y, ldy, (int)M, N, K, (char*)ws, stream);
    return run((const float*)x, ldx, (const signed char*)q, ldq, (const float*)s, (const float*)bias, (float*)y, ldy, (int)M, N, K, (char*)ws, stream);
}
