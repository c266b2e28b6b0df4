// K22: orthogonalisation of weight-shaped matrices by Newton-Schulz products (gfx950), K23: the optimizer step on top.
//
//   X_0 = G / max(|G|_F, eps)   as n x m with n <= m (a tall matrix is taken transposed)
//   A = X X^T,  P = b A + c A^2,  X <- a X + P X          `steps` times;  result: X, in G's orientation
//
// Arithmetic.  A perturbation of X in the directions of small singular values grows by a per step (485 over five steps
// with a = 3.4445), so where the products round decides the result's accuracy.  The matrix pipe runs fp16 at bf16's
// rate with three more bits, and every quantity here is bounded, so the operands are fp16, scaled by 2^12 (off the
// subnormals); two things are kept apart from them at no extra product:
//   * X is a pair of fp16 values hi + lo; products read hi, the term a X reads both;
//   * the diagonals of A and P stay in fp32 (near the end A is close to a multiple of 1: its diagonal carries all of
//     its rounding): with A = D + O,  A^2 = O^2 + (d_i + d_j) O + D^2, and P X = (a + diag P) X + offdiag(P) X_hi.
// Against 64 bits the result is 2e-4 .. 1e-3 off (2-norm; Gaussian, power-law, exponential, low-rank and gradient-like
// spectra), below half a bf16 step (1.7e-3 on average); bf16 operands throughout give 8e-3 .. 0.3, plain fp16 1e-3 .. 4e-2.
//
// A call takes up to 64 groups of equal matrices; all of them share each launch (a table of shapes and offsets travels by
// value in the kernel arguments, so a call can be captured or recorded and needs no copy to the device): sums of squares,
// packing, three products a step, result.  A matrix whose norm is below eps starts at X_0 = G / eps, far below 1: it is
// kept scaled by a further 2^e (shift_of), which falls from step to step as X can grow.  Workspace copies are padded to multiples of 64 with zeros, which the steps
// keep (0 = a 0 + 0), so the products have no edges.
#include "common.h"
#include <math.h>

namespace {

typedef _Float16 f16_t;
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int MAXG = 64;            // groups of a launch: one lane each in find_group
constexpr int PARTS = 1024;         // most partial sums of squares of a matrix
constexpr float SC = 4096.f, USC = 1.f / 4096.f;

struct IoGroup {                    // where a group's matrices come from / go to
    const void* p;                  // first matrix (K23: unused)
    long long bs;                   // elements from a matrix to the next (K23: offset in the arenas)
    int rs, cs;                     // strides of a row, of a column
    int r, c;
    int part_elems;                 // elements of a partial sum of squares
    unsigned xo;                    // first matrix in the workspace, in 64 elements
    unsigned po;                    // its first partial sum
    unsigned first;                 // first workgroup of the group in this launch
    unsigned mat;                   // its first matrix among all
};
struct IoTable { IoGroup g[MAXG]; int count; };

struct MulGroup {
    int np, mp;                     // padded sizes
    unsigned xo, ao, dof;           // first matrix in the X and A workspaces (64 elements), in the diagonals (elements)
    unsigned first;
    unsigned mat;
    int tiles;                      // workgroups of a matrix
    int batch;
};
struct MulTable { MulGroup g[MAXG]; int count; };

// the group whose workgroups contain `bid`: groups are in ascending order of `first`
template <typename T>
__device__ __forceinline__ int find_group(const T& t, unsigned bid) {
    const int lane = threadIdx.x & 63;
    const bool mine = lane < t.count && t.g[lane < t.count ? lane : 0].first <= bid;
    return __builtin_amdgcn_readfirstlane(__popcll(__ballot(mine)) - 1);
}

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

struct Muon {                       // K23: arenas of one parameter dtype
    const void* g;
    float* v;
    float* w;
    bf16_t* lowp;
    float lr, mu, wd;
    int nesterov;
    const float* lr_scale;
};

// X in the workspace is 2^(12 + e) X: e of a matrix after steps that let it grow by at most 2^down
__device__ __forceinline__ int shift_of(const int* ex, unsigned mat, int down) {
    const int e = ex[mat] - down;
    return e > 0 ? e : 0;
}

// ---- element (i, j) of the matrix that is orthogonalised --------------------------------------------------------------
// kind 0 / 1: an fp32 / bf16 tensor; 2 / 3: the momentum direction from an fp32 / bf16 gradient arena
template <int KIND>
__device__ __forceinline__ float load_u(const IoGroup& g, const Muon& mu, int b, int i, int j) {
    if (KIND >= 2) {
        const long long e = g.bs + (long long)i * g.c + j;
        const float v = mu.v[e];
        if (!mu.nesterov) return v;
        const float gr = KIND == 3 ? bf2f(((const bf16_t*)mu.g)[e]) : ((const float*)mu.g)[e];
        return gr + mu.mu * v;
    }
    const long long e = b * g.bs + (long long)i * g.rs + (long long)j * g.cs;
    return KIND == 1 ? bf2f(((const bf16_t*)g.p)[e]) : ((const float*)g.p)[e];
}

// sums of squares in 64 bits (an fp32 square overflows from 1.8e19 on and vanishes below 1e-23): one partial a workgroup
template <int KIND>
__global__ void __launch_bounds__(256) ortho_sqsum_kernel(const IoTable t, const Muon mu, double* __restrict__ part) {
    const int gi = find_group(t, blockIdx.x);
    const IoGroup g = t.g[gi];
    const long long numel = (long long)g.r * g.c;
    const int np = (int)((numel + g.part_elems - 1) / g.part_elems);
    const unsigned idx = blockIdx.x - g.first;
    const int b = idx / np, pi = idx - b * np;
    const long long lo = (long long)pi * g.part_elems, hi = lo + g.part_elems < numel ? lo + g.part_elems : numel;
    double s = 0.0;
    for (long long e = lo + threadIdx.x; e < hi; e += 256) {
        float u;
        if (KIND >= 2) {
            const long long at = g.bs + e;
            const float gr = KIND == 3 ? bf2f(((const bf16_t*)mu.g)[at]) : ((const float*)mu.g)[at];
            const float v = mu.mu * mu.v[at] + gr;
            mu.v[at] = v;
            u = mu.nesterov ? gr + mu.mu * v : v;
        } else {
            const int i = (int)(e / g.c), j = (int)(e - (long long)i * g.c);
            u = load_u<KIND>(g, mu, b, i, j);
        }
        s += (double)u * (double)u;
    }
    __shared__ double red[4];
    s = wave_sum_d(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) part[g.po + (unsigned)b * np + pi] = (red[0] + red[1]) + (red[2] + red[3]);
}

// hi + lo of the scaled, normalised matrix; one 64 x 64 tile of the padded workspace a workgroup
template <int KIND>
__global__ void __launch_bounds__(256) ortho_pack_kernel(const IoTable t, const Muon mu, const double* __restrict__ part, float eps,
                                                        int* __restrict__ ex, f16_t* __restrict__ xh, f16_t* __restrict__ xl) {
    __shared__ float tile[64][65];
    __shared__ double red[4];
    const int gi = find_group(t, blockIdx.x);
    const IoGroup g = t.g[gi];
    const bool turn = g.r > g.c;
    const int n = turn ? g.c : g.r, m = turn ? g.r : g.c;
    const int tn = (n + 63) >> 6, tm = (m + 63) >> 6;
    const unsigned idx = blockIdx.x - g.first;
    const int b = idx / (tn * tm), ti = (idx - b * (tn * tm)) / tm, tj = idx - b * (tn * tm) - ti * tm;
    const long long numel = (long long)g.r * g.c;
    const int np = (int)((numel + g.part_elems - 1) / g.part_elems);
    double s = 0.0;
    for (int k = threadIdx.x; k < np; k += 256) s += part[g.po + (unsigned)b * np + k];
    s = wave_sum_d(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    const double norm = sqrt((red[0] + red[1]) + (red[2] + red[3]));
    const bool small = norm < (double)eps && norm > 0.0;
    const int shift = small ? ilogb((double)eps / norm) : 0;
    const double inv = ldexp((double)SC, shift) / (norm > (double)eps ? norm : (norm == norm ? (double)eps : norm));   // (a NaN stays one)
    if (ti == 0 && tj == 0 && threadIdx.x == 0) ex[g.mat + b] = shift;
    const int x = threadIdx.x & 63, y0 = threadIdx.x >> 6;
    for (int y = y0; y < 64; y += 4) {
        // the lane index runs along the source's rows (its usual contiguous direction) in both orientations
        const int i = turn ? tj * 64 + y : ti * 64 + y, j = turn ? ti * 64 + x : tj * 64 + x;
        const float u = i < g.r && j < g.c ? (float)(load_u<KIND>(g, mu, b, i, j) * inv) : 0.f;
        if (turn) tile[x][y] = u; else tile[y][x] = u;
    }
    __syncthreads();
    const int mp = tm * 64;
    const long long base = (long long)g.xo * 64 + (long long)b * (tn * 64) * mp + (long long)(ti * 64) * mp + tj * 64;
    for (int y = y0; y < 64; y += 4) {
        const float u = tile[y][x];
        const f16_t h = (f16_t)u;
        xh[base + (long long)y * mp + x] = h;
        xl[base + (long long)y * mp + x] = (f16_t)(u - (float)h);
    }
}

// result of the last step -> the output tensor (bf16), or the weights (K23)
template <bool MUON>
__global__ void __launch_bounds__(256) ortho_unpack_kernel(const IoTable t, const Muon mu, const int* __restrict__ ex, int down,
                                                          const f16_t* __restrict__ xh, const f16_t* __restrict__ xl) {
    __shared__ float tile[64][65];
    const int gi = find_group(t, blockIdx.x);
    const IoGroup g = t.g[gi];
    const bool turn = g.r > g.c;
    const int n = turn ? g.c : g.r, m = turn ? g.r : g.c;
    const int tn = (n + 63) >> 6, tm = (m + 63) >> 6;
    const unsigned idx = blockIdx.x - g.first;
    const int b = idx / (tn * tm), ti = (idx - b * (tn * tm)) / tm, tj = idx - b * (tn * tm) - ti * tm;
    const int mp = tm * 64;
    const long long base = (long long)g.xo * 64 + (long long)b * (tn * 64) * mp + (long long)(ti * 64) * mp + tj * 64;
    const int x = threadIdx.x & 63, y0 = threadIdx.x >> 6;
    const float scale = ldexpf(USC, -shift_of(ex, g.mat + b, down));
    for (int y = y0; y < 64; y += 4) {
        const float u = ((float)xh[base + (long long)y * mp + x] + (float)xl[base + (long long)y * mp + x]) * scale;
        if (turn) tile[x][y] = u; else tile[y][x] = u;
    }
    __syncthreads();
    for (int y = y0; y < 64; y += 4) {
        const int i = turn ? tj * 64 + y : ti * 64 + y, j = turn ? ti * 64 + x : tj * 64 + x;
        if (i >= g.r || j >= g.c) continue;
        const float u = tile[y][x];
        if (MUON) {
            const float lr = mu.lr_scale ? mu.lr * *mu.lr_scale : mu.lr;
            const float s = lr * sqrtf(g.r > g.c ? (float)g.r / (float)g.c : 1.f);
            const long long e = g.bs + (long long)i * g.c + j;
            const float w = mu.w[e] * (1.f - lr * mu.wd) - s * u;
            mu.w[e] = w;
            if (mu.lowp) mu.lowp[e] = f2bf(w);
        } else {
            ((bf16_t*)g.p)[b * g.bs + (long long)i * g.rs + (long long)j * g.cs] = f2bf(u);
        }
    }
}

// ---- products ---------------------------------------------------------------------------------------------------------
// D = F S^T over K (a multiple of 32): 4 waves as 2 x 2, a BF x BS tile in steps of 32, NST stages filled by LDS-DMA (tile
// t + NST - 1 is on its way while tile t is multiplied; counted waits, one barrier a step).
//   S and, with TRF = false, F: row-major, k-contiguous rows.  LDS rows of 64 bytes, 16-byte chunk c of row r at c ^ -(r / 4)
//   (16 rows x one chunk are free of bank conflicts).
//   TRF = true: F is given transposed, [k][columns].  Its rows of k stay as they are in LDS and are read by the transposing
//   load: 16 lanes take 4 rows x 16 columns; a half-wave touches rows 0-3 and 8-11 (+ 4, + 16), whose 32-byte windows
//   the swizzle spreads over all banks.
// A lane ends with D[i][j][e]: F index 16 i + 4 (lane / 16) + e, S index 16 j + lane % 16 of its wave's quarter.
typedef __fp16 half4 __attribute__((ext_vector_type(4)));      // (the type that the transposing load is declared with)
typedef __attribute__((address_space(3))) half4* lds_half4_ptr;
constexpr unsigned OUT = 0x80000000u;      // an offset behind the descriptor's range: reads as zero

__device__ __forceinline__ int nt_off(int row, int ch) { return row * 64 + ((ch ^ ((0 - (row >> 2)) & 3)) << 4); }
template <int B>
__device__ __forceinline__ int tr_swz(int row) {
    return B == 128 ? (row & 3) | ((row >> 1) & 4) : ((row >> 1) & 1) | ((row >> 2) & 2);
}

template <int BF, int BS, int NST, bool TRF>
struct Mul {
    static constexpr int FBYTES = BF * 64, SBYTES = BS * 64, STAGE = FBYTES + SBYTES;
    static constexpr int FL = BF / 64, SL = BS / 64, L = FL + SL;       // LDS-DMA instructions of a wave and stage
    static constexpr int NF = BF / 32, NS = BS / 32;                    // fragments of a wave
    f32x4 acc[NF][NS];

    // f: first row (TRF: first column) of the tile, ldf its row length, fleft rows (columns) that exist; s likewise
    __device__ __forceinline__ void run(unsigned char* smem, const f16_t* f, long long ldf, int fleft, const f16_t* s, long long lds, int sleft, int K) {
        const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), w0 = wid >> 1, w1 = wid & 1;
        const int fr = lane & 15, fq = lane >> 4;
        const int KT = K / 32;
        const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) void*)smem;
        unsigned fo[FL], so[SL];
#pragma unroll
        for (int i = 0; i < FL; ++i) {
            const int slot = (i * 4 + wid) * 64 + lane;
            if (TRF) {
                constexpr int CPR = BF / 8;
                const int row = slot / CPR, ch = slot % CPR, c = (((ch >> 1) ^ tr_swz<BF>(row)) << 1) | (ch & 1);
                fo[i] = c * 8 < fleft ? (unsigned)((row * ldf + c * 8) * 2) : OUT;
            } else {
                const int row = slot >> 2, c = (slot & 3) ^ ((0 - (row >> 2)) & 3);
                fo[i] = row < fleft ? (unsigned)((row * ldf + c * 8) * 2) : OUT;
            }
        }
#pragma unroll
        for (int i = 0; i < SL; ++i) {
            const int slot = (i * 4 + wid) * 64 + lane, row = slot >> 2, c = (slot & 3) ^ ((0 - (row >> 2)) & 3);
            so[i] = row < sleft ? (unsigned)((row * lds + c * 8) * 2) : OUT;
        }
        // every stage is exactly L instructions a wave (zeros behind the end): the counted waits rely on it
        auto fetch = [&](int kt, int stage) {
            const bool live = kt < KT;
            const u32x4 rf = raw_rsrc(f + (live ? (TRF ? (long long)kt * 32 * ldf : (long long)kt * 32) : 0), OUT - 16);
            const u32x4 rs = raw_rsrc(s + (live ? (long long)kt * 32 : 0), OUT - 16);
            const unsigned at = lds0 + (unsigned)(stage * STAGE + wid * 1024);
#pragma unroll
            for (int i = 0; i < FL; ++i) lds_dma16(rf, at + i * 4096, live ? fo[i] : OUT, 0u);
#pragma unroll
            for (int i = 0; i < SL; ++i) lds_dma16(rs, at + FBYTES + i * 4096, live ? so[i] : OUT, 0u);
        };
        int foff[NF], soff[NS];
        const int trow = 8 * fq + ((lane >> 2) & 3);
#pragma unroll
        for (int i = 0; i < NF; ++i)
            foff[i] = TRF ? trow * (BF * 2) + (((w0 * NF + i) ^ tr_swz<BF>(trow)) * 32) + 8 * (lane & 3) : nt_off(w0 * (BF / 2) + i * 16 + fr, fq);
#pragma unroll
        for (int j = 0; j < NS; ++j) soff[j] = FBYTES + nt_off(w1 * (BS / 2) + j * 16 + fr, fq);
#pragma unroll
        for (int i = 0; i < NF; ++i)
#pragma unroll
            for (int j = 0; j < NS; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

#pragma unroll
        for (int k = 0; k < NST - 1; ++k) fetch(k, k);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NST - 2) * L) : "memory");
        __builtin_amdgcn_s_barrier();
        int cur = 0, nxt = NST - 1;
        for (int kt = 0; kt < KT; ++kt) {
            fetch(kt + NST - 1, nxt);          // into the stage whose reads ended before the last barrier
            unsigned char* st = smem + cur * STAGE;
            f16x8 a[NF], b[NS];
#pragma unroll
            for (int j = 0; j < NS; ++j) b[j] = *reinterpret_cast<const f16x8*>(st + soff[j]);
#pragma unroll
            for (int i = 0; i < NF; ++i) {
                if (TRF) {
                    // (row + 4 has the swizzle of row: bit 2 of the row does not take part in it)
                    const f16x4 lo = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_half4_ptr)(st + foff[i])));
                    const f16x4 hi = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_half4_ptr)(st + foff[i] + 4 * BF * 2)));
                    a[i] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                } else {
                    a[i] = *reinterpret_cast<const f16x8*>(st + foff[i]);
                }
            }
#pragma unroll
            for (int i = 0; i < NF; ++i)
#pragma unroll
                for (int j = 0; j < NS; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i], b[j], acc[i][j], 0, 0, 0);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NST - 2) * L) : "memory");
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            nxt = cur;
            cur = cur + 1 == NST ? 0 : cur + 1;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
};

// Tiles of a matrix in bands of 8 rows, a band column by column: the tiles that an XCD works on at a time are about as many
// rows as columns.  A matrix of many tiles is dealt to the XCDs (workgroup number modulo 8) in runs of neighbours.
__device__ __forceinline__ int deal(int idx, int tiles) {
    if (tiles < 64) return idx;
    const int q = tiles >> 3, r = tiles & 7, xcd = idx & 7;
    return xcd * q + (xcd < r ? xcd : r) + (idx >> 3);
}
__device__ __forceinline__ void band_tile(int idx, int rows, int cols, int& ti, int& tj) {
    const int band = idx / (8 * cols), rem = idx - band * 8 * cols, h = rows - band * 8 < 8 ? rows - band * 8 : 8;
    tj = rem / h;
    ti = band * 8 + rem - tj * h;
}
// the same of a lower triangle (ti >= tj): band b is 8 b whole columns and a triangle
__device__ __forceinline__ void tri_tile(int idx, int rows, int& ti, int& tj) {
    int band = (int)((sqrtf(16.f + 128.f * (float)idx) - 4.f) * (1.f / 64.f));
    while (32 * (band + 1) * (band + 1) + 4 * (band + 1) <= idx) ++band;
    while (32 * band * band + 4 * band > idx) --band;
    const int rem = idx - 32 * band * band - 4 * band, h = rows - band * 8 < 8 ? rows - band * 8 : 8;
    if (rem < h * 8 * band) {
        tj = rem / h;
        ti = band * 8 + rem - tj * h;
        return;
    }
    const int left = rem - h * 8 * band;
    int i = 0;
    while ((i + 1) * (i + 2) / 2 <= left) ++i;
    ti = band * 8 + i;
    tj = band * 8 + left - i * (i + 1) / 2;
}

// SQUARE = false: O, d of A = X X^T.  SQUARE = true: O, d of P = b A + c A^2 (diagonal: + a) from those of A
template <int B, int NST, bool SQUARE>
__global__ void __launch_bounds__(256, 2) ortho_sym_kernel(const MulTable t, const f16_t* __restrict__ in, const float* __restrict__ din,
                                                          f16_t* __restrict__ out, float* __restrict__ dout, const int* __restrict__ ex, int down,
                                                          float ca, float cb, float cc) {
    typedef Mul<B, B, NST, false> M;
    __shared__ __attribute__((aligned(16))) unsigned char smem[NST * M::STAGE];
    const int gi = find_group(t, blockIdx.x);
    const MulGroup g = t.g[gi];
    const unsigned idx = blockIdx.x - g.first;
    const int b = idx / g.tiles;
    if (b >= g.batch) return;              // (groups are padded to multiples of 8 workgroups)
    int ti, tj;
    tri_tile(deal(idx - b * g.tiles, g.tiles), (g.np + B - 1) / B, ti, tj);
    const int K = SQUARE ? g.np : g.mp;
    const long long ao = (long long)g.ao * 64 + (long long)b * g.np * g.np;
    const f16_t* src = SQUARE ? in + ao : in + (long long)g.xo * 64 + (long long)b * g.np * g.mp;
    M m;
    m.run(smem, src + (long long)ti * B * K, K, g.np - ti * B, src + (long long)tj * B * K, K, g.np - tj * B, K);
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, w0 = wid >> 1, w1 = wid & 1;
    const float* d = SQUARE ? din + g.dof + (long long)b * g.np : nullptr;
    const float unscale = SQUARE ? USC * USC : ldexpf(USC * USC, -2 * shift_of(ex, g.mat + b, down));
    f16_t* o = out + ao;
#pragma unroll
    for (int i = 0; i < M::NF; ++i)
#pragma unroll
        for (int j = 0; j < M::NS; ++j) {
            const int r = ti * B + w0 * (B / 2) + i * 16 + (lane >> 4) * 4, c = tj * B + w1 * (B / 2) + j * 16 + (lane & 15);
            if (B > 64 && (r >= g.np || c >= g.np)) continue;
            f32x4 v = m.acc[i][j] * unscale;
            if (SQUARE) {
                // (A is symmetric: its row c holds this lane's column)
                const f16x4 a = *reinterpret_cast<const f16x4*>(src + (long long)c * K + r);
                const f32x4 dr = *reinterpret_cast<const f32x4*>(d + r);
                const float dc = d[c];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float af = (float)a[e] * USC;
                    v[e] = r + e == c ? ca + cb * dc + cc * (v[e] + dc * dc) : cb * af + cc * (v[e] + (dr[e] + dc) * af);
                }
            }
            f16x4 h;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (r + e == c) dout[g.dof + (long long)b * g.np + c] = v[e];
                h[e] = r + e == c ? (f16_t)0.f : (f16_t)(v[e] * SC);
                if (ti != tj) o[(long long)(r + e) * g.np + c] = h[e];
            }
            *reinterpret_cast<f16x4*>(o + (long long)c * g.np + r) = h;
        }
}

// X' = pd X + offdiag(P) X_hi; tile: BF columns of X times BS rows of P
template <int BF, int BS, int NST>
__global__ void __launch_bounds__(256, 2) ortho_apply_kernel(const MulTable t, const f16_t* __restrict__ P, const float* __restrict__ pd,
                                                            const f16_t* __restrict__ xh, const f16_t* __restrict__ xl,
                                                            f16_t* __restrict__ yh, f16_t* __restrict__ yl,
                                                            const int* __restrict__ ex, int down, int down1) {
    typedef Mul<BF, BS, NST, true> M;
    __shared__ __attribute__((aligned(16))) unsigned char smem[NST * M::STAGE];
    const int gi = find_group(t, blockIdx.x);
    const MulGroup g = t.g[gi];
    const unsigned idx = blockIdx.x - g.first;
    const int b = idx / g.tiles;
    if (b >= g.batch) return;              // (groups are padded to multiples of 8 workgroups)
    int ti, tj;
    band_tile(deal(idx - b * g.tiles, g.tiles), (g.np + BS - 1) / BS, (g.mp + BF - 1) / BF, ti, tj);
    const f16_t* A = P + (long long)g.ao * 64 + (long long)b * g.np * g.np + (long long)ti * BS * g.np;
    const long long xo = (long long)g.xo * 64 + (long long)b * g.np * g.mp;
    M m;
    m.run(smem, xh + xo + tj * BF, g.mp, g.mp - tj * BF, A, g.np, g.np - ti * BS, g.np);
    const float rescale = ldexpf(1.f, shift_of(ex, g.mat + b, down1) - shift_of(ex, g.mat + b, down));
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, w0 = wid >> 1, w1 = wid & 1;
    const float* d = pd + g.dof + (long long)b * g.np;
#pragma unroll
    for (int j = 0; j < M::NS; ++j) {
        const int r = ti * BS + w1 * (BS / 2) + j * 16 + (lane & 15);
        if (BS > 64 && r >= g.np) continue;
        const float dr = d[r];
#pragma unroll
        for (int i = 0; i < M::NF; ++i) {
            const int c = tj * BF + w0 * (BF / 2) + i * 16 + (lane >> 4) * 4;
            if (BF > 64 && c >= g.mp) continue;
            const long long at = xo + (long long)r * g.mp + c;
            const f16x4 h0 = *reinterpret_cast<const f16x4*>(xh + at), l0 = *reinterpret_cast<const f16x4*>(xl + at);
            f16x4 h, l;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float v = (dr * ((float)h0[e] + (float)l0[e]) + m.acc[i][j][e] * USC) * rescale;
                h[e] = (f16_t)v;
                l[e] = (f16_t)(v - (float)h[e]);
            }
            *reinterpret_cast<f16x4*>(yh + at) = h;
            *reinterpret_cast<f16x4*>(yl + at) = l;
        }
    }
}

// ---- host -------------------------------------------------------------------------------------------------------------
// one group as the callers describe it: 11 int64 values
struct Desc { long long src, sb, srs, scs, dst, db, drs, dcs, r, c, batch; };

struct Plan {
    long long x_elems = 0, a_elems = 0, d_elems = 0, parts = 0, mats = 0;
    long long xa_h, xa_l, xb_h, xb_l, o, p, d, pd, part, ex, bytes;
};

long long part_elems_of(long long numel) {
    long long e = (numel + PARTS - 1) / PARTS;
    e = (e + 2047) / 2048 * 2048;
    return e < 4096 ? 4096 : e;
}
long long pad64(long long v) { return (v + 63) / 64 * 64; }

bool plan_of(const Desc* q, int count, Plan& pl) {
    if (count < 0 || count > MAXG || (count && !q)) return false;
    for (int i = 0; i < count; ++i) {
        const Desc& s = q[i];
        if (s.r <= 0 || s.c <= 0 || s.batch <= 0 || s.r > (1 << 20) || s.c > (1 << 20)) return false;
        if (s.batch > (1LL << 31) || (s.r * s.c) > (1LL << 33)) return false;
        const long long np = pad64(s.r < s.c ? s.r : s.c), mp = pad64(s.r < s.c ? s.c : s.r);
        pl.x_elems += s.batch * np * mp;
        pl.a_elems += s.batch * np * np;
        pl.d_elems += s.batch * np;
        pl.mats += s.batch;
        const long long pe = part_elems_of(s.r * s.c);
        pl.parts += s.batch * ((s.r * s.c + pe - 1) / pe);
        if (pl.x_elems > (1LL << 37) || pl.d_elems > 0x7fffffffLL || pl.parts > 0x7fffffffLL) return false;
    }
    auto up = [](long long b) { return (b + 255) / 256 * 256; };
    long long at = 0;
    pl.xa_h = at; at += up(pl.x_elems * 2);
    pl.xa_l = at; at += up(pl.x_elems * 2);
    pl.xb_h = at; at += up(pl.x_elems * 2);
    pl.xb_l = at; at += up(pl.x_elems * 2);
    pl.o = at; at += up(pl.a_elems * 2);
    pl.p = at; at += up(pl.a_elems * 2);
    pl.d = at; at += up(pl.d_elems * 4);
    pl.pd = at; at += up(pl.d_elems * 4);
    pl.part = at; at += up(pl.parts * 8);
    pl.ex = at; at += up(pl.mats * 4);
    pl.bytes = at;
    return true;
}

// The polynomial over [0, top], top = what the step before leaves: the largest |f(s)|, |b s^2 + c s^4| (X and P have to stay
// in fp16's range) and |f(s) / s|, the most that X grows by.  False: out of range
bool range_of(float a, float b, float c, int steps, double& growth) {
    double top = 1.0;
    growth = 1.0;
    for (int k = 0; k < steps; ++k) {
        double f = 0.0, p = 0.0, q = 0.0;
        for (int i = 0; i <= 4096; ++i) {
            const double s = top * i / 4096.0, l = s * s, r = fabs(a + b * l + c * l * l);
            f = fmax(f, s * r);
            p = fmax(p, fabs(b * l + c * l * l));
            q = fmax(q, r);
        }
        if (!(f * 1.02 <= 8.0) || !(p * 1.02 <= 15.0) || !(top * top <= 15.0) || !(q <= 1024.0)) return false;
        growth = fmax(growth, q);
        top = f * 1.02 > 1.0 ? f * 1.02 : 1.0;
    }
    return true;
}
int growth_bits(float a, float b, float c, int steps) {
    double growth;
    return range_of(a, b, c, steps, growth) ? (int)ceil(log2(growth)) : 0;
}

// kind as in load_u
int run_all(const Desc* q, int count, int kind, const Muon& mu, float a, float b, float c, int steps, float eps, char* ws, hipStream_t stream) {
    Plan pl;
    if (!plan_of(q, count, pl)) return DDL_EINVAL;
    IoTable in, tiles, outt;
    MulTable sym, app;
    static const int sb = getenv("ORTHO_SB") ? atoi(getenv("ORTHO_SB")) : 64, ab = getenv("ORTHO_AB") ? atoi(getenv("ORTHO_AB")) : 64;
    in.count = tiles.count = outt.count = sym.count = app.count = count;
    long long nin = 0, nio = 0, nsym = 0, napp = 0, xo = 0, ao = 0, dof = 0, po = 0, mat = 0;
    for (int i = 0; i < count; ++i) {
        const Desc& s = q[i];
        const long long n = s.r < s.c ? s.r : s.c, m = s.r < s.c ? s.c : s.r, np = pad64(n), mp = pad64(m), tn = np / 64, tm = mp / 64;
        const long long pe = part_elems_of(s.r * s.c), parts = (s.r * s.c + pe - 1) / pe;
        IoGroup io;
        io.p = (const void*)s.src; io.bs = s.sb; io.rs = (int)s.srs; io.cs = (int)s.scs; io.r = (int)s.r; io.c = (int)s.c;
        io.part_elems = (int)pe; io.xo = (unsigned)(xo / 64); io.po = (unsigned)po; io.mat = (unsigned)mat;
        io.first = (unsigned)nin; in.g[i] = io;
        io.first = (unsigned)nio; tiles.g[i] = io;
        if (kind < 2) { io.p = (const void*)s.dst; io.bs = s.db; io.rs = (int)s.drs; io.cs = (int)s.dcs; }
        outt.g[i] = io;
        MulGroup mg;
        mg.np = (int)np; mg.mp = (int)mp; mg.xo = (unsigned)(xo / 64); mg.ao = (unsigned)(ao / 64); mg.dof = (unsigned)dof; mg.mat = (unsigned)mat; mg.batch = (int)s.batch;
        const long long sn = (np + sb - 1) / sb, an = (np + ab - 1) / ab, am = (mp + ab - 1) / ab;
        mg.tiles = (int)(sn * (sn + 1) / 2); mg.first = (unsigned)nsym; sym.g[i] = mg;
        nsym += (s.batch * mg.tiles + 7) / 8 * 8;
        mg.tiles = (int)(an * am); mg.first = (unsigned)napp; app.g[i] = mg;
        napp += (s.batch * mg.tiles + 7) / 8 * 8;
        nin += s.batch * parts; nio += s.batch * tn * tm;
        xo += s.batch * np * mp; ao += s.batch * np * np; dof += s.batch * np; po += s.batch * parts; mat += s.batch;
        if (nin > 0x7fffffffLL || nio > 0x7fffffffLL || nsym > 0x7fffffffLL || napp > 0x7fffffffLL) return DDL_EINVAL;
    }
    f16_t *xh = (f16_t*)(ws + pl.xa_h), *xl = (f16_t*)(ws + pl.xa_l), *yh = (f16_t*)(ws + pl.xb_h), *yl = (f16_t*)(ws + pl.xb_l);
    f16_t *O = (f16_t*)(ws + pl.o), *P = (f16_t*)(ws + pl.p);
    float *d = (float*)(ws + pl.d), *pd = (float*)(ws + pl.pd);
    double* part = (double*)(ws + pl.part);
    int* ex = (int*)(ws + pl.ex);
    const int fall = growth_bits(a, b, c, steps);
    const dim3 block(256);
#define IO(K)                                                                                              \
    DDL_KLAUNCH(ortho_sqsum_kernel<K>, dim3((unsigned)nin), block, 0, stream, in, mu, part);               \
    DDL_KLAUNCH(ortho_pack_kernel<K>, dim3((unsigned)nio), block, 0, stream, tiles, mu, part, eps, ex, xh, xl)
    if (kind == 0) { IO(0); } else if (kind == 1) { IO(1); } else if (kind == 2) { IO(2); } else { IO(3); }
#undef IO
    for (int k = 0; k < steps; ++k) {
#define SYM(B, NST, SQ, IN, DIN, OUTP, DOUT, DOWN) DDL_KLAUNCH((ortho_sym_kernel<B, NST, SQ>), dim3((unsigned)nsym), block, 0, stream, sym, IN, DIN, OUTP, DOUT, ex, DOWN, a, b, c)
        if (sb == 64) { SYM(64, 4, false, xh, (const float*)nullptr, O, d, k * fall); SYM(64, 4, true, O, d, P, pd, 0); }
        else { SYM(128, 4, false, xh, (const float*)nullptr, O, d, k * fall); SYM(128, 4, true, O, d, P, pd, 0); }
        if (ab == 64) DDL_KLAUNCH((ortho_apply_kernel<64, 64, 4>), dim3((unsigned)napp), block, 0, stream, app, P, pd, xh, xl, yh, yl, ex, k * fall, (k + 1) * fall);
        else DDL_KLAUNCH((ortho_apply_kernel<128, 128, 4>), dim3((unsigned)napp), block, 0, stream, app, P, pd, xh, xl, yh, yl, ex, k * fall, (k + 1) * fall);
        f16_t* s = xh; xh = yh; yh = s;
        s = xl; xl = yl; yl = s;
    }
    if (kind < 2) DDL_KLAUNCH(ortho_unpack_kernel<false>, dim3((unsigned)nio), block, 0, stream, outt, mu, ex, steps * fall, xh, xl);
    else DDL_KLAUNCH(ortho_unpack_kernel<true>, dim3((unsigned)nio), block, 0, stream, outt, mu, ex, steps * fall, xh, xl);
    return ddl_launch_status();
}

bool strides_fit(long long rs, long long cs) { return rs >= 0 && cs >= 0 && rs < (1LL << 31) && cs < (1LL << 31); }

}  // namespace

extern "C" int ddl_ortho_max_groups() { return MAXG; }

// 1 when the steps keep every operand in the range of scaled fp16 (see range_of)
extern "C" int ddl_ortho_coefficients_ok(float a, float b, float c, int steps) {
    double growth;
    return isfinite(a) && isfinite(b) && isfinite(c) && steps >= 0 && steps <= 64 && range_of(a, b, c, steps, growth);
}

// bytes of workspace of a call with these groups (`desc`: count x 11 int64: source address, its batch / row / column
// strides, destination address and strides, rows, columns, matrices), -1: sizes out of range
extern "C" long long ddl_ortho_workspace(const long long* desc, int count) {
    Plan pl;
    return plan_of((const Desc*)desc, count, pl) ? pl.bytes : -1;
}

// kind 0 / 1: fp32 / bf16 sources; destinations are bf16
extern "C" int ddl_orthogonalize(const long long* desc, int count, int kind, float a, float b, float c, int steps, float eps, void* ws,
                                 long long ws_bytes, hipStream_t stream) {
    if (count == 0) return DDL_OK;
    Plan pl;
    const Desc* q = (const Desc*)desc;
    if (kind < 0 || kind > 1 || !ws || !plan_of(q, count, pl) || ws_bytes < pl.bytes) return DDL_EINVAL;
    if (!ddl_ortho_coefficients_ok(a, b, c, steps) || !(eps >= 1e-30f)) return DDL_EINVAL;
    if (reinterpret_cast<uintptr_t>(ws) & 255) return DDL_EALIGN;
    for (int i = 0; i < count; ++i)
        if (!q[i].src || !q[i].dst || !strides_fit(q[i].srs, q[i].scs) || !strides_fit(q[i].drs, q[i].dcs) || q[i].sb < 0 || q[i].db < 0)
            return DDL_EINVAL;
    return run_all(q, count, kind, Muon{}, a, b, c, steps, eps, (char*)ws, stream);
}

// K23.  `desc` as above; only the batch stride (= the matrix's offset in the arenas), rows and columns are read.
//   v = mu v + g; u = nesterov ? g + mu v : v; O = orthogonalize(u)
//   w = w (1 - lr wd) - lr sqrt(max(1, r / c)) O; lowp = bf16(w) where given
// lr: by value times *lr_scale where given
extern "C" int ddl_muon_step(const long long* desc, int count, void* w, const void* g, void* v, void* lowp, int grad_is_bf16, float lr, float mu,
                             float wd, int nesterov, const void* lr_scale, float a, float b, float c, int steps, float eps, void* ws,
                             long long ws_bytes, hipStream_t stream) {
    if (count == 0) return DDL_OK;
    Plan pl;
    const Desc* q = (const Desc*)desc;
    if (!w || !g || !v || !ws || !plan_of(q, count, pl) || ws_bytes < pl.bytes) return DDL_EINVAL;
    if (!ddl_ortho_coefficients_ok(a, b, c, steps) || !(eps >= 1e-30f)) return DDL_EINVAL;
    if ((reinterpret_cast<uintptr_t>(ws) & 255) || !ddl_aligned16(w) || !ddl_aligned16(g) || !ddl_aligned16(v) || (lowp && !ddl_aligned16(lowp)))
        return DDL_EALIGN;
    for (int i = 0; i < count; ++i)
        if (q[i].batch != 1 || q[i].sb < 0) return DDL_EINVAL;
    Muon m;
    m.g = g; m.v = (float*)v; m.w = (float*)w; m.lowp = (bf16_t*)lowp;
    m.lr = lr; m.mu = mu; m.wd = wd; m.nesterov = nesterov; m.lr_scale = (const float*)lr_scale;
    return run_all(q, count, grad_is_bf16 ? 3 : 2, m, a, b, c, steps, eps, (char*)ws, stream);
}
