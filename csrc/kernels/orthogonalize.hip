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
constexpr int LDK = 40;   // LDS row of 32 reduction elements, padded to 80 bytes

// 64 x 64 tile of rows a[..][k] times rows b[..][k] (both k-contiguous), 4 waves of 32 x 32
template <bool TRANS_B>
__device__ __forceinline__ void tile_mul(const f16_t* __restrict__ a, int lda, const f16_t* __restrict__ b, int ldb, int K, f16_t* As,
                                         f16_t* Bs, f32x4 (&acc)[2][2]) {
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, wm = wid >> 1, wn = wid & 1;
    const int row = tid >> 2, ch = tid & 3;
    for (int k0 = 0; k0 < K; k0 += 32) {
        const f16x8 va = *reinterpret_cast<const f16x8*>(a + (long long)row * lda + k0 + ch * 8);
        f16x8 vb;
        if (TRANS_B) vb = *reinterpret_cast<const f16x8*>(b + (long long)(k0 + (tid >> 3)) * ldb + (tid & 7) * 8);
        else vb = *reinterpret_cast<const f16x8*>(b + (long long)row * ldb + k0 + ch * 8);
        __syncthreads();
        *reinterpret_cast<f16x8*>(As + row * LDK + ch * 8) = va;
        if (TRANS_B) {
#pragma unroll
            for (int e = 0; e < 8; ++e) Bs[((tid & 7) * 8 + e) * LDK + (tid >> 3)] = vb[e];
        } else {
            *reinterpret_cast<f16x8*>(Bs + row * LDK + ch * 8) = vb;
        }
        __syncthreads();
        f16x8 fa[2], fb[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            fa[i] = *reinterpret_cast<const f16x8*>(As + (wm * 32 + i * 16 + (lane & 15)) * LDK + (lane >> 4) * 8);
            fb[i] = *reinterpret_cast<const f16x8*>(Bs + (wn * 32 + i * 16 + (lane & 15)) * LDK + (lane >> 4) * 8);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fa[i], fb[j], acc[i][j], 0, 0, 0);
    }
}

__device__ __forceinline__ void tri_tile(int idx, int& ti, int& tj) {    // idx -> (ti >= tj) of a lower triangle
    ti = (int)((sqrtf(8.f * (float)idx + 1.f) - 1.f) * 0.5f);
    while ((ti + 1) * (ti + 2) / 2 <= idx) ++ti;
    while (ti * (ti + 1) / 2 > idx) --ti;
    tj = idx - ti * (ti + 1) / 2;
}

// SQUARE = false: O, d of A = X X^T.  SQUARE = true: O, d of P = b A + c A^2 (diagonal: + a) from those of A
template <bool SQUARE>
__global__ void __launch_bounds__(256) ortho_sym_kernel(const MulTable t, const f16_t* __restrict__ in, const float* __restrict__ din,
                                                       f16_t* __restrict__ out, float* __restrict__ dout, const int* __restrict__ ex, int down,
                                                       float ca, float cb, float cc) {
    __shared__ __attribute__((aligned(16))) f16_t As[64 * LDK], Bs[64 * LDK];
    const int gi = find_group(t, blockIdx.x);
    const MulGroup g = t.g[gi];
    const unsigned idx = blockIdx.x - g.first;
    const int b = idx / g.tiles;
    int ti, tj;
    tri_tile(idx - b * g.tiles, ti, tj);
    const int K = SQUARE ? g.np : g.mp;
    const long long ao = (long long)g.ao * 64 + (long long)b * g.np * g.np;
    const f16_t* src = SQUARE ? in + ao : in + (long long)g.xo * 64 + (long long)b * g.np * g.mp;
    f32x4 acc[2][2] = {};
    tile_mul<false>(src + (long long)ti * 64 * K, K, src + (long long)tj * 64 * K, K, K, As, Bs, acc);
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, wm = wid >> 1, wn = wid & 1;
    const float* d = SQUARE ? din + g.dof + (long long)b * g.np : nullptr;
    const float unscale = SQUARE ? USC * USC : ldexpf(USC * USC, -2 * shift_of(ex, g.mat + b, down));
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = ti * 64 + wm * 32 + i * 16 + (lane >> 4) * 4 + e, c = tj * 64 + wn * 32 + j * 16 + (lane & 15);
                float v = acc[i][j][e] * unscale;
                if (SQUARE) {
                    const float o = (float)src[(long long)r * K + c] * USC;
                    const float dr = d[r], dc = d[c];
                    v = r == c ? ca + cb * dr + cc * (v + dr * dr) : cb * o + cc * (v + (dr + dc) * o);
                }
                if (r == c) dout[g.dof + (long long)b * g.np + r] = v;
                const f16_t h = r == c ? (f16_t)0.f : (f16_t)(v * SC);
                out[ao + (long long)r * g.np + c] = h;
                if (ti != tj) out[ao + (long long)c * g.np + r] = h;
            }
}

// X' = pd X + offdiag(P) X_hi
__global__ void __launch_bounds__(256) ortho_apply_kernel(const MulTable t, const f16_t* __restrict__ P, const float* __restrict__ pd,
                                                         const f16_t* __restrict__ xh, const f16_t* __restrict__ xl,
                                                         f16_t* __restrict__ yh, f16_t* __restrict__ yl,
                                                         const int* __restrict__ ex, int down, int down1) {
    __shared__ __attribute__((aligned(16))) f16_t As[64 * LDK], Bs[64 * LDK];
    const int gi = find_group(t, blockIdx.x);
    const MulGroup g = t.g[gi];
    const unsigned idx = blockIdx.x - g.first;
    const int b = idx / g.tiles, rem = idx - b * g.tiles, tm = g.mp >> 6;
    const int ti = rem / tm, tj = rem - ti * tm;
    const f16_t* A = P + (long long)g.ao * 64 + (long long)b * g.np * g.np + (long long)ti * 64 * g.np;
    const long long xo = (long long)g.xo * 64 + (long long)b * g.np * g.mp;
    f32x4 acc[2][2] = {};
    tile_mul<true>(A, g.np, xh + xo + tj * 64, g.mp, g.np, As, Bs, acc);
    const float rescale = ldexpf(1.f, shift_of(ex, g.mat + b, down1) - shift_of(ex, g.mat + b, down));
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, wm = wid >> 1, wn = wid & 1;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = ti * 64 + wm * 32 + i * 16 + (lane >> 4) * 4 + e, c = tj * 64 + wn * 32 + j * 16 + (lane & 15);
                const long long at = xo + (long long)r * g.mp + c;
                const float v = (pd[g.dof + (long long)b * g.np + r] * ((float)xh[at] + (float)xl[at]) + acc[i][j][e] * USC) * rescale;
                const f16_t h = (f16_t)v;
                yh[at] = h;
                yl[at] = (f16_t)(v - (float)h);
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
        mg.np = (int)np; mg.mp = (int)mp; mg.xo = (unsigned)(xo / 64); mg.ao = (unsigned)(ao / 64); mg.dof = (unsigned)dof; mg.mat = (unsigned)mat;
        mg.tiles = (int)(tn * (tn + 1) / 2); mg.first = (unsigned)nsym; sym.g[i] = mg;
        nsym += s.batch * mg.tiles;
        mg.tiles = (int)(tn * tm); mg.first = (unsigned)napp; app.g[i] = mg;
        napp += s.batch * mg.tiles;
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
        DDL_KLAUNCH(ortho_sym_kernel<false>, dim3((unsigned)nsym), block, 0, stream, sym, xh, (const float*)nullptr, O, d, ex, k * fall, a, b, c);
        DDL_KLAUNCH(ortho_sym_kernel<true>, dim3((unsigned)nsym), block, 0, stream, sym, O, d, P, pd, ex, 0, a, b, c);
        DDL_KLAUNCH(ortho_apply_kernel, dim3((unsigned)napp), block, 0, stream, app, P, pd, xh, xl, yh, yl, ex, k * fall, (k + 1) * fall);
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
