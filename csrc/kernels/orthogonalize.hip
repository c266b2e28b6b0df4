// K22: orthogonalisation of weight-shaped matrices by Newton-Schulz products (gfx950), K23: the optimizer step on top.
//
//   X_0 = G / max(|G|_F, eps)   as n x m with n <= m (a tall matrix is taken transposed)
//   A = X X^T,  P = b A + c A^2,  X <- a X + P X          `steps` times;  result: X, in G's orientation
//
// Arithmetic.  A perturbation of X in the directions of small singular values grows by a per step (485 over five steps
// with a = 3.4445), so where the products round decides the result's accuracy.  The matrix pipe runs fp16 at bf16's
// rate with three more bits, and every quantity here is bounded, so the operands are fp16, scaled by 2^12 (off the
// subnormals); two things are kept apart from them at no extra product:
//   * X is a pair of fp16 values hi + lo; products read hi, the term a X and, in the last two steps, diag(P) X read both (see low_by_a);
//   * the diagonals of A and P stay in fp32 (near the end A is close to a multiple of 1: its diagonal carries all of
//     its rounding): with A = D + O,  A^2 = O^2 + (d_i + d_j) O + D^2, and P X = (a + diag P) X + offdiag(P) X_hi.
// Against 64 bits the result is, before its rounding to bf16 (1.7e-3 itself), at most this much off (2-norm; Gaussian, power-law,
// exponential over six decades, rank 1, all but a sixteenth of the singular values a thousandth, gradient-like): 1e-4 .. 1.3e-3 from 33 rows
// on (bf16 operands throughout give 8e-3 .. 0.3, plain fp16 1e-3 .. 4e-2); up to 32 rows, which run in fp64, 1e-7 .. 5e-5.
//
// A call takes up to 64 groups of equal matrices.  The forms, by sizes alone; the groups of one form share its launches:
//   * up to 32 rows: all steps on the Gram matrix in fp64, a workgroup a matrix in one launch (ortho_few_kernel), long ones in four
//     (ortho_thin_*_kernel); see forms_of;
//   * if all others are of up to 64 x 768 or 128 x 384: a workgroup a matrix, one launch (ortho_small_kernel, all_small);
//   * else tiles: sums of squares (whose first workgroup writes the table of shapes and offsets, from the kernel's arguments: a
//     call can be captured or recorded and copies nothing to the device), packing, three products a step; the last product
//     writes the result or the weights.
// A matrix whose norm is below eps starts at X_0 = G / eps, far below 1: it is kept scaled by a further 2^e (shift_of), which
// falls from step to step as X can grow.  Workspace copies are padded to multiples of 64 with zeros, which the steps keep
// (0 = a 0 + 0), so the products have no edges.
#include "common.h"
#include "tile_mul.h"
#include <math.h>
#include <string.h>

namespace {

constexpr int MAXG = 64;            // groups of a call: one lane each where a workgroup looks its group up
constexpr int CHUNK = 32;           // groups that travel in one launch's arguments
constexpr int PARTS = 1024;         // most partial sums of squares of a matrix
constexpr float SC = 4096.f, USC = 1.f / 4096.f;

struct Group {                      // `batch` equal matrices
    const void* src;                // K23: unused
    bf16_t* dst;                    // dense
    long long sb;                   // elements from a matrix to the next (K23: offset in the arenas)
    int rs, cs;                     // strides of a row, of a column of src
    int r, c, np, mp;               // sizes; padded shorter and longer side
    int batch;
    short vec, flat;                // src (K23: the arenas) can be read 8 elements of a row at a time; src is one array from 16 bytes on
    int part_elems, parts;          // elements of a partial sum of squares, partial sums of a matrix
    unsigned xo, ao, dof, po, mat;  // first matrix in the X and square workspaces (64 elements), in the diagonals, the partial sums, among all
    int tsym, tapp;                 // tiles of a matrix in the symmetric products and in P X
    int hsym, happ;                 // the XCD that computes them, -1: all
    unsigned fin, fio;              // first workgroup of the sums, of the packing (thin form: of the chunks)
    union { int tcols; int split; };        // thin form: columns of a chunk; tiles: parts of a tile's sum in X X^T (see splits_of)
    union { int chunks; unsigned slab; };   // thin form: chunks of a matrix; tiles: the first part's slab and counter
};
struct Chunk { Group g[CHUNK]; int base, n, last; };

// What the kernels of a call read.  Workgroup w of a product runs on XCD w mod 8 as that XCD's item w / 8: fsym / fapp say at
// which item a group begins there.  Tiles of a small matrix all go to one XCD, whose L2 then holds it; those of a large one are
// cut into 8 runs of neighbours.
struct Table {
    Group g[MAXG];
    unsigned fin[MAXG], fio[MAXG], fsym[8][MAXG], fapp[8][MAXG];
    int batch[MAXG], np[MAXG], mp[MAXG], tsym[MAXG], tapp[MAXG], hsym[MAXG], happ[MAXG];      // copies out of g: a lane a group (find_tile)
    unsigned xo[MAXG], ao[MAXG], dof[MAXG], mat[MAXG], slab[MAXG];
    int split[MAXG], lone[MAXG];
};

__host__ __device__ __forceinline__ unsigned run_start(unsigned total, int home, int xcd) {
    return home < 0 ? (unsigned)((unsigned long long)total * xcd / 8) : (xcd > home ? total : 0u);
}

// One workgroup writes its chunk's groups; that of the last chunk also where the groups begin on each XCD.  1024 threads: one
// wave a prefix sum.
__device__ __forceinline__ void write_table(const Chunk& ch, Table* __restrict__ t, unsigned* __restrict__ counters, int slabs) {
    if (ch.last)
        for (int i = threadIdx.x; i < slabs; i += 1024) counters[i] = 0u;
    const unsigned* from = reinterpret_cast<const unsigned*>(ch.g);
    unsigned* to = reinterpret_cast<unsigned*>(t->g + ch.base);
    for (int i = threadIdx.x; i < ch.n * (int)(sizeof(Group) / 4); i += 1024) to[i] = from[i];
    if (!ch.last) return;
    const int lane = threadIdx.x & 63, k = threadIdx.x >> 6, count = ch.base + ch.n;
    const bool live = lane < count;
    // (groups of earlier chunks: written by earlier launches)
    Group g = {};
    if (lane < ch.base) g = t->g[lane];
    else if (live) g = ch.g[lane - ch.base];
    if (k == 0) {
        t->fin[lane] = live ? g.fin : 0xffffffffu;
        t->fio[lane] = live ? g.fio : 0xffffffffu;
        t->batch[lane] = g.batch; t->np[lane] = g.np; t->mp[lane] = g.mp;
        t->tsym[lane] = g.tsym; t->tapp[lane] = g.tapp; t->hsym[lane] = g.hsym; t->happ[lane] = g.happ;
        t->xo[lane] = g.xo; t->ao[lane] = g.ao; t->dof[lane] = g.dof; t->mat[lane] = live ? g.mat : 0xffffffffu;
        t->split[lane] = g.split; t->slab[lane] = g.slab; t->lone[lane] = g.r == 1 || g.c == 1;
    }
    const int xcd = k & 7, home = k < 8 ? g.hsym : g.happ;
    const unsigned total = live ? (unsigned)g.batch * (unsigned)(k < 8 ? g.tsym : g.tapp) : 0u;
    const unsigned mine = run_start(total, home, xcd + 1) - run_start(total, home, xcd);
    unsigned sum = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned v = __shfl_up(sum, o, 64);
        if (lane >= o) sum += v;
    }
    (k < 8 ? t->fsym : t->fapp)[xcd][lane] = live ? sum - mine : 0xffffffffu;
}

// the last of the groups that begin at or before `at`
__device__ __forceinline__ int find_group(const unsigned* first, unsigned at) {
    const bool mine = first[threadIdx.x & 63] <= at;
    return __builtin_amdgcn_readfirstlane(__popcll(__ballot(mine)) - 1);
}
// item of a product -> group, matrix, tile and what the product needs to know.  Every lane reads its group's values at once and
// the one that is meant is picked afterwards: a tile waits for one load, not for two in a row.
// What Item needs of a call's only group (ONE, tiles of 64): it travels in the arguments, a round trip to memory less in each launch
// (301 x 410 105 -> 101 us, 12 of 512 x 512 153 -> 149)
struct Single { int np, mp, batch, tsym, tapp, split, lone; };
template <bool ONE>
struct Item {
    int gi, b, tile, np, mp, part, split, lone;
    unsigned xo, ao, dof, mat, slab;
    __device__ __forceinline__ bool find(const Table* t, const Single& one, bool sym) {      // false: this XCD has no such item
        const unsigned xcd = blockIdx.x & 7, at = blockIdx.x >> 3;
        part = 0;
        split = 1;
        if (ONE) {
            gi = 0;
            np = one.np;
            lone = one.lone;
            mp = one.mp;
            xo = ao = dof = mat = slab = 0u;
            const unsigned tiles = sym ? one.tsym : one.tapp, total = (unsigned)one.batch * tiles, idx = at + run_start(total, -1, xcd);
            if (idx >= run_start(total, -1, xcd + 1)) return false;
            b = idx / tiles;
            tile = idx - b * tiles;
            if (sym) {
                split = one.split;
                const int whole = tile / split;
                part = tile - whole * split;
                slab = idx - part;
                tile = whole;
            }
            return true;
        }
        const int lane = threadIdx.x & 63;
        const unsigned first = sym ? t->fsym[xcd][lane] : t->fapp[xcd][lane];
        const int l_tiles = sym ? t->tsym[lane] : t->tapp[lane], l_home = sym ? t->hsym[lane] : t->happ[lane];
        const int l_np = t->np[lane], l_mp = t->mp[lane], l_xo = t->xo[lane], l_ao = t->ao[lane], l_dof = t->dof[lane], l_mat = t->mat[lane];
        const int l_batch = t->batch[lane], l_split = sym ? t->split[lane] : 1, l_lone = sym ? 0 : t->lone[lane];
        const unsigned l_slab = sym ? t->slab[lane] : 0u;
        gi = __builtin_amdgcn_readfirstlane(__popcll(__ballot(first <= at)) - 1);
        const unsigned tiles = __builtin_amdgcn_readlane(l_tiles, gi);
        const int home = __builtin_amdgcn_readlane(l_home, gi);
        np = __builtin_amdgcn_readlane(l_np, gi);
        mp = __builtin_amdgcn_readlane(l_mp, gi);
        lone = __builtin_amdgcn_readlane(l_lone, gi);
        xo = __builtin_amdgcn_readlane(l_xo, gi);
        ao = __builtin_amdgcn_readlane(l_ao, gi);
        dof = __builtin_amdgcn_readlane(l_dof, gi);
        mat = __builtin_amdgcn_readlane(l_mat, gi);
        const unsigned total = (unsigned)__builtin_amdgcn_readlane(l_batch, gi) * tiles;
        const unsigned idx = at - (unsigned)__builtin_amdgcn_readlane((int)first, gi) + run_start(total, home, xcd);
        if (idx >= run_start(total, home, xcd + 1)) return false;
        b = idx / tiles;
        tile = idx - b * tiles;
        if (sym) {
            split = __builtin_amdgcn_readlane(l_split, gi);
            const int whole = tile / split;
            part = tile - whole * split;
            slab = __builtin_amdgcn_readlane(l_slab, gi) + idx - part;
            tile = whole;
        }
        return true;
    }
};

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// What X_lo is multiplied with in the place of P = a + (P - a), whose product reads X_hi alone.  a leaves out (P - a) X_lo, which lies
// in the directions of large singular values: it is not amplified by later steps.  diag(P) comes nearer to P where P is almost a diagonal,
// but leaves out offdiag(P) X_lo, which later steps amplify by a each where singular values are small.  So: a, and diag(P) in
// the last two steps.  Rank 1, 64 x 768: 6e-4 (diag(P) throughout 9e-3); Gaussian 512 x 512: 8e-4 (a throughout 1.2e-3).
__host__ __device__ __forceinline__ bool low_by_a(int step, int steps) { return step < steps - 2; }

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

// ---- the matrix that is orthogonalised --------------------------------------------------------------------------------
// KIND 0 / 1: an fp32 / bf16 tensor; 2 / 3: the momentum direction from an fp32 / bf16 gradient arena
template <bool BF>
__device__ __forceinline__ void load8(const void* p, long long e, float (&v)[8]) {
    if (BF) {
        const bf16x8 b = *reinterpret_cast<const bf16x8*>((const bf16_t*)p + e);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = bf2f(b[j]);
    } else {
        load8f((const float*)p + e, v);
    }
}
template <bool BF>
__device__ __forceinline__ f32x4 load4(const void* p, long long e) {
    if (!BF) return *reinterpret_cast<const f32x4*>((const float*)p + e);
    const bf16x4 b = *reinterpret_cast<const bf16x4*>((const bf16_t*)p + e);
    return f32x4{bf2f(b[0]), bf2f(b[1]), bf2f(b[2]), bf2f(b[3])};
}
template <bool BF>
__device__ __forceinline__ float load1(const void* p, long long e) { return BF ? bf2f(((const bf16_t*)p)[e]) : ((const float*)p)[e]; }

__device__ __forceinline__ float momentum_of(const Muon& mu, float g, float v) { return mu.mu * v + g; }
__device__ __forceinline__ float direction_of(const Muon& mu, float g, float v) { return mu.nesterov ? g + mu.mu * v : v; }   // v: new

// sums of squares in 64 bits (an fp32 square overflows from 1.8e19 on and vanishes below 1e-23): one partial a workgroup.
// (The new momentum is not stored here: ortho_pack_kernel computes it again, and what this pass read may still be in the
// memory-side cache then.)
// A chunk of groups a launch; its first workgroup writes the table for the kernels behind it.  Bound by memory: ResNet-50's
// gradients and momentum (153 MB) 37 us.
template <int KIND>
__global__ void __launch_bounds__(1024) ortho_sqsum_kernel(const Chunk ch, const Muon mu, double* __restrict__ part, Table* __restrict__ t,
                                                           unsigned* __restrict__ counters, int slabs) {
    constexpr bool BF = KIND & 1;
    if (blockIdx.x == 0) {
        write_table(ch, t, counters, slabs);
        return;
    }
    const unsigned wg = blockIdx.x - 1 + ch.g[0].fin;
    const int lane = threadIdx.x & 63;
    const bool mine = lane < ch.n && ch.g[lane < CHUNK ? lane : 0].fin <= wg;
    const int gi = __builtin_amdgcn_readfirstlane(__popcll(__ballot(mine)) - 1);
    const Group& g = ch.g[gi];
    const long long numel = (long long)g.r * g.c;
    const unsigned idx = wg - g.fin;
    const int b = idx / g.parts, pi = idx - b * g.parts;
    const long long lo = (long long)pi * g.part_elems, hi = lo + g.part_elems < numel ? lo + g.part_elems : numel;
    double s = 0.0;
    if (KIND >= 2) {
        const long long end8 = lo + ((hi - lo) & ~7LL);
        for (long long e = lo + threadIdx.x * 8; e < end8; e += 8192) {
            float gr[8], v[8];
            load8<BF>(mu.g, g.sb + e, gr);
            load8f(mu.v + g.sb + e, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float u = direction_of(mu, gr[j], momentum_of(mu, gr[j], v[j]));
                s += (double)u * (double)u;
            }
        }
        if (threadIdx.x < hi - end8) {
            const long long e = g.sb + end8 + threadIdx.x;
            const float gr = load1<BF>(mu.g, e), u = direction_of(mu, gr, momentum_of(mu, gr, mu.v[e]));
            s += (double)u * (double)u;
        }
    } else if (g.flat) {
        const long long end8 = lo + ((hi - lo) & ~7LL);
        for (long long e = lo + threadIdx.x * 8; e < end8; e += 8192) {
            float u[8];
            load8<BF>(g.src, b * g.sb + e, u);
#pragma unroll
            for (int j = 0; j < 8; ++j) s += (double)u[j] * (double)u[j];
        }
        if (threadIdx.x < hi - end8) {
            const float u = load1<BF>(g.src, b * g.sb + end8 + threadIdx.x);
            s += (double)u * (double)u;
        }
    } else {
        for (long long e = lo + threadIdx.x; e < hi; e += 1024) {
            const unsigned i = (unsigned)e / (unsigned)g.c, j = (unsigned)e - i * (unsigned)g.c;
            const float u = load1<BF>(g.src, b * g.sb + (long long)i * g.rs + (long long)j * g.cs);
            s += (double)u * (double)u;
        }
    }
    __shared__ double red[16];
    s = wave_sum_d(s);
    if (lane == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double all = 0.0;
#pragma unroll
        for (int w = 0; w < 16; ++w) all += red[w];
        part[g.po + (unsigned)b * g.parts + pi] = all;
    }
}

// scale and further shift of a matrix of this norm: X in the workspace is 2^(12 + shift) X
__device__ __forceinline__ double inverse_of(double norm, float eps, int& shift) {
    shift = norm < (double)eps && norm > 0.0 ? ilogb((double)eps / norm) : 0;
    return ldexp((double)SC, shift) / (norm > (double)eps ? norm : (norm == norm ? (double)eps : norm));   // (a NaN stays one)
}

// hi + lo of the scaled, normalised matrix; one 64 x 64 tile of the padded workspace a workgroup.  A lane's 8 elements run along
// the source's rows in both orientations.  Bound by memory: ResNet-50 from bf16 (51 MB in, 102 MB out) 29 us; with its momentum
// (153 MB in, 204 MB out) 68 us.
template <int KIND>
__global__ void __launch_bounds__(256) ortho_pack_kernel(const Table* __restrict__ t, const Muon mu, const double* __restrict__ part, float eps,
                                                        int* __restrict__ ex, f16_t* __restrict__ xh, f16_t* __restrict__ xl) {
    constexpr bool BF = KIND & 1;
    __shared__ __attribute__((aligned(16))) float tile[64][68];
    __shared__ double red[4];
    const int gi = find_group(t->fio, blockIdx.x);
    const Group& g = t->g[gi];
    const bool turn = g.r > g.c;
    const int tn = g.np >> 6, tm = g.mp >> 6;
    const unsigned idx = blockIdx.x - t->fio[gi];
    const int b = idx / (tn * tm), ti = (idx - b * (tn * tm)) / tm, tj = idx - b * (tn * tm) - ti * tm;
    double s = 0.0;
    for (int k = threadIdx.x; k < g.parts; k += 256) s += part[g.po + (unsigned)b * g.parts + k];
    s = wave_sum_d(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    // the source: rows i0 .. i0 + 63, columns j0 .. j0 + 63
    const int i0 = (turn ? tj : ti) * 64, j0 = (turn ? ti : tj) * 64;
    const int x = (threadIdx.x & 7) * 8, y0 = threadIdx.x >> 3;
    float u[2][8];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int i = i0 + y0 + k * 32, j = j0 + x;
#pragma unroll
        for (int q = 0; q < 8; ++q) u[k][q] = 0.f;
        if (i >= g.r || j >= g.c) continue;
        const long long e = KIND >= 2 ? g.sb + (long long)i * g.c + j : b * g.sb + (long long)i * g.rs + (long long)j * g.cs;
        if (g.vec && j + 8 <= g.c) {
            if (KIND >= 2) {
                float v[8];
                load8<BF>(mu.g, e, u[k]);
                load8f(mu.v + e, v);
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    v[q] = momentum_of(mu, u[k][q], v[q]);
                    u[k][q] = direction_of(mu, u[k][q], v[q]);
                }
                *reinterpret_cast<f32x4*>(mu.v + e) = f32x4{v[0], v[1], v[2], v[3]};
                *reinterpret_cast<f32x4*>(mu.v + e + 4) = f32x4{v[4], v[5], v[6], v[7]};
            } else {
                load8<BF>(g.src, e, u[k]);
            }
        } else {
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                if (j + q >= g.c) continue;
                if (KIND >= 2) {
                    const float gr = load1<BF>(mu.g, e + q), v = momentum_of(mu, gr, mu.v[e + q]);
                    mu.v[e + q] = v;
                    u[k][q] = direction_of(mu, gr, v);
                } else {
                    u[k][q] = load1<BF>(g.src, e + (long long)q * g.cs);
                }
            }
        }
    }
    __syncthreads();
    int shift;
    const double inv = inverse_of(sqrt((red[0] + red[1]) + (red[2] + red[3])), eps, shift);
    if (ti == 0 && tj == 0 && threadIdx.x == 0) ex[g.mat + b] = shift;
    const long long base = (long long)g.xo * 64 + ((long long)b * g.np + ti * 64) * g.mp + tj * 64;
    if (turn) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int q = 0; q < 8; ++q) tile[x + q][y0 + k * 32] = (float)(u[k][q] * inv);
        __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int y = y0 + k * 32;
        f16x8 h, l;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const float v = turn ? tile[y][x + q] : (float)(u[k][q] * inv);
            h[q] = (f16_t)v;
            l[q] = (f16_t)(v - (float)h[q]);
        }
        *reinterpret_cast<f16x8*>(xh + base + (long long)y * g.mp + x) = h;
        *reinterpret_cast<f16x8*>(xl + base + (long long)y * g.mp + x) = l;
    }
}

// 8 consecutive elements of the result (row i from column j on, `live` of them inside) -> the output, or the weights (K23)
template <bool MUON>
__device__ __forceinline__ void store_result(const Group& g, const Muon& mu, int b, int i, int j, int live, float lr, float step, const float (&u)[8]) {
    if (MUON) {
        const long long e = g.sb + (long long)i * g.c + j;
        const float keep = 1.f - lr * mu.wd;
        if (g.vec && live == 8) {
            float w[8];
            load8f(mu.w + e, w);
            bf16x8 lo;
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                w[q] = w[q] * keep - step * u[q];
                lo[q] = f2bf(w[q]);
            }
            *reinterpret_cast<f32x4*>(mu.w + e) = f32x4{w[0], w[1], w[2], w[3]};
            *reinterpret_cast<f32x4*>(mu.w + e + 4) = f32x4{w[4], w[5], w[6], w[7]};
            if (mu.lowp) *reinterpret_cast<bf16x8*>(mu.lowp + e) = lo;
        } else {
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (q < live) {
                    const float w = mu.w[e + q] * keep - step * u[q];
                    mu.w[e + q] = w;
                    if (mu.lowp) mu.lowp[e + q] = f2bf(w);
                }
        }
    } else {
        bf16_t* o = g.dst + ((long long)b * g.r + i) * g.c + j;
        bf16x8 v;
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = f2bf(u[q]);
        if (live == 8 && (g.c & 7) == 0) {
            *reinterpret_cast<bf16x8*>(o) = v;
        } else {
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (q < live) o[q] = v[q];
        }
    }
}

// ---- products ---------------------------------------------------------------------------------------------------------
// Tiles of a matrix in bands of 8 rows, a band column by column: the tiles that an XCD works on at a time are about as many
// rows as columns.
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

// SQUARE = false: O, d of A = X X^T.  SQUARE = true: O, d of P = b A + c A^2 (diagonal: + a) from those of A.
// Only tiles on and below the diagonal are computed and written twice.  4096 x 8192: 166 and 100 us (tiles of 256, bound by the
// matrix pipe: 880 TFLOP/s in X X^T); 12 of 512 x 512: 8.6 and 9.8 us (432 tiles of 64, bound by the latency of their 8 stages).
template <int B, int W0, int W1, int NST, int KS, bool SQUARE, bool ONE>
__global__ void __launch_bounds__(KS * W0 * W1 * 64, B == 128 ? 4 : 2) ortho_sym_kernel(const Table* __restrict__ t, const Single one, const f16_t* __restrict__ in, const float* __restrict__ din,
                                                          f16_t* __restrict__ out, float* __restrict__ dout, const int* __restrict__ ex, int down,
                                                          float ca, float cb, float cc, float* __restrict__ slabs, unsigned* __restrict__ counters) {
    typedef TileMul<MulF16, B, B, W0, W1, NST, false, KS> M;
    __shared__ __attribute__((aligned(16))) unsigned char smem[M::LDS];
    Item<ONE> it;
    if (!it.find(t, one, true) || (SQUARE && it.part > 0)) return;
    const int np = it.np, lda = np, ld = SQUARE ? np : it.mp, b = it.b;
    const int each = SQUARE ? np / 64 : (ld / 64 + it.split - 1) / it.split, k0 = SQUARE ? 0 : it.part * each;
    const int stages = ld / 64 - k0 < each ? ld / 64 - k0 : each;
    int ti, tj;
    tri_tile(it.tile, (np + B - 1) / B, ti, tj);
    const long long ao = (long long)it.ao * 64 + (long long)b * np * lda;
    const f16_t* src = SQUARE ? in + ao : in + (long long)it.xo * 64 + (long long)b * np * ld;
    M m;
    m.run(smem, src + (long long)ti * B * ld + k0 * 64, ld * 2, np - ti * B, src + (long long)tj * B * ld + k0 * 64, ld * 2, np - tj * B, stages);
    const float* d = SQUARE ? din + it.dof + (long long)b * np : nullptr;
    const float unscale = SQUARE ? USC * USC : ldexpf(USC * USC, -2 * shift_of(ex, it.mat + b, down));
    f16_t* o = out + ao;
    float* dst = dout + it.dof + (long long)b * np;
    float* tile = reinterpret_cast<float*>(smem);
    bool joined = false;
    if constexpr (B == 64 && !SQUARE) {
        joined = it.split > 1;
        if (joined && !join_parts<float>(m, tile, slabs + (long long)it.slab * (B * B), counters + it.slab, it.part, it.split)) return;
    }
    // value (r, c) of the result from the product's
    auto value = [&](float v, int r, int c, float a, float dr, float dc) {
        v *= unscale;
        if (SQUARE) {
            a *= USC;
            v = r == c ? ca + cb * dc + cc * (v + dc * dc) : cb * a + cc * (v + (dr + dc) * a);
        }
        return v;
    };
#pragma unroll
    for (int pass = 0; pass < M::PASSES; ++pass) {
        if (M::PASSES > 1 && pass > 0) __syncthreads();
        if (!joined) m.to_lds(tile, pass);
        __syncthreads();
        // block (tj, ti): rows c, 8 of r a thread
        for (int k = threadIdx.x; k < M::ROWS * B / 8; k += M::THREADS) {
            const int s = k / (B / 8), q = (k % (B / 8)) * 2, c = tj * B + M::tile_row(s, pass), r = ti * B + q * 4;
            if (B > 64 && (c >= np || r >= np)) continue;
            const f32x4 v0 = M::at(tile, s, q), v1 = M::at(tile, s, q + 1);
            f16x8 av = {};
            f32x4 d0 = {}, d1 = {};
            float dc = 0.f;
            if (SQUARE) {
                av = *reinterpret_cast<const f16x8*>(src + (long long)c * ld + r);        // (A is symmetric)
                d0 = *reinterpret_cast<const f32x4*>(d + r);
                d1 = *reinterpret_cast<const f32x4*>(d + r + 4);
                dc = d[c];
            }
            f16x8 h;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float v = value(e < 4 ? v0[e & 3] : v1[e & 3], r + e, c, (float)av[e], e < 4 ? d0[e & 3] : d1[e & 3], dc);
                h[e] = r + e == c ? (f16_t)0.f : (f16_t)(v * SC);
                if (ti == tj && r + e == c) dst[c] = v;
            }
            *reinterpret_cast<f16x8*>(o + (long long)c * lda + r) = h;
        }
        if (ti == tj) continue;
        // block (ti, tj): 4 rows r x 8 of c a thread, 8 threads side by side along c
        for (int k = threadIdx.x; k < M::ROWS * B / 32; k += M::THREADS) {
            const int s = ((k & 7) + (k >> 3) % (M::ROWS / 64) * 8) * 8, q = (k >> 3) / (M::ROWS / 64);
            const int c = tj * B + M::tile_row(s, pass), r = ti * B + q * 4;
            if (B > 64 && (c >= np || r >= np)) continue;
            f32x4 v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = M::at(tile, s + e, q);
            f16x8 av[4] = {};
            f32x4 d0 = {}, d1 = {}, dr = {};
            if (SQUARE) {
#pragma unroll
                for (int i = 0; i < 4; ++i) av[i] = *reinterpret_cast<const f16x8*>(src + (long long)(r + i) * ld + c);
                d0 = *reinterpret_cast<const f32x4*>(d + c);
                d1 = *reinterpret_cast<const f32x4*>(d + c + 4);
                dr = *reinterpret_cast<const f32x4*>(d + r);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f16x8 h;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    h[e] = (f16_t)(value(v[e][i], r + i, c + e, (float)av[i][e], dr[i], e < 4 ? d0[e & 3] : d1[e & 3]) * SC);
                *reinterpret_cast<f16x8*>(o + (long long)(r + i) * lda + c) = h;
            }
        }
    }
}

// X' = pd X_hi + (pd or a) X_lo + offdiag(P) X_hi; tile: BF columns of X times BS rows of P.  FINAL 0: the next X; 1: the output; 2: the weights (K23).
// 4096 x 8192: 250 us (tiles of 256, bound by the matrix pipe: 1100 TFLOP/s); all of ResNet-50: 60 us (tiles of 128, bound by X's
// pairs, 204 MB in and out), 97 us where it writes the weights; 12 of 512 x 512: 12 us (768 tiles of 64, latency).
template <int BF, int BS, int W0, int W1, int NST, int KS, int FINAL, bool ONE>
__global__ void __launch_bounds__(KS * W0 * W1 * 64, BF == 128 ? 4 : 2) ortho_apply_kernel(const Table* __restrict__ t, const Single one, const Muon mu, const f16_t* __restrict__ P,
                                                            const float* __restrict__ pd, const f16_t* __restrict__ xh, const f16_t* __restrict__ xl,
                                                            f16_t* __restrict__ yh, f16_t* __restrict__ yl,
                                                            const int* __restrict__ ex, int down, int down1, int by_a, float ca) {
    typedef TileMul<MulF16, BF, BS, W0, W1, NST, true, KS> M;
    __shared__ __attribute__((aligned(16))) unsigned char smem[M::LDS];
    Item<ONE> it;
    if (!it.find(t, one, false)) return;
    const int np = it.np, mp = it.mp, b = it.b;
    int ti, tj;
    band_tile(it.tile, (np + BS - 1) / BS, (mp + BF - 1) / BF, ti, tj);
    const f16_t* A = P + (long long)it.ao * 64 + ((long long)b * np + ti * BS) * np;
    const long long xo = (long long)it.xo * 64 + (long long)b * np * mp;
    M m;
    m.run(smem, xh + xo + tj * BF, mp * 2, mp - tj * BF, A, np * 2, np - ti * BS, np / 64);
    const int e0 = shift_of(ex, it.mat + b, down), e1 = shift_of(ex, it.mat + b, down1);
    const float rescale = FINAL ? ldexpf(USC, -e0) : ldexpf(1.f, e1 - e0);
    const float* d = pd + it.dof + (long long)b * np;
    float* tile = reinterpret_cast<float*>(smem);
    const Group& g = t->g[it.gi];
    const bool turn = FINAL && g.r > g.c;
    float lr = 0.f, step = 0.f;
    if (FINAL == 2) {
        lr = mu.lr_scale ? mu.lr * *mu.lr_scale : mu.lr;
        step = lr * sqrtf(turn ? (float)g.r / (float)g.c : 1.f);
    }
#pragma unroll
    for (int pass = 0; pass < M::PASSES; ++pass) {
        if (M::PASSES > 1 && pass > 0) __syncthreads();
        m.to_lds(tile, pass);
        __syncthreads();
#pragma unroll 2
        for (int k = threadIdx.x; k < M::ROWS * BF / 8; k += M::THREADS) {
            const int s = k / (BF / 8), q = (k % (BF / 8)) * 2, r = ti * BS + M::tile_row(s, pass), c = tj * BF + q * 4;
            if ((BS > 64 && r >= np) || (BF > 64 && c >= mp)) continue;
            const long long at = xo + (long long)r * mp + c;
            const f16x8 h0 = *reinterpret_cast<const f16x8*>(xh + at), l0 = *reinterpret_cast<const f16x8*>(xl + at);
            const float dr = d[r], dl = by_a && !it.lone ? ca : dr;
            const f32x4 v0 = M::at(tile, s, q), v1 = M::at(tile, s, q + 1);
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = (dr * (float)h0[e] + dl * (float)l0[e] + (e < 4 ? v0[e & 3] : v1[e & 3]) * USC) * rescale;
            if (FINAL == 0) {
                f16x8 h, l;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    h[e] = (f16_t)v[e];
                    l[e] = (f16_t)(v[e] - (float)h[e]);
                }
                *reinterpret_cast<f16x8*>(yh + at) = h;
                *reinterpret_cast<f16x8*>(yl + at) = l;
            } else if (!turn) {
                if (r < g.r && c < g.c) store_result<FINAL == 2>(g, mu, b, r, c, g.c - c < 8 ? g.c - c : 8, lr, step, v);
            } else {
                M::put(tile, s, q, f32x4{v[0], v[1], v[2], v[3]});
                M::put(tile, s, q + 1, f32x4{v[4], v[5], v[6], v[7]});
            }
        }
        if (FINAL == 0 || !turn) continue;
        // a tall matrix: the tile's columns are the result's rows; 8 threads side by side along them
        __syncthreads();
#pragma unroll 1
        for (int k = threadIdx.x; k < M::ROWS * BF / 8; k += M::THREADS) {
            const int s = ((k & 7) + (k >> 3) % (M::ROWS / 64) * 8) * 8, f = (k >> 3) / (M::ROWS / 64);
            const int j = ti * BS + M::tile_row(s, pass), i = tj * BF + f;
            if (i >= g.r || j >= g.c) continue;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = M::at1(tile, s + e, f);
            store_result<FINAL == 2>(g, mu, b, i, j, g.c - j < 8 ? g.c - j : 8, lr, step, v);
        }
    }
}

// ---- small matrices: all steps in one launch ----------------------------------------------------------------------------
// One workgroup of 8 waves a matrix: np = NP padded rows, up to 128 CB columns.  X stays in registers in fp32 (in the layout of the
// products' results: wave w has the 16-column blocks w, w + 8, ..; a lane 4 columns of rows lane % 16 + 16 j), X_hi, O and
// P in LDS; pd X (lo: by a) is the accumulator that P X is added to.  What bounds it is latency: 64 x 64 takes 13 us here,
// and the tiles 17 launches of 5 us.
template <int NP, int CB, int KIND>
__global__ void __launch_bounds__(512, 2) ortho_small_kernel(const Chunk ch, const Muon mu, float ca, float cb, float cc, int steps, int fall, float eps) {
    constexpr bool BF = KIND & 1;
    constexpr int LDX = 128 * CB + 8, LDO = NP + 8, NS = NP / 16, GF = NS * NS / 8;      // GF: blocks of A a wave
    __shared__ __attribute__((aligned(16))) f16_t Xs[NP * LDX], Os[NP * LDO];
    __shared__ __attribute__((aligned(16))) float ds[NP], pds[NP];
    __shared__ double red[8];
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), fr = lane & 15, fq = lane >> 4;
    const bool mine = lane < ch.n && ch.g[lane < CHUNK ? lane : 0].fin <= blockIdx.x;
    const int gi = __builtin_amdgcn_readfirstlane(__popcll(__ballot(mine)) - 1);
    const Group g = ch.g[gi];
    const int b = blockIdx.x - g.fin;
    const bool turn = g.r > g.c;
    const int n = turn ? g.c : g.r, m = turn ? g.r : g.c;
    const int blocks = g.mp >> 4;
    // row r, columns c .. c + 3 of X in the source
    f32x4 x[CB][NS];
    double sq = 0.0;
    const long long rs = turn ? g.cs : g.rs, cs = turn ? g.rs : g.cs;
    const long long ar = turn ? 1 : g.c, ac = turn ? g.c : 1;             // the same strides in a dense array
#pragma unroll
    for (int k = 0; k < CB; ++k)
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            x[k][j] = f32x4{0.f, 0.f, 0.f, 0.f};
            const int r = j * 16 + fr, c = (wid + 8 * k) * 16 + fq * 4;
            if (r >= n) continue;
            if (!turn && g.vec) {                                         // (whole fours: the columns are a multiple of 8)
                if (c >= m) continue;
                f32x4 u;
                if (KIND >= 2) {
                    const long long at = g.sb + r * ar + c;
                    const f32x4 gr = load4<BF>(mu.g, at);
                    f32x4 v = *reinterpret_cast<const f32x4*>(mu.v + at);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        v[e] = momentum_of(mu, gr[e], v[e]);
                        u[e] = direction_of(mu, gr[e], v[e]);
                    }
                    *reinterpret_cast<f32x4*>(mu.v + at) = v;
                } else {
                    u = load4<BF>(g.src, b * g.sb + r * rs + c);
                }
                x[k][j] = u;
#pragma unroll
                for (int e = 0; e < 4; ++e) sq += (double)u[e] * (double)u[e];
                continue;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (c + e >= m) continue;
                float u;
                if (KIND >= 2) {
                    const long long at = g.sb + r * ar + (c + e) * ac;
                    const float gr = load1<BF>(mu.g, at), v = momentum_of(mu, gr, mu.v[at]);
                    mu.v[at] = v;
                    u = direction_of(mu, gr, v);
                } else {
                    u = load1<BF>(g.src, b * g.sb + r * rs + (c + e) * cs);
                }
                x[k][j][e] = u;
                sq += (double)u * (double)u;
            }
        }
    sq = wave_sum_d(sq);
    if (lane == 0) red[wid] = sq;
    __syncthreads();
    int shift;
    const double inv = inverse_of(sqrt(((red[0] + red[1]) + (red[2] + red[3])) + ((red[4] + red[5]) + (red[6] + red[7]))), eps, shift);
    auto put_x = [&]() {
#pragma unroll
        for (int k = 0; k < CB; ++k)
            if (wid + 8 * k < blocks)
#pragma unroll
                for (int j = 0; j < NS; ++j) {
                    f16x4 h;
#pragma unroll
                    for (int e = 0; e < 4; ++e) h[e] = (f16_t)x[k][j][e];
                    *reinterpret_cast<f16x4*>(Xs + (j * 16 + fr) * LDX + (wid + 8 * k) * 16 + fq * 4) = h;
                }
    };
#pragma unroll
    for (int k = 0; k < CB; ++k)
#pragma unroll
        for (int j = 0; j < NS; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[k][j][e] = (float)(x[k][j][e] * inv);
    put_x();
    __syncthreads();
    const int fi = wid * NS / 8, s0 = NP == 64 ? (wid & 1) * 2 : 0;          // this wave's blocks of A: row block fi, columns s0 .. s0 + GF - 1
#pragma unroll 1
    for (int step = 0; step < steps; ++step) {
        const int e0 = shift > step * fall ? shift - step * fall : 0, e1 = shift > (step + 1) * fall ? shift - (step + 1) * fall : 0;
        // A
        f32x4 acc[GF];
#pragma unroll
        for (int j = 0; j < GF; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int k0 = 0; k0 < g.mp; k0 += 32) {
            const f16x8 a = *reinterpret_cast<const f16x8*>(Xs + (fi * 16 + fr) * LDX + k0 + fq * 8);
#pragma unroll
            for (int j = 0; j < GF; ++j) {
                const f16x8 q = *reinterpret_cast<const f16x8*>(Xs + ((s0 + j) * 16 + fr) * LDX + k0 + fq * 8);
                acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, q, acc[j], 0, 0, 0);
            }
        }
        const int r0 = fi * 16 + fq * 4;
        const float unscale = ldexpf(USC * USC, -2 * e0);
        f32x4 av[GF];                                                         // A's values, rows r0 .. r0 + 3, column (s0 + j) 16 + fr
#pragma unroll
        for (int j = 0; j < GF; ++j) {
            const int c = (s0 + j) * 16 + fr;
            f16x4 h;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                av[j][e] = acc[j][e] * unscale;
                if (r0 + e == c) ds[c] = av[j][e];
                h[e] = r0 + e == c ? (f16_t)0.f : (f16_t)(av[j][e] * SC);
            }
            *reinterpret_cast<f16x4*>(Os + c * LDO + r0) = h;                 // (symmetric)
        }
        __syncthreads();
        // P
#pragma unroll
        for (int j = 0; j < GF; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k0 = 0; k0 < NP; k0 += 32) {
            const f16x8 a = *reinterpret_cast<const f16x8*>(Os + (fi * 16 + fr) * LDO + k0 + fq * 8);
#pragma unroll
            for (int j = 0; j < GF; ++j) {
                const f16x8 q = *reinterpret_cast<const f16x8*>(Os + ((s0 + j) * 16 + fr) * LDO + k0 + fq * 8);
                acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, q, acc[j], 0, 0, 0);
            }
        }
        const f32x4 dr = *reinterpret_cast<const f32x4*>(ds + r0);
        float dc[GF];
#pragma unroll
        for (int j = 0; j < GF; ++j) dc[j] = ds[(s0 + j) * 16 + fr];
        __syncthreads();
#pragma unroll
        for (int j = 0; j < GF; ++j) {
            const int c = (s0 + j) * 16 + fr;
            f16x4 h;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float v = acc[j][e] * (USC * USC), o = av[j][e];
                if (r0 + e == c) pds[c] = ca + cb * dc[j] + cc * (v + dc[j] * dc[j]);
                h[e] = r0 + e == c ? (f16_t)0.f : (f16_t)((cb * o + cc * (v + (dr[e] + dc[j]) * o)) * SC);
            }
            *reinterpret_cast<f16x4*>(Os + c * LDO + r0) = h;
        }
        __syncthreads();
        // X: D rows = columns of X, D columns = rows of P
        const float rescale = ldexpf(USC, e1 - e0);
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            const float pd = pds[j * 16 + fr] * SC, pl = low_by_a(step, steps) && n > 1 ? ca * SC : pd;
#pragma unroll
            for (int k = 0; k < CB; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[k][j][e] = pl * x[k][j][e] + (pd - pl) * (float)(f16_t)x[k][j][e];
                }
        }
#pragma unroll
        for (int h = 0; h < NP / 32; ++h) {
            f16x8 q[NS];
#pragma unroll
            for (int j = 0; j < NS; ++j) q[j] = *reinterpret_cast<const f16x8*>(Os + (j * 16 + fr) * LDO + h * 32 + fq * 8);
#pragma unroll
            for (int k = 0; k < CB; ++k) {
                if (wid + 8 * k >= blocks) continue;
                f16_t* at = Xs + (h * 32 + 8 * fq + ((lane >> 2) & 3)) * LDX + (wid + 8 * k) * 16 + 4 * (lane & 3);
                const f16x4 lo = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_half4_ptr)at));
                const f16x4 hi = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_half4_ptr)(at + 4 * LDX)));
                const f16x8 a = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                for (int j = 0; j < NS; ++j) x[k][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, q[j], x[k][j], 0, 0, 0);
            }
        }
#pragma unroll
        for (int k = 0; k < CB; ++k)
#pragma unroll
            for (int j = 0; j < NS; ++j) x[k][j] *= rescale;
        if (step == steps - 1) break;
        __syncthreads();
        put_x();
        __syncthreads();
    }
    const float scale = ldexpf(USC, -(shift > steps * fall ? shift - steps * fall : 0));
    float lr = 0.f, by = 0.f;
    if (KIND >= 2) {
        lr = mu.lr_scale ? mu.lr * *mu.lr_scale : mu.lr;
        by = lr * sqrtf(turn ? (float)g.r / (float)g.c : 1.f);
    }
#pragma unroll
    for (int k = 0; k < CB; ++k)
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            const int r = j * 16 + fr, c = (wid + 8 * k) * 16 + fq * 4;
            if (r >= n) continue;
            if (!turn && g.vec) {
                if (c >= m) continue;
                const long long at = (KIND >= 2 ? g.sb : (long long)b * g.r * g.c) + r * ar + c;
                bf16x4 o;
                if (KIND >= 2) {
                    f32x4 w = *reinterpret_cast<const f32x4*>(mu.w + at);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        w[e] = w[e] * (1.f - lr * mu.wd) - by * (x[k][j][e] * scale);
                        o[e] = f2bf(w[e]);
                    }
                    *reinterpret_cast<f32x4*>(mu.w + at) = w;
                    if (mu.lowp) *reinterpret_cast<bf16x4*>(mu.lowp + at) = o;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] = f2bf(x[k][j][e] * scale);
                    *reinterpret_cast<bf16x4*>(g.dst + at) = o;
                }
                continue;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (c + e >= m) continue;
                const long long at = r * ar + (c + e) * ac;
                const float u = x[k][j][e] * scale;
                if (KIND >= 2) {
                    const float w = mu.w[g.sb + at] * (1.f - lr * mu.wd) - by * u;
                    mu.w[g.sb + at] = w;
                    if (mu.lowp) mu.lowp[g.sb + at] = f2bf(w);
                } else {
                    g.dst[(long long)b * g.r * g.c + at] = f2bf(u);
                }
            }
        }
}

// ---- thin matrices: all steps on the Gram matrix ------------------------------------------------------------------------
// Up to 32 rows of any length.  X_k = Q_k X_0 with Q_k and A_k polynomials in A_0: A <- P A P, Q <- P Q on np x np matrices, so the
// long side is read twice and never iterated on: Gram matrix a chunk of columns a workgroup, all steps in one workgroup a matrix,
// result a chunk of columns a workgroup.  An error of A_0 grows by up to a^(2 steps) = 2.3e5 where a singular value vanishes, so A and Q are
// computed in fp64 (its matrix instruction); Q reaches a^steps = 485 with cancelling entries: the result's product is fp32.
// Bound by latency: of four launches, or of a workgroup's loads and fp64 products (ortho_few_kernel; which one: forms_of).
// Error against 64 bits: 1e-5 before the rounding to bf16.
typedef double f64x4 __attribute__((ext_vector_type(4)));

// value of X (before its scale) at row r, column c; STORE: the new momentum is stored
template <int KIND, bool STORE>
__device__ __forceinline__ float thin_value(const Group& g, const Muon& mu, int b, bool turn, int r, int c) {
    constexpr bool BF = KIND & 1;
    const int i = turn ? c : r, j = turn ? r : c;
    if (KIND >= 2) {
        const long long at = g.sb + (long long)i * g.c + j;
        const float gr = load1<BF>(mu.g, at), v = momentum_of(mu, gr, mu.v[at]);
        if (STORE) mu.v[at] = v;
        return direction_of(mu, gr, v);
    }
    return load1<BF>(g.src, b * g.sb + (long long)i * g.rs + (long long)j * g.cs);
}
__device__ __forceinline__ double thin_scale(const Group& g, const double* __restrict__ part, int b, float eps) {   // by one whole wave
    double s = 0.0;
    for (int k = threadIdx.x & 63; k < g.parts; k += 64) s += part[g.po + (unsigned)b * g.parts + k];
    const double norm = sqrt(wave_sum_d(s));
    return 1.0 / (norm > (double)eps ? norm : (norm == norm ? (double)eps : norm));
}

// slab [NP][NP] of X X^T over a chunk of columns.  A lane has 4 columns of a row; the e-th of all lanes are the reduction's 4
// values of one matrix instruction (the columns' order does not matter).  Its result: rows lane / 16 + 4 e, column lane % 16.
template <int NP, int KIND>
__global__ void __launch_bounds__(256) ortho_thin_gram_kernel(const Table* __restrict__ t, const Muon mu, const double* __restrict__ part, float eps,
                                                             double* __restrict__ slabs) {
    constexpr int NS = NP / 16;
    __shared__ double red[4][NP][NP + 2];
    const int gi = find_group(t->fio, blockIdx.x);
    const Group& g = t->g[gi];
    const bool turn = g.r > g.c;
    const int n = turn ? g.c : g.r, m = turn ? g.r : g.c, chunks = g.chunks, width = g.tcols;
    const unsigned idx = blockIdx.x - t->fio[gi];
    const int b = idx / chunks, c0 = (idx - b * chunks) * width, end = c0 + width < m ? c0 + width : m;
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, fr = lane & 15, fq = lane >> 4;
    const double scale = thin_scale(g, part, b, eps);
    f64x4 acc[NS][NS];
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int j = 0; j < NS; ++j) acc[i][j] = f64x4{0.0, 0.0, 0.0, 0.0};
    for (int k = c0 + wid * 16; k < end; k += 64) {
        f32x4 x[NS];
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = i * 16 + fr, c = k + fq * 4 + e;
                x[i][e] = r < n && c < end ? (float)(thin_value<KIND, false>(g, mu, b, turn, r, c) * scale) : 0.f;
            }
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int i = 0; i < NS; ++i)
#pragma unroll
                for (int j = 0; j <= i; ++j) acc[i][j] = __builtin_amdgcn_mfma_f64_16x16x4f64((double)x[i][e], (double)x[j][e], acc[i][j], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int j = 0; j <= i; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = i * 16 + fq + 4 * e, c = j * 16 + fr;
                red[wid][r][c] = acc[i][j][e];
                if (i != j) red[wid][c][r] = acc[i][j][e];
            }
    __syncthreads();
    double* out = slabs + (long long)blockIdx.x * NP * NP;
    for (int k = threadIdx.x; k < NP * NP; k += 256) {
        const int r = k / NP, c = k % NP;
        out[k] = (red[0][r][c] + red[1][r][c]) + (red[2][r][c] + red[3][r][c]);
    }
}

// C = M N for symmetric N, all [NP][NP + 2] in LDS; lower block triangle, mirrored (products of polynomials in A are symmetric).
// post(r, c, value) gives what is stored.
template <int NP, typename F>
__device__ __forceinline__ void thin_mul(const double (*M)[NP + 2], const double (*N)[NP + 2], double (*C)[NP + 2], F post) {
    constexpr int NS = NP / 16, BLOCKS = NS * (NS + 1) / 2;
    const int lane = threadIdx.x & 63, blk = threadIdx.x >> 6, fr = lane & 15, fq = lane >> 4;
    if (blk < BLOCKS) {
        const int i = blk > 0, j = blk > 1;
        f64x4 acc = {0.0, 0.0, 0.0, 0.0}, odd = acc;  // two sums: half the instruction's latency
#pragma unroll
        for (int k = 0; k < NP; k += 8) {
            acc = __builtin_amdgcn_mfma_f64_16x16x4f64(M[i * 16 + fr][k + fq], N[j * 16 + fr][k + fq], acc, 0, 0, 0);
            odd = __builtin_amdgcn_mfma_f64_16x16x4f64(M[i * 16 + fr][k + 4 + fq], N[j * 16 + fr][k + 4 + fq], odd, 0, 0, 0);
        }
        acc += odd;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = i * 16 + fq + 4 * e, c = j * 16 + fr;
            const double v = post(r, c, acc[e]);
            C[r][c] = v;
            if (i != j) C[c][r] = v;
        }
    }
    __syncthreads();
}

// All steps on np x np matrices in LDS: A holds A_0; returns which of Q holds their product.
template <int NP, typename Mat>
__device__ __forceinline__ int thin_steps_of(Mat& A, Mat& P, Mat& T, Mat* Q, float ca, float cb, float cc, int steps) {
    const double da = ca, db = cb, dc = cc;
    auto same = [](int, int, double v) { return v; };
    auto poly = [&](int r, int c, double v) { return db * A[r][c] + dc * v + (r == c ? da : 0.0); };
    thin_mul<NP>(A, A, Q[0], poly);
    int at = 0;
#pragma unroll 1
    for (int k = 1; k < steps; ++k) {
        // A <- P A P; P of the first step is Q
        const Mat& last = k == 1 ? Q[0] : P;
        thin_mul<NP>(A, last, T, same);
        thin_mul<NP>(last, T, A, same);
        thin_mul<NP>(A, A, P, poly);
        thin_mul<NP>(P, Q[at], Q[at ^ 1], same);
        at ^= 1;
    }
    return at;
}

template <int NP>
__global__ void __launch_bounds__(256) ortho_thin_steps_kernel(const Table* __restrict__ t, const double* __restrict__ slabs, float* __restrict__ Qout, float ca,
                                                              float cb, float cc, int steps) {
    typedef double Mat[NP][NP + 2];
    __shared__ Mat A, P, T, Q[2];
    const int gi = find_group(t->mat, blockIdx.x);
    const Group& g = t->g[gi];
    const int b = blockIdx.x - g.mat, chunks = g.chunks;
    const double* from = slabs + ((long long)g.fio + (long long)b * chunks) * NP * NP;
    for (int k = threadIdx.x; k < NP * NP; k += 256) {
        double s = 0.0;
#pragma unroll 8
        for (int i = 0; i < chunks; ++i) s += from[(long long)i * NP * NP + k];
        A[k / NP][k % NP] = s;
    }
    __syncthreads();
    const int at = thin_steps_of<NP>(A, P, T, Q, ca, cb, cc, steps);
    float* out = Qout + (long long)blockIdx.x * NP * NP;
    for (int k = threadIdx.x; k < NP * NP; k += 256) out[k] = (float)Q[at][k / NP][k % NP];
}

// result = Q X, columns k0, k0 + stride, .. (16 each) before `end`: D rows = columns of X (4 a lane), D columns = rows
template <int NP, int KIND>
__device__ __forceinline__ void thin_columns(const Group& g, const Muon& mu, int b, bool turn, const float (*Q)[NP + 4], double scale, int k0, int stride, int end) {
    constexpr int NS = NP / 16;
    const int n = turn ? g.c : g.r, lane = threadIdx.x & 63, fr = lane & 15, fq = lane >> 4;
    float lr = 0.f, by = 0.f;
    if (KIND >= 2) {
        lr = mu.lr_scale ? mu.lr * *mu.lr_scale : mu.lr;
        by = lr * sqrtf(turn ? (float)g.r / (float)g.c : 1.f);
    }
#pragma unroll 1
    for (int k = k0; k < end; k += stride) {
        f32x4 acc[NS];
        float x[NS][4];
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = i * 16 + fq * 4 + e, c = k + fr;
                x[i][e] = r < n && c < end ? (float)(thin_value<KIND, true>(g, mu, b, turn, r, c) * scale) : 0.f;
            }
        }
#pragma unroll
        for (int i = 0; i < NS; ++i) {
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                const f32x4 q = *reinterpret_cast<const f32x4*>(&Q[j * 16 + fr][i * 16 + fq * 4]);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i][e], q[e], acc[j], 0, 0, 0);
            }
        }
#pragma unroll
        for (int j = 0; j < NS; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = j * 16 + fr, c = k + fq * 4 + e;
                if (r >= n || c >= end) continue;
                const long long at = turn ? (long long)c * g.c + r : (long long)r * g.c + c;
                if (KIND >= 2) {
                    const float w = mu.w[g.sb + at] * (1.f - lr * mu.wd) - by * acc[j][e];
                    mu.w[g.sb + at] = w;
                    if (mu.lowp) mu.lowp[g.sb + at] = f2bf(w);
                } else {
                    g.dst[(long long)b * g.r * g.c + at] = f2bf(acc[j][e]);
                }
            }
    }
}

template <int NP, int KIND>
__global__ void __launch_bounds__(256) ortho_thin_apply_kernel(const Table* __restrict__ t, const Muon mu, const double* __restrict__ part, float eps,
                                                              const float* __restrict__ Qin) {
    __shared__ __attribute__((aligned(16))) float Q[NP][NP + 4];
    const int gi = find_group(t->fio, blockIdx.x);
    const Group& g = t->g[gi];
    const bool turn = g.r > g.c;
    const int m = turn ? g.r : g.c, chunks = g.chunks, width = g.tcols;
    const unsigned idx = blockIdx.x - t->fio[gi];
    const int b = idx / chunks, c0 = (idx - b * chunks) * width, end = c0 + width < m ? c0 + width : m;
    const float* from = Qin + ((long long)g.mat + b) * NP * NP;
    for (int k = threadIdx.x; k < NP * NP; k += 256) Q[k / NP][k % NP] = from[k];
    const double scale = thin_scale(g, part, b, eps);
    __syncthreads();
    thin_columns<NP, KIND>(g, mu, b, turn, Q, scale, c0 + (threadIdx.x >> 6) * 16, 64, end);
}

// The same in one launch, a workgroup of 8 waves a matrix: the Gram matrix of the values as they are (products of fp32 values are exact
// in fp64), whose trace is the square of the norm; all steps; the result from a second read.
template <int NP, int KIND>
__global__ void __launch_bounds__(512) ortho_few_kernel(const Chunk ch, const Muon mu, float ca, float cb, float cc, int steps, float eps) {
    constexpr int NS = NP / 16, W = 8, EL = (NP * NP + 511) / 512;
    typedef double Mat[NP][NP + 2];
    __shared__ Mat mats[W];                              // the waves' sums; then A, P, T, Q[2]
    __shared__ __attribute__((aligned(16))) float Qf[NP][NP + 4];
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), fr = lane & 15, fq = lane >> 4;
    const bool mine = lane < ch.n && ch.g[lane < CHUNK ? lane : 0].fin <= blockIdx.x;
    const int gi = __builtin_amdgcn_readfirstlane(__popcll(__ballot(mine)) - 1);
    const Group g = ch.g[gi];
    const int b = blockIdx.x - g.fin;
    const bool turn = g.r > g.c;
    const int n = turn ? g.c : g.r, m = turn ? g.r : g.c;
    f64x4 acc[NS][NS];
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int j = 0; j < NS; ++j) acc[i][j] = f64x4{0.0, 0.0, 0.0, 0.0};
    struct Cols { float x[NS][4]; };
    auto load = [&](int k) {
        Cols v;
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = i * 16 + fr, c = k + fq * 4 + e;
                v.x[i][e] = r < n && c < m ? thin_value<KIND, false>(g, mu, b, turn, r, c) : 0.f;
            }
        return v;
    };
    Cols now = load(wid * 16);
    for (int k = wid * 16; k < m; k += W * 16) {
        const Cols next = load(k + W * 16);              // (behind the end: zeros)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int i = 0; i < NS; ++i)
#pragma unroll
                for (int j = 0; j <= i; ++j) acc[i][j] = __builtin_amdgcn_mfma_f64_16x16x4f64((double)now.x[i][e], (double)now.x[j][e], acc[i][j], 0, 0, 0);
        now = next;
    }
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int j = 0; j <= i; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = i * 16 + fq + 4 * e, c = j * 16 + fr;
                mats[wid][r][c] = acc[i][j][e];
                if (i != j) mats[wid][c][r] = acc[i][j][e];
            }
    __syncthreads();
    double sum[EL];
#pragma unroll
    for (int q = 0; q < EL; ++q) {
        const int k = threadIdx.x + q * 512, r = k / NP, c = k % NP;
        sum[q] = 0.0;
        if (k < NP * NP)
#pragma unroll
            for (int w = 0; w < W; ++w) sum[q] += mats[w][r][c];
    }
    double trace = 0.0;
    if (lane < NP)
#pragma unroll
        for (int w = 0; w < W; ++w) trace += mats[w][lane][lane];
    const double norm = sqrt(wave_sum_d(trace)), scale = 1.0 / (norm > (double)eps ? norm : (norm == norm ? (double)eps : norm));
    __syncthreads();
    Mat& A = mats[0];
#pragma unroll
    for (int q = 0; q < EL; ++q) {
        const int k = threadIdx.x + q * 512;
        if (k < NP * NP) A[k / NP][k % NP] = sum[q] * scale * scale;
    }
    __syncthreads();
    const int at = thin_steps_of<NP>(A, mats[1], mats[2], mats + 3, ca, cb, cc, steps);
    for (int k = threadIdx.x; k < NP * NP; k += 512) Qf[k / NP][k % NP] = (float)mats[3 + at][k / NP][k % NP];
    __syncthreads();
    thin_columns<NP, KIND>(g, mu, b, turn, Qf, scale, wid * 16, W * 16, m);
}

// ---- host -------------------------------------------------------------------------------------------------------------
// one group as the callers describe it: 11 int64 values
struct Desc { long long src, sb, srs, scs, dst, db, drs, dcs, r, c, batch; };

// most workgroups of a launch: their threads are counted in 32 bits
constexpr long long most_wgs(int threads) { return 0xffffffffLL / threads; }

struct Plan {
    long long x_elems = 0, a_elems = 0, d_elems = 0, parts = 0, mats = 0;
    long long table = 0, xa_h = 0, xa_l = 0, xb_h = 0, xb_l = 0, o = 0, p = 0, d = 0, pd = 0, part = 0, ex = 0, bytes = 0;
    int thin = 0;                   // padded rows of the thin form, 0: not taken
    long long slabs = 0;            // thin form: of all chunks; tiles: of the parts of long sums
    long long slab = 0, cnt = 0;    // (tiles)
};

long long part_elems_of(long long numel) {
    long long e = (numel + PARTS - 1) / PARTS;
    e = (e + 8191) / 8192 * 8192;
    return e < 16384 ? 16384 : e;
}
long long pad64(long long v) { return (v + 63) / 64 * 64; }

// Padded rows of the thin form, or 0: some matrix has more than 32
int thin_rows(const Desc* q, int count) {
    long long most = 0;
    for (int i = 0; i < count; ++i) {
        const long long n = q[i].r < q[i].c ? q[i].r : q[i].c;
        if (n > most) most = n;
    }
    return most > 32 ? 0 : most > 16 ? 32 : 16;
}

// columns of a chunk: a 16-column block for each of a workgroup's waves, but 128 chunks at most
long long thin_cols(long long m) { return (m + 8191) / 8192 * 64; }

void tiles_of(const Desc* q, int count, int& sym, int& app);
long long splits_of(const Desc* q, int count, int sym, int* split);

bool plan_of(const Desc* q, int count, bool thin, Plan& pl) {
    if (count < 0 || count > MAXG || (count && !q)) return false;
    for (int i = 0; i < count; ++i) {
        const Desc& s = q[i];
        if (s.r <= 0 || s.c <= 0 || s.batch <= 0 || s.r >= (1LL << 30) || s.c >= (1LL << 30)) return false;
        const long long np = pad64(s.r < s.c ? s.r : s.c), mp = pad64(s.r < s.c ? s.c : s.r);
        if (s.batch > 0x7fffffffLL || np * mp >= (1LL << 30)) return false;        // (a matrix's byte offsets have 31 bits)
        pl.x_elems += s.batch * np * mp;
        pl.a_elems += s.batch * np * np;
        pl.d_elems += s.batch * np;
        pl.mats += s.batch;
        const long long pe = part_elems_of(s.r * s.c);
        pl.parts += s.batch * ((s.r * s.c + pe - 1) / pe);
        if (pl.x_elems > (1LL << 37) || pl.d_elems > 0x7fffffffLL || pl.parts >= most_wgs(1024) || pl.mats > most_wgs(512)) return false;
    }
    auto up = [](long long b) { return (b + 255) / 256 * 256; };
    long long at = 0;
    pl.table = at; at += up(sizeof(Table));
    if (thin && (pl.thin = thin_rows(q, count)) != 0) {
        for (int i = 0; i < count; ++i) {
            const long long m = q[i].r > q[i].c ? q[i].r : q[i].c, w = thin_cols(m);
            pl.slabs += q[i].batch * ((m + w - 1) / w);
        }
        if (pl.slabs > most_wgs(256)) return false;
        pl.part = at; at += up(pl.parts * 8);
        pl.o = at; at += up(pl.slabs * pl.thin * pl.thin * 8);
        pl.p = at; at += up(pl.mats * pl.thin * pl.thin * 4);
        pl.bytes = at;
        return true;
    }
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
    int sym, app, split[MAXG];
    tiles_of(q, count, sym, app);
    pl.slabs = splits_of(q, count, sym, split);
    pl.slab = at; at += up(pl.slabs * 64 * 64 * 4);
    pl.cnt = at; at += up(pl.slabs * 4);
    pl.bytes = at;
    return true;
}

// whether the source's rows (K23: the arenas', whose offsets are checked) can be read 8 elements at a time
bool vec_of(const Desc& s, int kind) {
    if (kind >= 2) return s.c % 8 == 0;
    return s.scs == 1 && s.srs % 8 == 0 && (s.batch == 1 || s.sb % 8 == 0) && ((uintptr_t)s.src & 15) == 0;
}

// XCDs for the groups' tiles, the costliest first: a group of more than a sixteenth of all cost is cut over all of them, another
// goes to the one with the least so far.  Returns the workgroups of the launch.
long long homes(Group* g, int count, bool sym, const double* cost) {
    double all = 0.0, load[8] = {};
    int order[MAXG];
    for (int i = 0; i < count; ++i) { all += cost[i]; order[i] = i; }
    for (int i = 1; i < count; ++i)
        for (int k = i; k > 0 && cost[order[k]] > cost[order[k - 1]]; --k) { const int s = order[k]; order[k] = order[k - 1]; order[k - 1] = s; }
    for (int k = 0; k < count; ++k) {
        int home = -1;
        if (cost[order[k]] * 16.0 <= all) {
            home = 0;
            for (int x = 1; x < 8; ++x) if (load[x] < load[home]) home = x;
            load[home] += cost[order[k]];
        }
        (sym ? g[order[k]].hsym : g[order[k]].happ) = home;
    }
    long long most = 0;
    for (int x = 0; x < 8; ++x) {
        long long items = 0;
        for (int i = 0; i < count; ++i) {
            const unsigned total = (unsigned)g[i].batch * (unsigned)(sym ? g[i].tsym : g[i].tapp);
            const int home = sym ? g[i].hsym : g[i].happ;
            items += run_start(total, home, x + 1) - run_start(total, home, x);
        }
        if (items > most) most = items;
    }
    return most * 8;
}

// The polynomial over [0, top], top = what the step before leaves (1 at first): the largest |f(s)| and |b s^2 + c s^4| (X and P
// have to stay in fp16's range) and |f(s) / s|, the most that X grows by - at the ends or where a derivative vanishes.
// False: out of range
bool range_of(double a, double b, double c, int steps, double& growth) {
    double top = 1.0;
    growth = 1.0;
    for (int k = 0; k < steps; ++k) {
        const double end = top * top;
        double l[4] = {0.0, end, 0.0, 0.0};                            // squares of the candidates
        double f = 0.0, p = 0.0, q = 0.0;
        const double root = 9.0 * b * b - 20.0 * a * c;               // f' = a + 3 b l + 5 c l^2
        if (c != 0.0) {
            if (root >= 0.0) { l[2] = (-3.0 * b + sqrt(root)) / (10.0 * c); l[3] = (-3.0 * b - sqrt(root)) / (10.0 * c); }
        } else if (b != 0.0) {
            l[2] = -a / (3.0 * b);
        }
        for (int i = 0; i < 4; ++i) {
            const double s = l[i] >= 0.0 && l[i] <= end ? l[i] : 0.0;
            f = fmax(f, sqrt(s) * fabs(a + b * s + c * s * s));
        }
        const double mid = c != 0.0 && -b / (2.0 * c) > 0.0 && -b / (2.0 * c) < end ? -b / (2.0 * c) : 0.0;
        p = fmax(fabs(b * end + c * end * end), fabs(b * mid + c * mid * mid));
        q = fmax(fmax(fabs(a), fabs(a + b * end + c * end * end)), fabs(a + b * mid + c * mid * mid));
        // (the products' roundings may pass the exact range by a little)
        if (!(f * 1.02 <= 8.0) || !(p * 1.02 <= 15.0) || !(end <= 15.0) || !(q <= 1024.0)) return false;
        growth = fmax(growth, q);
        top = f * 1.02 > 1.0 ? f * 1.02 : 1.0;
    }
    return true;
}
int growth_bits(float a, float b, float c, int steps) {
    double growth;
    return range_of(a, b, c, steps, growth) ? (int)ceil(log2(growth)) : 0;
}

// Whether the thin form serves these steps: the Gram matrix's rounding, 2^-53, grows by the square of what X grows by (3.4445 ^ 10 =
// 2^18 for five steps of the usual coefficients), and Q, rounded to fp32, by what X grows by (485)
bool thin_steps(float a, float b, float c, int steps) {
    double growth;
    return steps >= 1 && steps <= 64 && range_of(a, b, c, steps, growth) && steps * log2(growth) <= 10.0;
}

// Tile sizes of a call.  Larger tiles need less LDS and L2 traffic a product (256 CUs full: 64 x 64 650, 128 x 128 890, 256 x 256
// 1050 TFLOP/s), smaller ones fill the chip with less work.  Measured (us, 64 / 128 / 256): P X of 12 512 x 512 (768 tiles of 64)
// 12.3 / 14.2 / 25.6, of 2048 x 2048 (1024) 35 / 32 / 55, of all of ResNet-50 (6200) 75 / 65 / 72, of 4096 x 8192 (8192; 512
// of 256) 468 / 311 / 274; A and A^2 of ResNet-50 (880) 52 / 79 / 134, of 2048 x 2048 (528) 51 / 56 / 108, of two
// 2048 x 4096 and 1000 x 4096 (1192) 116 / 107 / 152, of 4096 x 8192 (2080; 136 of 256) 374 / 318 / 311.
// Tiles of 64 that have a CU each (up to 256) are computed by two groups of waves: 512 x 4608 alone 201 -> 182 us in all.
void tiles_of(const Desc* q, int count, int& sym, int& app) {
    long long s64 = 0, s256 = 0, a64 = 0, a256 = 0;
    for (int i = 0; i < count; ++i) {
        const long long n = q[i].r < q[i].c ? q[i].r : q[i].c, m = q[i].r < q[i].c ? q[i].c : q[i].r;
        const long long n64 = (n + 63) / 64, n256 = (n + 255) / 256;
        s64 += q[i].batch * n64 * (n64 + 1) / 2;
        s256 += q[i].batch * n256 * (n256 + 1) / 2;
        a64 += q[i].batch * n64 * ((m + 63) / 64);
        a256 += q[i].batch * n256 * ((m + 255) / 256);
    }
    sym = s256 >= 128 && s64 >= 12 * s256 ? 256 : (s64 >= 1100 ? 128 : 64);      // (12 of 16: the larger tiles are mostly filled)
    app = a256 >= 512 && a64 >= 12 * a256 ? 256 : (a64 >= 1024 ? 128 : 64);
}

// Parts of the tiles' sums in X X^T (tiles of 64); returns the parts of all tiles that have more than one.  A workgroup alone on
// its CU takes 0.15 us per 64 columns, the join 4 us and 0.3 us a part: sqrt(stages / 2) parts from 96 stages on, of at least a
// 512th of the launch's work each, and no more than leave each workgroup a CU of its own if the tiles do.  Measured, whole calls:
// 500 x 10000 281 -> 236 us, 128 x 20000 328 -> 166, 64 x 100000 1189 -> 226; shorter sums in parts of 16:
// 512 x 4608 185 -> 177, 1000 x 2048 164 -> 222, all of ResNet-50 597 -> 632.
long long splits_of(const Desc* q, int count, int sym, int* split) {
    long long tiles[MAXG], stages[MAXG], whole = 0, items = 0, slabs = 0;
    double all = 0.0;
    for (int i = 0; i < count; ++i) {
        const long long n64 = ((q[i].r < q[i].c ? q[i].r : q[i].c) + 63) / 64;
        tiles[i] = q[i].batch * (n64 * (n64 + 1) / 2);
        stages[i] = ((q[i].r < q[i].c ? q[i].c : q[i].r) + 63) / 64;
        whole += tiles[i];
        all += (double)tiles[i] * (double)stages[i];
    }
    for (int i = 0; i < count; ++i) {
        const double most = fmin(64.0, fmin(sqrt(0.5 * (double)stages[i]), 512.0 * (double)stages[i] / all));
        split[i] = sym == 64 && stages[i] >= 96 && most >= 2.0 ? (int)most : 1;
        items += tiles[i] * split[i];
    }
    while (whole <= 256 && items > 256) {
        int top = 0;
        for (int i = 1; i < count; ++i)
            if (split[i] > split[top]) top = i;
        --split[top];
        items -= tiles[top];
    }
    for (int i = 0; i < count; ++i) {
        const long long each = (stages[i] + split[i] - 1) / split[i];
        split[i] = (int)((stages[i] + each - 1) / each);               // none of them empty
        if (split[i] > 1) slabs += tiles[i] * split[i];
    }
    return slabs;
}

// Calls that ortho_small_kernel serves: every matrix of up to 64 rows (its shorter side) and 768 columns, or 128 and 384 (more
// do not fit the registers and, 128 rows, LDS).  Tiles against it: 64 x 576 79 -> 37 us, 64 x 768 80 -> 43, 128 x 384 85 -> 66, 1000 of 64 x 600
// 651 -> 169, 1000 of 128 x 384 832 -> 309.  All are computed in the largest's size, as each size is a launch that takes as long as its steps
// (64 x 64 1.8 us a step and 4.3, 64 x 576 4.9 and 12, 128 x 384 10.3 and 14): 64 x 147, 64 x 64, 64 x 576, 256 x 64 and 64 x 256 82 -> 36.  Returns 0: not served; else 8 * padded rows / 64 + the number
// of the least columns, 128, 256, ..
int all_small(const Desc* q, int count) {
    long long most = 0, wide = 0;
    for (int i = 0; i < count; ++i) {
        const long long n = q[i].r < q[i].c ? q[i].r : q[i].c, m = q[i].r < q[i].c ? q[i].c : q[i].r;
        most = n > most ? n : most;
        wide = m > wide ? m : wide;
    }
    if (most <= 64 && wide <= 768) return 8 + (wide <= 128 ? 0 : wide <= 256 ? 1 : wide <= 512 ? 2 : 3);
    if (most <= 128 && wide <= 384) return 16 + (wide <= 128 ? 0 : wide <= 256 ? 1 : 2);
    return 0;
}
template <int KIND>
int launch_small(int cls, const Chunk& ch, unsigned grid, const Muon& mu, float a, float b, float c, int steps, int fall, float eps, hipStream_t stream) {
#define SMALL(NP, CB) DDL_KLAUNCH((ortho_small_kernel<NP, CB, KIND>), dim3(grid), dim3(512), 0, stream, ch, mu, a, b, c, steps, fall, eps)
    switch (cls) {
        case 8: SMALL(64, 1); break;
        case 9: SMALL(64, 2); break;
        case 10: SMALL(64, 4); break;
        case 11: SMALL(64, 6); break;
        case 16: SMALL(128, 1); break;
        case 17: SMALL(128, 2); break;
        default: SMALL(128, 3); break;
    }
#undef SMALL
    return ddl_launch_status();
}
int run_small(const Desc* q, int count, int cls, int kind, const Muon& mu, float a, float b, float c, int steps, float eps, hipStream_t stream) {
    const int fall = growth_bits(a, b, c, steps);
    for (int base = 0; base < count; base += CHUNK) {
        Chunk ch;
        memset(&ch, 0, sizeof(ch));
        long long grid = 0;
        for (int i = base; i < count && i < base + CHUNK; ++i) {
            Group& o = ch.g[ch.n++];
            const Desc& s = q[i];
            o.src = (const void*)s.src; o.dst = (bf16_t*)s.dst; o.sb = s.sb; o.rs = (int)s.srs; o.cs = (int)s.scs;
            o.r = (int)s.r; o.c = (int)s.c; o.batch = (int)s.batch;
            o.vec = vec_of(s, kind) && s.c % 8 == 0;
            o.np = (int)pad64(s.r < s.c ? s.r : s.c); o.mp = (int)pad64(s.r < s.c ? s.c : s.r);
            o.fin = (unsigned)grid;
            grid += s.batch;
        }
        const int rc = kind == 0 ? launch_small<0>(cls, ch, (unsigned)grid, mu, a, b, c, steps, fall, eps, stream)
                     : kind == 1 ? launch_small<1>(cls, ch, (unsigned)grid, mu, a, b, c, steps, fall, eps, stream)
                     : kind == 2 ? launch_small<2>(cls, ch, (unsigned)grid, mu, a, b, c, steps, fall, eps, stream)
                                 : launch_small<3>(cls, ch, (unsigned)grid, mu, a, b, c, steps, fall, eps, stream);
        if (rc != DDL_OK) return rc;
    }
    return DDL_OK;
}

// matrices that ortho_few_kernel serves, whatever their number
int run_few(const Desc* q, int count, int kind, const Muon& mu, float a, float b, float c, int steps, float eps, hipStream_t stream) {
    const int rows = thin_rows(q, count);
    for (int base = 0; base < count; base += CHUNK) {
        Chunk ch;
        memset(&ch, 0, sizeof(ch));
        long long grid = 0;
        for (int i = base; i < count && i < base + CHUNK; ++i) {
            Group& o = ch.g[ch.n++];
            const Desc& s = q[i];
            o.src = (const void*)s.src; o.dst = (bf16_t*)s.dst; o.sb = s.sb; o.rs = (int)s.srs; o.cs = (int)s.scs;
            o.r = (int)s.r; o.c = (int)s.c; o.batch = (int)s.batch;
            o.fin = (unsigned)grid;
            grid += s.batch;
        }
        if (grid > most_wgs(512)) return DDL_EINVAL;
#define FEW(NP, K) DDL_KLAUNCH((ortho_few_kernel<NP, K>), dim3((unsigned)grid), dim3(512), 0, stream, ch, mu, a, b, c, steps, eps)
#define FEW1(K) { if (rows == 16) FEW(16, K); else FEW(32, K); }
        if (kind == 0) FEW1(0) else if (kind == 1) FEW1(1) else if (kind == 2) FEW1(2) else FEW1(3)
#undef FEW1
#undef FEW
        const int rc = ddl_launch_status();
        if (rc != DDL_OK) return rc;
    }
    return DDL_OK;
}

// A call's groups by form.  Up to 32 rows the fp16 products of the other forms would leave 1e-3 .. 3e-3 (few values to average over), so
// where the steps allow it (thin_steps) such matrices always run on their Gram matrix: `few` in one launch, `thin` in four that spread
// long rows over the chip.  Measured (us, few / thin): 16 x 64 8.5 / 15.7, 16 x 512 17 / 18, 16 x 1024 26 / 19, 32 x 256 23 / 28,
// 32 x 512 32 / 28, 64 of 16 x 2048 45 / 30, 1000 of 16 x 2048 128 / 212, 1000 of 32 x 8192 1370 / 2380: few up to 512 columns (above 16 rows
// 256) or where a stack has a matrix for each CU; the rest of a call's then share thin's launches.
// One row has no offdiagonal values: it is exact in every form and goes along with the others, if they are of one form.
struct Forms {
    Desc few[MAXG], thin[MAXG], rest[MAXG];
    int nfew = 0, nthin = 0, nrest = 0;
};
void forms_of(const Desc* q, int count, bool steps_fit, Forms& f) {
    bool gram = false, other = false, spread = false;
    for (int i = 0; i < count; ++i) {
        const long long n = q[i].r < q[i].c ? q[i].r : q[i].c, m = q[i].r < q[i].c ? q[i].c : q[i].r;
        gram = gram || (n > 1 && n <= 32);
        other = other || n > 32;
        spread = spread || (n <= 32 && q[i].batch < 256 && m > (n > 16 ? 256 : 512));
    }
    for (int i = 0; i < count; ++i) {
        const long long n = q[i].r < q[i].c ? q[i].r : q[i].c;
        if (!steps_fit || n > 32 || (n == 1 && other && !gram)) f.rest[f.nrest++] = q[i];
        else if (q[i].batch >= 256 || !spread) f.few[f.nfew++] = q[i];
        else f.thin[f.nthin++] = q[i];
    }
}

// the forms that have a table in the workspace: thin, or tiles; kind as in load8
int run_table(const Desc* q, int count, bool thin, int kind, const Muon& mu, float a, float b, float c, int steps, float eps, char* ws, hipStream_t stream) {
    Plan pl;
    if (!plan_of(q, count, thin, pl)) return DDL_EINVAL;
    int sb = 64, ab = 64, split[MAXG];
    tiles_of(q, count, sb, ab);
    splits_of(q, count, sb, split);
    long long slabs = 0, squares = 0;
    // the groups with the longest sums first
    int order[MAXG];
    for (int i = 0; i < count; ++i) order[i] = i;
    auto longer = [&](int i) { return q[i].r > q[i].c ? q[i].r : q[i].c; };
    for (int i = 1; i < count; ++i)
        for (int k = i; k > 0 && longer(order[k]) > longer(order[k - 1]); --k) { const int s = order[k]; order[k] = order[k - 1]; order[k - 1] = s; }
    Group g[MAXG];
    double csym[MAXG], capp[MAXG];
    long long nin = 0, nio = 0, nsym = 0, napp = 0, xo = 0, ao = 0, dof = 0, po = 0, mat = 0;
    for (int i = 0; i < count; ++i) {
        const Desc& s = q[order[i]];
        Group& o = g[i];
        const long long n = s.r < s.c ? s.r : s.c, m = s.r < s.c ? s.c : s.r, np = pad64(n), mp = pad64(m);
        const long long pe = part_elems_of(s.r * s.c), parts = (s.r * s.c + pe - 1) / pe;
        const long long sn = (np + sb - 1) / sb, an = (np + ab - 1) / ab, am = (mp + ab - 1) / ab;
        o.src = (const void*)s.src; o.dst = (bf16_t*)s.dst; o.sb = s.sb; o.rs = (int)s.srs; o.cs = (int)s.scs;
        o.r = (int)s.r; o.c = (int)s.c; o.np = (int)np; o.mp = (int)mp; o.batch = (int)s.batch;
        o.vec = vec_of(s, kind);
        o.flat = s.scs == 1 && s.srs == s.c && (s.batch == 1 || s.sb % 8 == 0) && ((uintptr_t)s.src & 15) == 0;
        o.part_elems = (int)pe; o.parts = (int)parts;
        o.xo = (unsigned)(xo / 64); o.ao = (unsigned)(ao / 64); o.dof = (unsigned)dof; o.po = (unsigned)po; o.mat = (unsigned)mat;
        const long long whole = sn * (sn + 1) / 2;
        o.tsym = (int)(whole * (pl.thin ? 1 : split[order[i]])); o.tapp = (int)(an * am);
        o.fin = (unsigned)nin; o.fio = (unsigned)nio;
        csym[i] = (double)s.batch * whole * (double)(np + mp + 512);      // (512: what a tile costs beside its sum)
        capp[i] = (double)s.batch * o.tapp * (double)(np + 512);
        if (pl.thin) {
            o.tcols = (int)thin_cols(m);
            o.chunks = (int)((m + o.tcols - 1) / o.tcols);
        } else {
            o.split = split[order[i]];
            o.slab = (unsigned)slabs;
            if (o.split > 1) slabs += s.batch * o.tsym;
        }
        squares += s.batch * whole;
        nin += s.batch * parts; nio += s.batch * (pl.thin ? o.chunks : (np / 64) * (mp / 64));
        nsym += s.batch * o.tsym; napp += s.batch * o.tapp;
        xo += s.batch * np * mp; ao += s.batch * np * np; dof += s.batch * np; po += s.batch * parts; mat += s.batch;
        if (nio > most_wgs(256) || nsym > most_wgs(512) || napp > most_wgs(512)) return DDL_EINVAL;
    }
    nsym = homes(g, count, true, csym);
    napp = homes(g, count, false, capp);
    if (nsym > most_wgs(512) || napp > most_wgs(512)) return DDL_EINVAL;
    const Single one = count == 1 ? Single{g[0].np, g[0].mp, g[0].batch, g[0].tsym, g[0].tapp, g[0].split, g[0].r == 1 || g[0].c == 1} : Single{};
    Table* t = (Table*)(ws + pl.table);
    f16_t *xh = (f16_t*)(ws + pl.xa_h), *xl = (f16_t*)(ws + pl.xa_l), *yh = (f16_t*)(ws + pl.xb_h), *yl = (f16_t*)(ws + pl.xb_l);
    f16_t *O = (f16_t*)(ws + pl.o), *P = (f16_t*)(ws + pl.p);
    float *d = (float*)(ws + pl.d), *pd = (float*)(ws + pl.pd);
    double* part = (double*)(ws + pl.part);
    int* ex = (int*)(ws + pl.ex);
    float* slab = (float*)(ws + pl.slab);
    unsigned* counters = (unsigned*)(ws + pl.cnt);
    const int fall = growth_bits(a, b, c, steps);
    for (int base = 0; base < count; base += CHUNK) {
        Chunk ch;
        ch.base = base;
        ch.n = count - base < CHUNK ? count - base : CHUNK;
        ch.last = base + CHUNK >= count;
        memcpy(ch.g, g + base, ch.n * sizeof(Group));
        memset(ch.g + ch.n, 0, (CHUNK - ch.n) * sizeof(Group));
        const dim3 grid((unsigned)((ch.last ? nin : g[base + CHUNK].fin) - g[base].fin) + 1);
#define SUMS(K) DDL_KLAUNCH(ortho_sqsum_kernel<K>, grid, dim3(1024), 0, stream, ch, mu, part, t, counters, (int)(pl.thin ? 0 : pl.slabs))
        if (kind == 0) SUMS(0); else if (kind == 1) SUMS(1); else if (kind == 2) SUMS(2); else SUMS(3);
#undef SUMS
    }
    if (pl.thin) {
        double* slabs = (double*)(ws + pl.o);
        float* Q = (float*)(ws + pl.p);
#define THIN1(NP, K)                                                                                                             \
        {                                                                                                                        \
            DDL_KLAUNCH((ortho_thin_gram_kernel<NP, K>), dim3((unsigned)nio), dim3(256), 0, stream, t, mu, part, eps, slabs);    \
            DDL_KLAUNCH(ortho_thin_steps_kernel<NP>, dim3((unsigned)mat), dim3(256), 0, stream, t, slabs, Q, a, b, c, steps);    \
            DDL_KLAUNCH((ortho_thin_apply_kernel<NP, K>), dim3((unsigned)nio), dim3(256), 0, stream, t, mu, part, eps, Q);       \
        }
#define THIN(K) { if (pl.thin == 16) THIN1(16, K) else THIN1(32, K) }
        if (kind == 0) THIN(0) else if (kind == 1) THIN(1) else if (kind == 2) THIN(2) else THIN(3)
#undef THIN
#undef THIN1
        return ddl_launch_status();
    }
#define PACK(K) DDL_KLAUNCH(ortho_pack_kernel<K>, dim3((unsigned)nio), dim3(256), 0, stream, t, mu, part, eps, ex, xh, xl)
    if (kind == 0) PACK(0); else if (kind == 1) PACK(1); else if (kind == 2) PACK(2); else PACK(3);
#undef PACK
    for (int k = 0; k < steps; ++k) {
        const int fin = k < steps - 1 ? 0 : (kind < 2 ? 1 : 2);
#define SYM(B, W0, W1, NST, KS, SQ, ONE, IN, DIN, OUTP, DOUT, DOWN) DDL_KLAUNCH((ortho_sym_kernel<B, W0, W1, NST, KS, SQ, ONE>), dim3((unsigned)nsym), dim3(KS * W0 * W1 * 64), 0, stream, t, one, IN, DIN, OUTP, DOUT, ex, DOWN, a, b, c, slab, counters)
#define SYM1(B, W0, W1, NST, KS, ONE) SYM(B, W0, W1, NST, KS, false, ONE, xh, (const float*)nullptr, O, d, k * fall)
#define SYM2(B, W0, W1, NST, KS, ONE) SYM(B, W0, W1, NST, KS, true, ONE, O, d, P, pd, 0)
#define APP1(B, W0, W1, NST, KS, FIN, ONE) DDL_KLAUNCH((ortho_apply_kernel<B, B, W0, W1, NST, KS, FIN, ONE>), dim3((unsigned)napp), dim3(KS * W0 * W1 * 64), 0, stream, t, one, mu, P, pd, xh, xl, yh, yl, ex, k * fall, (k + 1) * fall, low_by_a(k, steps), a)
#define APP(B, W0, W1, NST, KS, ONE) { if (fin == 0) APP1(B, W0, W1, NST, KS, 0, ONE); else if (fin == 1) APP1(B, W0, W1, NST, KS, 1, ONE); else APP1(B, W0, W1, NST, KS, 2, ONE); }
#define TILES64(ONE)                                                                                                         \
        {                                                                                                                    \
            if (sb == 64) {                                                                                                  \
                if (nsym <= 256) SYM1(64, 2, 2, 3, 2, ONE); else SYM1(64, 2, 2, 3, 1, ONE);                                  \
                if (squares <= 256) SYM2(64, 2, 2, 3, 2, ONE); else SYM2(64, 2, 2, 3, 1, ONE);                               \
            }                                                                                                                \
        }
        if (one.np) TILES64(true) else TILES64(false)
        if (sb == 128) {
            SYM1(128, 2, 4, 2, 1, false);
            SYM2(128, 2, 4, 2, 1, false);
        } else if (sb == 256) {
            SYM1(256, 2, 4, 2, 1, false);
            SYM2(256, 2, 4, 2, 1, false);
        }
        if (ab == 64 && one.np) { if (napp <= 256) APP(64, 2, 2, 3, 2, true) else APP(64, 2, 2, 3, 1, true) }
        else if (ab == 64) { if (napp <= 256) APP(64, 2, 2, 3, 2, false) else APP(64, 2, 2, 3, 1, false) }
        else if (ab == 128) APP(128, 2, 4, 2, 1, false)
        else APP(256, 2, 4, 2, 1, false)
        f16_t* s = xh; xh = yh; yh = s;
        s = xl; xl = yl; yl = s;
    }
    return ddl_launch_status();
}

int run_all(const Desc* q, int count, int kind, const Muon& mu, float a, float b, float c, int steps, float eps, char* ws, hipStream_t stream) {
    Forms f;
    forms_of(q, count, thin_steps(a, b, c, steps), f);
    int rc = DDL_OK;
    // (one after another in the stream: they share the workspace)
    if (f.nfew) rc = run_few(f.few, f.nfew, kind, mu, a, b, c, steps, eps, stream);
    if (rc == DDL_OK && f.nthin) rc = run_table(f.thin, f.nthin, true, kind, mu, a, b, c, steps, eps, ws, stream);
    if (rc == DDL_OK && f.nrest) {
        if (const int cls = all_small(f.rest, f.nrest)) rc = run_small(f.rest, f.nrest, cls, kind, mu, a, b, c, steps, eps, stream);
        else rc = run_table(f.rest, f.nrest, false, kind, mu, a, b, c, steps, eps, ws, stream);
    }
    return rc;
}

// -1: sizes out of range
long long workspace_of(const Desc* q, int count, float a, float b, float c, int steps) {
    Plan whole, gram;              // (of one form each: what either takes)
    if (!plan_of(q, count, true, gram) || !plan_of(q, count, false, whole)) return -1;
    Forms f;
    forms_of(q, count, thin_steps(a, b, c, steps), f);
    Plan thin, tiles;
    if (f.nthin && !plan_of(f.thin, f.nthin, true, thin)) return -1;
    if (f.nrest && !all_small(f.rest, f.nrest) && !plan_of(f.rest, f.nrest, false, tiles)) return -1;
    return thin.bytes > tiles.bytes ? thin.bytes : tiles.bytes;
}

bool strides_fit(long long rs, long long cs) { return rs >= 0 && cs >= 0 && rs < (1LL << 31) && cs < (1LL << 31); }

}  // namespace

extern "C" int ddl_ortho_max_groups() { return MAXG; }

// 1 when the steps keep every operand in the range of scaled fp16 (see range_of)
extern "C" int ddl_ortho_coefficients_ok(float a, float b, float c, int steps) {
    double growth;
    return isfinite(a) && isfinite(b) && isfinite(c) && steps >= 1 && steps <= 64 && range_of(a, b, c, steps, growth);
}

// bytes of workspace of a call with these groups (`desc`: count x 11 int64: source address, its batch / row / column
// strides, destination address and strides, rows, columns, matrices) and steps, 0: none, -1: sizes out of range
extern "C" long long ddl_ortho_workspace(const long long* desc, int count, float a, float b, float c, int steps) {
    return workspace_of((const Desc*)desc, count, a, b, c, steps);
}

// kind 0 / 1: fp32 / bf16 sources; destinations are dense bf16 (other strides are refused)
extern "C" int ddl_orthogonalize(const long long* desc, int count, int kind, float a, float b, float c, int steps, float eps, void* ws,
                                 long long ws_bytes, hipStream_t stream) {
    if (count == 0) return DDL_OK;
    const Desc* q = (const Desc*)desc;
    const long long need = workspace_of(q, count, a, b, c, steps);
    if (kind < 0 || kind > 1 || need < 0 || ws_bytes < need || (need > 0 && !ws)) return DDL_EINVAL;
    if (!ddl_ortho_coefficients_ok(a, b, c, steps) || !(eps >= 1e-30f && eps <= 3.1e38f)) return DDL_EINVAL;
    if (reinterpret_cast<uintptr_t>(ws) & 255) return DDL_EALIGN;
    for (int i = 0; i < count; ++i)
        if (!q[i].src || !q[i].dst || !strides_fit(q[i].srs, q[i].scs) || q[i].sb < 0 || q[i].drs != q[i].c || q[i].dcs != 1 ||
            (q[i].batch > 1 && q[i].db != q[i].r * q[i].c))
            return DDL_EINVAL;
    for (int i = 0; i < count; ++i)
        if (!ddl_aligned16((const void*)q[i].dst)) return DDL_EALIGN;
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
    const Desc* q = (const Desc*)desc;
    const long long need = workspace_of(q, count, a, b, c, steps);
    if (!w || !g || !v || need < 0 || ws_bytes < need || (need > 0 && !ws)) return DDL_EINVAL;
    if (!ddl_ortho_coefficients_ok(a, b, c, steps) || !(eps >= 1e-30f && eps <= 3.1e38f)) return DDL_EINVAL;
    if ((reinterpret_cast<uintptr_t>(ws) & 255) || !ddl_aligned16(w) || !ddl_aligned16(g) || !ddl_aligned16(v) || (lowp && !ddl_aligned16(lowp)))
        return DDL_EALIGN;
    for (int i = 0; i < count; ++i)
        if (q[i].batch != 1 || q[i].sb < 0 || q[i].sb % 8) return DDL_EINVAL;
    Muon m;
    m.g = g; m.v = (float*)v; m.w = (float*)w; m.lowp = (bf16_t*)lowp;
    m.lr = lr; m.mu = mu; m.wd = wd; m.nesterov = nesterov; m.lr_scale = (const float*)lr_scale;
    return run_all(q, count, grad_is_bf16 ? 3 : 2, m, a, b, c, steps, eps, (char*)ws, stream);
}
