// Tile product on the matrix pipe, shared by the kernels whose operands are rows of 16-bit or 8-bit values (gfx950).
//
// D = F S^T: W0 x W1 waves, a BF x BS tile, NST stages of 128 bytes of every row (64 fp16 or 128 int8 values) filled by LDS-DMA
// (64-byte pieces fetched each line twice), counted waits, one barrier a stage.
//   S and, with TRF = false, F: row-major, k-contiguous rows.  16-byte chunk c of row r lies at c ^ (r / 2 mod 8): the 16 rows x
//   one chunk that a quarter of a wave reads are free of bank conflicts.
//   TRF = true (fp16): F is given transposed, [k][columns].  Its rows of k stay as they are in LDS and are read by the transposing
//   load: 16 lanes take 4 rows x 16 columns; a half-wave touches rows 0-3 and 8-11 (+ 4, + 16), whose 32-byte windows
//   the swizzle spreads over all banks.
// A lane ends with D[i][j][e]: F index 16 i + 4 (lane / 16) + e, S index 16 j + lane % 16 of its wave's part.
#pragma once
#include "common.h"

typedef _Float16 f16_t;
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

namespace {

typedef __fp16 half4 __attribute__((ext_vector_type(4)));      // (the type that the transposing load is declared with)
typedef __attribute__((address_space(3))) half4* lds_half4_ptr;
// Whether the scalar offset of a buffer load counts in its range check is left open here: every descriptor has the same range, longer than
// any sum of both offsets; lanes that must not read have OUT as their own offset, behind that range (zeros); all others are inside
// their array.
constexpr unsigned OUT = 0x80000000u, DESC_BYTES = OUT - 16;

__device__ __forceinline__ int nt_off(int row, int ch) { return row * 128 + ((ch ^ ((row >> 1) & 7)) << 4); }
template <int B>
__host__ __device__ __forceinline__ int tr_swz(int row) {
    return B >= 128 ? (row & 3) | ((row >> 1) & 4) : ((row >> 1) & 1) | ((row >> 2) & 2);
}

struct MulF16 {
    typedef f16x8 frag;
    typedef f32x4 acc;
    static constexpr bool CUT = false;         // rows of f are whole stages
    static __device__ __forceinline__ acc mma(frag a, frag b, acc c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
struct MulI8 {
    typedef i32x4 frag;
    typedef i32x4 acc;
    static constexpr bool CUT = true;          // rows of f are the caller's: they end inside the last stage
    static __device__ __forceinline__ acc mma(frag a, frag b, acc c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
};

// Stages of a group of waves: it issues the loads of `count`, of which `live` exist and `last` (if any) is the sum's last one.
struct Stages { int first, count, live, last; };
__host__ __device__ __forceinline__ Stages stages_of(int total, int ks, int group) {
    if (ks == 1) return Stages{0, total, total, total - 1};
    const int half = (total + 1) >> 1;                  // (the second group may have a stage less)
    return group ? Stages{half, half, total - half, total - 1 - half} : Stages{0, half, half, total - 1};
}

// KS = 2: two such groups of waves with stages of their own take half of the sum each and are added at the end - a tile
// that has a CU to itself is bound by the latency of its stages, one after another, not by their bytes.
template <typename OP, int BF, int BS, int W0, int W1, int NST, bool TRF, int KS = 1>
struct TileMul {
    typedef typename OP::frag frag;
    typedef typename OP::acc vec;
    static constexpr int WAVES = W0 * W1, THREADS = KS * WAVES * 64, TILE = BF * BS;
    static constexpr int FBYTES = BF * 128, SBYTES = BS * 128, STAGE = FBYTES + SBYTES, LDS = KS * NST * STAGE;
    static constexpr int FL = BF / 8 / WAVES, SL = BS / 8 / WAVES, L = FL + SL;         // LDS-DMA instructions of a wave and stage
    static constexpr int NF = BF / W0 / 16, NS = BS / W1 / 16;                          // fragments of a wave
    static_assert(FL * 8 * WAVES == BF && SL * 8 * WAVES == BS, "whole instructions");
    static_assert(NST >= 2 && LDS <= 160 * 1024 && KS <= 2, "LDS");
    vec acc[NF][NS];

    static __device__ __forceinline__ u32x4 uniform(u32x4 r) {               // (it is: tells the compiler so)
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = __builtin_amdgcn_readfirstlane(r[i]);
        return r;
    }
    // The lane's offset of a wave's i-th load of f and of s (the same in every stage), and what is or-ed to f's in the last stage: OUT
    // where the 16 bytes begin at or behind byte `fend` of the stage's 128 (the swizzle has whole turns in WAVES * 8 rows: any i).
    static __host__ __device__ __forceinline__ unsigned f_offset(int i, int wid, int lane, unsigned ldf, int fleft) {
        const int slot = (i * WAVES + wid) * 64 + lane;
        if (TRF) {
            constexpr int CPR = BF / 8;
            const int row = slot / CPR, ch = slot % CPR, c = (((ch >> 1) ^ tr_swz<BF>(row)) << 1) | (ch & 1);
            return c * 8 < fleft ? row * ldf + c * 16 : OUT;
        }
        const int row = slot >> 3, c = (slot & 7) ^ ((row >> 1) & 7);
        return row < fleft ? row * ldf + c * 16 : OUT;
    }
    static __host__ __device__ __forceinline__ unsigned s_offset(int i, int wid, int lane, unsigned lds, int sleft) {
        const int slot = (i * WAVES + wid) * 64 + lane, row = slot >> 3, c = (slot & 7) ^ ((row >> 1) & 7);
        return row < sleft ? row * lds + c * 16 : OUT;
    }
    static __host__ __device__ __forceinline__ unsigned f_behind(int wid, int lane, int fend) {
        static_assert(WAVES % 2 == 0, "swizzle");
        const int slot = wid * 64 + lane, c = (slot & 7) ^ ((slot >> 4) & 7);
        return c * 16 < fend ? 0u : OUT;
    }
    // f: first row (TRF: first column) of the tile, ldf bytes from a row to the next, fleft rows (columns) that exist (behind them:
    // zeros), of which the last stage is read up to byte `fend` (a multiple of 16; OP::CUT: behind it zeros, else 128); s likewise, in
    // whole stages; `total` stages.  All offsets < 2^31 - 16.
    __device__ __forceinline__ void run(unsigned char* smem, const void* f, unsigned ldf, int fleft, const void* s, unsigned lds, int sleft, int total,
                                        int fend = 128) {
        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wid = wave % WAVES, w0 = wid / W1, w1 = wid % W1;
        const Stages mine = stages_of(total, KS, wave / WAVES);
        const int KT = mine.count, live = mine.live;
        if (KS == 2 && wave >= WAVES) {
            smem += NST * STAGE;
            f = (const char*)f + (size_t)mine.first * (TRF ? ldf * 64u : 128u);
            s = (const char*)s + (size_t)mine.first * 128u;
        }
        const int fr = lane & 15, fq = lane >> 4;
        const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) void*)smem;
        unsigned vo[L];
#pragma unroll
        for (int i = 0; i < FL; ++i) vo[i] = f_offset(i, wid, lane, ldf, fleft);
#pragma unroll
        for (int i = 0; i < SL; ++i) vo[FL + i] = s_offset(i, wid, lane, lds, sleft);
        const unsigned cut = OP::CUT ? f_behind(wid, lane, fend) : 0u;
        const u32x4 rf = uniform(raw_rsrc(f, DESC_BYTES)), rs = uniform(raw_rsrc(s, DESC_BYTES));
        const unsigned fstep = TRF ? ldf * 64u : 128u;                         // bytes from a tile to the next
        // every stage is exactly L instructions a wave (behind the end: the last tile again): the counted waits rely on it
        auto piece = [&](unsigned kt, unsigned at, int i) {                    // at: LDS address of the wave's part of the stage
            unsigned o = KS == 1 || (int)kt < live ? vo[i] : OUT;              // (a stage that the second group does not have: zeros)
            if (OP::CUT && i < FL && (int)kt == mine.last) o |= cut;
            if (i < FL) lds_dma16(rf, at + i * WAVES * 1024, o, kt * fstep);
            else lds_dma16(rs, at + FBYTES + (i - FL) * WAVES * 1024, o, kt * 128u);
        };
        // a fragment's offset in a stage, half h: i-th of f at fbase[h] + 2048 i (TRF: foff[i] + 64 BF h), of s at sbase[h] + 2048 j
        int fbase[2], sbase[2], foff[NF];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            fbase[h] = nt_off(w0 * (BF / W0) + fr, h * 4 + fq);
            sbase[h] = FBYTES + nt_off(w1 * (BS / W1) + fr, h * 4 + fq);
        }
        const int trow = 8 * fq + ((lane >> 2) & 3);
#pragma unroll
        for (int i = 0; i < NF; ++i) foff[i] = trow * (BF * 2) + (((w0 * NF + i) ^ tr_swz<BF>(trow)) * 32) + 8 * (lane & 3);
        auto read_f = [&](unsigned char* st, int h, int i) -> frag {
            if constexpr (!TRF) {
                return *reinterpret_cast<const frag*>(st + fbase[h] + i * 2048);
            } else {
            // (row + 4 has the swizzle of row: bit 2 of the row takes no part in it; nor does bit 5)
            unsigned char* p = st + foff[i] + h * (BF * 64);
            const f16x4 lo = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_half4_ptr)p));
            const f16x4 hi = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_half4_ptr)(p + 4 * BF * 2)));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            }
        };
        auto read_s = [&](unsigned char* st, int h, int j) -> frag { return *reinterpret_cast<const frag*>(st + sbase[h] + j * 2048); };
#pragma unroll
        for (int i = 0; i < NF; ++i)
#pragma unroll
            for (int j = 0; j < NS; ++j) acc[i][j] = vec{0, 0, 0, 0};

        // The fragments of the next half are read while a half is multiplied: s into a second set of registers, each of f into
        // its own behind its last use.  A stage is free once both halves are in registers: behind the barrier that ends
        // the first one, tile t + NST goes where tile t was.  (Higher priority around the products: 256 x 256 in 8 waves, where
        // two waves of one workgroup share a SIMD, 271 -> 260 us for 4096 x 4096 x 8192; 128 x 128 loses 5 %.)
        const unsigned at0 = lds0 + wid * 1024;
#pragma unroll
        for (int k = 0; k < NST; ++k)
#pragma unroll
            for (int i = 0; i < L; ++i) piece(k < KT ? k : KT - 1, at0 + k * STAGE, i);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NST - 1) * L) : "memory");
        __builtin_amdgcn_s_barrier();
        frag a[NF], b0[NS], b1[NS];
#pragma unroll
        for (int j = 0; j < NS; ++j) b0[j] = read_s(smem, 0, j);
#pragma unroll
        for (int i = 0; i < NF; ++i) a[i] = read_f(smem, 0, i);
        int cur = 0;                               // offset of tile kt's stage
        for (int kt = 0; kt < KT; ++kt) {
            unsigned char* st = smem + cur;
#pragma unroll
            for (int j = 0; j < NS; ++j) b1[j] = read_s(st, 1, j);
#pragma unroll
            for (int i = 0; i < NF; ++i) {
                if (WAVES == 8) __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int j = 0; j < NS; ++j) acc[i][j] = OP::mma(a[i], b0[j], acc[i][j]);
                if (WAVES == 8) __builtin_amdgcn_s_setprio(0);
                a[i] = read_f(st, 1, i);
            }
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NST - 2) * L) : "memory");
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            const int ns = cur + STAGE == NST * STAGE ? 0 : cur + STAGE;
            const unsigned next = kt + NST < KT ? kt + NST : KT - 1;
            unsigned char* sn = smem + ns;
#pragma unroll
            for (int j = 0; j < NS; ++j) b0[j] = read_s(sn, 0, j);
#pragma unroll
            for (int i = 0; i < NF; ++i) {
                if (WAVES == 8) __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int j = 0; j < NS; ++j) acc[i][j] = OP::mma(a[i], b1[j], acc[i][j]);
                if (WAVES == 8) __builtin_amdgcn_s_setprio(0);
                a[i] = read_f(sn, 0, i);
#pragma unroll
                for (int q = i * L / NF; q < (i + 1) * L / NF; ++q) piece(next, at0 + cur, q);
                __builtin_amdgcn_sched_barrier(0);
            }
            cur = ns;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();              // the LDS is the epilogue's from here
    }

    // The epilogues go through LDS (32-bit values, rows of S, 16-byte chunk q of row s at q ^ fold(s)): whole rows are read back and
    // written, and their loops stay rolled - a tile's code runs once, so its length is paid for in instruction fetches
    // (an unrolled epilogue of 8 KB took 4 us).  PASSES parts of BS / PASSES rows where the tile is larger than the stages.
    static constexpr int PASSES = BF * BS * 4 > LDS ? BF * BS * 4 / LDS : 1;
    static_assert(NS % PASSES == 0 && (KS == 1 || PASSES == 1), "whole fragments a pass");
    static constexpr int ROWS = BS / PASSES;       // rows of a pass: those of fragments j with j / (NS / PASSES) == pass of every wave
    __device__ __forceinline__ void to_lds(void* t, int pass) const {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wid = wave % WAVES, w0 = wid / W1, w1 = wid % W1;
        const int s0 = w1 * (ROWS / W1) + (lane & 15), f0 = w0 * (BF / W0 / 4) + (lane >> 4);
        auto place = [&](int i, int j) { return reinterpret_cast<vec*>((unsigned*)t + (s0 + j * 16) * BF + (((f0 + i * 4) ^ fold(s0 + j * 16)) * 4)); };
        if (KS == 2) {
            if (wave >= WAVES) {
#pragma unroll
                for (int j = 0; j < NS; ++j)
#pragma unroll
                    for (int i = 0; i < NF; ++i) *place(i, j) = acc[i][j];
            }
            __syncthreads();
            if (wave >= WAVES) return;
        }
#pragma unroll
        for (int p = 0; p < PASSES; ++p)
            if (p == pass)
#pragma unroll
                for (int j = 0; j < NS / PASSES; ++j)
#pragma unroll
                    for (int i = 0; i < NF; ++i) {
                        if (KS == 2) *place(i, j) += acc[i][j];
                        else *place(i, j) = acc[i][p * (NS / PASSES) + j];
                    }
    }
    static __device__ __forceinline__ int fold(int s) { return (s ^ (s >> 3)) & 15; }     // rows 1 apart and rows 8 apart on different banks
    // row of the tile that row `s` of a pass holds
    static __device__ __forceinline__ int tile_row(int s, int pass) { return (s / (ROWS / W1)) * (BS / W1) + pass * (ROWS / W1) + s % (ROWS / W1); }
    static __device__ __forceinline__ void put(float* t, int s, int q, f32x4 v) { *reinterpret_cast<f32x4*>(t + s * BF + ((q ^ fold(s)) * 4)) = v; }
    static __device__ __forceinline__ float at1(const float* t, int s, int f) { return t[s * BF + (((f >> 2) ^ fold(s)) * 4) + (f & 3)]; }
    static __device__ __forceinline__ vec at(const void* t, int s, int q) { return *reinterpret_cast<const vec*>((const unsigned*)t + s * BF + ((q ^ fold(s)) * 4)); }
};

// A part of a tile's sum.  The workgroup that ends last adds the parts, in their order, into LDS (as to_lds leaves them) and
// returns true; the others are done.  The parts pass from XCD to XCD by stores and loads of the device's scope, each wave waiting
// for its stores before the counter is raised (a fence would write back and empty a whole L2: 316 us in the place of 177 for
// an orthogonalisation of 512 x 4608).  `slabs`: `split` tiles; `counter`: zero, and zero again afterwards.
template <typename V, typename M>
__device__ __forceinline__ bool join_parts(const M& m, void* tile, V* slabs, unsigned* counter, int part, int split) {
    typedef unsigned long long u64;
    constexpr int PAIRS = M::TILE / 2;
    static_assert(sizeof(V) == 4 && M::PASSES == 1, "32-bit sums, the tile in LDS at once");
    __shared__ unsigned before;
    u64 *all = reinterpret_cast<u64*>(slabs), *pairs = reinterpret_cast<u64*>(tile);
    m.to_lds(tile, 0);
    __syncthreads();
    for (int k = threadIdx.x; k < PAIRS; k += M::THREADS) __hip_atomic_store(all + part * PAIRS + k, pairs[k], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) before = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (before != (unsigned)split - 1u) return false;
    for (int k = threadIdx.x; k < PAIRS; k += M::THREADS) {
        V s0 = 0, s1 = 0;
#pragma unroll 8
        for (int p = 0; p < split; ++p) {
            const u64 v = __hip_atomic_load(all + p * PAIRS + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            s0 += __builtin_bit_cast(V, (unsigned)v);
            s1 += __builtin_bit_cast(V, (unsigned)(v >> 32));
        }
        pairs[k] = (u64)__builtin_bit_cast(unsigned, s1) << 32 | __builtin_bit_cast(unsigned, s0);
    }
    if (threadIdx.x == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    return true;
}

}  // namespace
