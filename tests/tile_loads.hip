// Every load of TileMul::run, walked on the host with the header's own offset functions: what a lane reads must lie in its array
// whether or not the buffer's range check counts the scalar offset, and a value that exists must not be left out.
#include "tile_mul.h"

#include <cstdio>

static const char* what = "";
static long long cases = 0;

static void fail(const char* why, long long a, long long b) {
    printf("%s: %s (%lld, %lld)\n", what, why, a, b);
    exit(1);
}

// rows of an operand from this tile on: `left` exist, `ld` bytes apart; `row_end` bytes of a row may be read from the first stage on
struct Side { long long ld, left, row_end; };

template <typename M>
static void walk(Side f, Side s, int total, int fend, int ks, bool trf, int bf) {
    ++cases;
    const long long f_end = trf ? (total * 64 - 1) * f.ld + f.left * 2 : ((f.left < bf ? f.left : bf) - 1) * f.ld + f.row_end;
    const long long s_end = (s.left - 1) * s.ld + s.row_end;
    for (int group = 0; group < ks; ++group) {
        const Stages st = stages_of(total, ks, group);
        const long long fstep = trf ? f.ld * 64 : 128;
        for (int kt = 0; kt < st.count; ++kt)
            for (int wid = 0; wid < M::WAVES; ++wid)
                for (int lane = 0; lane < 64; ++lane)
                    for (int i = 0; i < M::L; ++i) {
                        const bool is_f = i < M::FL;
                        const unsigned own = is_f ? M::f_offset(i, wid, lane, (unsigned)f.ld, (int)f.left) : M::s_offset(i - M::FL, wid, lane, (unsigned)s.ld, (int)s.left);
                        unsigned o = ks == 1 || kt < st.live ? own : OUT;
                        if (is_f && kt == st.last) o |= M::f_behind(wid, lane, fend);
                        const long long scalar = kt * (is_f ? fstep : 128), at = st.first * (is_f ? fstep : 128) + scalar;
                        if (scalar >= (long long)DESC_BYTES) fail("scalar offset beyond the range", scalar, kt);
                        if (o < OUT) {
                            if (o + scalar + 16 > (long long)DESC_BYTES) fail("a value that exists is behind the range", o, scalar);
                            if (at + o + 16 > (is_f ? f_end : s_end)) fail("reads behind its array", at + o + 16, is_f ? f_end : s_end);
                        } else {
                            if (kt < st.live && own < OUT && !trf) {           // left out: only what is behind the row's end
                                const int slot = ((is_f ? i : i - M::FL) * M::WAVES + wid) * 64 + lane;
                                const long long col = ((slot & 7) ^ ((slot >> 4) & 7)) * 16 + at;
                                if (col < (is_f ? f.row_end : s.row_end)) fail("a value that exists is left out", col, own);
                            }
                        }
                    }
    }
}

// codes [N][K], rows padded to `pad` bytes, times rows of a workspace [.][Kp]
template <typename M>
static void codes(int n_left, int K, int pad, int ks, int bf, int bs) {
    const int Kp = (K + 127) / 128 * 128, ld = (K + pad - 1) / pad * pad, K16 = (K + 15) / 16 * 16;
    walk<M>(Side{ld, n_left, K16}, Side{Kp, bs, Kp}, Kp / 128, K16 - (Kp - 128), ks, false, bf);
}

template <typename M>
static void halves(int np, int mp, int ks, bool trf, int b) {
    for (int first = 0; first < np; first += b)
        for (int other = 0; other < (trf ? mp : np); other += b) {
            if (trf) walk<M>(Side{mp * 2LL, mp - other, 0}, Side{np * 2LL, np - first < b ? np - first : b, np * 2LL}, np / 64, 128, ks, true, b);
            else walk<M>(Side{mp * 2LL, np - first, mp * 2LL}, Side{mp * 2LL, np - other < b ? np - other : b, mp * 2LL}, mp / 64, 128, ks, false, b);
        }
}

int main() {
    const int ks_[] = {1, 15, 16, 17, 63, 64, 65, 100, 127, 128, 129, 192, 193, 256, 257, 300, 320, 321, 385, 513, 2047, 2048, 2049};
    for (int K : ks_)
        for (int left : {1, 2, 17, 63, 64, 65, 127, 128, 129, 1000})
            for (int pad : {16, 64}) {
                what = "int8, 64, two groups";
                codes<TileMul<MulI8, 64, 64, 2, 2, 3, false, 2>>(left, K, pad, 2, 64, 64);
                what = "int8, 64";
                codes<TileMul<MulI8, 64, 64, 2, 2, 3, false, 1>>(left, K, pad, 1, 64, 64);
                what = "int8, 128";
                codes<TileMul<MulI8, 128, 128, 2, 2, 2, false, 1>>(left, K, pad, 1, 128, 128);
            }
    for (int np : {64, 128, 192, 320, 576})
        for (int mp : {64, 128, 192, 320, 576, 1088}) {
            if (mp < np) continue;
            what = "fp16, 64, two groups";
            halves<TileMul<MulF16, 64, 64, 2, 2, 3, false, 2>>(np, mp, 2, false, 64);
            halves<TileMul<MulF16, 64, 64, 2, 2, 3, true, 2>>(np, mp, 2, true, 64);
            what = "fp16, 64";
            halves<TileMul<MulF16, 64, 64, 2, 2, 3, false, 1>>(np, mp, 1, false, 64);
            halves<TileMul<MulF16, 64, 64, 2, 2, 3, true, 1>>(np, mp, 1, true, 64);
            what = "fp16, 128";
            halves<TileMul<MulF16, 128, 128, 2, 4, 2, false, 1>>(np, mp, 1, false, 128);
            halves<TileMul<MulF16, 128, 128, 2, 4, 2, true, 1>>(np, mp, 1, true, 128);
            what = "fp16, 256";
            halves<TileMul<MulF16, 256, 256, 2, 4, 2, false, 1>>(np, mp, 1, false, 256);
            halves<TileMul<MulF16, 256, 256, 2, 4, 2, true, 1>>(np, mp, 1, true, 256);
        }
    printf("ok %lld\n", cases);
    return 0;
}
