// 8-bit block-scaled convolutions, wide layers: 256 channels x 256 (or 192) pixels per workgroup, two
// groups of four waves one barrier apart (gfx950).  The mathematics, layouts and exponents are
// those of conv_blockscaled.hip; the results are bit-identical to its kernel's.
//
// One K tile (128 input channels of one tap) is 32 MFMAs of 32 cycles per wave, 2 048 cycles of a SIMD's
// matrix pipe for its two waves, against 64 KB of operands: what a CU pulls from its L2 in the
// same time.  So the two kernels here keep the pipe fed in two ways:
//
//   schedule   a wave alternates between an interval of loads (fragment reads, LDS-DMA issue, counted
//              waits) and one of 16 MFMAs, four intervals per K tile; the second group runs one
//              barrier behind, so on every SIMD one wave computes while the other loads
//   operands   3x3 stride 1 (f8_slab_tile): the input pixels of all nine taps of a block of 128
//              channels are one run of TP + 2 W + 2 pixels, staged once ("slab", two in LDS, the next
//              block's fetched behind the current one's taps); tap (r, c) of pixel n reads row
//              n + r W + c, taps outside the image a row of zeros.  36 KB of DMA per K tile
//              instead of 64.  Other windows and strides (f8_stag_tile): both operands per K tile
//
// LDS rows are 128 bytes, 16-byte chunk c of row r in slot c ^ (r & 7).  DMA instructions per wave and K
// tile are constant (what has nothing to fetch reads out of range), so the waits can count them.
#include <algorithm>

#include "conv_blockscaled.h"

namespace ymx {

typedef unsigned int f8_u32x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) const f8_u32x4_t *f8_lds16_t;
typedef __attribute__((address_space(3))) const unsigned char *f8_lds8_t;

constexpr unsigned F8_OOB = 0x80000000u;
constexpr int F8_PIECE = 128 * 128;                         // 128 rows of 128 bytes

// A raw barrier (no implied drain of the memory counters) that the compiler may not move LDS reads across.
__device__ __forceinline__ void f8_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Fragments and accumulators of one wave: 128 channels (halves of four 16-row blocks) x 16 NJ pixels.
template <int NJ> struct F8Wave {
    f32x4_t acc[8][NJ];
    i32x8_t w[4], x[NJ];
    int ws[4], xs[NJ];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    // a weight piece's blocks (rows +16 each) and their exponents
    __device__ __forceinline__ void load_w(const char *rows, const char *exps, int swz0, int swz1) {
#pragma unroll
        for (int ib = 0; ib < 4; ++ib) {
            w[ib] = f8_frag(*(const int4 *)(rows + ib * 2048 + swz0), *(const int4 *)(rows + ib * 2048 + swz1));
            ws[ib] = *(const unsigned char *)(exps + ib * 16);
        }
    }
    // The accumulators pass through an empty asm statement behind the MFMAs: without it the compiler, for which a
    // barrier does not order them, moves an interval's MFMAs into the next one.
    template <int MH> __device__ __forceinline__ void mfma() {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int ib = 0; ib < 4; ++ib)
#pragma unroll
            for (int j = 0; j < NJ; ++j) acc[MH * 4 + ib][j] = f8_mfma(w[ib], x[j], acc[MH * 4 + ib][j], ws[ib], xs[j]);
#pragma unroll
        for (int ib = 0; ib < 4; ++ib)
#pragma unroll
            for (int j = 0; j < NJ; ++j) asm volatile("" : "+v"(acc[MH * 4 + ib][j]));
        __builtin_amdgcn_s_setprio(0);
    }
};

// ---- 3x3, stride 1: input slab resident over the taps --------------------------------------------------
// LDS: 2 slabs of npieces KB | 4 weight pieces (slot (kt & 1) 2 + half) | zero KB | 4 x 256 weight exponents
// | 2 x 512 pixel exponents
template <int NJ>
__device__ __forceinline__ void f8_slab_tile(const F8Args &g, const int p0, const int q0, const int ncb, const int npieces) {
    constexpr int WP = 16 * NJ;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const ConvArgs &a = g.a;
    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wq = wave & 1, wp = wave >> 1, group = wave >> 2;
    const int nk = ncb * 9;
    const i32x4_t xr = make_rsrc(a.x, a.x_bytes), wr = make_rsrc(a.w, a.w_bytes);
    const i32x4_t xsr = make_rsrc(g.xs, g.xs_bytes), wsr = make_rsrc(g.ws, g.ws_bytes);
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char *)smem;
    const int slab_bytes = npieces * 1024;
    const unsigned ring0 = lds0 + 2u * (unsigned)slab_bytes, zero0 = ring0 + 4u * F8_PIECE;
    const unsigned wexp0 = zero0 + 1024u, xexp0 = wexp0 + 1024u;
    const char *ring = smem + 2 * slab_bytes, *wexp = ring + 4 * F8_PIECE + 1024;

    const int srow = lane >> 3, chunk = (lane & 7) ^ srow;
    // slab piece i = rows 8 i .. 8 i + 7 = pixels p0 - W - 1 + 8 i + srow (a pixel before the tensor wraps to an
    // offset beyond it and reads zeros); channels past the input's last read zeros
    const unsigned slab_off0 = (unsigned)(p0 - a.W - 1 + srow) * (unsigned)a.Cin + (unsigned)(chunk * 16);
    const unsigned slab_step = 8u * (unsigned)a.Cin;
    const unsigned row_bytes = (unsigned)(nk * 128);
    unsigned woff[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = 16 * wave + 8 * i + srow;             // piece row r = channel (r >> 6) 128 + half 64 + (r & 63)
        woff[i] = (unsigned)(q0 + (r >> 6) * 128 + (r & 63)) * row_bytes + (unsigned)(chunk * 16);
    }
    const unsigned whalf = 64u * row_bytes;
    auto issue_w = [&](int kt, int half) {
        const unsigned dst = ring0 + (unsigned)(((kt & 1) * 2 + half) * F8_PIECE + wave * 2048);
        const unsigned base = (unsigned)kt * 128u + (half ? whalf : 0u);
#pragma unroll
        for (int i = 0; i < 2; ++i) f8_dma16(wr, dst + (unsigned)(i * 1024), kt < nk ? base + woff[i] : F8_OOB);
    };
    // loop form: offsets of W(m1) of tile kt + 1 and of W(m0) of tile kt + 2; tiles past the end fetch what lies
    // behind the row into slots that nothing reads any more
    unsigned wcur[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) { wcur[0][i] = woff[i] + 256u; wcur[1][i] = woff[i] + whalf + 128u; }
    // slab piece idx of block cb, or nothing; all conditions are selects, a branch would cost the interval
    auto issue_slab = [&](int cb, int idx) {
        const bool real = idx < npieces && cb < ncb;
        const unsigned dst = real ? lds0 + (unsigned)((cb & 1) * slab_bytes + idx * 1024) : zero0;
        const unsigned src = slab_off0 + ((unsigned)idx * slab_step + (unsigned)cb * 128u);
        f8_dma16(xr, dst, cb * 128 + chunk * 16 < (real ? a.Cin : 0) ? src : F8_OOB);
    };
    // exponents: wave 0 those of the 256 channels of a K tile (esrc: of tile kt + 2), waves 1 and 2 those of a block's slab
    // pixels, from the first one's number rounded down to 4 (esrc: of block cb + 1), the others nothing
    const int first = p0 - a.W - 1, xlow = first & ~3;
    const bool e_w = wave == 0, e_x = wave == 1 || wave == 2;
    i32x4_t er;
#pragma unroll
    for (int i = 0; i < 4; ++i) er[i] = e_x ? xsr[i] : wsr[i];
    unsigned esrc = e_w ? (unsigned)(q0 + lane * 4) : (unsigned)(xlow + (wave - 1) * 256 + lane * 4);
    auto issue_exp = [&](int kt, int cb, bool pixels) {
        const bool take = e_x && pixels && cb < ncb;
        const unsigned xdst = xexp0 + (unsigned)((cb & 1) * 512 + (wave - 1) * 256), wdst = wexp0 + (unsigned)((kt & 3) * 256);
        f8_dma4(er, e_w ? wdst : take ? xdst : zero0, e_w || take ? esrc : F8_OOB);
        esrc += e_w ? (unsigned)g.rows : take ? g.plane : 0u;
    };

    f8_dma_ready();
#pragma unroll
    for (int jj = 0; jj < 6; ++jj) issue_slab(0, jj * 8 + wave);
    f8_dma16(xr, zero0, F8_OOB);                           // the zero KB starts out (and stays) zero
    issue_w(0, 0);
    issue_w(0, 1);
    issue_w(1, 0);
    issue_exp(0, 0, true);
    issue_exp(1, 0, false);

    // the lane's pixels (16-pixel blocks j of the wave's) and which taps they have
    unsigned fmask[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        int unused;
        pixel_geometry(a, p0 + wp * WP + j * 16 + (lane & 15), unused, fmask[j]);
    }
    const int hb0 = wp * WP + (lane & 15), q4 = lane >> 4;
    const int swz0 = (q4 ^ (lane & 7)) << 4, swz1 = ((4 + q4) ^ (lane & 7)) << 4;
    const int a_row = (wq * 64 + (lane & 15)) * 128, a_exp = wq * 128 + (lane & 15);
    F8Wave<NJ> v;
    v.clear();

    auto load_x = [&](int cb, int shift, int tap) {
        const int hb = hb0 + shift;
        const unsigned base = lds0 + (unsigned)((cb & 1) * slab_bytes) + (unsigned)(hb * 128 + ((q4 ^ (hb & 7)) << 4));
        const unsigned e = xexp0 + (unsigned)((cb & 1) * 512 + (first & 3) + hb);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const unsigned in = (unsigned)__builtin_amdgcn_sbfe((int)fmask[j], (unsigned)tap, 1u);     // all ones inside the image
            const unsigned off = ((base + (unsigned)(j * 2048)) & in) | (zero0 & ~in);
            v.x[j] = f8_frag(__builtin_bit_cast(int4, *(f8_lds16_t)(uintptr_t)off), __builtin_bit_cast(int4, *(f8_lds16_t)(uintptr_t)(off ^ 64u)));
            v.xs[j] = *(f8_lds8_t)(uintptr_t)(e + (unsigned)(j * 16));
        }
    };

    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    f8_barrier();
    if (group == 1) f8_barrier();                           // the second group runs one barrier behind

    // Per K tile and wave six DMA instructions, all in load 2: W(m1) x 2 of the next tile, W(m0) x 2 of the one after,
    // a slab piece, exponents of the tile after next.  vmcnt(4) at the end of load 1 = "W(m1) of this tile has
    // landed" (read in load 2, one barrier later; the other group's same wait lies before that barrier too);
    // vmcnt(6) at the end of load 2 = "everything issued before this load 2 has landed": W(m0) and the exponents of the
    // next tile.  A slab's last piece is issued three tiles before its block begins.  Load intervals end with
    // lgkmcnt(0): what they read may be overwritten from the next interval on.
    int cb = 0, tap = 0;
    for (int kt = 0; kt < nk; ++kt) {
        const int tr = (tap * 11) >> 5, shift = tr * a.W + (tap - tr * 3);             // tap / 3 for tap < 9
        // load 1
        v.load_w(ring + ((kt & 1) * 2) * F8_PIECE + a_row, wexp + (kt & 3) * 256 + a_exp, swz0, swz1);
        load_x(cb, shift, tap);
        asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        f8_barrier();
        v.template mfma<0>();
        f8_barrier();
        // load 2
        v.load_w(ring + ((kt & 1) * 2 + 1) * F8_PIECE + a_row, wexp + (kt & 3) * 256 + 64 + a_exp, swz0, swz1);
        {
            const unsigned d1 = ring0 + (unsigned)((((kt + 1) & 1) * 2 + 1) * F8_PIECE + wave * 2048);
            const unsigned d0 = ring0 + (unsigned)(((kt & 1) * 2) * F8_PIECE + wave * 2048);
#pragma unroll
            for (int i = 0; i < 2; ++i) f8_dma16(wr, d1 + (unsigned)(i * 1024), wcur[1][i]);
#pragma unroll
            for (int i = 0; i < 2; ++i) f8_dma16(wr, d0 + (unsigned)(i * 1024), wcur[0][i]);
            issue_slab(tap < 6 ? cb + 1 : ncb, tap * 8 + wave);
            issue_exp(kt + 2, cb + 1, tap == 0);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) { wcur[0][i] += 128u; wcur[1][i] += 128u; }
        asm volatile("s_waitcnt vmcnt(6)" ::: "memory");
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        f8_barrier();
        v.template mfma<1>();
        f8_barrier();
        if (++tap == 9) { tap = 0; ++cb; }
    }
    if (group == 0) f8_barrier();
    f8_vmcnt<0>();
    __syncthreads();
    f8_epilogue<bf16_t, 8, NJ>(a, v.acc, smem, wave, q0 + wq * 128, p0 + wp * WP, lane);
}

// ---- any window and stride: both operands per K tile ------------------------------------------------------
// LDS: 8 pieces (slot (kt & 1) 4 + {W(m0), X(n0), X(n1), W(m1)}) | 4 x (256 weight exponents, 256 dwords of pixel ones)
// | 256 bytes that nothing reads
constexpr int F8_STAG_EXP = 256 + 1024, F8_STAG_LDS = 8 * F8_PIECE + 4 * F8_STAG_EXP + 256;

template <int NJ>
__device__ __forceinline__ void f8_stag_tile(const F8Args &g, const int p0, const int q0) {
    constexpr int WP = 16 * NJ;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const ConvArgs &a = g.a;
    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wq = wave & 1, wp = wave >> 1, group = wave >> 2;
    const int nk = g.nkt;
    const i32x4_t xr = make_rsrc(a.x, a.x_bytes), wr = make_rsrc(a.w, a.w_bytes);
    const i32x4_t xsr = make_rsrc(g.xs, g.xs_bytes), wsr = make_rsrc(g.ws, g.ws_bytes);
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char *)smem;
    const unsigned exp0 = lds0 + 8u * F8_PIECE, dump = exp0 + 4u * F8_STAG_EXP;

    const int srow = lane >> 3, chunk = (lane & 7) ^ srow;
    // Row r of a W piece is channel (r >> 6) 128 + half 64 + (r & 63), of an X piece pixel (r >> 5) WP + half 32 +
    // (r & 31) of the tile (rows past the wave's WP pixels stay empty).  This wave fills rows 16 wave + 8 i + srow.
    unsigned xoff[2][2], xmask[2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = 16 * wave + 8 * i + srow, n = h * 32 + (r & 31);
            int pix;
            pixel_geometry(a, p0 + (r >> 5) * WP + n, pix, xmask[h][i]);
            if (n >= WP) xmask[h][i] = 0u;
            xoff[h][i] = (unsigned)pix * (unsigned)a.Cin + (unsigned)(chunk * 16);
        }
    const unsigned row_bytes = (unsigned)(nk * 128);
    unsigned woff[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = 16 * wave + 8 * i + srow;
        woff[i] = (unsigned)(q0 + (r >> 6) * 128 + (r & 63)) * row_bytes + (unsigned)(chunk * 16);
    }
    const unsigned whalf = 64u * row_bytes;
    // exponents: waves 0 .. NJ - 1 those of 64 pixels each, wave 4 those of the 256 channels, the others nothing
    int spix = 0;
    unsigned smask = 0;
    if (wave < NJ) pixel_geometry(a, p0 + wave * 64 + lane, spix, smask);

    // tap of a K tile, the same for every lane: its pixel step, mask bit (0 past the end) and first channel
    auto decode = [&](int kt, int &tpix, unsigned &bit, int &blk) {
        blk = g.taps == 1 ? kt : (int)(((unsigned)kt * 7282u) >> 16);                  // kt / 9 for kt < 32768
        const int tap = kt - blk * g.taps, tr = g.taps == 1 ? 0 : (tap * 11) >> 5;     // tap / 3 for tap < 9
        tpix = tr * a.W + (tap - tr * 3);
        bit = kt < nk ? 1u << tap : 0u;
    };
    auto issue_x = [&](int kt, int half, int tpix, unsigned bit, int blk) {
        const unsigned dst = lds0 + (unsigned)(((kt & 1) * 4 + 1 + half) * F8_PIECE + wave * 2048);
        const unsigned step = (unsigned)tpix * (unsigned)a.Cin + (unsigned)blk * 128u;
        const unsigned ok = blk * 128 + chunk * 16 < a.Cin ? bit : 0u;
#pragma unroll
        for (int i = 0; i < 2; ++i) f8_dma16(xr, dst + (unsigned)(i * 1024), (xmask[half][i] & ok) ? xoff[half][i] + step : F8_OOB);
    };
    auto issue_w = [&](int kt, int half) {
        const unsigned dst = lds0 + (unsigned)(((kt & 1) * 4 + (half ? 3 : 0)) * F8_PIECE + wave * 2048);
        const unsigned base = (unsigned)kt * 128u + (half ? whalf : 0u);
#pragma unroll
        for (int i = 0; i < 2; ++i) f8_dma16(wr, dst + (unsigned)(i * 1024), kt < nk ? base + woff[i] : F8_OOB);
    };
    const bool e_w = wave == 4, e_x = wave < NJ;
    auto issue_exp = [&](int kt, int tpix, unsigned bit, int blk) {
        const unsigned slot = exp0 + (unsigned)((kt & 3) * F8_STAG_EXP);
        if (e_w) {
            f8_dma4(wsr, slot, kt < nk ? (unsigned)(kt * g.rows + q0) + (unsigned)(lane * 4) : F8_OOB);
        } else {
            const unsigned src = (unsigned)spix + ((unsigned)blk * g.plane + (unsigned)tpix);
            f8_dma_u8(xsr, e_x ? slot + 256u + (unsigned)(wave * 256) : dump, (smask & (e_x ? bit : 0u)) ? src : F8_OOB);
        }
    };
    auto first_half = [&](int kt) {                          // W(m0), X(n0), exponents
        int tpix, blk;
        unsigned bit;
        decode(kt, tpix, bit, blk);
        issue_w(kt, 0);
        issue_x(kt, 0, tpix, bit, blk);
        issue_exp(kt, tpix, bit, blk);
    };
    auto second_half = [&](int kt) {                         // X(n1), W(m1)
        int tpix, blk;
        unsigned bit;
        decode(kt, tpix, bit, blk);
        issue_x(kt, 1, tpix, bit, blk);
        issue_w(kt, 1);
    };
    f8_dma_ready();
    first_half(0);
    second_half(0);
    first_half(1);

    const int q4 = lane >> 4;
    const int swz0 = (q4 ^ (lane & 7)) << 4, swz1 = ((4 + q4) ^ (lane & 7)) << 4;
    const int a_row = (wq * 64 + (lane & 15)) * 128, a_exp = wq * 128 + (lane & 15);
    const int b_row = (wp * 32 + (lane & 15)) * 128, b_exp = 256 + (wp * WP + (lane & 15)) * 4;
    F8Wave<NJ> v;
    v.clear();
    f8_vmcnt<7>();
    f8_barrier();
    if (group == 1) f8_barrier();

    // Nine DMA instructions per wave and K tile: X(n1), W(m1) of the next tile in load 1, W(m0), X(n0) and the exponents of
    // the one after in load 2.  vmcnt(9) at the end of load 1 = "W(m1) of this tile has landed", vmcnt(7) at the end of
    // load 2 = "W(m0), X(n0), X(n1) and the exponents of the next tile have".
    for (int kt = 0; kt < nk; ++kt) {
        const char *piece = smem + (kt & 1) * 4 * F8_PIECE, *exps = smem + 8 * F8_PIECE + (kt & 3) * F8_STAG_EXP;
        v.load_w(piece + a_row, exps + a_exp, swz0, swz1);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const char *row = piece + (1 + (j >> 1)) * F8_PIECE + b_row + (j & 1) * 2048;
            v.x[j] = f8_frag(*(const int4 *)(row + swz0), *(const int4 *)(row + swz1));
            v.xs[j] = *(const int *)(exps + b_exp + j * 64);
        }
        second_half(kt + 1);
        f8_vmcnt<9>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        f8_barrier();
        v.template mfma<0>();
        f8_barrier();
        v.load_w(piece + 3 * F8_PIECE + a_row, exps + 64 + a_exp, swz0, swz1);
        first_half(kt + 2);
        f8_vmcnt<7>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        f8_barrier();
        v.template mfma<1>();
        f8_barrier();
    }
    if (group == 0) f8_barrier();
    f8_vmcnt<0>();
    __syncthreads();
    f8_epilogue<bf16_t, 8, NJ>(a, v.acc, smem, wave, q0 + wq * 128, p0 + wp * WP, lane);
}

// Both tile forms in one launch, see plan_wide_tiles: workgroups below nbig take 256-pixel tiles over the first pbig
// pixels, the rest 192-pixel tiles from there on (nbig 0: only those; a huge pbig: only the former).
template <bool SLAB>
__global__ void __launch_bounds__(512, 2)
conv_f8_wide_kernel(const F8Args g, const int ntq, const int ncb, const int np4, const int np3, const int nbig, const int pbig) {
    const int b = blockIdx.x;
    if (b < nbig) {
        const int id = xcd_remap(b, nbig);
        if constexpr (SLAB) f8_slab_tile<4>(g, (id / ntq) * 256, (id % ntq) * 256, ncb, np4);
        else f8_stag_tile<4>(g, (id / ntq) * 256, (id % ntq) * 256);
    } else {
        const int id = xcd_remap(b - nbig, (int)gridDim.x - nbig);
        if constexpr (SLAB) f8_slab_tile<3>(g, pbig + (id / ntq) * 192, (id % ntq) * 256, ncb, np3);
        else f8_stag_tile<3>(g, pbig + (id / ntq) * 192, (id % ntq) * 256);
    }
}

static int slab_pieces(int W, int tp) { return (tp + 2 * W + 2 + 7) / 8; }
static int slab_lds(int pieces) { return 2 * pieces * 1024 + 4 * F8_PIECE + 1024 + 1024 + 1024; }
// Slabs of 192-pixel tiles fit for rows up to 87 pixels, of 256-pixel tiles up to 55.
static bool slab_fits(const F8Args &g) { return g.taps == 9 && g.a.stride == 1 && slab_lds(slab_pieces(g.a.W, 192)) <= 160 * 1024; }

// Layers for these kernels: bf16 outputs, 160 tiles and more, 256-channel tiles no more than a quarter wider than
// 64-channel ones would be (64 x 26^2 512 -> 300 3x3: 124 us here, 90 in tiles of 128), more than two K tiles (16 x 52^2
// 144 -> 200 1x1: 21.4, 18.8), and, where both operands are fetched per K tile, not between one round of the chip and two
// (64 x 26^2 1024 -> 512 1x1, 338 tiles: 47.6, 44.1; 64 x 52^2, 1352 tiles: 156, 194).
bool conv_f8_wide(const F8Args &g) {
    const long long nq = (g.a.Cout + 255) / 256, n64 = (g.a.Cout + 63) / 64;
    const long long tiles = (long long)((g.a.P + 255) / 256) * nq;
    return g.a.out_dtype == YMX_BF16 && nq * 16 <= n64 * 5 && tiles >= 160 && g.nkt > 2 && (slab_fits(g) || tiles <= 256 || tiles >= 512);
}

static TilePlan wide_plan(const F8Args &g, bool slab) {
    if (slab && slab_lds(slab_pieces(g.a.W, 256)) > 160 * 1024) return TilePlan{192, 0, 0};
    return plan_wide_tiles(g.a.P, (g.a.Cout + 255) / 256, 0.85, 0, 0);
}
const char *conv_f8_wide_tile(const F8Args &g) {
    const bool slab = slab_fits(g);
    const int px = wide_plan(g, slab).pixels;
    if (slab) return px == 256 ? "256x256 slab" : px == 192 ? "256x192 slab" : "256x256 and 256x192 slab";
    return px == 256 ? "256x256" : px == 192 ? "256x192" : "256x256 and 256x192";
}

template <bool SLAB> static int launch_wide(const F8Args &g, hipStream_t s) {
    const int ntq = (g.a.Cout + 255) / 256, np4 = slab_pieces(g.a.W, 256), np3 = slab_pieces(g.a.W, 192);
    const TilePlan pl = wide_plan(g, SLAB);
    const long long t4 = ((long long)g.a.P + 255) / 256;
    int nbig = 0, pbig = 0;
    if (pl.pixels == 256) { nbig = (int)(t4 * ntq); pbig = g.a.P; }
    if (pl.pixels == 448) { nbig = pl.big_tiles; pbig = pl.big_pixels; }
    const long long rest = (long long)g.a.P - pbig;
    const long long grid = nbig + (rest > 0 ? (rest + 191) / 192 * ntq : 0);
    if (grid > 0x7fffffffLL) return fail(YMX_EUNSUPPORTED, "conv_f8: grid too large");
    const int epi = 8 * EpiGeom<8, 64, 64>::LDS_BYTES;
    const int lds = SLAB ? std::max(epi, slab_lds(nbig ? np4 : np3)) : std::max(epi, F8_STAG_LDS);
    auto kern = conv_f8_wide_kernel<SLAB>;
    static LdsReserve reserved;
    if (const int rc = reserve_lds(reserved, (const void *)kern, 160 * 1024, "conv_f8 (wide)")) return rc;
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(512), lds, s, g, ntq, (g.a.Cin + 127) / 128, np4, np3, nbig, pbig);
    return check_launch("conv_f8 (wide)");
}

int launch_conv_f8_wide(const F8Args &g, hipStream_t s) {
    return slab_fits(g) ? launch_wide<true>(g, s) : launch_wide<false>(g, s);
}

}  // namespace ymx
