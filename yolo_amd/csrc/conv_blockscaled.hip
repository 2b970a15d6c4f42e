// Convolution blocks in 8-bit floating point with a scale for each block of 128 channels (gfx950).
//
//   y = act( sum_{tap, c} x(pixel + tap, c) w(tap, c, channel) * scale + shift ) + residual
//
// x and w are held as e4m3 numbers (3 bits behind the leading one, largest 448) and one power of
// two for each block of up to 128 input channels: of one pixel for x, of one tap and one output
// channel for w.  The block's exponent is the smallest k (>= -126) with |largest| <= 448 * 2^k (0
// for a block of zeros); what is stored is value / 2^k rounded to nearest even, NaN and infinities
// become NaN.  Powers of two make three things exact: the division, the way back, and the joining
// of blocks -- v_mfma_scale_f32_16x16x128_f8f6f4 takes one exponent byte per row and column and
// applies both to the 128 products it sums, so the scaled blocks are added in the fp32 accumulators
// of the matrix pipe with no other instruction.
//
// What the 8-bit pipe keeps: it adds products in groups of eight aligned to the group's largest, of
// which 13 bits below its leading one survive, and the groups in fp32 (measured with single products;
// 5e-5 of the result's magnitude on random operands).  That is a thirtieth of bf16's half step, so
// bf16 outputs take it.  32-bit outputs (the logits) would show it: they run the same tiles through the
// bf16 instructions at half the rate, whose products are exact and whose sums are fp32: a scaled e4m3
// number is a bf16 number, one conversion instruction per pair.
//
// Quantised map (ymx_quantize_blocks):  [pixel][C] e4m3 bytes (padded to 256), then one plane of
// exponent bytes (k + 127) per block of channels, [block][pixels rounded up to 4], the padding zero.
// Packed kernel (ymx_pack_weights):  [channel, padded to 256][K tile][128] bytes, then
// [K tile][channel] exponent bytes.  K tile = (block of 128 input channels) * taps + tap, so that
// the taps of a block, which read the same pixels, follow one another; channels past the input's
// last are zeros.
#include <algorithm>

#include "conv_blockscaled.h"

namespace ymx {

// ---- quantisation ---------------------------------------------------------------------------------
// The block's exponent from the bits of its largest finite magnitude: 1.75 * 2^8 = 448.
__device__ __forceinline__ int f8_exponent(uint32_t amax_bits) {
    const int k = (int)(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return amax_bits == 0u ? 0 : (k < -126 ? -126 : k);
}
__device__ __forceinline__ float f8_factor(int k) { return __uint_as_float((uint32_t)(127 - k) << 23); }   // 2^-k, -126 <= k <= 120
// Magnitude bits of a finite value, 0 for NaN and infinities (they take no part in the maximum).
__device__ __forceinline__ uint32_t f8_mag(float v) {
    const uint32_t m = __float_as_uint(v) & 0x7fffffffu;
    return m < 0x7f800000u ? m : 0u;
}
__device__ __forceinline__ float f8_scaled(float v, float f) {
    return (__float_as_uint(v) & 0x7fffffffu) < 0x7f800000u ? v * f : __uint_as_float(0x7fc00000u);
}
__device__ __forceinline__ uint32_t f8_pack4(float a, float b, float c, float d) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
    return (uint32_t)r;
}

static size_t f8_map_bytes(long long n_pix, int C) { return ((size_t)n_pix * C + 255) / 256 * 256; }
static long long f8_plane(long long n_pix) { return (n_pix + 3) / 4 * 4; }
size_t quant_bytes(long long n_pix, int C) { return f8_map_bytes(n_pix, C) + (size_t)f8_plane(n_pix) * ((C + 127) / 128); }

// GL lanes of 8 channels share a block of one pixel (16 lanes = 128 channels; 8 or 4 where the map has no more
// than 64 or 32); a wave takes 64 / GL neighbouring pixels of one block, so that four exponents leave as a dword.
// Reads 2 or 4 bytes a value, writes one: bound by memory (5.4 TB/s on a 177 MB map).
template <typename T, int GL>
__global__ void __launch_bounds__(256)
quantize_kernel(const T *__restrict__ x, int x_ld, unsigned char *__restrict__ q, unsigned char *__restrict__ scales, long long n_pix,
                int C, int nb, long long plane) {
    constexpr int NPX = 64 / GL;
    const long long units = (n_pix + NPX - 1) / NPX * nb;
    const int lane = threadIdx.x & 63, gl = lane % GL;
    for (long long u = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); u < units; u += (long long)gridDim.x * 4) {
        const long long run = nb == 1 ? u : u / nb;
        const int blk = nb == 1 ? 0 : (int)(u - run * nb);
        const long long p = run * NPX + lane / GL;
        const int c = blk * 128 + gl * 8;
        const bool on = c < C && p < n_pix;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
        if (on) {
            const T *src = x + (size_t)p * x_ld + c;
            if constexpr (sizeof(T) == 2) {
                const uint4 r = *(const uint4 *)src;
                const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[2 * i] = __uint_as_float(w[i] << 16);
                    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
                }
            } else {
                const float4 a = *(const float4 *)src, b = *(const float4 *)(src + 4);
                v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
                v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
            }
        }
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, f8_mag(v[i]));
#pragma unroll
        for (int o = GL / 2; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o));
        const int k = f8_exponent(m);
        const float f = f8_factor(k);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = f8_scaled(v[i], f);
        if (on) *(uint2 *)(q + (size_t)p * C + c) = uint2{f8_pack4(v[0], v[1], v[2], v[3]), f8_pack4(v[4], v[5], v[6], v[7])};
        // exponents of four neighbouring pixels -> the first one's leading lane (0 behind the last pixel)
        uint32_t e = p < n_pix ? (uint32_t)(k + 127) : 0u;
        e |= (uint32_t)__shfl_down((int)e, GL) << 8;
        e |= (uint32_t)__shfl_down((int)e, 2 * GL) << 16;
        if (lane % (4 * GL) == 0 && p < n_pix) *(uint32_t *)(scales + (size_t)blk * plane + p) = e;
    }
}

int launch_quantize(const void *x, int x_ld, void *q, long long n_pix, int C, int dtype, hipStream_t s) {
    const int nb = (C + 127) / 128;
    unsigned char *sc = (unsigned char *)q + f8_map_bytes(n_pix, C);
    auto go = [&](auto ttag, auto gtag) {
        typedef decltype(ttag) T;
        constexpr int GL = decltype(gtag)::value;
        const long long units = (n_pix + 64 / GL - 1) / (64 / GL) * nb;
        hipLaunchKernelGGL((quantize_kernel<T, GL>), dim3((unsigned)std::min<long long>((units + 3) / 4, 16384)), dim3(256), 0, s, (const T *)x, x_ld,
                           (unsigned char *)q, sc, n_pix, C, nb, f8_plane(n_pix));
    };
    auto lanes = [&](auto ttag) {
        if (C > 64) go(ttag, std::integral_constant<int, 16>{});
        else if (C > 32) go(ttag, std::integral_constant<int, 8>{});
        else go(ttag, std::integral_constant<int, 4>{});
    };
    if (dtype == YMX_BF16) lanes(bf16_t{});
    else lanes(float{});
    return check_launch("quantize_blocks");
}

// ---- packed kernels -------------------------------------------------------------------------------
static int f8_rows(int Cout) { return (Cout + 255) / 256 * 256; }
static int f8_tiles(int k, int Cin) { return (Cin + 127) / 128 * k * k; }
size_t packed_f8_bytes(int k, int Cin, int Cout) { return (size_t)f8_rows(Cout) * f8_tiles(k, Cin) * (128 + 1); }

// One thread per (output channel, K tile); neighbouring threads read neighbouring channels, the block's 128 values at once
// (512 -> 1024 3x3 in 12 us; one after the other, twice, 55).
__global__ void __launch_bounds__(256)
pack_f8_kernel(const float *__restrict__ w, unsigned char *__restrict__ out, unsigned char *__restrict__ scales, int taps, int Cin, int Cout, int rows, int nkt) {
    const int co = blockIdx.x * 256 + threadIdx.x, kt = blockIdx.y;
    const int blk = kt / taps, tap = kt - blk * taps;
    const int c0 = blk * 128, nc = min(128, Cin - c0);
    const float *__restrict__ src = w + ((size_t)tap * Cin + c0) * Cout + co;
    float v[128];
#pragma unroll
    for (int c = 0; c < 128; ++c) v[c] = co < Cout && c < nc ? src[(size_t)c * Cout] : 0.0f;
    uint32_t m = 0;
#pragma unroll
    for (int c = 0; c < 128; ++c) m = max(m, f8_mag(v[c]));
    const int k = f8_exponent(m);
    const float f = f8_factor(k);
    uint4 *dst = (uint4 *)(out + ((size_t)co * nkt + kt) * 128);
#pragma unroll
    for (int c = 0; c < 128; c += 16) {
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            o[i] = f8_pack4(f8_scaled(v[c + 4 * i], f), f8_scaled(v[c + 4 * i + 1], f), f8_scaled(v[c + 4 * i + 2], f), f8_scaled(v[c + 4 * i + 3], f));
        dst[c >> 4] = uint4{o[0], o[1], o[2], o[3]};
    }
    scales[(size_t)kt * rows + co] = (unsigned char)(k + 127);
}

int launch_pack_f8(const float *w_hwio, void *packed, int k, int Cin, int Cout, hipStream_t s) {
    const int rows = f8_rows(Cout), nkt = f8_tiles(k, Cin);
    unsigned char *out = (unsigned char *)packed;
    hipLaunchKernelGGL(pack_f8_kernel, dim3(rows / 256, nkt), dim3(256), 0, s, w_hwio, out, out + (size_t)rows * nkt * 128, k * k, Cin, Cout, rows,
                       nkt);
    return check_launch("pack_weights");
}

// ---- quantisation inside the product ------------------------------------------------------------------
// 16 bf16 values -> e4m3 numbers and the exponent byte of their block, which eight neighbouring lanes share: the values
// and bytes that quantize_kernel gives.
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u16x2_t f8_max2(u16x2_t a, uint32_t b) { return __builtin_elementwise_max(a, __builtin_bit_cast(u16x2_t, b)); }
__device__ __forceinline__ uint4 f8_quantize16(uint32_t (&w)[8], int &e) {
    u16x2_t m = {0, 0};
#pragma unroll
    for (int n = 0; n < 8; ++n) m = f8_max2(m, w[n] & 0x7fff7fffu);
    if (__any(max((uint32_t)m.x, (uint32_t)m.y) >= 0x7f80u)) {   // NaN and infinities: NaN, and no part in the maximum
        m = u16x2_t{0, 0};
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            const bool lo = (w[n] & 0x7fffu) >= 0x7f80u, hi = (w[n] & 0x7fff0000u) >= 0x7f800000u;
            m = f8_max2(m, w[n] & ((lo ? 0u : 0x7fffu) | (hi ? 0u : 0x7fff0000u)));
            w[n] |= (lo ? 0x7fffu : 0u) | (hi ? 0x7fff0000u : 0u);
        }
    }
    uint32_t p = max((uint32_t)m.x, (uint32_t)m.y);
    p = max(p, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)p, 0xb1, 0xf, 0xf, false));       // lane ^ 1
    p = max(p, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)p, 0x4e, 0xf, 0xf, false));       // lane ^ 2
    p = max(p, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)p, 0x141, 0xf, 0xf, false));      // 7 - lane of eight
    e = f8_exponent(p << 16) + 127;
    const float f = __uint_as_float((uint32_t)e << 23);
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    typedef short s2 __attribute__((ext_vector_type(2)));
    uint32_t o[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        s2 v = {0, 0};
        v = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(v, __builtin_bit_cast(bf2, w[2 * n]), f, false);
        v = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(v, __builtin_bit_cast(bf2, w[2 * n + 1]), f, true);
        o[n] = __builtin_bit_cast(uint32_t, v);
    }
    return uint4{o[0], o[1], o[2], o[3]};
}

// ---- the product ----------------------------------------------------------------------------------
// NWQ x NWP waves, each 16 NI channels x 16 NJ pixels; K tiles of 128 channels of one tap through NSTAGE stages
// of LDS, filled by LDS-DMA NSTAGE - 1 tiles ahead, one barrier per tile.  Rows are 128 bytes (one pixel's or one
// channel's 128 values), the 16-byte chunk c of row r in slot c ^ (r & 7): the lanes that read one fragment then
// touch 16 different slots.  A lane's 32 values of a fragment are the chunks q and q + 4 of its row, q = lane / 16,
// for pixels and channels alike (the order inside a block does not matter: one exponent covers it).
//
// RAW: x is a bf16 map, staged as such (256 bytes per pixel and K tile, chunk c of row r in slot c ^ (r & 15)).  While
// tile kt is multiplied, the threads quantise tile kt + 1, 16 channels each, into one of two further row buffers (32-bit
// outputs: in place, as the bf16 numbers that their products take).
template <bool RAW, typename OT, int NWQ, int NWP, int NI, int NJ, int NSTAGE> struct F8Tile {
    static constexpr int NW = NWQ * NWP, TQ = NWQ * NI * 16, TP = NWP * NJ * 16;
    static constexpr int XROW = RAW ? 256 : 128, XPER = 1024 / XROW;                // bytes of a pixel, pixels per instruction
    static constexpr int NXI = TP / XPER / NW, NWI = TQ / 8 / NW;                       // DMA instructions per wave: rows ...
    static constexpr int SX = RAW ? 0 : (TP + 63) / 64, NS = SX + (TQ + 63) / 64;              // ... and, in all, exponents
    static constexpr int NSI = (NS + NW - 1) / NW;                                   // (per wave)
    static constexpr int XB = TP * XROW, WB = TQ * 128, STAGE = XB + WB + NS * 256, PIECES = NXI + NWI + NSI;
    static constexpr int EPI = NW * EpiGeom<NI, 64, 16 * NJ>::LDS_BYTES;
    static constexpr int XQ = RAW && sizeof(OT) == 2 ? TP * 132 : 0, USED = NSTAGE * STAGE + 2 * XQ, LDS = USED > EPI ? USED : EPI;     // (rows and exponents)
    static constexpr int AHEAD = NSTAGE - (RAW ? 3 : 2);                             // K tiles in flight behind the one waited for
    static_assert(TP % (XPER * NW) == 0 && TQ % (8 * NW) == 0, "whole instructions per wave");
};
template <bool RAW, typename OT, int NWQ, int NWP, int NI, int NJ, int NSTAGE>
__global__ void __launch_bounds__(64 * NWQ * NWP, 2)
conv_f8_kernel(const F8Args g, const int ntile_q) {
    typedef F8Tile<RAW, OT, NWQ, NWP, NI, NJ, NSTAGE> C;
    constexpr int NXI = C::NXI, NWI = C::NWI, NSI = C::NSI, SX = C::SX, XB = C::XB, WB = C::WB, STAGE = C::STAGE;
    constexpr bool EXACT = sizeof(OT) == 4, ROUNDED = RAW && EXACT;
    constexpr unsigned OOB = 0x80000000u;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const ConvArgs &a = g.a;
    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wq = wave % NWQ, wp = wave / NWQ;
    const int id = xcd_remap(blockIdx.x, gridDim.x);
    const int tq = id % ntile_q, tp = id / ntile_q;
    const int p0 = tp * C::TP, q0 = tq * C::TQ;
    const i32x4_t xr = make_rsrc(a.x, a.x_bytes), wr = make_rsrc(a.w, a.w_bytes);
    const i32x4_t xsr = make_rsrc(g.xs, g.xs_bytes), wsr = make_rsrc(g.ws, g.ws_bytes);
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char *)smem;

    const int srow = lane >> 3, chunk = (lane & 7) ^ srow;
    unsigned xoff[NXI], xmask[NXI];
    int xch[NXI];                                            // first channel, within the block, of the 16 bytes
#pragma unroll
    for (int i = 0; i < NXI; ++i) {
        int pix;
        const int row = (wave * NXI + i) * C::XPER + (RAW ? lane >> 4 : srow), ck = RAW ? (lane & 15) ^ (row & 15) : chunk;
        pixel_geometry(a, p0 + row, pix, xmask[i]);
        xoff[i] = (unsigned)pix * g.pitch + (unsigned)(ck * 16);
        xch[i] = ck * (RAW ? 8 : 16);
    }
    const unsigned row_bytes = (unsigned)(g.nkt * 128);
    const unsigned woff = (unsigned)(q0 + wave * NWI * 8 + srow) * row_bytes + (unsigned)chunk * 16u;
    // exponents: instructions 0 .. SX - 1 fetch those of 64 pixels, the others those of 64 channels; instructions past the
    // last repeat it
    int si[NSI];
    unsigned smask[NSI], ebase[NSI];
    i32x4_t er[NSI];
#pragma unroll
    for (int e = 0; e < NSI; ++e) {
        si[e] = min(wave + e * C::NW, C::NS - 1);
        const bool s_x = si[e] < SX;
        int pix = 0;
        smask[e] = 0;
        if (s_x) {
            pixel_geometry(a, p0 + si[e] * 64 + lane, pix, smask[e]);
            if (si[e] * 64 + lane >= C::TP) smask[e] = 0u;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) er[e][i] = s_x ? xsr[i] : wsr[i];
        const int ch = (si[e] - SX) * 64 + lane;                 // channel of the tile
        ebase[e] = s_x ? (unsigned)pix : ch < C::TQ ? (unsigned)(q0 + ch) : OOB;
    }

    // the K tile issued next: its block, its tap's row and column
    int kn = 0, blk = 0, tr = 0, tc = 0;
    auto dma = [&](int stage) {
        const unsigned sb = lds0 + (unsigned)(stage * STAGE);
        const int tpix = tr * a.W + tc;
        const bool on = kn < g.nkt;
        const unsigned bit = on ? 1u << (tr * a.k + tc) : 0u;
        const unsigned step = (unsigned)tpix * g.pitch + (unsigned)(blk * C::XROW);
#pragma unroll
        for (int i = 0; i < NXI; ++i)
            f8_dma16(xr, sb + (unsigned)((wave * NXI + i) * 1024), (xmask[i] & (blk * 128 + xch[i] < a.Cin ? bit : 0u)) ? xoff[i] + step : OOB);
        const unsigned wk = on ? woff + (unsigned)kn * 128u : OOB;
#pragma unroll
        for (int i = 0; i < NWI; ++i) f8_dma16(wr, sb + (unsigned)(XB + (wave * NWI + i) * 1024), wk + (unsigned)i * 8u * row_bytes);
#pragma unroll
        for (int e = 0; e < NSI; ++e) {
            const bool s_x = si[e] < SX;
            const unsigned es = s_x ? (unsigned)blk * g.plane + (unsigned)tpix : (unsigned)(kn * g.rows);
            const bool eon = s_x ? (smask[e] & bit) != 0u : on && ebase[e] != OOB;
            f8_dma_u8(er[e], sb + (unsigned)(XB + WB + si[e] * 256), eon ? ebase[e] + es : OOB);
        }
        ++kn;
        tc = tc + 1 == a.k ? 0 : tc + 1;
        tr = tc != 0 ? tr : tr + 1 == a.k ? 0 : tr + 1;
        blk += tc == 0 && tr == 0 ? 1 : 0;
    };

    f32x4_t acc[NI][NJ];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    const int frow = lane & 15, q = lane >> 4;
    const int s0 = (q ^ (frow & 7)) << 4, s1 = ((q + 4) ^ (frow & 7)) << 4;
    const int a_off = XB + (wq * NI * 16 + frow) * 128, b_off = (wp * NJ * 16 + frow) * (ROUNDED ? 256 : 128);
    const int as_off = XB + WB + (SX * 64 + wq * NI * 16 + frow) * 4, bs_off = (RAW ? C::TP * 128 : XB + WB) + (wp * NJ * 16 + frow) * 4;

    auto frag = [&](const char *p) { return f8_frag(*(const int4 *)(p + s0), *(const int4 *)(p + s1)); };
    // Fragments of a tile: all pixels', and the channels' where there are few of them (PRE), before the next DMA is issued,
    // which then runs under the reads' latency.
    constexpr int PRE = NI <= 2 ? NI : 1;
    i32x8_t b[NJ], w[PRE];
    bf16x8_t bb[EXACT ? NJ : 1][4];                              // 32-bit outputs: the same fragments, scaled, as bf16
    int bs[NJ], ws[PRE];
    auto load_w = [&](const char *base, int i, i32x8_t &f, int &e) {
        f = frag(base + a_off + i * 2048);
        e = *(const int *)(base + as_off + i * 64);
    };
    auto load = [&](const char *base, const char *xbase) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            if constexpr (ROUNDED) {
#pragma unroll
                for (int h = 0; h < 4; ++h) bb[j][h] = *(const bf16x8_t *)(xbase + b_off + j * 4096 + (((2 * q + (h & 1) + (h & 2) * 4) ^ frow) << 4));
            } else {
                b[j] = frag(xbase + b_off + j * 2048);
                bs[j] = *(const int *)(xbase + bs_off + j * 64);
            }
        }
#pragma unroll
        for (int i = 0; i < PRE; ++i) load_w(base, i, w[i], ws[i]);
    };
    // RAW: tile kt's pixels t / 8, t / 8 + 8 NW, ...: 16 channels a thread.  For 32-bit outputs the values go back as scaled bf16
    // numbers to where they were, once for all waves.
    char *xq = smem + NSTAGE * STAGE;
    auto quantize = [&](char *base, char *to) {
#pragma unroll
        for (int n = 0; n < C::TP / (8 * C::NW); ++n) {
            const int row = n * 8 * C::NW + (t >> 3), part = t & 7;
            uint4 *lo = (uint4 *)(base + row * 256 + (((2 * part) ^ (row & 15)) << 4)), *hi = (uint4 *)(base + row * 256 + (((2 * part + 1) ^ (row & 15)) << 4));
            const uint4 l = *lo, h = *hi;
            uint32_t v[8] = {l.x, l.y, l.z, l.w, h.x, h.y, h.z, h.w};
            int e;
            const uint4 o = f8_quantize16(v, e);
            if constexpr (ROUNDED) {
                f8_words_to_bf16(o.x, o.y, e, *lo);
                f8_words_to_bf16(o.z, o.w, e, *hi);
            } else {
                *(uint4 *)(to + row * 128 + ((part ^ (row & 7)) << 4)) = o;
                if (part == 0) *(int *)(to + C::TP * 128 + row * 4) = e;
            }
        }
    };
    auto compute = [&](const char *base) {
        if constexpr (EXACT && !RAW)
#pragma unroll
            for (int j = 0; j < NJ; ++j) f8_to_bf16(b[j], bs[j], bb[j]);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            i32x8_t wf;
            int we;
            if (i < PRE) {
                wf = w[i < PRE ? i : 0];
                we = ws[i < PRE ? i : 0];
            } else {
                load_w(base, i, wf, we);
            }
            if constexpr (EXACT) {
                bf16x8_t wb[4];
                f8_to_bf16(wf, we, wb);
#pragma unroll
                for (int h = 0; h < 4; ++h)
#pragma unroll
                    for (int j = 0; j < NJ; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb[h], bb[j][h], acc[i][j], 0, 0, 0);
            } else {
#pragma unroll
                for (int j = 0; j < NJ; ++j) acc[i][j] = f8_mfma(wf, b[j], acc[i][j], we, bs[j]);
            }
        }
    };

    f8_dma_ready();
#pragma unroll
    for (int i = 0; i < NSTAGE - 1; ++i) dma(i);
    f8_vmcnt<C::PIECES * C::AHEAD>();
    __syncthreads();
    if constexpr (RAW) {
        quantize(smem, xq);
        __syncthreads();
    }
    int st = 0;
    for (int kt = 0; kt < g.nkt; ++kt) {
        char *base = smem + st * STAGE;
        const int next = st + 1 == NSTAGE ? 0 : st + 1;
        load(base, RAW && !ROUNDED ? xq + (kt & 1) * C::XQ : base);
        dma(st == 0 ? NSTAGE - 1 : st - 1);
        if constexpr (RAW) quantize(smem + next * STAGE, xq + (kt + 1 & 1) * C::XQ);
        compute(base);
        f8_vmcnt<C::PIECES * C::AHEAD>();
        __syncthreads();
        st = next;
    }
    f8_vmcnt<0>();
    __syncthreads();
    f8_epilogue<OT, NI, NJ>(a, acc, smem, wave, q0 + wq * NI * 16, p0 + wp * NJ * 16, lane);
}

template <typename OT, int NWQ, int NWP, int NI, int NJ, int NSTAGE, bool RAW = false> static int launch_f8_cfg(const F8Args &g, hipStream_t s) {
    typedef F8Tile<RAW, OT, NWQ, NWP, NI, NJ, NSTAGE> C;
    auto kern = conv_f8_kernel<RAW, OT, NWQ, NWP, NI, NJ, NSTAGE>;
    static LdsReserve reserved;
    if (const int rc = reserve_lds(reserved, (const void *)kern, C::LDS, "conv_f8")) return rc;
    const int ntq = (g.a.Cout + C::TQ - 1) / C::TQ;
    const long long grid = (long long)((g.a.P + C::TP - 1) / C::TP) * ntq;
    if (grid > 0x7fffffffLL) return fail(YMX_EUNSUPPORTED, "conv_f8: grid too large");
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(64 * C::NW), C::LDS, s, g, ntq);
    return check_launch("conv_f8");
}

// The tile, by how many there are.  Measured (us, batch x map, in -> out channels, window):
//   256 x 256, staggered (conv_blockscaled_wide.hip): 160 tiles and more (16 x 104^2 128 -> 256 3x3 stride 2: 25.2, 64 x 128 30.3)
//   128 ch x 128 px, eight waves, two workgroups a CU: from 300 tiles that are no more than a quarter wider than needed, bf16
//       outputs (64 x 26^2 144 -> 768 3x3 stride 2: 26.5, 64 x 128 38.4)
//   64 ch x 128 px, two stages, three workgroups a CU: from 512 tiles.  64 x 104^2 128 -> 64 1x1: 48, in tiles of
//       128 x 128 75, of 64 x 64 82; up to 32 channels as 32 x 128 (64 x 208^2 64 -> 32 1x1: 142 against 170)
//   64 x 64, two stages, four workgroups a CU: from 200 (52^2 512 -> 1024 3x3: 30.8, 64 x 128 34.5)
//   64 x 64, four stages: fewer (26^2 512 -> 1024 3x3: 19.2, two stages 27.3)
//   64 x 32, four stages: where even that leaves half the CUs idle (13^2 512 -> 1024 3x3: 15.1, 64 x 64 18.0), and for
//       32-bit outputs, whose conversions weigh more, wherever there are few tiles (8 x 26^2 1024 -> 255 1x1: 12.3, 14.4)
enum class F8Shape { WIDE, T128x128, T64x128, T32x128, T64x64_TWO_STAGES, T64x64, T64x32 };
static F8Shape f8_shape(const F8Args &g) {
    if (conv_f8_wide(g)) return F8Shape::WIDE;
    const bool bf16 = g.a.out_dtype == YMX_BF16;
    const long long np = g.a.P, nq = (g.a.Cout + 63) / 64, n128 = (g.a.Cout + 127) / 128;
    const long long tiles = (np + 127) / 128 * nq;
    if (bf16 && n128 * 8 <= nq * 5 && (np + 127) / 128 * n128 >= 300) return F8Shape::T128x128;
    if (tiles >= 512) return g.a.Cout <= 32 ? F8Shape::T32x128 : F8Shape::T64x128;
    if (bf16 && tiles >= 200) return F8Shape::T64x64_TWO_STAGES;
    return !bf16 || (np + 63) / 64 * nq <= 128 ? F8Shape::T64x32 : F8Shape::T64x64;
}
template <typename OT> static int launch_f8_shape(const F8Args &g, hipStream_t s) {
    const F8Shape shape = f8_shape(g);
    if constexpr (sizeof(OT) == 2) {                             // (shapes that 32-bit outputs never take)
        if (shape == F8Shape::WIDE) return launch_conv_f8_wide(g, s);
        if (shape == F8Shape::T128x128) return launch_f8_cfg<OT, 4, 2, 2, 4, 2>(g, s);
        if (shape == F8Shape::T64x64_TWO_STAGES) return launch_f8_cfg<OT, 4, 1, 1, 4, 2>(g, s);
        if (shape == F8Shape::T64x64) return launch_f8_cfg<OT, 4, 1, 1, 4, 4>(g, s);
    }
    if (shape == F8Shape::T64x128) return launch_f8_cfg<OT, 2, 2, 2, 4, 2>(g, s);
    if (shape == F8Shape::T32x128) return launch_f8_cfg<OT, 2, 2, 1, 4, 2>(g, s);
    return launch_f8_cfg<OT, 4, 1, 1, 2, 4>(g, s);
}

// Whether a layer on a bf16 map quantises it in its own kernel, in tiles of 64 x 32.  Every tile of channels and every tap
// quantises its pixels again, so where there are few of them: 1x1 windows, up to 176 tiles of 64 x 64; up to 768 for 32-bit
// outputs, which save the waves' own conversions.  Measured (us, one launch against two): 13^2 1024 -> 512 11.8, 12.4; 26^2 256 ->
// 512 8.5, 10.9; 8 x 13^2 1024 -> 512 (176 tiles) 13.2, 13.6; 8 x 13^2 1024 -> 1024 (352) 19.7, 15.0; to fp32: 8 x 26^2 1024 -> 255
// 17.5, 21.4; 64 x 13^2 1024 -> 255 (676) 30.1, 33.2; 8 x 52^2 256 -> 255 (1352) 27.8, 26.1; 3x3: 13^2 512 -> 1024 25.8, 20.2.
bool conv_f8_raw(long long P, int Cout, int k, int out_dtype) {
    return k == 1 && (P + 63) / 64 * ((Cout + 63) / 64) <= (out_dtype == YMX_F32 ? 768 : 176);
}

// a: geometry of the convolution with x_ld = Cin; x = quantised map, or a bf16 one
// where conv_f8_raw says so; w = packed kernel.
static int f8_args(const ConvArgs &args, long long in_pix, F8Args &g) {
    g.a = args;
    g.a.x_ld = 1;
    g.taps = args.k * args.k;
    g.nkt = f8_tiles(args.k, args.Cin);
    g.rows = f8_rows(args.Cout);
    g.plane = (unsigned)f8_plane(in_pix);
    set_fastdiv((unsigned)g.taps, g.taps_m, g.taps_s);
    const bool raw = args.x_dtype == YMX_BF16;
    g.pitch = raw ? (unsigned)args.x_ld * 2u : (unsigned)args.Cin;
    const unsigned long long xb = raw ? ((unsigned long long)(in_pix - 1) * args.x_ld + args.Cin) * 2 : (unsigned long long)in_pix * args.Cin, wb = (unsigned long long)g.rows * g.nkt * 128;
    if (xb >= (1ull << 31) || wb >= (1ull << 31) || (unsigned long long)g.plane * ((args.Cin + 127) / 128) >= (1ull << 31))
        return fail(YMX_EUNSUPPORTED, "conv2d: more than 2 GiB of 8-bit input or kernel");
    g.a.x_bytes = (unsigned)xb;
    g.a.w_bytes = (unsigned)wb;
    g.xs = raw ? nullptr : (const char *)args.x + f8_map_bytes(in_pix, args.Cin);
    g.xs_bytes = raw ? 0u : g.plane * (unsigned)((args.Cin + 127) / 128);
    g.ws = (const char *)args.w + wb;
    g.ws_bytes = (unsigned)(g.nkt * g.rows);
    if (args.res && args.out_dtype == YMX_BF16) {
        const long long rb = ((long long)(args.P - 1) * args.res_ld + args.Cout) * 2;
        g.a.res_bytes = rb < 0x80000000LL ? (unsigned)rb : 0u;
    }
    return YMX_OK;
}
int launch_conv_f8(const ConvArgs &args, long long in_pix, hipStream_t s) {
    F8Args g;
    if (const int rc = f8_args(args, in_pix, g)) return rc;
    if (args.x_dtype == YMX_BF16) return args.out_dtype == YMX_BF16 ? launch_f8_cfg<bf16_t, 4, 1, 1, 2, 3, true>(g, s) : launch_f8_cfg<float, 4, 1, 1, 2, 3, true>(g, s);
    return args.out_dtype == YMX_BF16 ? launch_f8_shape<bf16_t>(g, s) : launch_f8_shape<float>(g, s);
}
const char *conv_f8_tile(const ConvArgs &args, long long in_pix) {
    F8Args g;
    if (f8_args(args, in_pix, g)) return nullptr;
    if (args.x_dtype == YMX_BF16) return "64x32 raw";
    switch (f8_shape(g)) {
        case F8Shape::WIDE: return conv_f8_wide_tile(g);
        case F8Shape::T128x128: return "128x128";
        case F8Shape::T64x128: return "64x128";
        case F8Shape::T32x128: return "32x128";
        case F8Shape::T64x64_TWO_STAGES: return "64x64, two stages";
        case F8Shape::T64x64: return "64x64";
        default: return "64x32";
    }
}

}  // namespace ymx
