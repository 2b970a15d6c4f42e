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
// bf16 instructions, whose products and sums are exact to fp32 (e4m3 numbers are bf16 numbers), at half
// the rate, the block's sum being scaled by v_ldexp on its way into the accumulator.
//
// Quantised map (ymx_quantize_blocks):  [pixel][C] e4m3 bytes (padded to 256), then
// [pixel][4 ceil(nb / 4)] exponent bytes (k + 127; nb = ceil(C / 128)).
// Packed kernel (ymx_pack_weights):  [channel, padded to 256][K tile][128] bytes, then
// [K tile][channel] exponents as dwords.  K tile = (block of 128 input channels) * taps + tap, so
// that the taps of a block, which read the same pixels, follow one another; channels past the
// input's last are zeros.
#include <algorithm>
#include <type_traits>

#include "conv_epilogue.h"

namespace ymx {

typedef __attribute__((ext_vector_type(8))) int i32x8_t;

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
static int f8_scale_ld(int C) { return ((C + 127) / 128 + 3) / 4 * 4; }
size_t quant_bytes(long long n_pix, int C) { return f8_map_bytes(n_pix, C) + (size_t)n_pix * f8_scale_ld(C); }

// GL lanes of 8 channels share a block of one pixel (16 lanes = 128 channels; 8 or 4 where the map has no more
// than 64 or 32).  Reads 2 or 4 bytes a value, writes one: bound by memory.
template <typename T, int GL>
__global__ void __launch_bounds__(256)
quantize_kernel(const T *__restrict__ x, int x_ld, unsigned char *__restrict__ q, unsigned char *__restrict__ scales, long long n_pix,
                int C, int nb, int s_ld) {
    const long long groups = n_pix * nb;
    const int gl = threadIdx.x % GL;
    for (long long g = ((long long)blockIdx.x * 256 + threadIdx.x) / GL; g < groups; g += (long long)gridDim.x * (256 / GL)) {
        const long long p = nb == 1 ? g : g / nb;
        const int blk = nb == 1 ? 0 : (int)(g - p * nb);
        const int c = blk * 128 + gl * 8;
        const bool on = c < C;
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
        if (gl == 0) scales[(size_t)p * s_ld + blk] = (unsigned char)(k + 127);
    }
}

int launch_quantize(const void *x, int x_ld, void *q, long long n_pix, int C, int dtype, hipStream_t s) {
    const int nb = (C + 127) / 128;
    unsigned char *sc = (unsigned char *)q + f8_map_bytes(n_pix, C);
    auto go = [&](auto ttag, auto gtag) {
        typedef decltype(ttag) T;
        constexpr int GL = decltype(gtag)::value;
        const long long wgs = (n_pix * nb * GL + 255) / 256;
        hipLaunchKernelGGL((quantize_kernel<T, GL>), dim3((unsigned)std::min<long long>(wgs, 16384)), dim3(256), 0, s, (const T *)x, x_ld,
                           (unsigned char *)q, sc, n_pix, C, nb, f8_scale_ld(C));
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
size_t packed_f8_bytes(int k, int Cin, int Cout) { return (size_t)f8_rows(Cout) * f8_tiles(k, Cin) * (128 + 4); }

// One thread per (output channel, K tile); neighbouring threads read neighbouring channels.
__global__ void __launch_bounds__(256)
pack_f8_kernel(const float *__restrict__ w, unsigned char *__restrict__ out, uint32_t *__restrict__ scales, int taps, int Cin, int Cout, int rows, int nkt) {
    const int co = blockIdx.x * 256 + threadIdx.x, kt = blockIdx.y;
    const int blk = kt / taps, tap = kt - blk * taps;
    const int c0 = blk * 128, nc = min(128, Cin - c0);
    const float *__restrict__ src = w + ((size_t)tap * Cin + c0) * Cout + co;
    uint32_t m = 0;
    if (co < Cout)
        for (int c = 0; c < nc; ++c) m = max(m, f8_mag(src[(size_t)c * Cout]));
    const int k = f8_exponent(m);
    const float f = f8_factor(k);
    uint32_t *dst = (uint32_t *)(out + ((size_t)co * nkt + kt) * 128);
    for (int c = 0; c < 128; c += 4) {
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (co < Cout && c + i < nc) ? f8_scaled(src[(size_t)(c + i) * Cout], f) : 0.0f;
        dst[c >> 2] = f8_pack4(v[0], v[1], v[2], v[3]);
    }
    scales[(size_t)kt * rows + co] = (uint32_t)(k + 127);
}

int launch_pack_f8(const float *w_hwio, void *packed, int k, int Cin, int Cout, hipStream_t s) {
    const int rows = f8_rows(Cout), nkt = f8_tiles(k, Cin);
    unsigned char *out = (unsigned char *)packed;
    hipLaunchKernelGGL(pack_f8_kernel, dim3(rows / 256, nkt), dim3(256), 0, s, w_hwio, out, (uint32_t *)(out + (size_t)rows * nkt * 128), k * k, Cin, Cout,
                       rows, nkt);
    return check_launch("pack_weights");
}

// ---- the product ----------------------------------------------------------------------------------
// One LDS-DMA wave-instruction of dwords: lane l's 4 bytes land at lds_addr + 4 l (see lds_dma16).
__device__ __forceinline__ void lds_dma4(const i32x4_t rsrc, unsigned lds_addr, unsigned voff) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\t"
                 "s_mov_b32 m0, %2\n\t"
                 "s_nop 4\n\t"
                 "buffer_load_dword %1, %3, 0 offen lds\n\t"
                 "s_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "v"(voff), "s"(lds_addr), "s"(rsrc)
                 : "memory");
}
template <int N> __device__ __forceinline__ void f8_vmcnt() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

struct F8Args {
    ConvArgs a;                  // x_ld = 1: pixel_geometry then counts pixels; k_m, k_s as in ConvArgs
    const void *xs, *ws;         // exponents of the map and of the kernel
    unsigned xs_bytes, ws_bytes;
    int s_ld, rows, nkt, taps;   // exponent bytes per pixel, padded output channels, K tiles
    unsigned taps_m, taps_s;     // fastdiv of the taps
};

// A fragment's 32 values as bf16, which holds every e4m3 number: eight at a time, in the order they lie in.
__device__ __forceinline__ void f8_to_bf16(const i32x8_t &v, bf16x8_t (&o)[4]) {
#pragma unroll
    for (int h = 0; h < 4; ++h) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            w[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)v[2 * h + i], 1.0f, false));
            w[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)v[2 * h + i], 1.0f, true));
        }
        o[h] = __builtin_bit_cast(bf16x8_t, uint4{w[0], w[1], w[2], w[3]});
    }
}

// Finished rows from a wave's accumulators (16 NI channels x 64 pixels, a lane holding 4 channels of one
// pixel per block), by way of a private LDS image as in conv_epilogue.h.  The residual has the output's type.
template <typename OT, int NI>
__device__ __forceinline__ void f8_epilogue(const ConvArgs &a, f32x4_t (&acc)[NI][4], char *tbase, int cbase, int pbase, int lane) {
    constexpr int HQ = NI * 16 < 64 ? NI * 16 : 64, NH = NI * 16 / HQ, SLOTS = HQ / 4, LPP = SLOTS / 2, PPI = 64 / LPP, NPASS = 64 / PPI;
    OT *__restrict__ y = (OT *)a.y;
    const OT *__restrict__ res = (const OT *)a.res;
    const int sl = lane % LPP;
    const bool vec = (a.Cout & 7) == 0 && (a.y_ld & 7) == 0 && ((uintptr_t)y & 15) == 0 &&
                     (res == nullptr || ((a.res_ld & 7) == 0 && ((uintptr_t)res & 15) == 0));
    auto rows = [&](auto act_tag, auto vec_tag) {
        constexpr int ACT = decltype(act_tag)::value;
        constexpr bool VEC = decltype(vec_tag)::value;
#pragma unroll
        for (int half = 0; half < NH; ++half) {
#pragma unroll
            for (int il = 0; il < HQ / 16; ++il) {
                const int slot = il * 4 + (lane >> 4);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int px = j * 16 + (lane & 15);
                    *(f32x4_t *)(tbase + px * (HQ * 4) + ((slot ^ (px & (SLOTS - 1))) << 4)) = acc[half * (HQ / 16) + il][j];
                }
            }
            const int co = cbase + half * HQ + sl * 8;
            float sc[8], sh[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                const bool in = co + r < a.Cout;
                sc[r] = in ? (a.scale ? a.scale[co + r] : 1.0f) : 0.0f;
                sh[r] = (in && a.shift) ? a.shift[co + r] : 0.0f;
            }
#pragma unroll 2
            for (int n = 0; n < NPASS; ++n) {
                const int px = n * PPI + lane / LPP, p = pbase + px;
                const char *row = tbase + px * (HQ * 4);
                const int sw = px & (SLOTS - 1);
                const float4 v0 = *(const float4 *)(row + (((2 * sl) ^ sw) << 4));
                const float4 v1 = *(const float4 *)(row + (((2 * sl + 1) ^ sw) << 4));
                float v[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
                if (p >= a.P || co >= a.Cout) continue;
#pragma unroll
                for (int r = 0; r < 8; ++r) v[r] = act_c<ACT>(affine_f(v[r], sc[r], sh[r]));
                OT *yp = y + (size_t)p * a.y_ld + co;
                const OT *rp = res + (size_t)p * a.res_ld + co;
                if constexpr (VEC) {
                    if constexpr (sizeof(OT) == 2) {
                        if (res) {
                            const uint4 q = *(const uint4 *)rp;
                            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                v[2 * r] += __uint_as_float(w[r] << 16);
                                v[2 * r + 1] += __uint_as_float(w[r] & 0xffff0000u);
                            }
                        }
                        store_stream16(yp, pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3]), pack2_bf16(v[4], v[5]), pack2_bf16(v[6], v[7]));
                    } else {
                        if (res) {
                            const float4 q0 = *(const float4 *)rp, q1 = *(const float4 *)(rp + 4);
                            v[0] += q0.x; v[1] += q0.y; v[2] += q0.z; v[3] += q0.w;
                            v[4] += q1.x; v[5] += q1.y; v[6] += q1.z; v[7] += q1.w;
                        }
                        store_stream16(yp, v[0], v[1], v[2], v[3]);
                        store_stream16(yp + 4, v[4], v[5], v[6], v[7]);
                    }
                } else {
#pragma unroll
                    for (int r = 0; r < 8; ++r)
                        if (co + r < a.Cout) elem<OT>::store(yp + r, res ? v[r] + elem<OT>::load(rp + r) : v[r]);
                }
            }
        }
    };
    auto pick = [&](auto act_tag) {
        if (vec) rows(act_tag, std::true_type{});
        else rows(act_tag, std::false_type{});
    };
    if (a.act == YMX_ACT_MISH) pick(std::integral_constant<int, YMX_ACT_MISH>{});
    else if (a.act == YMX_ACT_LEAKY) pick(std::integral_constant<int, YMX_ACT_LEAKY>{});
    else pick(std::integral_constant<int, YMX_ACT_NONE>{});
}

// NWQ x NWP waves, each 16 NI channels x 64 pixels; K tiles of 128 channels of one tap through NSTAGE stages
// of LDS, filled by LDS-DMA NSTAGE - 1 tiles ahead, one barrier per tile.  Rows are 128 bytes (one pixel's or one
// channel's 128 values), the 16-byte chunk c of row r in slot c ^ (r & 7): the lanes that read one fragment then
// touch 16 different slots.  A lane's 32 values of a fragment are the chunks q and q + 4 of its row, q = lane / 16,
// for pixels and channels alike (the order inside a block does not matter: one exponent covers it).
template <typename OT, int NWQ, int NWP, int NI, int NSTAGE>
__global__ void __launch_bounds__(64 * NWQ * NWP, 2)
conv_f8_kernel(const F8Args g, const int ntile_q) {
    constexpr int NW = NWQ * NWP, TQ = NWQ * NI * 16, TP = NWP * 64, NJ = 4;
    constexpr int NXI = TP / 8 / NW, NWI = TQ / 8 / NW, NS = (TP + TQ) / 64;         // DMA instructions: rows per wave; exponents in all
    static_assert(TP % (8 * NW) == 0 && TQ % (8 * NW) == 0 && NS <= NW, "whole instructions per wave, one of exponents");
    constexpr int XB = TP * 128, WB = TQ * 128, STAGE = XB + WB + NS * 256, PIECES = NXI + NWI + 1;
    constexpr unsigned OOB = 0x80000000u;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const ConvArgs &a = g.a;
    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wq = wave % NWQ, wp = wave / NWQ;
    const int id = xcd_remap(blockIdx.x, gridDim.x);
    const int tq = id % ntile_q, tp = id / ntile_q;
    const int p0 = tp * TP, q0 = tq * TQ;
    const i32x4_t xr = make_rsrc(a.x, a.x_bytes), wr = make_rsrc(a.w, a.w_bytes);
    const i32x4_t xsr = make_rsrc(g.xs, g.xs_bytes), wsr = make_rsrc(g.ws, g.ws_bytes);
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char *)smem;

    const int srow = lane >> 3, chunk = (lane & 7) ^ srow;
    int xpix[NXI];
    unsigned xmask[NXI];
#pragma unroll
    for (int i = 0; i < NXI; ++i) pixel_geometry(a, p0 + (wave * NXI + i) * 8 + srow, xpix[i], xmask[i]);
    const unsigned woff = (unsigned)(q0 + wave * NWI * 8 + srow) * (unsigned)(g.nkt * 128) + (unsigned)chunk * 16u;
    const unsigned wstep = 8u * (unsigned)(g.nkt * 128);
    // exponents: instructions 0 .. TP/64 - 1 fetch a dword (four blocks) per pixel, the others a dword per channel;
    // waves past the last one repeat it
    const int si = min(wave, NS - 1);
    int spix = 0;
    unsigned smask = 0;
    if (si < TP / 64) pixel_geometry(a, p0 + si * 64 + lane, spix, smask);

    auto dma = [&](int kt, int stage) {
        const unsigned sb = lds0 + (unsigned)(stage * STAGE);
        const int blk = fastdiv(kt, g.taps_m, g.taps_s), tap = kt - blk * g.taps;
        const int tr = fastdiv(tap, a.k_m, a.k_s), tc = tap - tr * a.k;
        const int tpix = tr * a.W + tc;
        const bool on = kt < g.nkt;
        const unsigned bit = on ? 1u << tap : 0u;
        const int c = blk * 128 + chunk * 16;
        const unsigned cbit = c < a.Cin ? bit : 0u;
#pragma unroll
        for (int i = 0; i < NXI; ++i)
            lds_dma16(xr, sb + (unsigned)((wave * NXI + i) * 1024), (xmask[i] & cbit) ? (unsigned)(xpix[i] + tpix) * (unsigned)a.Cin + (unsigned)c : OOB);
#pragma unroll
        for (int i = 0; i < NWI; ++i)
            lds_dma16(wr, sb + (unsigned)(XB + (wave * NWI + i) * 1024), on ? woff + (unsigned)i * wstep + (unsigned)kt * 128u : OOB);
        unsigned so;
        i32x4_t sr;
        if (si < TP / 64) {
            so = (smask & bit) ? (unsigned)(spix + tpix) * (unsigned)g.s_ld + (unsigned)(blk & ~3) : OOB;
            sr = xsr;
        } else {
            so = on ? ((unsigned)kt * (unsigned)g.rows + (unsigned)(q0 + (si - TP / 64) * 64 + lane)) * 4u : OOB;
            sr = wsr;
        }
        lds_dma4(sr, sb + (unsigned)(XB + WB + si * 256), so);
    };

    f32x4_t acc[NI][NJ];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    const int frow = lane & 15, q = lane >> 4;
    const int s0 = (q ^ (frow & 7)) << 4, s1 = ((q + 4) ^ (frow & 7)) << 4;
    const int a_off = XB + (wq * NI * 16 + frow) * 128, b_off = (wp * 64 + frow) * 128;
    const int as_off = XB + WB + (TP + wq * NI * 16 + frow) * 4, bs_off = XB + WB + (wp * 64 + frow) * 4;

    auto frag = [&](const char *p) {
        const int4 lo = *(const int4 *)(p + s0), hi = *(const int4 *)(p + s1);
        return i32x8_t{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    };
    // 32-bit outputs: the same fragments as bf16 (exact), the block's sum scaled and added by the vector unit
    auto compute_exact = [&](int kt, int stage) {
        const char *base = smem + stage * STAGE;
        const int sh = (fastdiv(kt, g.taps_m, g.taps_s) & 3) * 8;
        bf16x8_t b[NJ][4];
        int bs[NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            f8_to_bf16(frag(base + b_off + j * 2048), b[j]);
            bs[j] = (int)((*(const uint32_t *)(base + bs_off + j * 64) >> sh) & 255u) - 254;
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            bf16x8_t w[4];
            f8_to_bf16(frag(base + a_off + i * 2048), w);
            const int4 ws = *(const int4 *)(base + XB + WB + (TP + (wq * NI + i) * 16 + q * 4) * 4);     // of the lane's four results
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int h = 0; h < 4; ++h) sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[h], b[j][h], sum, 0, 0, 0);
                acc[i][j][0] += __builtin_ldexpf(sum[0], ws.x + bs[j]);
                acc[i][j][1] += __builtin_ldexpf(sum[1], ws.y + bs[j]);
                acc[i][j][2] += __builtin_ldexpf(sum[2], ws.z + bs[j]);
                acc[i][j][3] += __builtin_ldexpf(sum[3], ws.w + bs[j]);
            }
        }
    };
    auto compute = [&](int kt, int stage) {
        if constexpr (sizeof(OT) == 4) return compute_exact(kt, stage);
        const char *base = smem + stage * STAGE;
        const int sh = (fastdiv(kt, g.taps_m, g.taps_s) & 3) * 8;
        i32x8_t b[NJ];
        int bs[NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            b[j] = frag(base + b_off + j * 2048);
            bs[j] = (int)(*(const uint32_t *)(base + bs_off + j * 64) >> sh);
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const i32x8_t w = frag(base + a_off + i * 2048);
            const int ws = *(const int *)(base + as_off + i * 64);
#pragma unroll
            for (int j = 0; j < NJ; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, b[j], acc[i][j], 0, 0, 0, ws, 0, bs[j]);
        }
    };

#pragma unroll
    for (int i = 0; i < NSTAGE - 1; ++i) dma(i, i);
    f8_vmcnt<PIECES * (NSTAGE - 2)>();
    __syncthreads();
    int st = 0;
    for (int kt = 0; kt < g.nkt; ++kt) {
        dma(kt + NSTAGE - 1, st == 0 ? NSTAGE - 1 : st - 1);
        compute(kt, st);
        f8_vmcnt<PIECES * (NSTAGE - 2)>();
        __syncthreads();
        st = st + 1 == NSTAGE ? 0 : st + 1;
    }
    f8_vmcnt<0>();
    __syncthreads();
    constexpr int EPI = 64 * (NI * 16 < 64 ? NI * 16 : 64) * 4;
    f8_epilogue<OT, NI>(a, acc, smem + wave * EPI, q0 + wq * NI * 16, p0 + wp * 64, lane);
}

template <typename OT, int NWQ, int NWP, int NI, int NSTAGE> static int launch_f8_cfg(const F8Args &g, hipStream_t s) {
    constexpr int TQ = NWQ * NI * 16, TP = NWP * 64, NW = NWQ * NWP;
    constexpr int PIPE = NSTAGE * ((TP + TQ) * 128 + (TP + TQ) / 64 * 256), EPI = NW * 64 * (NI * 16 < 64 ? NI * 16 : 64) * 4;
    constexpr int LDS = PIPE > EPI ? PIPE : EPI;
    auto kern = conv_f8_kernel<OT, NWQ, NWP, NI, NSTAGE>;
    static LdsReserve reserved;
    if (const int rc = reserve_lds(reserved, (const void *)kern, LDS, "conv_f8")) return rc;
    const int ntq = (g.a.Cout + TQ - 1) / TQ;
    const long long grid = (long long)((g.a.P + TP - 1) / TP) * ntq;
    if (grid > 0x7fffffffLL) return fail(YMX_EUNSUPPORTED, "conv_f8: grid too large");
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(64 * NW), LDS, s, g, ntq);
    return check_launch("conv_f8");
}

template <typename OT> static int launch_f8_shape(const F8Args &g, hipStream_t s) {
    const long long big = (long long)((g.a.P + 255) / 256) * ((g.a.Cout + 255) / 256);
    const long long mid = (long long)((g.a.P + 127) / 128) * ((g.a.Cout + 127) / 128);
    if constexpr (sizeof(OT) == 2)
        if (big >= 160) return launch_f8_cfg<OT, 2, 4, 8, 2>(g, s);
    if (mid >= 160) return launch_f8_cfg<OT, 2, 2, 4, 2>(g, s);
    return launch_f8_cfg<OT, 4, 1, 1, 4>(g, s);
}

// a: geometry of the convolution with x_ld = Cin; x = quantised map, w = packed kernel.
int launch_conv_f8(const ConvArgs &args, long long in_pix, hipStream_t s) {
    F8Args g;
    g.a = args;
    g.a.x_ld = 1;
    g.taps = args.k * args.k;
    g.nkt = f8_tiles(args.k, args.Cin);
    g.rows = f8_rows(args.Cout);
    g.s_ld = f8_scale_ld(args.Cin);
    set_fastdiv((unsigned)g.taps, g.taps_m, g.taps_s);
    const unsigned long long xb = (unsigned long long)in_pix * args.Cin, wb = (unsigned long long)g.rows * g.nkt * 128;
    if (xb >= (1ull << 31) || wb >= (1ull << 31) || (unsigned long long)in_pix * g.s_ld >= (1ull << 31))
        return fail(YMX_EUNSUPPORTED, "conv2d: more than 2 GiB of 8-bit input or kernel");
    g.a.x_bytes = (unsigned)xb;
    g.a.w_bytes = (unsigned)wb;
    g.xs = (const char *)args.x + f8_map_bytes(in_pix, args.Cin);
    g.xs_bytes = (unsigned)(in_pix * g.s_ld);
    g.ws = (const char *)args.w + wb;
    g.ws_bytes = (unsigned)((size_t)g.nkt * g.rows * 4);
    return args.out_dtype == YMX_BF16 ? launch_f8_shape<bf16_t>(g, s) : launch_f8_shape<float>(g, s);
}

}  // namespace ymx
