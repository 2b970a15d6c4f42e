// Shared by the 8-bit block-scaled convolution kernels: argument block, exponent DMA, fragments, epilogue.
#pragma once
#include <type_traits>

#include "conv_epilogue.h"

namespace ymx {

typedef __attribute__((ext_vector_type(8))) int i32x8_t;

struct F8Args {
    ConvArgs a;                  // x_ld = 1: pixel_geometry then counts pixels
    const void *xs, *ws;         // exponents of the map [block][plane] and of the kernel [K tile][rows], bytes
    unsigned xs_bytes, ws_bytes;
    unsigned plane;              // pixels of the map, rounded up to 4
    unsigned pitch;              // bytes from pixel to pixel of the map
    int rows, nkt, taps;         // padded output channels, K tiles, filter taps
    unsigned taps_m, taps_s;     // fastdiv of the taps
};

template <int N> __device__ __forceinline__ void f8_vmcnt() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// One LDS-DMA wave-instruction: lane l's 16 bytes (4 bytes; one byte, zero-extended to 4) at buffer offset voff land at
// lds_addr + 16 l (4 l), zeros where voff is out of range.  Inline asm on purpose, see lds_dma16; the caller counts them
// (vmcnt) and waits before a barrier.  M0 is not restored: the compiler reserves it and sets it before each use of its own.
// That, and one wait state instead of five, makes 30 cycles less of the issue of each; operands are scalars computed long
// before (f8_dma_ready before the first).
#define YMX_F8_DMA(NAME, OP)                                                                                     \
    __device__ __forceinline__ void NAME(const i32x4_t rsrc, unsigned lds_addr, unsigned voff) {                 \
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\t" OP " %0, %2, 0 offen lds"                                \
                     :: "v"(voff), "s"(lds_addr), "s"(rsrc) : "memory");                                         \
    }
YMX_F8_DMA(f8_dma16, "buffer_load_dwordx4")
YMX_F8_DMA(f8_dma4, "buffer_load_dword")
YMX_F8_DMA(f8_dma_u8, "buffer_load_ubyte")
#undef YMX_F8_DMA
__device__ __forceinline__ void f8_dma_ready() { asm volatile("s_nop 7" ::: "memory"); }

__device__ __forceinline__ i32x8_t f8_frag(const int4 &lo, const int4 &hi) {
    return i32x8_t{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
}
// 16 x 16 results += 128 products each, scaled by the row's and the column's power of two.
__device__ __forceinline__ f32x4_t f8_mfma(const i32x8_t &w, const i32x8_t &x, const f32x4_t &c, int ws, int xs) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 0, 0, 0, ws, 0, xs);
}

// Two words of e4m3 numbers times 2^(exponent byte - 127) as eight bf16 ones.  Exact down to 2^-126, bf16 having e4m3's
// digits and fp32's exponents.
__device__ __forceinline__ void f8_words_to_bf16(uint32_t a, uint32_t b, int exponent, uint4 &o) {
    const float f = __uint_as_float((uint32_t)exponent << 23);
    o.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, f, false));
    o.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, f, true));
    o.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, f, false));
    o.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, f, true));
}
// A fragment's 32 values, eight at a time, in the order they lie in.
__device__ __forceinline__ void f8_to_bf16(const i32x8_t &v, int exponent, bf16x8_t (&o)[4]) {
#pragma unroll
    for (int h = 0; h < 4; ++h) {
        uint4 w;
        f8_words_to_bf16((uint32_t)v[2 * h], (uint32_t)v[2 * h + 1], exponent, w);
        o[h] = __builtin_bit_cast(bf16x8_t, w);
    }
}

// Rows of the fp32 accumulator image in LDS (see conv_epilogue.h for the layout) with 32-bit outputs, whose residual is
// 32-bit too, and of any output whose channel count or pixel stride is no multiple of 8 (the 255 channels
// of the logits): there a lane takes a few neighbouring channels of a pixel, whose address need not be aligned.
template <typename OT, int NI, int NJ>
__device__ __forceinline__ void f8_epilogue_rows(const ConvArgs &a, f32x4_t (&acc)[NI][NJ], char *tbase, int cbase, int pbase, int lane) {
    constexpr int HQ = NI * 16 < 64 ? NI * 16 : 64, NH = NI * 16 / HQ, SLOTS = HQ / 4, LPP = SLOTS / 2, PPI = 64 / LPP, NPASS = 16 * NJ / PPI;
    OT *__restrict__ y = (OT *)a.y;
    const OT *__restrict__ res = (const OT *)a.res;
    const bool vec = sizeof(OT) == 4 && epi_vec_ok(a);
    auto rows = [&](auto act_tag) {
        constexpr int ACT = decltype(act_tag)::value;
#pragma unroll
        for (int half = 0; half < NH; ++half) {
#pragma unroll
            for (int il = 0; il < HQ / 16; ++il) {
                const int slot = il * 4 + (lane >> 4);
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const int px = j * 16 + (lane & 15);
                    *(f32x4_t *)(tbase + px * (HQ * 4) + ((slot ^ (px & (SLOTS - 1))) << 4)) = acc[half * (HQ / 16) + il][j];
                }
            }
            const int c0 = cbase + half * HQ;
            if (sizeof(OT) == 4 && vec) {
                const int sl = lane % LPP, co = c0 + sl * 8;
                float sc[8], sh[8];
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    const bool in = co + r < a.Cout;
                    sc[r] = in ? (a.scale ? a.scale[co + r] : 1.0f) : 0.0f;
                    sh[r] = (in && a.shift) ? a.shift[co + r] : 0.0f;
                }
                constexpr int U = NPASS < 4 ? NPASS : 4;             // residuals of U passes in flight
                for (int n0 = 0; n0 < NPASS; n0 += U) {
                    float4 q[U][2];
                    if (res)
#pragma unroll
                        for (int u = 0; u < U; ++u) {
                            const int p = pbase + (n0 + u) * PPI + lane / LPP;
                            const float *rp = (const float *)res + (size_t)p * a.res_ld + co;
                            if (p < a.P && co < a.Cout) { q[u][0] = *(const float4 *)rp; q[u][1] = *(const float4 *)(rp + 4); }
                        }
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const int px = (n0 + u) * PPI + lane / LPP, p = pbase + px, sw = px & (SLOTS - 1);
                        const char *row = tbase + px * (HQ * 4);
                        const float4 v0 = *(const float4 *)(row + (((2 * sl) ^ sw) << 4));
                        const float4 v1 = *(const float4 *)(row + (((2 * sl + 1) ^ sw) << 4));
                        float v[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
                        if (p >= a.P || co >= a.Cout) continue;
#pragma unroll
                        for (int r = 0; r < 8; ++r) v[r] = act_c<ACT>(affine_f(v[r], sc[r], sh[r]));
                        if (res) {
                            const float4 q0 = q[u][0], q1 = q[u][1];
                            v[0] = __fadd_rn(v[0], q0.x); v[1] = __fadd_rn(v[1], q0.y); v[2] = __fadd_rn(v[2], q0.z); v[3] = __fadd_rn(v[3], q0.w);
                            v[4] = __fadd_rn(v[4], q1.x); v[5] = __fadd_rn(v[5], q1.y); v[6] = __fadd_rn(v[6], q1.z); v[7] = __fadd_rn(v[7], q1.w);
                        }
                        float *yp = (float *)y + (size_t)p * a.y_ld + co;
                        store_stream16(yp, v[0], v[1], v[2], v[3]);
                        store_stream16(yp + 4, v[4], v[5], v[6], v[7]);
                    }
                }
            } else {
                // two bf16 or four fp32 channels a lane, one access at any address; the last ones of a pixel one by one (6 x 122^2
                // 128 -> 959 3x3 with shortcut 287 us, a channel a lane 514, 960 channels 190; 64 x 52^2 1024 -> 255 to fp32 161, 184)
                constexpr int CH = sizeof(OT) == 4 ? 4 : 2, HL = HQ / CH, PP = 64 / HL, N = 16 * NJ / PP;
                constexpr int B = N % (16 / CH) == 0 ? 16 / CH : N % 4 == 0 ? 4 : N % 2 == 0 ? 2 : 1;
                struct __attribute__((packed, aligned(sizeof(OT)))) few_t { OT v[CH]; };
                typedef float tvec_t __attribute__((ext_vector_type(CH)));
                typedef std::conditional_t<sizeof(OT) == 4, tvec_t, uint32_t> word_t;
                typedef word_t any_word_t __attribute__((aligned(sizeof(OT))));
                const int cl = lane % HL * CH, co = c0 + cl, nc = min(a.Cout - co, CH);
                float sc[CH], sh[CH];
#pragma unroll
                for (int r = 0; r < CH; ++r) {
                    sc[r] = r < nc && a.scale ? a.scale[co + r] : 1.0f;
                    sh[r] = r < nc && a.shift ? a.shift[co + r] : 0.0f;
                }
                for (int n0 = 0; n0 < N; n0 += B) {
                    few_t q[B];                                          // residuals of B passes in flight
                    if (res)
#pragma unroll
                        for (int u = 0; u < B; ++u) {
                            const int p = pbase + (n0 + u) * PP + lane / HL;
                            const OT *rp = res + (size_t)p * a.res_ld + co;
                            if (p >= a.P) continue;
                            if (nc >= CH) q[u] = *(const few_t *)rp;
                            else
#pragma unroll
                                for (int r = 0; r < CH - 1; ++r)
                                    if (r < nc) q[u].v[r] = rp[r];
                        }
#pragma unroll
                    for (int u = 0; u < B; ++u) {
                        const int px = (n0 + u) * PP + lane / HL, p = pbase + px;
                        const tvec_t t = *(const tvec_t *)(tbase + px * (HQ * 4) + (((cl >> 2) ^ (px & (SLOTS - 1))) << 4) + (cl & 3) * 4);
                        if (p >= a.P || nc <= 0) continue;
                        tvec_t v;
#pragma unroll
                        for (int r = 0; r < CH; ++r) {
                            v[r] = act_c<ACT>(affine_f(t[r], sc[r], sh[r]));
                            if (res) v[r] = __fadd_rn(v[r], elem<OT>::load(&q[u].v[r]));
                        }
                        OT *yp = y + (size_t)p * a.y_ld + co;
                        if (nc >= CH) {
                            if constexpr (sizeof(OT) == 4) *(any_word_t *)yp = v;
                            else *(any_word_t *)yp = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, epi_bf16x2_t));
                        } else
#pragma unroll
                            for (int r = 0; r < CH - 1; ++r)
                                if (r < nc) elem<OT>::store(yp + r, v[r]);
                    }
                }
            }
        }
    };
    if (a.act == YMX_ACT_MISH) rows(std::integral_constant<int, YMX_ACT_MISH>{});
    else if (a.act == YMX_ACT_LEAKY) rows(std::integral_constant<int, YMX_ACT_LEAKY>{});
    else rows(std::integral_constant<int, YMX_ACT_NONE>{});
}

// The end of a tile, after every wave's last LDS read: acc -> finished rows, by way of the wave's own part of LDS.
template <typename OT, int NI, int NJ>
__device__ __forceinline__ void f8_epilogue(const ConvArgs &a, f32x4_t (&acc)[NI][NJ], char *smem, int wave, int cbase, int pbase, int lane) {
    typedef EpiGeom<NI, 64, 16 * NJ> Epi;
    char *tbase = smem + wave * Epi::LDS_BYTES;
    constexpr bool WIDE = sizeof(OT) == 2 && NJ >= 3;
    if (WIDE && epi_vec_ok(a) && (a.res == nullptr || a.res_bytes != 0)) {
      if constexpr (WIDE) {
        epi_u32x4_t rpre[Epi::NH][Epi::NPASS];
        if (epi_res_pre(a)) {
            epi_load_res<NI, 64, 16 * NJ>(a, 0, cbase, pbase, lane, rpre[0]);
        } else {
#pragma unroll
            for (int n = 0; n < Epi::NPASS; ++n) rpre[0][n] = epi_u32x4_t{0u, 0u, 0u, 0u};
        }
        epi_run<bf16_t, NI, NJ>(a, acc, tbase, cbase, pbase, lane, rpre);
      }
    } else {
        f8_epilogue_rows<OT, NI, NJ>(a, acc, tbase, cbase, pbase, lane);
    }
}

bool conv_f8_wide(const F8Args &g);
int launch_conv_f8_wide(const F8Args &g, hipStream_t s);
const char *conv_f8_wide_tile(const F8Args &g);

}  // namespace ymx
