// Counter-based random words: Philox4x32 with 10 rounds (Salmon, Moraes, Dror and Shaw, "Parallel
// random numbers: as easy as 1, 2, 3", 2011).  Words 4 j .. 4 j + 3 of call `call` under `seed` are
// the output for the counter (j lo, j hi, call lo, call hi) and the key (seed lo, seed hi), so a
// mask is a function of (seed, call, element) alone: the backward pass computes it again and
// nothing is stored.
#pragma once
#include "common.h"

namespace ymx {

// 10 x (two 32 x 32 -> 64 bit products and four xors) for four words.
__device__ __forceinline__ uint4 philox4(unsigned long long j, const uint4 &sc) {      // sc = (seed lo, seed hi, call lo, call hi)
    uint32_t c0 = (uint32_t)j, c1 = (uint32_t)(j >> 32), c2 = sc.z, c3 = sc.w, k0 = sc.x, k1 = sc.y;
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const unsigned long long p0 = (unsigned long long)c0 * 0xD2511F53u, p1 = (unsigned long long)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)p1;
        c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return uint4{c0, c1, c2, c3};
}

// Dropout of one launch.  state (device memory) = (seed, call); an element is kept iff its word
// is >= threshold = floor(rate * 2^32), and kept values are multiplied by 1 / (1 - rate).
struct DropArgs {
    const uint32_t *state;
    uint32_t threshold;
    float keep_scale;
};

// Which of V consecutive elements from linear index i0 (a multiple of V where V > 1) are kept.  The caller selects (a
// dropped element is 0 whatever it held).
template <int V> __device__ __forceinline__ void drop_keep(const DropArgs &d, const uint4 &sc, unsigned long long i0, bool (&keep)[V]) {
    if constexpr (V >= 4) {
#pragma unroll
        for (int q = 0; q < V / 4; ++q) {
            const uint4 w = philox4((i0 >> 2) + q, sc);
            keep[4 * q] = w.x >= d.threshold;
            keep[4 * q + 1] = w.y >= d.threshold;
            keep[4 * q + 2] = w.z >= d.threshold;
            keep[4 * q + 3] = w.w >= d.threshold;
        }
    } else {
        static_assert(V == 1, "vectors of 1, 4 or 8 elements");
        const uint4 w = philox4(i0 >> 2, sc);
        const uint32_t lo = (i0 & 1) ? w.y : w.x, hi = (i0 & 1) ? w.w : w.z;
        keep[0] = ((i0 & 2) ? hi : lo) >= d.threshold;
    }
}

// V consecutive elements of a map as floats: 16-byte accesses for whole vectors (streaming stores: group norm over 16 x
// 208^2 x 64 forward 79.5 -> 74.4 us, backward 105.8 -> 100.4), scalar ones for V = 1.
template <typename T, int V> struct vec_io;
template <> struct vec_io<bf16_t, 8> {
    typedef uint4 raw;
    __device__ static __forceinline__ raw load(const bf16_t *p) { return *(const uint4 *)p; }
    __device__ static __forceinline__ void unpack(const raw &r, float (&v)[8]) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    __device__ static __forceinline__ uint32_t pack(float lo, float hi) {          // one v_cvt_pk_bf16_f32
        typedef __bf16 pair_t __attribute__((ext_vector_type(2)));
        const f32x2_t v = {lo, hi};
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, pair_t));
    }
    __device__ static __forceinline__ void store(bf16_t *p, const float (&v)[8]) {
        store_stream16(p, pack(v[0], v[1]), pack(v[2], v[3]), pack(v[4], v[5]), pack(v[6], v[7]));
    }
};
template <> struct vec_io<bf16_t, 4> {
    typedef uint2 raw;
    __device__ static __forceinline__ raw load(const bf16_t *p) { return *(const uint2 *)p; }
    __device__ static __forceinline__ void unpack(const raw &r, float (&v)[4]) {
        v[0] = __uint_as_float(r.x << 16);
        v[1] = __uint_as_float(r.x & 0xffff0000u);
        v[2] = __uint_as_float(r.y << 16);
        v[3] = __uint_as_float(r.y & 0xffff0000u);
    }
    __device__ static __forceinline__ void store(bf16_t *p, const float (&v)[4]) {
        *(uint2 *)p = uint2{vec_io<bf16_t, 8>::pack(v[0], v[1]), vec_io<bf16_t, 8>::pack(v[2], v[3])};
    }
};
template <> struct vec_io<float, 4> {
    typedef float4 raw;
    __device__ static __forceinline__ raw load(const float *p) { return *(const float4 *)p; }
    __device__ static __forceinline__ void unpack(const raw &r, float (&v)[4]) { v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w; }
    __device__ static __forceinline__ void store(float *p, const float (&v)[4]) { store_stream16(p, v[0], v[1], v[2], v[3]); }
};
template <typename T> struct vec_io<T, 1> {
    typedef T raw;
    __device__ static __forceinline__ raw load(const T *p) { return *p; }
    __device__ static __forceinline__ void unpack(const raw &r, float (&v)[1]) { v[0] = elem<T>::load(&r); }
    __device__ static __forceinline__ void store(T *p, const float (&v)[1]) { elem<T>::store(p, v[0]); }
};

}  // namespace ymx
