// Group norm over channels-last maps with an activation, dropout and a shortcut in the same pass,
// and its gradients.  x [B][P][C] dense (P pixels), G groups of D = C / G channels, N = P D:
//
//   forward   mean, var of every (sample, group);  r = 1 / sqrt(var + eps)
//             h = (x - mean) r,  t = gamma h + beta,  y = keep * act(t) / (1 - rate) + shortcut
//   backward  dt = keep * dy / (1 - rate) * act'(t)
//             dbeta = sum dt,  dgamma = sum dt h            (over samples and pixels)
//             S1 = sum gamma dt,  S2 = sum gamma dt h       (over one group)
//             dx = r (gamma dt - (S1 + h S2) / N)
//
// Everything here is bound by memory: about 20 operations per element forward and 35 backward
// against 4 and 6 bytes in bf16.  t, dt and the dropout mask are computed again where they are
// needed instead of being stored.
//
// Chunked form: the pixels of a sample are cut into chunks, a workgroup per chunk.  Pass 1 leaves one
// pair of numbers per (chunk, group) -- mean and centred sum of squares (in 64 bits), or S1 and S2 -- and, backward,
// one per (chunk, channel); every workgroup of pass 2 first joins the pairs of its sample (a few
// hundred, from L2), then reads the map again and writes.  Slab form: see gn_slab_kernel.  All sums
// are fp32 or wider, added in a fixed order: no result depends on the order workgroups run in.
#include <algorithm>
#include <type_traits>

#include "philox.h"

namespace ymx {

// Where a thread of the chunked kernels works: V channels from c0 of the pixels p, p + R, ... < p1 of sample b.  A
// workgroup covers wc channels from cb: whole groups, or (nsub > 1) one of the nsub parts of a group that
// is wider than 256 vectors.
struct GnWork {
    int cvb, R, nzb;             // channel vectors per workgroup, pixels side by side, channel blocks
    int nsub;                    // blocks per group where a group needs several, else 1
    int nchunk, per;             // chunks per sample, pixels per chunk
};
template <int V> struct GnPos {
    int b, chunk, cb, wc, cv, r, c0, p, p1;
    int g0, sub, D;              // first group, part of it, channels per group of this block
    bool on;
    __device__ __forceinline__ GnPos(const GnArgs &a, const GnWork &w, int first = 0) {
        int id = blockIdx.x - first;
        const int zb = id % w.nzb, W = w.cvb * V;
        id /= w.nzb;
        chunk = id % w.nchunk;
        b = id / w.nchunk;
        if (w.nsub > 1) {
            g0 = zb / w.nsub;
            sub = zb - g0 * w.nsub;
            cb = g0 * a.D + sub * W;
            D = wc = min(W, a.D - sub * W);
        } else {
            cb = zb * W;
            wc = min(W, a.C - cb);
            g0 = cb / a.D;
            sub = 0;
            D = a.D;
        }
        cv = threadIdx.x % w.cvb;
        r = threadIdx.x / w.cvb;
        c0 = cb + cv * V;
        on = r < w.R && cv * V < wc;
        p = chunk * w.per + r;
        p1 = min(a.P, (chunk + 1) * w.per);
    }
    __device__ __forceinline__ size_t pair(const GnArgs &a, const GnWork &w) const {      // of group g0 in the table of pairs
        return (((size_t)b * w.nchunk + chunk) * w.nsub + sub) * a.G + g0;
    }
};

// A sum of squares that rounding may have taken below zero; NaN stays NaN (an infinity in the map makes the variance one).
template <typename F> __device__ __forceinline__ F gn_squares(F v) { return v < (F)0 ? (F)0 : v; }
__device__ __forceinline__ double gn_rstd(double var, float eps) { return 1.0 / sqrt(gn_squares(var) + (double)eps); }
// Statistics for the backward pass: mean, 1 / sqrt(var + eps) and what their rounding left out.
__device__ __forceinline__ void gn_keep_stats(const GnArgs &a, int b, int g, double mean, double rstd) {
    const float m = (float)mean, r = (float)rstd;
    ((float4 *)a.stats)[(size_t)b * a.G + g] = float4{m, r, (float)(mean - m), (float)(rstd - r)};
}

// Calls use(p, load(p)) for p, p + R, ... < p1, U loads in flight at a time.
template <int U, typename L, typename F> __device__ __forceinline__ void gn_rows(int p, int p1, int R, L load, F use) {
    for (; p + (U - 1) * R < p1; p += U * R) {
        decltype(load(p)) v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = load(p + u * R);
#pragma unroll
        for (int u = 0; u < U; ++u) use(p + u * R, v[u]);
    }
    for (; p < p1; p += R) use(p, load(p));
}

// Sum over the D channels of a group of f(channel), every group of the workgroup's W channels handed to done(group,
// sum): a thread per group for narrow groups, a wave per group for wide ones.  `sum` returns a float2.
template <typename F, typename D2> __device__ __forceinline__ void gn_over_groups(int W, int D, F f, D2 done) {
    const int ng = W / D;
    if (D <= 16) {
        for (int g = threadIdx.x; g < ng; g += 256) {
            float2 s = {0.0f, 0.0f};
            for (int c = 0; c < D; ++c) {
                const float2 v = f(g * D + c);
                s.x += v.x;
                s.y += v.y;
            }
            done(g, s);
        }
    } else {
        const int lane = threadIdx.x & 63;
        for (int g = threadIdx.x >> 6; g < ng; g += 4) {
            float2 s = {0.0f, 0.0f};
            for (int c = lane; c < D; c += 64) {
                const float2 v = f(g * D + c);
                s.x += v.x;
                s.y += v.y;
            }
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) {
                s.x += __shfl_xor(s.x, o);
                s.y += __shfl_xor(s.y, o);
            }
            if (lane == 0) done(g, s);
        }
    }
}

// Pass 1, forward: part[((b nchunk + chunk) nsub + sub) G + g] = (mean, sum of squares about it) of the block's values.
// A thread sums about its own first value, so what cancels in s2 - s1^2 / n is at most n eps of the result; the threads' means
// stay (first value, rest) until they are joined in 64 bits, so that what is lost is small against the spread, wherever the
// mean lies (rounded to fp32 each: 3e-6 of the spread at a mean of 100 spreads; the leaky derivative shows that, see gn_mend).
template <typename T, int V>
__global__ void __launch_bounds__(256) gn_stats_kernel(const GnArgs a, const GnWork w, double2 *__restrict__ part) {
    __shared__ float2 red[256 * V];                              // [R][W] (mean - first value, squares); row 0 then holds the channels' pairs
    __shared__ __attribute__((aligned(16))) T first[256 * V];    // [R][W]; row 0 then holds what is missing from the channels' means
    const GnPos<V> g(a, w);
    typedef vec_io<T, V> IO;
    const T *__restrict__ x = (const T *)a.x + (size_t)g.b * a.P * a.C + g.c0;
    const int W = w.cvb * V;
    if (g.on) {
        float piv[V], s1[V], s2[V];
        typename IO::raw q0 = {};
#pragma unroll
        for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.0f;
        if (g.p < g.p1) q0 = IO::load(x + (size_t)g.p * a.C);
        IO::unpack(q0, piv);
        gn_rows<4>(g.p, g.p1, w.R, [&](int p) { return IO::load(x + (size_t)p * a.C); },
                   [&](int, const typename IO::raw &q) {
                       float v[V];
                       IO::unpack(q, v);
#pragma unroll
                       for (int i = 0; i < V; ++i) {
                           const float d = v[i] - piv[i];
                           s1[i] += d;
                           s2[i] += d * d;
                       }
                   });
        const int n = g.p < g.p1 ? (g.p1 - g.p + w.R - 1) / w.R : 0;
        const float inv = n > 0 ? 1.0f / (float)n : 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) red[g.r * W + g.cv * V + i] = float2{s1[i] * inv, gn_squares(s2[i] - s1[i] * s1[i] * inv)};
        *(typename IO::raw *)&first[g.r * W + g.cv * V] = q0;
    }
    __syncthreads();
    const int np = g.p1 - g.chunk * w.per;                       // pixels of the chunk
    const int rows = min(w.R, np);
    // The n values of row r: the chunk's pixels r, r + R, ...
    const int each = np / w.R, more = np - each * w.R;
    auto row = [&](int r, int c, double &n, double &m, float &m2) {
        const float2 q = red[r * W + c];
        n = each + (r < more ? 1 : 0);
        m = (double)elem<T>::load(&first[r * W + c]) + q.x;
        m2 = q.y;
    };
    for (int c = threadIdx.x; c < g.wc; c += 256) {
        double mean = 0.0, sq = 0.0, n, m;
        float m2;
        for (int r = 0; r < rows; ++r) {
            row(r, c, n, m, m2);
            mean += n * m;
        }
        mean /= np;
        for (int r = 0; r < rows; ++r) {
            row(r, c, n, m, m2);
            sq += m2 + n * ((m - mean) * (m - mean));
        }
        const float hi = (float)mean;
        red[c] = float2{hi, (float)sq};
        elem<T>::store(&first[c], (float)(mean - hi));
    }
    __syncthreads();
    const double inv_d = 1.0 / g.D;
    double2 *dst = part + g.pair(a, w);
    const int ng = g.wc / g.D, lane = threadIdx.x & 63;
    const int c0 = g.D <= 16 ? 0 : lane, step = g.D <= 16 ? 1 : 64;       // a thread per narrow group, a wave per wide one
    auto group_sum = [&](double v) {
        if (step == 64)
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
        return v;
    };
    for (int gr = step == 1 ? threadIdx.x : threadIdx.x >> 6; gr < ng; gr += step == 1 ? 256 : 4) {
        const float2 *ch = red + gr * g.D;
        const T *rest = first + gr * g.D;
        double mean = 0.0, sq = 0.0;
        for (int c = c0; c < g.D; c += step) mean += (double)ch[c].x + elem<T>::load(&rest[c]);
        mean = group_sum(mean) * inv_d;
        for (int c = c0; c < g.D; c += step) {
            const double d = (double)ch[c].x + elem<T>::load(&rest[c]) - mean;
            sq += ch[c].y + np * (d * d);
        }
        sq = group_sum(sq);
        if (step == 1 || lane == 0) dst[gr] = double2{mean, sq};
    }
}

// Pass 2 begins: the pairs of the sample's blocks joined for every group, all threads of the workgroup taking
// part (256: group lanes x block lanes).  out[g] in LDS; scratch holds 256 pairs.
//   forward   (mean, 1 / sqrt(var + eps)); one workgroup of the sample keeps it in stats
//   backward  (S1, S2) / N
template <bool BWD, int V, typename Pair>
__device__ __forceinline__ void gn_join(const GnArgs &a, const GnWork &w, int b, bool keep, const Pair *__restrict__ part,
                                        float2 *__restrict__ out, double2 *__restrict__ scratch) {
    const int gl = min(a.G, 256), cl = 256 / gl, lane = threadIdx.x % gl, row = threadIdx.x / gl, blocks = w.nchunk * w.nsub;
    const Pair *__restrict__ src = part + (size_t)b * blocks * a.G;
    const double inv_n = 1.0 / ((double)a.P * a.D);
    auto values = [&](int k) {                                   // how many block k holds of a group
        const int chunk = w.nsub == 1 ? k : k / w.nsub, sub = k - chunk * w.nsub;
        const int pix = min(w.per, a.P - chunk * w.per), wid = w.nsub == 1 ? a.D : min(w.cvb * V, a.D - sub * w.cvb * V);
        return (double)pix * wid;
    };
    for (int g0 = 0; g0 < a.G; g0 += gl) {
        const int g = g0 + lane;
        const bool on = row < cl && g < a.G;
        double2 s = {0.0, 0.0};
        double piv = 0.0;                                        // forward: sums about the first block's mean
        if (on) {
            if (!BWD) piv = src[g].x;
            auto add = [&](int k, const Pair &v) {
                if (BWD) {
                    s.x += v.x;
                    s.y += v.y;
                } else {
                    const double n = values(k), d = v.x - piv;
                    s.x += n * d;
                    s.y += v.y + n * d * d;
                }
            };
            int k = row;
            for (; k + 7 * cl < blocks; k += 8 * cl) {
                Pair v[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) v[u] = src[(size_t)(k + u * cl) * a.G + g];
#pragma unroll
                for (int u = 0; u < 8; ++u) add(k + u * cl, v[u]);
            }
            for (; k < blocks; k += cl) add(k, src[(size_t)k * a.G + g]);
        }
        __syncthreads();
        if (on) scratch[row * gl + lane] = s;
        __syncthreads();
        if (on && row == 0) {
            for (int r = 1; r < cl; ++r) {
                s.x += scratch[r * gl + lane].x;
                s.y += scratch[r * gl + lane].y;
            }
            if (BWD) {
                out[g] = float2{(float)(s.x * inv_n), (float)(s.y * inv_n)};
            } else {
                const double shift = s.x * inv_n, mean = piv + shift, rstd = gn_rstd(s.y * inv_n - shift * shift, a.eps);
                out[g] = float2{(float)mean, (float)rstd};
                if (keep && a.stats) gn_keep_stats(a, b, g, mean, rstd);
            }
        }
    }
    __syncthreads();
}

// The numbers of a thread's V channels: d = x - mean first (exact next to the mean, so that a map without
// spread gives beta itself), then h = d r and t = d (gamma r) + beta.
template <int V> struct GnChannels {
    float mean[V], r[V], ta[V], be[V];
    __device__ __forceinline__ void set(int i, float m, float rstd, float gamma, float beta) {
        mean[i] = m;
        r[i] = rstd;
        ta[i] = gamma * rstd;
        be[i] = beta;
    }
    template <typename S> __device__ __forceinline__ void load(const GnArgs &a, const S *st, int c0) {      // st: of the sample's groups
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const S m = st[(c0 + i) / a.D];
            set(i, m.x, m.y, a.gamma[c0 + i], a.beta[c0 + i]);
        }
    }
    // a t smaller than this may have the wrong sign (0 where nothing has been rounded: gamma = beta = 0, or a mean and a beta
    // of 0; such a channel may hold nothing but t = 0, and has no doubtful one)
    __device__ __forceinline__ float near(int i) const { return 4e-7f * (fabsf(be[i]) + fabsf(mean[i] * ta[i])); }
    __device__ __forceinline__ bool doubtful(float low) const {
        float n = near(0);
#pragma unroll
        for (int i = 1; i < V; ++i) n = fmaxf(n, near(i));
        return low < n;
    }
    __device__ __forceinline__ float t(int i, float x) const { return __builtin_fmaf(x - mean[i], ta[i], be[i]); }
};

// Bit i: element i0 + i is kept.
template <int V> __device__ __forceinline__ unsigned gn_keep_bits(const DropArgs &drop, const uint4 &key, unsigned long long i0) {
    bool keep[V];
    drop_keep<V>(drop, key, i0, keep);
    unsigned m = 0u;
#pragma unroll
    for (int i = 0; i < V; ++i) m |= keep[i] ? 1u << i : 0u;
    return m;
}

// Single elements (V = 1) would compute four random words each for one: their bits come from a pass of its own over the flat
// map, byte j those of elements 8 j ... 8 j + 7 (16 x 52^2 x 255, rate 0.1: forward/backward 36.4/44.7 us, 50.6/77.5 without).
__global__ void __launch_bounds__(256) gn_mask_kernel(const DropArgs drop, unsigned long long n, unsigned char *__restrict__ mask) {
    const uint4 key = {drop.state[0], drop.state[1], drop.state[2], drop.state[3]};
    for (unsigned long long j = (unsigned long long)blockIdx.x * 256 + threadIdx.x; j * 8 < n; j += (unsigned long long)gridDim.x * 256)
        mask[j] = (unsigned char)gn_keep_bits<8>(drop, key, j * 8);
}
__device__ __forceinline__ unsigned gn_mask_bit(const unsigned char *mask, size_t i) { return mask[i >> 3] >> (i & 7) & 1u; }

// Pass 2, forward.
template <typename T, int V, int ACT, bool DROP>
__global__ void __launch_bounds__(256) gn_apply_kernel(const GnArgs a, const GnWork w, const double2 *__restrict__ part,
                                                       const unsigned char *__restrict__ mask) {
    extern __shared__ __attribute__((aligned(16))) float2 joined[];      // [G, even], then 256 pairs of doubles
    const GnPos<V> g(a, w);
    gn_join<false, V>(a, w, g.b, g.chunk == 0 && g.cb == 0, part, joined, (double2 *)(joined + (a.G + 1 & ~1)));
    if (!g.on) return;
    typedef vec_io<T, V> IO;
    GnChannels<V> ch;
    ch.load(a, joined, g.c0);
    const size_t base = (size_t)g.b * a.P * a.C + g.c0;
    const T *__restrict__ x = (const T *)a.x + base, *__restrict__ res = (const T *)a.res + base;
    T *__restrict__ y = (T *)a.y + base;
    const bool has_res = a.res != nullptr;
    const DropArgs drop = {a.state, a.threshold, a.keep_scale};
    uint4 key = {};
    if constexpr (DROP && V > 1) key = uint4{a.state[0], a.state[1], a.state[2], a.state[3]};
    struct Row { typename IO::raw x, s; unsigned keep; };
    gn_rows<V == 1 ? 4 : 2>(g.p, g.p1, w.R, [&](int p) {
                   Row q;
                   q.x = IO::load(x + (size_t)p * a.C);
                   if constexpr (DROP && V == 1) q.keep = gn_mask_bit(mask, base + (size_t)p * a.C);
                   if (has_res) q.s = IO::load(res + (size_t)p * a.C);
                   return q;
               },
               [&](int p, const Row &q) {
                   float v[V], s[V];
                   bool keep[V];
                   IO::unpack(q.x, v);
                   if constexpr (DROP && V == 1) keep[0] = q.keep;
                   else if constexpr (DROP) drop_keep<V>(drop, key, base + (size_t)p * a.C, keep);
#pragma unroll
                   for (int i = 0; i < V; ++i) {
                       v[i] = act_c<ACT>(ch.t(i, v[i]));
                       if constexpr (DROP) v[i] = keep[i] ? v[i] * drop.keep_scale : 0.0f;
                   }
                   if (has_res) {
                       IO::unpack(q.s, s);
#pragma unroll
                       for (int i = 0; i < V; ++i) v[i] += s[i];
                   }
                   IO::store(y + (size_t)p * a.C, v);
               });
}

// dt of one vector of a map and its gradient; bit i of keep: element i is kept.  low (leaky): the least |t| so far.
template <int V, int ACT, bool DROP>
__device__ __forceinline__ void gn_dt(const GnChannels<V> &ch, float keep_scale, unsigned keep, const float (&x)[V], const float (&dy)[V],
                                      float (&dt)[V], float &low) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float d = dy[i];
        if constexpr (DROP) d = (keep >> i & 1u) ? d * keep_scale : 0.0f;
        const float t = ch.t(i, x[i]);
        if constexpr (ACT == YMX_ACT_LEAKY) low = fminf(low, fabsf(t));
        dt[i] = d * act_grad_c<ACT>(t);
    }
}

// dx of V values: r (gamma dt - (m1 + h m2)) = ta dt + d b + c with the group's m1 = S1 / N, m2 = S2 / N.
template <int V> struct GnGradient {
    float b[V], c[V];
    __device__ __forceinline__ void set(const GnChannels<V> &ch, int i, float m1, float m2) {
        b[i] = -ch.r[i] * ch.r[i] * m2;
        c[i] = -ch.r[i] * m1;
    }
    __device__ __forceinline__ float dx(const GnChannels<V> &ch, int i, float x, float dt) const {
        return __builtin_fmaf(ch.ta[i], dt, __builtin_fmaf(x - ch.mean[i], b[i], c[i]));
    }
};

// The leaky derivative jumps at t = 0, and one element in ten million (mean and spread alike; in proportion to the mean) has a t
// whose fp32 sign is not that of the formula: off by the whole jump.  So a thread that met a doubtful t (one element in a
// million has one, or more where |beta| + |gamma mean| r is above 1) goes over its rows once more: for each of its elements
// whose sign 64-bit arithmetic on the kept statistics turns round, use(i, p, x, right dt - wrong dt, right dt, its channel).
// Those are off by about 5e-9 of the spread (fp32 sums of differences from a value of the map, joined in 64 bits), wherever
// the mean lies; one sign in a hundred million elements stays undecided.
template <typename T, int V, bool DROP, typename F>
__device__ __forceinline__ void gn_mend(const GnArgs &a, const GnChannels<V> &ch, int b, int c0, int p, int p1, int R, F use) {
    // everything is computed and loaded again: not to cost the rest registers
    asm volatile("" : "+v"(c0), "+v"(p)::"memory");
    typedef vec_io<T, V> IO;
    const size_t base = (size_t)b * a.P * a.C + c0;
    const T *__restrict__ x = (const T *)a.x + base, *__restrict__ dy = (const T *)a.dy + base;
    gn_rows<8>(p, p1, R, [&](int q) { return IO::load(x + (size_t)q * a.C); }, [&](int q, const typename IO::raw &r) {
        float v[V];
        IO::unpack(r, v);
        unsigned doubt = 0u;
#pragma unroll
        for (int i = 0; i < V; ++i) doubt |= fabsf(ch.t(i, v[i])) < ch.near(i) ? 1u << i : 0u;
        while (doubt) {
            const int i = __builtin_ctz(doubt), c = c0 + i;
            doubt &= doubt - 1u;
            const float4 *st = (const float4 *)a.stats + (size_t)b * a.G;
            const float4 own = st[c / a.D];
            GnChannels<1> one;
            one.load(a, st, c);
            const size_t at = (size_t)q * a.C + i;
            const float w = elem<T>::load(x + at);
            const double h = ((double)w - own.x - own.z) * ((double)own.y + own.w), exact = a.gamma[c] * h + a.beta[c];
            if ((exact > 0.0) == (one.t(0, w) > 0.0f)) continue;
            float d = elem<T>::load(dy + at);
            if constexpr (DROP) {
                bool keep[1];
                const DropArgs drop = {a.state, a.threshold, a.keep_scale};
                drop_keep<1>(drop, uint4{a.state[0], a.state[1], a.state[2], a.state[3]}, base + at, keep);
                d = keep[0] ? d * a.keep_scale : 0.0f;
            }
            const float right = d * (exact > 0.0 ? 1.0f : 0.1f), wrong = d * (exact > 0.0 ? 0.1f : 1.0f);
            use(i, q, w, right - wrong, right, one);
        }
    });
}

// Pass 1, backward: part[(b nchunk + chunk) C + c] = (sum dt, sum dt h) of the chunk's pixels, and
// gpart[((b nchunk + chunk) nsub + sub) G + g] = (S1, S2) of the block's values.  With dropout, mask (V > 1) receives a byte
// of kept elements per vector for pass 2: the random words are a fifth of this pass (16 x 208^2 x 64, rate 0.1: backward
// 126.8 us with the words in both passes, 117.0 with the bytes).
template <typename T, int V, int ACT, bool DROP>
__global__ void __launch_bounds__(256) gn_bwd_sums_kernel(const GnArgs a, const GnWork w, float2 *__restrict__ part,
                                                          float2 *__restrict__ gpart, unsigned char *__restrict__ mask) {
    __shared__ float2 red[256 * V];                              // [R][W]; row 0 then holds gamma times the channels' pairs
    const GnPos<V> g(a, w);
    typedef vec_io<T, V> IO;
    const int W = w.cvb * V;
    if (g.on) {
        GnChannels<V> ch;
        ch.load(a, (const float4 *)a.stats + (size_t)g.b * a.G, g.c0);
        const size_t base = (size_t)g.b * a.P * a.C + g.c0;
        const T *__restrict__ x = (const T *)a.x + base, *__restrict__ dy = (const T *)a.dy + base;
        const DropArgs drop = {a.state, a.threshold, a.keep_scale};
        uint4 key = {};
        if constexpr (DROP) key = uint4{a.state[0], a.state[1], a.state[2], a.state[3]};
        float s1[V], s2[V];
        float low = __builtin_inff();
#pragma unroll
        for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.0f;
        struct Row { typename IO::raw x, d; unsigned keep; };
        gn_rows<4>(g.p, g.p1, w.R, [&](int p) {
                       Row q = {IO::load(x + (size_t)p * a.C), IO::load(dy + (size_t)p * a.C), 0u};
                       if constexpr (DROP && V == 1) q.keep = gn_mask_bit(mask, base + (size_t)p * a.C);
                       return q;
                   },
                   [&](int p, const Row &q) {
                       float v[V], d[V], dt[V];
                       IO::unpack(q.x, v);
                       IO::unpack(q.d, d);
                       unsigned keep = 0u;
                       if constexpr (DROP && V == 1) keep = q.keep;
                       else if constexpr (DROP) {
                           const size_t at = base + (size_t)p * a.C;
                           keep = gn_keep_bits<V>(drop, key, at);
                           mask[at / V] = (unsigned char)keep;
                       }
                       gn_dt<V, ACT, DROP>(ch, drop.keep_scale, keep, v, d, dt, low);
#pragma unroll
                       for (int i = 0; i < V; ++i) {
                           s1[i] += dt[i];
                           s2[i] += dt[i] * (v[i] - ch.mean[i]);
                       }
                   });
        if constexpr (ACT == YMX_ACT_LEAKY)
            if (ch.doubtful(low))
                gn_mend<T, V, DROP>(a, ch, g.b, g.c0, g.p, g.p1, w.R, [&](int i, int, float v, float more, float, const GnChannels<1> &c) {
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        s1[k] += k == i ? more : 0.0f;
                        s2[k] += k == i ? more * (v - c.mean[0]) : 0.0f;
                    }
                });
#pragma unroll
        for (int i = 0; i < V; ++i) red[g.r * W + g.cv * V + i] = float2{s1[i], s2[i] * ch.r[i]};
    }
    __syncthreads();
    for (int c = threadIdx.x; c < g.wc; c += 256) {
        double d1 = 0.0, d2 = 0.0;
        for (int r = 0; r < w.R; ++r) {
            const float2 q = red[r * W + c];
            d1 += q.x;
            d2 += q.y;
        }
        const float2 s = {(float)d1, (float)d2};
        part[((size_t)g.b * w.nchunk + g.chunk) * a.C + g.cb + c] = s;
        const float ga = a.gamma[g.cb + c];
        red[c] = float2{ga * s.x, ga * s.y};
    }
    __syncthreads();
    float2 *dst = gpart + g.pair(a, w);
    gn_over_groups(g.wc, g.D, [&](int c) { return red[c]; }, [&](int gr, float2 t) { dst[gr] = t; });
}

// dbeta and dgamma of 16 channels from `rows` pairs each, by a workgroup of 16 * RL threads: RL row lanes (four chains
// each) and those by a tree, in 64 bits: the sums run over a whole batch of maps, and there are few of them.
// red: 16 * (RL + 1) pairs of doubles.
template <int RL>
__device__ __forceinline__ void gn_param_grads(const GnArgs &a, int block, int rows, const float2 *__restrict__ part, double2 *__restrict__ red) {
    const int cl = threadIdx.x & 15, row = threadIdx.x >> 4, c = block * 16 + cl;
    double2 s[4] = {};
    if (c < a.C) {
        int i = row;
        for (; i + 3 * RL < rows; i += 4 * RL) {
            float2 v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = part[(size_t)(i + RL * u) * a.C + c];
#pragma unroll
            for (int u = 0; u < 4; ++u) { s[u].x += v[u].x; s[u].y += v[u].y; }
        }
        for (; i < rows; i += RL) {
            const float2 v = part[(size_t)i * a.C + c];
            s[0].x += v.x;
            s[0].y += v.y;
        }
    }
    red[cl * (RL + 1) + row] = double2{(s[0].x + s[1].x) + (s[2].x + s[3].x), (s[0].y + s[1].y) + (s[2].y + s[3].y)};
    __syncthreads();
    // RL lanes per channel, channels dealt to the groups of RL threads
    const int lane = threadIdx.x % RL, cw = threadIdx.x / RL;
    double2 t = red[cw * (RL + 1) + lane];
#pragma unroll
    for (int o = RL / 2; o > 0; o >>= 1) {
        t.x += __shfl_xor(t.x, o);
        t.y += __shfl_xor(t.y, o);
    }
    if (lane == 0 && block * 16 + cw < a.C) {
        a.dbeta[block * 16 + cw] = (float)t.x;
        a.dgamma[block * 16 + cw] = (float)t.y;
    }
}
__global__ void __launch_bounds__(1024) gn_param_grads_kernel(const GnArgs a, int rows, const float2 *__restrict__ part) {
    __shared__ double2 red[16 * 65];
    gn_param_grads<64>(a, blockIdx.x, rows, part, red);
}

// Pass 2, backward.
template <typename T, int V, int ACT, bool DROP>
__global__ void __launch_bounds__(256) gn_bwd_apply_kernel(const GnArgs a, const GnWork w, const float2 *__restrict__ part,
                                                           const float2 *__restrict__ gpart, const unsigned char *__restrict__ mask, int nparam) {
    extern __shared__ __attribute__((aligned(16))) float2 joined[];      // [G, even], then 256 pairs of doubles; or 16 * 17 of them
    if ((int)blockIdx.x < nparam) {                              // the first workgroups: parameter gradients, 16 channels each
        gn_param_grads<16>(a, blockIdx.x, a.B * w.nchunk, part, (double2 *)joined);
        return;
    }
    const GnPos<V> g(a, w, nparam);
    gn_join<true, V>(a, w, g.b, false, gpart, joined, (double2 *)(joined + (a.G + 1 & ~1)));
    if (!g.on) return;
    typedef vec_io<T, V> IO;
    GnChannels<V> ch;
    GnGradient<V> gr;
    ch.load(a, (const float4 *)a.stats + (size_t)g.b * a.G, g.c0);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float2 m = joined[(g.c0 + i) / a.D];
        gr.set(ch, i, m.x, m.y);
    }
    const size_t base = (size_t)g.b * a.P * a.C + g.c0;
    const T *__restrict__ x = (const T *)a.x + base, *__restrict__ dy = (const T *)a.dy + base;
    T *__restrict__ dx = (T *)a.dx + base;
    float low = __builtin_inff();
    struct Row { typename IO::raw x, d; unsigned keep; };
    gn_rows<4>(g.p, g.p1, w.R, [&](int p) {
                   Row q = {IO::load(x + (size_t)p * a.C), IO::load(dy + (size_t)p * a.C), 0u};
                   if constexpr (DROP && V == 1) q.keep = gn_mask_bit(mask, base + (size_t)p * a.C);
                   else if constexpr (DROP) q.keep = mask[(base + (size_t)p * a.C) / V];
                   return q;
               },
               [&](int p, const Row &q) {
                   float v[V], d[V], dt[V];
                   IO::unpack(q.x, v);
                   IO::unpack(q.d, d);
                   gn_dt<V, ACT, DROP>(ch, a.keep_scale, q.keep, v, d, dt, low);
#pragma unroll
                   for (int i = 0; i < V; ++i) v[i] = gr.dx(ch, i, v[i], dt[i]);
                   IO::store(dx + (size_t)p * a.C, v);
               });
    if constexpr (ACT == YMX_ACT_LEAKY)
        if (ch.doubtful(low))
            gn_mend<T, V, DROP>(a, ch, g.b, g.c0, g.p, g.p1, w.R, [&](int i, int p, float v, float, float right, const GnChannels<1> &c) {
                const float2 m = joined[(g.c0 + i) / a.D];
                GnGradient<1> one;
                one.set(c, 0, m.x, m.y);
                elem<T>::store(dx + (size_t)p * a.C + i, one.dx(c, 0, v, right));
            });
}

// ---- one pass: the pixels of a sample's channel slab stay in registers ------------------------------
// A workgroup of 512 threads owns sv V neighbouring channels (whole groups) of one sample: thread (row, cv) holds
// the vectors of pixels row, row + R, ..., R = 512 / sv, so the map is read once, the statistics are taken in two
// steps (mean, then squares about it) from registers, and one launch does what the chunked form needs three for.
// sv is a power of two up to 64 and D one up to 64, so sums over rows are lane exchanges and one LDS step.
struct GnSlab { int sv, nslab; };

// sum[i] (channel cv V + i of this thread) -> totals over the workgroup's rows; tot[c] for thread c < sv V.
template <int V> __device__ __forceinline__ double gn_slab_total(const float (&v)[V], int sv, float *red) {
    float s[V];
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = v[i];
    for (int o = sv; o < 64; o <<= 1)
#pragma unroll
        for (int i = 0; i < V; ++i) s[i] += __shfl_xor(s[i], o);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, W = sv * V;
    __syncthreads();                                             // (the scratch may still be read)
    if (lane < sv)
#pragma unroll
        for (int i = 0; i < V; ++i) red[wave * W + lane * V + i] = s[i];
    __syncthreads();
    double t = 0.0;
    if ((int)threadIdx.x < W)
        for (int w = 0; w < 8; ++w) t += red[w * W + threadIdx.x];
    return t;
}
// Sum over the D neighbouring threads of a group.
__device__ __forceinline__ double gn_group_sum(double t, int D) {
    for (int o = 1; o < D; o <<= 1) t += __shfl_xor(t, o);
    return t;
}

template <typename T, int V, int NV, int ACT, bool DROP>
__global__ void __launch_bounds__(512) gn_slab_kernel(const GnArgs a, const GnSlab w) {
    extern __shared__ float red[];                               // [8][sv V] partial sums, then [sv V] of a channel's group
    typedef vec_io<T, V> IO;
    const int W = w.sv * V, cv = threadIdx.x % w.sv, row = threadIdx.x / w.sv, R = 512 / w.sv;
    const int id = xcd_remap(blockIdx.x, gridDim.x), slab = id % w.nslab, b = id / w.nslab;
    const size_t base = (size_t)b * a.P * a.C + slab * W + cv * V;
    const T *__restrict__ x = (const T *)a.x + base, *__restrict__ res = (const T *)a.res + base;
    T *__restrict__ y = (T *)a.y + base;
    float *grp = red + 8 * W;
    // sums about the first pixel's values, so that what they lose is small against the spread
    const typename IO::raw q0 = IO::load(x);
    const float c0 = (int)threadIdx.x < W ? elem<T>::load((const T *)a.x + (size_t)b * a.P * a.C + slab * W + threadIdx.x) : 0.0f;
    typename IO::raw q[NV];
#pragma unroll
    for (int n = 0; n < NV; ++n)
        if (row + n * R < a.P) q[n] = IO::load(x + (size_t)(row + n * R) * a.C);
    const double inv_n = 1.0 / ((double)a.P * a.D);
    float s[V], mean[V];
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = 0.0f;
    IO::unpack(q0, mean);
#pragma unroll
    for (int n = 0; n < NV; ++n) {
        float v[V];
        IO::unpack(q[n], v);
        if (row + n * R < a.P)
#pragma unroll
            for (int i = 0; i < V; ++i) s[i] += v[i] - mean[i];
    }
    const double m = gn_group_sum(gn_slab_total<V>(s, w.sv, red) + (double)a.P * c0, a.D) * inv_n, off = m - (float)m;
    if ((int)threadIdx.x < W) grp[threadIdx.x] = (float)m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) {
        mean[i] = grp[cv * V + i];
        s[i] = 0.0f;
    }
#pragma unroll
    for (int n = 0; n < NV; ++n) {
        float v[V];
        IO::unpack(q[n], v);
        if (row + n * R < a.P)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = v[i] - mean[i];
                s[i] += d * d;
            }
    }
    const double rstd = gn_rstd(gn_group_sum(gn_slab_total<V>(s, w.sv, red), a.D) * inv_n - off * off, a.eps);
    if ((int)threadIdx.x < W) {
        grp[threadIdx.x] = (float)rstd;
        if (a.stats && threadIdx.x % a.D == 0) gn_keep_stats(a, b, (slab * W + threadIdx.x) / a.D, m, rstd);
    }
    __syncthreads();
    GnChannels<V> ch;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = cv * V + i;
        ch.set(i, mean[i], grp[c], a.gamma[slab * W + c], a.beta[slab * W + c]);
    }
    const bool has_res = a.res != nullptr;
    const DropArgs drop = {a.state, a.threshold, a.keep_scale};
    uint4 key = {};
    if constexpr (DROP) key = uint4{a.state[0], a.state[1], a.state[2], a.state[3]};
#pragma unroll
    for (int n = 0; n < NV; ++n) {
        const int p = row + n * R;
        if (p >= a.P) continue;
        float v[V], r[V];
        bool keep[V];
        typename IO::raw qs;
        if (has_res) qs = IO::load(res + (size_t)p * a.C);
        IO::unpack(q[n], v);
        if constexpr (DROP) drop_keep<V>(drop, key, base + (size_t)p * a.C, keep);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            v[i] = act_c<ACT>(ch.t(i, v[i]));
            if constexpr (DROP) v[i] = keep[i] ? v[i] * drop.keep_scale : 0.0f;
        }
        if (has_res) {
            IO::unpack(qs, r);
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] += r[i];
        }
        IO::store(y + (size_t)p * a.C, v);
    }
}

// Backward: x stays as it was read, dt as computed (fp32); the sums over a sample of each channel go to
// part[b C + c] for the parameters' gradients; those of a single sample are the gradients (13^2 x 1024: 9.3 -> 6.4 us).
template <typename T, int V, int NV, int ACT, bool DROP>
__global__ void __launch_bounds__(512) gn_slab_bwd_kernel(const GnArgs a, const GnSlab w, float2 *__restrict__ part) {
    extern __shared__ float red[];                               // [8][sv V], then two of [sv V]
    typedef vec_io<T, V> IO;
    const int W = w.sv * V, cv = threadIdx.x % w.sv, row = threadIdx.x / w.sv, R = 512 / w.sv;
    const int id = xcd_remap(blockIdx.x, gridDim.x), slab = id % w.nslab, b = id / w.nslab;
    const size_t base = (size_t)b * a.P * a.C + slab * W + cv * V;
    const T *__restrict__ x = (const T *)a.x + base, *__restrict__ dy = (const T *)a.dy + base;
    T *__restrict__ dx = (T *)a.dx + base;
    float *g1 = red + 8 * W, *g2 = g1 + W;
    typename IO::raw q[NV], qd[NV];
#pragma unroll
    for (int n = 0; n < NV; ++n)
        if (row + n * R < a.P) {
            q[n] = IO::load(x + (size_t)(row + n * R) * a.C);
            qd[n] = IO::load(dy + (size_t)(row + n * R) * a.C);
        }
    GnChannels<V> ch;
    ch.load(a, (const float4 *)a.stats + (size_t)b * a.G, slab * W + cv * V);
    const DropArgs drop = {a.state, a.threshold, a.keep_scale};
    uint4 key = {};
    if constexpr (DROP) key = uint4{a.state[0], a.state[1], a.state[2], a.state[3]};
    float dt[NV][V], s1[V], s2[V];
    float low = __builtin_inff();
#pragma unroll
    for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.0f;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
        const int p = row + n * R;
        if (p < a.P) {
            float v[V], d[V];
            IO::unpack(q[n], v);
            IO::unpack(qd[n], d);
            unsigned keep = 0u;
            if constexpr (DROP) keep = gn_keep_bits<V>(drop, key, base + (size_t)p * a.C);
            gn_dt<V, ACT, DROP>(ch, drop.keep_scale, keep, v, d, dt[n], low);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                s1[i] += dt[n][i];
                s2[i] += dt[n][i] * (v[i] - ch.mean[i]);
            }
        }
    }
    if constexpr (ACT == YMX_ACT_LEAKY)
        if (ch.doubtful(low))
            gn_mend<T, V, DROP>(a, ch, b, slab * W + cv * V, row, a.P, R, [&](int i, int, float v, float more, float, const GnChannels<1> &c) {
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    s1[k] += k == i ? more : 0.0f;
                    s2[k] += k == i ? more * (v - c.mean[0]) : 0.0f;
                }
            });
#pragma unroll
    for (int i = 0; i < V; ++i) s2[i] *= ch.r[i];
    const double t1 = gn_slab_total<V>(s1, w.sv, red), t2 = gn_slab_total<V>(s2, w.sv, red);
    const double inv_n = 1.0 / ((double)a.P * a.D);
    double ga = 0.0;
    if ((int)threadIdx.x < W) {
        const int c = slab * W + threadIdx.x;
        if (a.B == 1) {                                          // the sums over all samples: no second launch
            a.dbeta[c] = (float)t1;
            a.dgamma[c] = (float)t2;
        } else {
            part[(size_t)b * a.C + c] = float2{(float)t1, (float)t2};
        }
        ga = a.gamma[slab * W + threadIdx.x] * inv_n;
    }
    const double u1 = gn_group_sum(ga * t1, a.D), u2 = gn_group_sum(ga * t2, a.D);
    if ((int)threadIdx.x < W) {
        g1[threadIdx.x] = (float)u1;
        g2[threadIdx.x] = (float)u2;
    }
    __syncthreads();
    GnGradient<V> gr;
#pragma unroll
    for (int i = 0; i < V; ++i) gr.set(ch, i, g1[cv * V + i], g2[cv * V + i]);
#pragma unroll
    for (int n = 0; n < NV; ++n) {
        const int p = row + n * R;
        if (p >= a.P) continue;
        float v[V];
        IO::unpack(q[n], v);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = gr.dx(ch, i, v[i], dt[n][i]);
        IO::store(dx + (size_t)p * a.C, v);
    }
    if constexpr (ACT == YMX_ACT_LEAKY)
        if (ch.doubtful(low))
            gn_mend<T, V, DROP>(a, ch, b, slab * W + cv * V, row, a.P, R, [&](int i, int p, float v, float, float right, const GnChannels<1> &c) {
                GnGradient<1> one;
                one.set(c, 0, g1[cv * V + i], g2[cv * V + i]);
                elem<T>::store(dx + (size_t)p * a.C + i, one.dx(c, 0, v, right));
            });
}

// ---- host side -----------------------------------------------------------------------------------
// Chunks of a sample: about 2048 workgroups (eight of 256 threads on each of 256 CUs), none with less than 16 K
// elements to read while that leaves 512 of them, else 4 K (16 x 52^2 x 256 forward 27.4 us at 16 K, 36.9 at 4 K;
// 52^2 x 256 alone 13.6 and 11.6, backward 17.3 and 11.2); at most 256, whose pairs every workgroup of pass 2 joins.
static int gn_chunks(int B, int P, int C) {
    const long long n = (long long)P * C;
    const long long most = std::max<long long>(n / 16384, std::min<long long>(n / 4096, 512 / B));
    const long long want = std::max(1, 2048 / B);
    return (int)std::min<long long>(std::max<long long>(1, std::min<long long>(256, std::min(most, want))), P);
}
// Channels are cut into blocks of whole groups of at most 256 vectors; a wider group into equal parts.
template <int V> static GnWork gn_work(const GnArgs &a) {
    GnWork w;
    const int cv = a.C / V;
    int unit = 1;                                                // vectors in the least run of whole groups
    while ((long long)unit * V % a.D) ++unit;
    w.nsub = 1;
    if (cv <= 256) {
        w.cvb = cv;
        w.nzb = 1;
    } else if (unit <= 256) {
        w.cvb = 256 / unit * unit;
        w.nzb = (cv + w.cvb - 1) / w.cvb;
    } else {                                                     // D > 256 V, a multiple of V (gn_pick)
        w.nsub = (a.D / V + 255) / 256;
        w.cvb = (a.D / V + w.nsub - 1) / w.nsub;
        w.nzb = a.G * w.nsub;
    }
    w.R = 256 / w.cvb;
    w.per = (a.P + gn_chunks(a.B, a.P, a.C) - 1) / gn_chunks(a.B, a.P, a.C);
    w.nchunk = (a.P + w.per - 1) / w.per;
    return w;
}
// Pairs: one per (chunk, channel) and one per (chunk, group or part of one); the forward pass has the latter alone, of twice
// the size, and there are no more groups' parts than channels.  Behind them the bytes of kept elements, one for
// four or eight.
static size_t gn_pairs(int G, int C) { return (size_t)G * ((C / G + 255) / 256); }
static size_t gn_pair_bytes(int B, int P, int C, int G) { return (size_t)B * gn_chunks(B, P, C) * (C + gn_pairs(G, C)) * sizeof(float2); }
size_t group_norm_workspace_bytes(int B, int P, int C, int G) {
    return gn_pair_bytes(B, P, C, G) + (size_t)B * P * C / 4 + 8;
}
template <int V> static unsigned char *gn_mask(const GnArgs &a, void *ws, hipStream_t s) {
    unsigned char *mask = (unsigned char *)ws + gn_pair_bytes(a.B, a.P, a.C, a.G);
    if (V == 1 && a.state) {
        const unsigned long long n = (unsigned long long)a.B * a.P * a.C;
        hipLaunchKernelGGL(gn_mask_kernel, dim3((unsigned)std::min<unsigned long long>((n + 2047) / 2048, 16384)), dim3(256), 0, s, DropArgs{a.state, a.threshold, a.keep_scale}, n, mask);
    }
    return mask;
}

// The one-pass form's slabs, or sv = 0 where the chunked form runs: groups of a power of two of at most 64
// channels in whole vectors, 64 bytes or more of a pixel (narrower slabs fetch every line several times: 16 x 52^2 x
// 256 forward 32 us in slabs of 32 bytes, 27 in chunks), the slab's pixels in at most `most` vectors a
// thread.  The widest of 64, 128 and 256 bytes that gives a thread at most six vectors and every CU a workgroup
// (64 x 13^2 x 1024 forward: 25.5, 22.0, 19.2 us; 64 x 26^2 x 512: 40.2 us at six vectors, 41.8 at eleven), else the
// narrowest.
template <int V> static GnSlab gn_slab(const GnArgs &a, int most) {
    const int cv = a.C / V;
    GnSlab best = {0, 0};
    if (a.D > 64 || (a.D & (a.D - 1))) return best;
    for (int sv = 4; sv <= 16 && cv % sv == 0; sv *= 2) {
        if (sv * V % a.D || (long long)a.P * sv > 512ll * most || (long long)a.B * (cv / sv) > (1 << 22)) continue;   // (a grid has 2^32 threads)
        if (best.sv && ((long long)a.B * (cv / sv) < 256 || (long long)a.P * sv > 512 * 6)) break;
        best.sv = sv;
        best.nslab = cv / sv;
    }
    return best;
}

// Calls f(vector width, activation, dropout) as types.
template <int V, typename F> static void gn_pick_act(const GnArgs &a, F f) {
    auto drop = [&](auto act) {
        if (a.state) f(std::integral_constant<int, V>{}, act, std::true_type{});
        else f(std::integral_constant<int, V>{}, act, std::false_type{});
    };
    if (a.act == YMX_ACT_MISH) drop(std::integral_constant<int, YMX_ACT_MISH>{});
    else if (a.act == YMX_ACT_LEAKY) drop(std::integral_constant<int, YMX_ACT_LEAKY>{});
    else drop(std::integral_constant<int, YMX_ACT_NONE>{});
}
// Vectors of V elements where the channel count and every map's address allow them and blocks of whole groups, or parts of
// a group, are whole vectors: 16 bytes, else 8 of bf16 (16 x 52^2 x 260 forward/backward 24.8/35.2 us, in single elements
// 35.9/50.8), else one element at a time.
template <int V, typename T> static bool gn_vectors(const GnArgs &a) {
    auto ok = [](const void *p) { return ((uintptr_t)p & (V * sizeof(T) - 1)) == 0; };
    int unit = a.D;
    for (int v = V; v > 1 && unit % 2 == 0; v /= 2) unit /= 2;   // vectors in the least run of whole groups
    const bool blocks = a.C <= 256 * V || unit <= 256 || a.D % V == 0;
    return a.C % V == 0 && blocks && ok(a.x) && ok(a.res) && ok(a.dy) && ok(a.y) && ok(a.dx);
}
template <typename T, typename F> static void gn_pick(const GnArgs &a, F f) {
    if (gn_vectors<16 / sizeof(T), T>(a)) return gn_pick_act<16 / sizeof(T)>(a, f);
    if constexpr (sizeof(T) == 2)
        if (gn_vectors<4, T>(a)) return gn_pick_act<4>(a, f);
    gn_pick_act<1>(a, f);
}

static size_t gn_join_lds(int G) { return (G + 1 & ~1) * sizeof(float2) + 256 * sizeof(double2); }

template <typename T> static int gn_forward(const GnArgs &a, void *ws, hipStream_t s) {
    gn_pick<T>(a, [&](auto v, auto act, auto drop) {
        constexpr int V = decltype(v)::value, ACT = decltype(act)::value;
        constexpr bool DROP = decltype(drop)::value;
        if constexpr (V * sizeof(T) == 16) {
            const GnSlab sl = gn_slab<V>(a, 16);
            if (sl.sv) {
                const int nv = (a.P * sl.sv + 511) / 512, lds = 9 * sl.sv * V * 4;
                const dim3 grid((unsigned)(a.B * sl.nslab));
                if (nv <= 2) hipLaunchKernelGGL((gn_slab_kernel<T, V, 2, ACT, DROP>), grid, dim3(512), lds, s, a, sl);
                else if (nv <= 4) hipLaunchKernelGGL((gn_slab_kernel<T, V, 4, ACT, DROP>), grid, dim3(512), lds, s, a, sl);
                else if (nv <= 8) hipLaunchKernelGGL((gn_slab_kernel<T, V, 8, ACT, DROP>), grid, dim3(512), lds, s, a, sl);
                else if (nv <= 12) hipLaunchKernelGGL((gn_slab_kernel<T, V, 12, ACT, DROP>), grid, dim3(512), lds, s, a, sl);
                else hipLaunchKernelGGL((gn_slab_kernel<T, V, 16, ACT, DROP>), grid, dim3(512), lds, s, a, sl);
                return;
            }
        }
        const GnWork w = gn_work<V>(a);
        const dim3 grid((unsigned)(a.B * w.nchunk * w.nzb));
        double2 *part = (double2 *)ws;                           // (the room of the channels' pairs, which only the backward pass has)
        const unsigned char *mask = gn_mask<V>(a, ws, s);
        hipLaunchKernelGGL((gn_stats_kernel<T, V>), grid, dim3(256), 0, s, a, w, part);
        hipLaunchKernelGGL((gn_apply_kernel<T, V, ACT, DROP>), grid, dim3(256), gn_join_lds(a.G), s, a, w, part, mask);
    });
    return check_launch("group_norm_forward");
}
template <typename T> static int gn_backward(const GnArgs &a, void *ws, hipStream_t s) {
    gn_pick<T>(a, [&](auto v, auto act, auto drop) {
        constexpr int V = decltype(v)::value, ACT = decltype(act)::value;
        constexpr bool DROP = decltype(drop)::value;
        if constexpr (V * sizeof(T) == 16) {
            const GnSlab sl = gn_slab<V>(a, 12);
            if (sl.sv) {
                const int nv = (a.P * sl.sv + 511) / 512, lds = 10 * sl.sv * V * 4;
                const dim3 grid((unsigned)(a.B * sl.nslab));
                float2 *part = (float2 *)ws;
                if (nv <= 2) hipLaunchKernelGGL((gn_slab_bwd_kernel<T, V, 2, ACT, DROP>), grid, dim3(512), lds, s, a, sl, part);
                else if (nv <= 4) hipLaunchKernelGGL((gn_slab_bwd_kernel<T, V, 4, ACT, DROP>), grid, dim3(512), lds, s, a, sl, part);
                else if (nv <= 6) hipLaunchKernelGGL((gn_slab_bwd_kernel<T, V, 6, ACT, DROP>), grid, dim3(512), lds, s, a, sl, part);
                else hipLaunchKernelGGL((gn_slab_bwd_kernel<T, V, 12, ACT, DROP>), grid, dim3(512), lds, s, a, sl, part);
                if (a.B > 1) hipLaunchKernelGGL(gn_param_grads_kernel, dim3((unsigned)((a.C + 15) / 16)), dim3(1024), 0, s, a, a.B, part);
                return;
            }
        }
        const GnWork w = gn_work<V>(a);
        const dim3 grid((unsigned)(a.B * w.nchunk * w.nzb));
        float2 *gpart = (float2 *)ws, *part = gpart + (size_t)a.B * w.nchunk * w.nsub * a.G;
        unsigned char *mask = gn_mask<V>(a, ws, s);
        const int nparam = (a.C + 127) / 128 * 8;                // whole eights: a chunk stays on the XCD that pass 1 read it on
        hipLaunchKernelGGL((gn_bwd_sums_kernel<T, V, ACT, DROP>), grid, dim3(256), 0, s, a, w, part, gpart, mask);
        hipLaunchKernelGGL((gn_bwd_apply_kernel<T, V, ACT, DROP>), dim3(grid.x + nparam), dim3(256),
                           std::max(gn_join_lds(a.G), 16 * 17 * sizeof(double2)), s, a, w,
                           part, gpart, mask, nparam);
    });
    return check_launch("group_norm_backward");
}

int launch_group_norm_forward(const GnArgs &a, void *ws, hipStream_t s) {
    return a.dtype == YMX_BF16 ? gn_forward<bf16_t>(a, ws, s) : gn_forward<float>(a, ws, s);
}
int launch_group_norm_backward(const GnArgs &a, void *ws, hipStream_t s) {
    return a.dtype == YMX_BF16 ? gn_backward<bf16_t>(a, ws, s) : gn_backward<float>(a, ws, s);
}

// ---- dropout alone: y = keep * x / (1 - rate) (+ shortcut), over a flat map ------------------------
// Bound by memory (two or three maps); ten Philox rounds serve four elements.  The last n % V
// elements, and maps that are not 16-byte aligned, go one at a time.
template <typename T, int V>
__global__ void __launch_bounds__(256)
dropout_kernel(const T *__restrict__ x, const T *__restrict__ res, T *__restrict__ y, unsigned long long n, const DropArgs drop) {
    const uint4 key = {drop.state[0], drop.state[1], drop.state[2], drop.state[3]};
    const unsigned long long step = (unsigned long long)gridDim.x * 256 * V;
    unsigned long long i = ((unsigned long long)blockIdx.x * 256 + threadIdx.x) * V;
    auto one = [&](unsigned long long j, auto vtag) {
        constexpr int W = decltype(vtag)::value;
        typedef vec_io<T, W> W_IO;
        float v[W], s[W];
        bool keep[W];
        const typename W_IO::raw q = W_IO::load(x + j);
        typename W_IO::raw qs;
        if (res) qs = W_IO::load(res + j);
        drop_keep<W>(drop, key, j, keep);
        W_IO::unpack(q, v);
#pragma unroll
        for (int k = 0; k < W; ++k) v[k] = keep[k] ? v[k] * drop.keep_scale : 0.0f;
        if (res) {
            W_IO::unpack(qs, s);
#pragma unroll
            for (int k = 0; k < W; ++k) v[k] += s[k];
        }
        W_IO::store(y + j, v);
    };
    for (; i + V <= n; i += step) one(i, std::integral_constant<int, V>{});
    if constexpr (V > 1)
        for (; i < n; ++i) one(i, std::integral_constant<int, 1>{});
}

template <typename T> static void dropout_pick(const void *x, const void *res, void *y, long long n, const DropArgs &d, hipStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const bool vec = aligned16(x) && aligned16(y) && (res == nullptr || aligned16(res));
    const unsigned long long per = 256ull * (vec ? V : 1);
    const dim3 grid((unsigned)std::min<unsigned long long>(((unsigned long long)n + per - 1) / per, 8192));
    if (vec) hipLaunchKernelGGL((dropout_kernel<T, V>), grid, dim3(256), 0, s, (const T *)x, (const T *)res, (T *)y, (unsigned long long)n, d);
    else hipLaunchKernelGGL((dropout_kernel<T, 1>), grid, dim3(256), 0, s, (const T *)x, (const T *)res, (T *)y, (unsigned long long)n, d);
}
int launch_dropout(const void *x, const void *res, void *y, long long n, int dtype, unsigned threshold, float keep_scale,
                   const unsigned *state, hipStream_t s) {
    const DropArgs d = {state, threshold, keep_scale};
    if (dtype == YMX_BF16) dropout_pick<bf16_t>(x, res, y, n, d, s);
    else dropout_pick<float>(x, res, y, n, d, s);
    return check_launch("dropout");
}

}  // namespace ymx
