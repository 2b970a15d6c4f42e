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
// Form: the pixels of a sample are cut into chunks, a workgroup per chunk.  Pass 1 leaves one pair
// of numbers per (chunk, channel) -- mean and centred sum of squares, or sum dt and sum dt h --
// a small launch adds them per group (and per channel) in a fixed order, pass 2 reads the map
// again and writes.  All sums are fp32 and no result depends on the order workgroups run in.
#include <algorithm>
#include <type_traits>

#include "philox.h"

namespace ymx {

// Where a thread of the chunked kernels works: V channels from c0 of the pixels p, p + R, ... < p1 of sample b.
struct GnWork {
    int cvb, R, nzb;             // channel vectors per workgroup, pixels side by side, channel blocks
    int nchunk, per;             // chunks per sample, pixels per chunk
};
template <int V> struct GnPos {
    int b, chunk, zb, cv, r, c0, p, p1;
    bool on;
    __device__ __forceinline__ GnPos(const GnArgs &a, const GnWork &w) {
        int id = blockIdx.x;
        zb = id % w.nzb;
        id /= w.nzb;
        chunk = id % w.nchunk;
        b = id / w.nchunk;
        cv = threadIdx.x % w.cvb;
        r = threadIdx.x / w.cvb;
        c0 = (zb * w.cvb + cv) * V;
        on = r < w.R && c0 < a.C;
        p = chunk * w.per + r;
        p1 = min(a.P, (chunk + 1) * w.per);
    }
};

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

__device__ __forceinline__ int gn_chunk_pixels(int P, int per, int k) { return min(P - k * per, per); }

// Pass 1, forward: part[(b nchunk + chunk) C + c] = (mean, sum of squares about it) of the chunk's pixels.
// A thread sums about its own first value, so what cancels in s2 - s1^2 / n is at most n eps of the result.
template <typename T, int V>
__global__ void __launch_bounds__(256) gn_stats_kernel(const GnArgs a, const GnWork w, float2 *__restrict__ part) {
    __shared__ float2 red[256 * V];
    const GnPos<V> g(a, w);
    typedef vec_io<T, V> IO;
    const T *__restrict__ x = (const T *)a.x + (size_t)g.b * a.P * a.C + g.c0;
    const int W = w.cvb * V;
    if (g.on) {
        float piv[V], s1[V], s2[V];
#pragma unroll
        for (int i = 0; i < V; ++i) piv[i] = s1[i] = s2[i] = 0.0f;
        if (g.p < g.p1) IO::unpack(IO::load(x + (size_t)g.p * a.C), piv);
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
        for (int i = 0; i < V; ++i)
            red[g.r * W + g.cv * V + i] = float2{piv[i] + s1[i] * inv, fmaxf(s2[i] - s1[i] * s1[i] * inv, 0.0f)};
    }
    __syncthreads();
    const int np = g.p1 - g.chunk * w.per;                       // pixels of the chunk
    const int rows = min(w.R, np);
    for (int c = threadIdx.x; c < W && g.zb * W + c < a.C; c += 256) {
        float mean = 0.0f, m2 = 0.0f;
        for (int r = 0; r < rows; ++r) mean += (float)((np - r + w.R - 1) / w.R) * red[r * W + c].x;
        mean /= (float)np;
        for (int r = 0; r < rows; ++r) {
            const float2 q = red[r * W + c];
            const float d = q.x - mean;
            m2 += q.y + (float)((np - r + w.R - 1) / w.R) * d * d;
        }
        part[((size_t)g.b * w.nchunk + g.chunk) * a.C + g.zb * W + c] = float2{mean, m2};
    }
}

// Sum of v over the workgroup, the same value on every thread; scratch holds one float per wave.
__device__ __forceinline__ float gn_block_sum(float v, float *scratch) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    const int nw = blockDim.x >> 6;
    if (nw == 1) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.0f;
    for (int i = 0; i < nw; ++i) s += scratch[i];
    return s;
}

// One workgroup per (sample, group): the chunks' pairs -> (mean, 1 / sqrt(var + eps)).
__global__ void __launch_bounds__(1024) gn_stats_join_kernel(const GnArgs a, const GnWork w, const float2 *__restrict__ part) {
    __shared__ float scratch[16];
    const int b = blockIdx.x / a.G, g = blockIdx.x % a.G;
    const float2 *__restrict__ q = part + (size_t)b * w.nchunk * a.C + g * a.D;
    const int items = w.nchunk * a.D;
    const float N = (float)a.P * (float)a.D;
    float s = 0.0f;
    for (int i = threadIdx.x; i < items; i += blockDim.x) {
        const int k = i / a.D, c = i - k * a.D;
        s += (float)gn_chunk_pixels(a.P, w.per, k) * q[(size_t)k * a.C + c].x;
    }
    const float mean = gn_block_sum(s, scratch) / N;
    s = 0.0f;
    for (int i = threadIdx.x; i < items; i += blockDim.x) {
        const int k = i / a.D, c = i - k * a.D;
        const float2 v = q[(size_t)k * a.C + c];
        const float d = v.x - mean;
        s += v.y + (float)gn_chunk_pixels(a.P, w.per, k) * d * d;
    }
    const float var = gn_block_sum(s, scratch) / N;
    if (threadIdx.x == 0) ((float2 *)a.stats)[blockIdx.x] = float2{mean, 1.0f / sqrtf(var + a.eps)};
}

// The numbers of a thread's V channels: h = (x - mean) r, t = gamma h + beta.
template <int V> struct GnChannels {
    float mean[V], r[V], ga[V], be[V];
    __device__ __forceinline__ GnChannels(const GnArgs &a, int b, int c0) {
        const float2 *__restrict__ st = (const float2 *)a.stats + (size_t)b * a.G;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float2 m = st[(c0 + i) / a.D];
            mean[i] = m.x;
            r[i] = m.y;
            ga[i] = a.gamma[c0 + i];
            be[i] = a.beta[c0 + i];
        }
    }
};

// Pass 2, forward.
template <typename T, int V, int ACT, bool DROP>
__global__ void __launch_bounds__(256) gn_apply_kernel(const GnArgs a, const GnWork w) {
    const GnPos<V> g(a, w);
    if (!g.on) return;
    typedef vec_io<T, V> IO;
    const GnChannels<V> ch(a, g.b, g.c0);
    const size_t base = (size_t)g.b * a.P * a.C + g.c0;
    const T *__restrict__ x = (const T *)a.x + base, *__restrict__ res = (const T *)a.res + base;
    T *__restrict__ y = (T *)a.y + base;
    const bool has_res = a.res != nullptr;
    const DropArgs drop = {a.state, a.threshold, a.keep_scale};
    uint4 key = {};
    if constexpr (DROP) key = uint4{a.state[0], a.state[1], a.state[2], a.state[3]};
    struct Row { typename IO::raw x, s; };
    gn_rows<2>(g.p, g.p1, w.R, [&](int p) {
                   Row q;
                   q.x = IO::load(x + (size_t)p * a.C);
                   if (has_res) q.s = IO::load(res + (size_t)p * a.C);
                   return q;
               },
               [&](int p, const Row &q) {
                   float v[V], s[V];
                   bool keep[V];
                   IO::unpack(q.x, v);
                   if constexpr (DROP) drop_keep<V>(drop, key, base + (size_t)p * a.C, keep);
#pragma unroll
                   for (int i = 0; i < V; ++i) {
                       const float h = (v[i] - ch.mean[i]) * ch.r[i];
                       v[i] = act_c<ACT>(__builtin_fmaf(ch.ga[i], h, ch.be[i]));
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

// dt and h of one vector of a map and its gradient.
template <int V, int ACT, bool DROP>
__device__ __forceinline__ void gn_dt(const GnChannels<V> &ch, const DropArgs &drop, const uint4 &key, unsigned long long i0,
                                      const float (&x)[V], const float (&dy)[V], float (&dt)[V], float (&h)[V]) {
    bool keep[V];
    if constexpr (DROP) drop_keep<V>(drop, key, i0, keep);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        h[i] = (x[i] - ch.mean[i]) * ch.r[i];
        float d = dy[i];
        if constexpr (DROP) d = keep[i] ? d * drop.keep_scale : 0.0f;
        dt[i] = d * act_grad_c<ACT>(__builtin_fmaf(ch.ga[i], h[i], ch.be[i]));
    }
}

// Pass 1, backward: part[(b nchunk + chunk) C + c] = (sum dt, sum dt h) of the chunk's pixels.
template <typename T, int V, int ACT, bool DROP>
__global__ void __launch_bounds__(256) gn_bwd_sums_kernel(const GnArgs a, const GnWork w, float2 *__restrict__ part) {
    __shared__ float2 red[256 * V];
    const GnPos<V> g(a, w);
    typedef vec_io<T, V> IO;
    const int W = w.cvb * V;
    if (g.on) {
        const GnChannels<V> ch(a, g.b, g.c0);
        const size_t base = (size_t)g.b * a.P * a.C + g.c0;
        const T *__restrict__ x = (const T *)a.x + base, *__restrict__ dy = (const T *)a.dy + base;
        const DropArgs drop = {a.state, a.threshold, a.keep_scale};
        uint4 key = {};
        if constexpr (DROP) key = uint4{a.state[0], a.state[1], a.state[2], a.state[3]};
        float s1[V], s2[V];
#pragma unroll
        for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.0f;
        struct Row { typename IO::raw x, d; };
        gn_rows<2>(g.p, g.p1, w.R, [&](int p) { return Row{IO::load(x + (size_t)p * a.C), IO::load(dy + (size_t)p * a.C)}; },
                   [&](int p, const Row &q) {
                       float v[V], d[V], dt[V], h[V];
                       IO::unpack(q.x, v);
                       IO::unpack(q.d, d);
                       gn_dt<V, ACT, DROP>(ch, drop, key, base + (size_t)p * a.C, v, d, dt, h);
#pragma unroll
                       for (int i = 0; i < V; ++i) {
                           s1[i] += dt[i];
                           s2[i] += dt[i] * h[i];
                       }
                   });
#pragma unroll
        for (int i = 0; i < V; ++i) red[g.r * W + g.cv * V + i] = float2{s1[i], s2[i]};
    }
    __syncthreads();
    for (int c = threadIdx.x; c < W && g.zb * W + c < a.C; c += 256) {
        float2 s = {0.0f, 0.0f};
        for (int r = 0; r < w.R; ++r) {
            const float2 q = red[r * W + c];
            s.x += q.x;
            s.y += q.y;
        }
        part[((size_t)g.b * w.nchunk + g.chunk) * a.C + g.zb * W + c] = s;
    }
}

// Workgroups 0 .. B G - 1: gsum[b][g] = (S1, S2) / N.  The others, 32 channels each: dbeta and dgamma,
// the B nchunk pairs of a channel added by 8 row lanes and those in order.
__global__ void __launch_bounds__(256) gn_bwd_join_kernel(const GnArgs a, const GnWork w, const float2 *__restrict__ part,
                                                          float2 *__restrict__ gsum) {
    __shared__ float2 red[256];
    if ((int)blockIdx.x < a.B * a.G) {
        const int b = blockIdx.x / a.G, g = blockIdx.x % a.G;
        const float2 *__restrict__ q = part + (size_t)b * w.nchunk * a.C + g * a.D;
        const int items = w.nchunk * a.D;
        float s1 = 0.0f, s2 = 0.0f;
        for (int i = threadIdx.x; i < items; i += 256) {
            const int k = i / a.D, c = i - k * a.D;
            const float2 v = q[(size_t)k * a.C + c];
            const float ga = a.gamma[g * a.D + c];
            s1 += ga * v.x;
            s2 += ga * v.y;
        }
        s1 = gn_block_sum(s1, (float *)red);
        s2 = gn_block_sum(s2, (float *)red + 16);
        const float inv = 1.0f / ((float)a.P * (float)a.D);
        if (threadIdx.x == 0) gsum[blockIdx.x] = float2{s1 * inv, s2 * inv};
    } else {
        const int c = ((int)blockIdx.x - a.B * a.G) * 32 + (threadIdx.x & 31), row = threadIdx.x >> 5;
        float2 s = {0.0f, 0.0f};
        if (c < a.C) {
            const int rows = a.B * w.nchunk;
            for (int i = row; i < rows; i += 8) {
                const float2 v = part[(size_t)i * a.C + c];
                s.x += v.x;
                s.y += v.y;
            }
        }
        red[threadIdx.x] = s;
        __syncthreads();
        if (row == 0 && c < a.C) {
            for (int i = 1; i < 8; ++i) {
                s.x += red[i * 32 + threadIdx.x].x;
                s.y += red[i * 32 + threadIdx.x].y;
            }
            a.dbeta[c] = s.x;
            a.dgamma[c] = s.y;
        }
    }
}

// Pass 2, backward.
template <typename T, int V, int ACT, bool DROP>
__global__ void __launch_bounds__(256) gn_bwd_apply_kernel(const GnArgs a, const GnWork w, const float2 *__restrict__ gsum) {
    const GnPos<V> g(a, w);
    if (!g.on) return;
    typedef vec_io<T, V> IO;
    const GnChannels<V> ch(a, g.b, g.c0);
    float m1[V], m2[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float2 m = gsum[(size_t)g.b * a.G + (g.c0 + i) / a.D];
        m1[i] = m.x;
        m2[i] = m.y;
    }
    const size_t base = (size_t)g.b * a.P * a.C + g.c0;
    const T *__restrict__ x = (const T *)a.x + base, *__restrict__ dy = (const T *)a.dy + base;
    T *__restrict__ dx = (T *)a.dx + base;
    const DropArgs drop = {a.state, a.threshold, a.keep_scale};
    uint4 key = {};
    if constexpr (DROP) key = uint4{a.state[0], a.state[1], a.state[2], a.state[3]};
    struct Row { typename IO::raw x, d; };
    gn_rows<2>(g.p, g.p1, w.R, [&](int p) { return Row{IO::load(x + (size_t)p * a.C), IO::load(dy + (size_t)p * a.C)}; },
               [&](int p, const Row &q) {
                   float v[V], d[V], dt[V], h[V];
                   IO::unpack(q.x, v);
                   IO::unpack(q.d, d);
                   gn_dt<V, ACT, DROP>(ch, drop, key, base + (size_t)p * a.C, v, d, dt, h);
#pragma unroll
                   for (int i = 0; i < V; ++i) v[i] = ch.r[i] * (ch.ga[i] * dt[i] - (m1[i] + h[i] * m2[i]));
                   IO::store(dx + (size_t)p * a.C, v);
               });
}

// ---- host side -----------------------------------------------------------------------------------
// About 2048 workgroups (eight of 256 threads on each of 256 CUs), none with less than 16 K elements to read.
static int gn_chunks(int B, int P, int C) {
    const long long most = std::max<long long>(1, (long long)P * C / 16384);
    const long long want = std::max(1, 2048 / B);
    return (int)std::min<long long>(std::min(most, want), P);
}
template <int V> static GnWork gn_work(const GnArgs &a) {
    GnWork w;
    const int cv = (a.C + V - 1) / V;
    w.nzb = (cv + 255) / 256;
    w.cvb = (cv + w.nzb - 1) / w.nzb;
    w.R = 256 / w.cvb;
    w.per = (a.P + gn_chunks(a.B, a.P, a.C) - 1) / gn_chunks(a.B, a.P, a.C);
    w.nchunk = (a.P + w.per - 1) / w.per;
    return w;
}
size_t group_norm_workspace_bytes(int B, int P, int C, int G) {
    return ((size_t)B * gn_chunks(B, P, C) * C + (size_t)B * G) * sizeof(float2);
}
static int gn_join_threads(const GnArgs &a, const GnWork &w) {
    const long long items = (long long)w.nchunk * a.D;
    return items <= 256 ? 64 : items <= 4096 ? 256 : 1024;
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
// 16-byte vectors where the channel count and every map's address allow them, else one element at a time.
template <typename T, typename F> static void gn_pick(const GnArgs &a, F f) {
    constexpr int V = 16 / sizeof(T);
    auto ok = [](const void *p) { return p == nullptr || aligned16(p); };
    if (a.C % V == 0 && ok(a.x) && ok(a.res) && ok(a.dy) && ok(a.y) && ok(a.dx)) gn_pick_act<V>(a, f);
    else gn_pick_act<1>(a, f);
}

template <typename T> static int gn_forward(const GnArgs &a, void *ws, hipStream_t s) {
    float2 *part = (float2 *)ws;
    gn_pick<T>(a, [&](auto v, auto act, auto drop) {
        constexpr int V = decltype(v)::value;
        const GnWork w = gn_work<V>(a);
        const dim3 grid((unsigned)(a.B * w.nchunk * w.nzb));
        hipLaunchKernelGGL((gn_stats_kernel<T, V>), grid, dim3(256), 0, s, a, w, part);
        hipLaunchKernelGGL(gn_stats_join_kernel, dim3((unsigned)(a.B * a.G)), dim3(gn_join_threads(a, w)), 0, s, a, w, part);
        hipLaunchKernelGGL((gn_apply_kernel<T, V, decltype(act)::value, decltype(drop)::value>), grid, dim3(256), 0, s, a, w);
    });
    return check_launch("group_norm_forward");
}
template <typename T> static int gn_backward(const GnArgs &a, void *ws, hipStream_t s) {
    gn_pick<T>(a, [&](auto v, auto act, auto drop) {
        constexpr int V = decltype(v)::value;
        const GnWork w = gn_work<V>(a);
        const dim3 grid((unsigned)(a.B * w.nchunk * w.nzb));
        float2 *gsum = (float2 *)ws, *part = gsum + (size_t)a.B * a.G;
        hipLaunchKernelGGL((gn_bwd_sums_kernel<T, V, decltype(act)::value, decltype(drop)::value>), grid, dim3(256), 0, s, a, w, part);
        hipLaunchKernelGGL(gn_bwd_join_kernel, dim3((unsigned)(a.B * a.G + (a.C + 31) / 32)), dim3(256), 0, s, a, w, part, gsum);
        hipLaunchKernelGGL((gn_bwd_apply_kernel<T, V, decltype(act)::value, decltype(drop)::value>), grid, dim3(256), 0, s, a, w, gsum);
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
