// Group normalisation + activation (+ dropout) (+ shortcut), channels last, forward and backward.
//
//   mean, var over one image's HW pixels and one group's Cg = C / G channels;  r = 1 / sqrt(var + eps)
//   z = gamma (x - mean) r + beta,   y = res + drop(act(z))
//   dz = drop(dy) act'(z),  xh = (x - mean) r,   dbeta = sum dz,  dgamma = sum dz xh
//   dx = r (gamma dz - S1 - xh S2),   S1, S2 = group means of gamma dz and gamma dz xh
//
// Three launches per direction: partial sums per (image, pixel range, column), a fold, the element pass.  No atomics: a call's
// results do not depend on scheduling.
//
// A block works on one image n, one span of chunk columns and one range of pixels; thread = (row = t / width, chunk = t % width).
#include "layer_common.hpp"

namespace {

struct Shape {
    long HW, ppb;          // pixels per image / per block
    int N, C, G, Cg;
    int cpr;               // chunks (V elements) per pixel
    int nspan, width;      // chunk columns are cut into nspan spans of `width` (the last may be narrower)
    int nblk;              // pixel ranges per image
};

struct Where {
    int n, blk, chunk, row, rows, width;      // width: chunk columns of this block's span; rows: pixels it takes per pass
    bool on;                           // this thread has a column
    long p0, p1;
};

__device__ __forceinline__ Where where(const Shape& sh) {
    Where w;
    const int b = blockIdx.x;
    const int span = (b / sh.nblk) % sh.nspan;
    w.n = b / (sh.nblk * sh.nspan);
    w.blk = b % sh.nblk;
    const int left = sh.cpr - span * sh.width;
    w.width = left < sh.width ? left : sh.width;
    w.rows = 256 / w.width;
    w.row = threadIdx.x / w.width;
    w.chunk = span * sh.width + threadIdx.x % w.width;
    w.on = w.row < w.rows;
    w.p0 = w.blk * sh.ppb;
    w.p1 = w.p0 + sh.ppb < sh.HW ? w.p0 + sh.ppb : sh.HW;
    return w;
}

// smallest power of two >= n
__device__ __forceinline__ int pow2_up(int n) { return n <= 1 ? 1 : 1 << (32 - __clz(n - 1)); }

// Statistics of a column: NACC = 1 -- a chunk lies in one group, one (mean, sum of squares) per thread; NACC = V -- one per channel.
// Every thread sums deviations from the FIRST value it reads: that value is one of the column's own, so the square of its distance
// to the mean is at most the column's sum of squares and the subtraction q - s^2 / n loses at most a factor of the (small) number
// of values a thread holds -- whatever the mean of the data.  Threads are merged by mean and centred sum of squares.
template <typename T, int V, int NACC>
__global__ void __launch_bounds__(256) gn_stats_kernel(const T* x, int ldx, Shape sh, float* part) {
    __shared__ float s_m[256 * NACC], s_q[256 * NACC], s_n[256];
    const Where w = where(sh);
    float K[NACC], s[NACC], q[NACC];
#pragma unroll
    for (int a = 0; a < NACC; ++a) K[a] = s[a] = q[a] = 0.f;
    int cnt = 0;
    if (w.on) {
        const T* src = x + (long)w.n * sh.HW * ldx + w.chunk * V;
        for (long p = w.p0 + w.row; p < w.p1; p += w.rows) {
            float f[V];
            load_v<T, V>(src + p * ldx, f);
            if (cnt == 0) {
#pragma unroll
                for (int a = 0; a < NACC; ++a) K[a] = f[a];
            }
            ++cnt;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int a = NACC == 1 ? 0 : i;
                const float d = f[i] - K[a];
                s[a] += d;
                q[a] += d * d;
            }
        }
    }
    float n = (float)cnt * (V / NACC);
    float m[NACC];
#pragma unroll
    for (int a = 0; a < NACC; ++a) {
        const float sm = n > 0.f ? s[a] / n : 0.f;
        m[a] = K[a] + sm;
        q[a] = q[a] - s[a] * sm;
        s_m[threadIdx.x * NACC + a] = m[a];
        s_q[threadIdx.x * NACC + a] = q[a];
    }
    s_n[threadIdx.x] = n;
    __syncthreads();
    for (int h = pow2_up(w.rows) >> 1; h > 0; h >>= 1) {
        if (w.row < h && w.row + h < w.rows) {
            const int o = threadIdx.x + h * w.width;
            const float nb = s_n[o], na = s_n[threadIdx.x], nt = na + nb;
            if (nb > 0.f) {
                const float fb = nb / nt;
#pragma unroll
                for (int a = 0; a < NACC; ++a) {
                    const float d = s_m[o * NACC + a] - s_m[threadIdx.x * NACC + a];
                    s_m[threadIdx.x * NACC + a] += d * fb;
                    s_q[threadIdx.x * NACC + a] += s_q[o * NACC + a] + d * d * na * fb;
                }
                s_n[threadIdx.x] = nt;
            }
        }
        __syncthreads();
    }
    if (w.row == 0) {
        float* dst = part + (((long)w.n * sh.nblk + w.blk) * sh.cpr + w.chunk) * NACC * 2;
#pragma unroll
        for (int a = 0; a < NACC; ++a) {
            dst[2 * a] = s_m[threadIdx.x * NACC + a];
            dst[2 * a + 1] = s_q[threadIdx.x * NACC + a];
        }
    }
}

// One wave per (image, group): the group's columns over all pixel ranges -> (mean, r).  Double, two passes over the partials
// (weighted mean, then centred sum of squares).
__global__ void __launch_bounds__(256) gn_fold_kernel(const float* part, Shape sh, int cols_per_group, int per_col, float eps,
                                                     float* stats) {
    const long job = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (job >= (long)sh.N * sh.G) return;
    const int n = (int)(job / sh.G), g = (int)(job % sh.G);
    const int cols = cols_per_group * sh.G;
    const float2* src = reinterpret_cast<const float2*>(part) + (long)n * sh.nblk * cols + g * cols_per_group;
    const int E = sh.nblk * cols_per_group;
    double sum = 0.0;
    for (int i = lane; i < E; i += 64) {
        const int blk = i / cols_per_group, k = i - blk * cols_per_group;
        const long px = blk == sh.nblk - 1 ? sh.HW - blk * sh.ppb : sh.ppb;
        sum += (double)px * (double)src[(long)blk * cols + k].x;
    }
    const double total = (double)sh.HW * cols_per_group;
    const double mean = wave_sum_d(sum) / total;
    double m2 = 0.0;
    for (int i = lane; i < E; i += 64) {
        const int blk = i / cols_per_group, k = i - blk * cols_per_group;
        const long px = blk == sh.nblk - 1 ? sh.HW - blk * sh.ppb : sh.ppb;
        const float2 v = src[(long)blk * cols + k];
        const double d = (double)v.x - mean;
        m2 += (double)v.y + (double)px * per_col * d * d;
    }
    m2 = wave_sum_d(m2);
    if (lane == 0) {
        double var = m2 / (total * per_col);
        if (var < 0.0) var = 0.0;
        stats[2 * job] = (float)mean;
        stats[2 * job + 1] = (float)(1.0 / sqrt(var + (double)eps));
    }
}

// act < 0: chosen at run time (the one-element kernels)
template <int ACT, bool FAST>
__device__ __forceinline__ float act_any(float z, int act) {
    if constexpr (ACT >= 0) return act_f<ACT, FAST>(z);
    else return act == CY_ACT_MISH ? act_f<CY_ACT_MISH, FAST>(z) : act == CY_ACT_LEAKY ? act_f<CY_ACT_LEAKY, FAST>(z) : z;
}
template <int ACT, bool FAST>
__device__ __forceinline__ float act_grad_any(float z, int act) {
    if constexpr (ACT >= 0) return act_grad<ACT, FAST>(z);
    else return act == CY_ACT_MISH ? act_grad<CY_ACT_MISH, FAST>(z) : act == CY_ACT_LEAKY ? act_grad<CY_ACT_LEAKY, FAST>(z) : 1.f;
}

// xh = (x - mean) r and z = gamma xh + beta with every operation rounded (no contraction), in both directions: which side of the leaky
// activation's kink a value falls on is then a function of the inputs and the statistics alone, the same in the forward and the
// backward pass.  (The mean is subtracted first: folding it into the shift loses |mean| / deviation in accuracy.)
__device__ __forceinline__ float norm_xh(float x, float mean, float r) {
#pragma clang fp contract(off)
    const float d = x - mean;
    return d * r;
}
__device__ __forceinline__ float norm_z(float xh, float gamma, float beta) {
#pragma clang fp contract(off)
    const float g = xh * gamma;
    return g + beta;
}

template <typename T, int V, int ACT, bool DROP>
__global__ void __launch_bounds__(256) gn_apply_kernel(const T* x, int ldx, T* y, int ldy, const T* res, int ldres, Shape sh,
                                                      const float* stats, const float* gamma, const float* beta, int act,
                                                      DropRng rng) {
    constexpr bool FAST = sizeof(T) == 2;
    const Where w = where(sh);
    if (!w.on) return;
    DropKey key;
    if constexpr (DROP) key = drop_key(rng);
    float mu[V], rs[V], ga[V], be[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = w.chunk * V + i;
        const float* st = stats + 2 * ((long)w.n * sh.G + c / sh.Cg);
        mu[i] = st[0];
        rs[i] = st[1];
        ga[i] = gamma[c];
        be[i] = beta[c];
    }
    for (long p = w.p0 + w.row; p < w.p1; p += w.rows) {
        const long px = (long)w.n * sh.HW + p;
        float f[V];
        load_v<T, V>(x + px * ldx + w.chunk * V, f);
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = act_any<ACT, FAST>(norm_z(norm_xh(f[i], mu[i], rs[i]), ga[i], be[i]), act);
        if constexpr (DROP) drop_apply<V>(key, rng.q, rng.scale, (unsigned long long)px * sh.C + w.chunk * V, f);
        if (res) {
            float r[V];
            load_v<T, V>(res + px * ldres + w.chunk * V, r);
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] += r[i];
        }
        store_v<T, V>(y + px * ldy + w.chunk * V, f);
    }
}

// Partial sums of dz and dz * xh per (image, pixel range, channel)
template <typename T, int V, int ACT, bool DROP>
__global__ void __launch_bounds__(256) gn_bwd_sums_kernel(const T* x, int ldx, const T* dy, int lddy, Shape sh, const float* stats,
                                                         const float* gamma, const float* beta, int act, DropRng rng,
                                                         float* part) {
    constexpr bool FAST = sizeof(T) == 2;
    __shared__ float red[256 * V * 2];
    const Where w = where(sh);
    float a[V], b[V];
#pragma unroll
    for (int i = 0; i < V; ++i) a[i] = b[i] = 0.f;
    if (w.on) {
        DropKey key;
        if constexpr (DROP) key = drop_key(rng);
        float mu[V], rs[V], ga[V], be[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = w.chunk * V + i;
            const float* st = stats + 2 * ((long)w.n * sh.G + c / sh.Cg);
            mu[i] = st[0]; rs[i] = st[1]; ga[i] = gamma[c]; be[i] = beta[c];
        }
        for (long p = w.p0 + w.row; p < w.p1; p += w.rows) {
            const long px = (long)w.n * sh.HW + p;
            float f[V], g[V];
            load_v<T, V>(x + px * ldx + w.chunk * V, f);
            load_v<T, V>(dy + px * lddy + w.chunk * V, g);
            if constexpr (DROP) drop_apply<V>(key, rng.q, rng.scale, (unsigned long long)px * sh.C + w.chunk * V, g);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float xh = norm_xh(f[i], mu[i], rs[i]);
                const float dz = g[i] * act_grad_any<ACT, FAST>(norm_z(xh, ga[i], be[i]), act);
                a[i] += dz;
                b[i] += dz * xh;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
        red[(threadIdx.x * V + i) * 2] = a[i];
        red[(threadIdx.x * V + i) * 2 + 1] = b[i];
    }
    __syncthreads();
    for (int h = pow2_up(w.rows) >> 1; h > 0; h >>= 1) {
        if (w.row < h && w.row + h < w.rows) {
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) red[threadIdx.x * 2 * V + i] += red[(threadIdx.x + h * w.width) * 2 * V + i];
        }
        __syncthreads();
    }
    if (w.row == 0) {
        float* dst = part + ((((long)w.n * sh.nblk + w.blk) * sh.C) + w.chunk * V) * 2;
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) dst[i] = red[threadIdx.x * 2 * V + i];
    }
}

// One wave per (image, group): channel sums over the pixel ranges -> chan[n][c] = (sum dz, sum dz xh), and the group's S1, S2.
// P = lanes side by side on channels (a power of two, at most 64); the other 64 / P take pixel ranges in turn.
__global__ void __launch_bounds__(256) gn_bwd_fold_kernel(const float* part, Shape sh, const float* gamma, float* chan, float* s12) {
    const long job = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (job >= (long)sh.N * sh.G) return;
    const int n = (int)(job / sh.G), g = (int)(job % sh.G);
    const int up = pow2_up(sh.Cg), P = up < 64 ? up : 64;
    const float2* src = reinterpret_cast<const float2*>(part) + (long)n * sh.nblk * sh.C + (long)g * sh.Cg;
    double s1 = 0.0, s2 = 0.0;
    for (int c0 = 0; c0 < sh.Cg; c0 += P) {
        const int c = c0 + (lane & (P - 1));
        double a = 0.0, b = 0.0;
        if (c < sh.Cg)
            for (int k = lane / P; k < sh.nblk; k += 64 / P) {
                const float2 v = src[(long)k * sh.C + c];
                a += (double)v.x;
                b += (double)v.y;
            }
        for (int o = P; o < 64; o <<= 1) {
            a += __shfl_xor(a, o, 64);
            b += __shfl_xor(b, o, 64);
        }
        if (c < sh.Cg && lane < P) {
            const int cc = g * sh.Cg + c;
            chan[2 * ((long)n * sh.C + cc)] = (float)a;
            chan[2 * ((long)n * sh.C + cc) + 1] = (float)b;
            s1 += (double)gamma[cc] * a;
            s2 += (double)gamma[cc] * b;
        }
    }
    s1 = wave_sum_d(s1);
    s2 = wave_sum_d(s2);
    if (lane == 0) {
        const double m = (double)sh.HW * sh.Cg;
        s12[2 * job] = (float)(s1 / m);
        s12[2 * job + 1] = (float)(s2 / m);
    }
}

template <typename T, int V, int ACT, bool DROP>
__global__ void __launch_bounds__(256) gn_bwd_apply_kernel(const T* x, int ldx, const T* dy, int lddy, T* dx, int lddx, T* resg,
                                                          int ldrg, int res_accum, Shape sh, const float* stats,
                                                          const float* gamma, const float* beta, const float* chan,
                                                          const float* s12, float* ggamma, float* gbeta, float gscale,
                                                          int accumulate, int act, DropRng rng) {
    constexpr bool FAST = sizeof(T) == 2;
    const Where w = where(sh);
    if (!w.on) return;
    if (w.n == 0 && w.blk == 0 && w.row == 0) {      // parameter gradients of this span: image order, double
#pragma unroll 1
        for (int i = 0; i < V; ++i) {
            const int c = w.chunk * V + i;
            double a = 0.0, b = 0.0;
            for (int n = 0; n < sh.N; ++n) {
                a += (double)chan[2 * ((long)n * sh.C + c)];
                b += (double)chan[2 * ((long)n * sh.C + c) + 1];
            }
            if (gbeta) gbeta[c] = (accumulate ? gbeta[c] : 0.f) + gscale * (float)a;
            if (ggamma) ggamma[c] = (accumulate ? ggamma[c] : 0.f) + gscale * (float)b;
        }
    }
    DropKey key;
    if constexpr (DROP) key = drop_key(rng);
    float mu[V], rs[V], ga[V], be[V], m1[V], m2[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = w.chunk * V + i;
        const long j = 2 * ((long)w.n * sh.G + c / sh.Cg);
        mu[i] = stats[j]; rs[i] = stats[j + 1]; ga[i] = gamma[c]; be[i] = beta[c];
        m1[i] = s12[j]; m2[i] = s12[j + 1];
    }
    for (long p = w.p0 + w.row; p < w.p1; p += w.rows) {
        const long px = (long)w.n * sh.HW + p;
        float f[V], g[V];
        load_v<T, V>(x + px * ldx + w.chunk * V, f);
        load_v<T, V>(dy + px * lddy + w.chunk * V, g);
        if (resg) {      // the shortcut branch's gradient is dy itself
            float o[V];
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = 0.f;
            if (res_accum) load_v<T, V>(resg + px * ldrg + w.chunk * V, o);
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] += g[i];
            store_v<T, V>(resg + px * ldrg + w.chunk * V, o);
        }
        if constexpr (DROP) drop_apply<V>(key, rng.q, rng.scale, (unsigned long long)px * sh.C + w.chunk * V, g);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float xh = norm_xh(f[i], mu[i], rs[i]);
            const float dz = g[i] * act_grad_any<ACT, FAST>(norm_z(xh, ga[i], be[i]), act);
            f[i] = rs[i] * (ga[i] * dz - m1[i] - xh * m2[i]);
        }
        store_v<T, V>(dx + px * lddx + w.chunk * V, f);
    }
}

// no pixels at all: the parameter gradients are zero sums
__global__ void gn_no_pixels_kernel(float* ggamma, float* gbeta, int C) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= C) return;
    if (ggamma) ggamma[c] = 0.f;
    if (gbeta) gbeta[c] = 0.f;
}

// ---- host ------------------------------------------------------------------------------------------------------------------
// Blocks for eight waves per SIMD on 256 compute units; a thread takes at least four pixels of its column.
constexpr long TARGET_BLOCKS = 2048;

Shape make_shape(int N, long HW, int C, int G, int V) {
    Shape sh;
    sh.N = N; sh.HW = HW; sh.C = C; sh.G = G; sh.Cg = C / G;
    sh.cpr = C / V;
    sh.nspan = (sh.cpr + 255) / 256;
    sh.width = (sh.cpr + sh.nspan - 1) / sh.nspan;
    const long rows = 256 / sh.width;
    long nblk = TARGET_BLOCKS / ((long)N * sh.nspan);
    const long most = (HW + 4 * rows - 1) / (4 * rows);
    if (nblk > most) nblk = most;
    if (nblk < 1) nblk = 1;
    sh.ppb = (HW + nblk - 1) / nblk;
    sh.ppb = (sh.ppb + rows - 1) / rows * rows;
    sh.nblk = (int)((HW + sh.ppb - 1) / sh.ppb);
    return sh;
}

bool sizes_ok(int N, int64_t HW, int C, int G, int dtype) {
    return N >= 0 && HW >= 0 && C >= 1 && G >= 1 && C % G == 0 && (dtype == CY_F16 || dtype == CY_BF16 || dtype == CY_F32);
}

// floats: partials (two per image, pixel range and channel) + (mean, r) or (S1, S2) per group + two per image and channel
int64_t need_floats(const Shape& sh) {
    return 2 * ((int64_t)sh.N * sh.nblk * sh.C + (int64_t)sh.N * sh.G + (int64_t)sh.N * sh.C);
}

bool grid_ok(const Shape& sh) { return (int64_t)sh.N * sh.nspan * sh.nblk < (1ll << 31) && ((int64_t)sh.N * sh.G + 3) / 4 < (1ll << 31); }

template <typename T, int V>
int forward(const T* x, int ldx, T* y, int ldy, const T* res, int ldres, const Shape& sh, const float* gamma, const float* beta,
            float eps, int act, const DropRng& rng, float* stats, float* ws, hipStream_t s) {
    if (!grid_ok(sh)) return CY_ERR_ARG;
    float* part = ws;
    if (!stats) stats = ws + 2 * (int64_t)sh.N * sh.nblk * sh.C;
    const dim3 grid((unsigned)((long)sh.N * sh.nspan * sh.nblk)), fgrid((unsigned)(((long)sh.N * sh.G + 3) / 4));
    const bool one = sh.Cg % V == 0;
    if (one) hipLaunchKernelGGL((gn_stats_kernel<T, V, 1>), grid, dim3(256), 0, s, x, ldx, sh, part);
    else hipLaunchKernelGGL((gn_stats_kernel<T, V, V>), grid, dim3(256), 0, s, x, ldx, sh, part);
    CY_LAUNCH_CHECK();
    hipLaunchKernelGGL(gn_fold_kernel, fgrid, dim3(256), 0, s, part, sh, one ? sh.Cg / V : sh.Cg, one ? V : 1, eps, stats);
    CY_LAUNCH_CHECK();
#define CY_GNA(A_, D_)                                                                                                         \
    hipLaunchKernelGGL((gn_apply_kernel<T, V, A_, D_>), grid, dim3(256), 0, s, x, ldx, y, ldy, res, ldres, sh, stats, gamma, beta, act, rng)
#define CY_GNA_ACT(A_)             \
    do {                           \
        if (rng.q) CY_GNA(A_, true); \
        else CY_GNA(A_, false);    \
    } while (0)
    if constexpr (V == 1) CY_GNA_ACT(-1);
    else if (act == CY_ACT_MISH) CY_GNA_ACT(CY_ACT_MISH);
    else if (act == CY_ACT_LEAKY) CY_GNA_ACT(CY_ACT_LEAKY);
    else CY_GNA_ACT(CY_ACT_LINEAR);
#undef CY_GNA_ACT
#undef CY_GNA
    CY_LAUNCH_CHECK();
    return 0;
}

template <typename T, int V>
int backward(const T* x, int ldx, const T* dy, int lddy, T* dx, int lddx, T* resg, int ldrg, int res_accum, const Shape& sh,
             const float* gamma, const float* beta, const float* stats, int act, const DropRng& rng, float* ggamma, float* gbeta,
             float gscale, int accumulate, float* ws, hipStream_t s) {
    if (!grid_ok(sh)) return CY_ERR_ARG;
    float* part = ws;
    float* s12 = part + 2 * (int64_t)sh.N * sh.nblk * sh.C;
    float* chan = s12 + 2 * (int64_t)sh.N * sh.G;
    const dim3 grid((unsigned)((long)sh.N * sh.nspan * sh.nblk)), fgrid((unsigned)(((long)sh.N * sh.G + 3) / 4));
#define CY_GNB(A_, D_)                                                                                                        \
    do {                                                                                                                      \
        hipLaunchKernelGGL((gn_bwd_sums_kernel<T, V, A_, D_>), grid, dim3(256), 0, s, x, ldx, dy, lddy, sh, stats, gamma, beta, \
                           act, rng, part);                                                                                   \
        CY_LAUNCH_CHECK();                                                                                                    \
        hipLaunchKernelGGL(gn_bwd_fold_kernel, fgrid, dim3(256), 0, s, part, sh, gamma, chan, s12);                            \
        CY_LAUNCH_CHECK();                                                                                                    \
        hipLaunchKernelGGL((gn_bwd_apply_kernel<T, V, A_, D_>), grid, dim3(256), 0, s, x, ldx, dy, lddy, dx, lddx, resg, ldrg, \
                           res_accum, sh, stats, gamma, beta, chan, s12, ggamma, gbeta, gscale, accumulate, act, rng);         \
    } while (0)
#define CY_GNB_ACT(A_)             \
    do {                           \
        if (rng.q) CY_GNB(A_, true); \
        else CY_GNB(A_, false);    \
    } while (0)
    if constexpr (V == 1) CY_GNB_ACT(-1);
    else if (act == CY_ACT_MISH) CY_GNB_ACT(CY_ACT_MISH);
    else if (act == CY_ACT_LEAKY) CY_GNB_ACT(CY_ACT_LEAKY);
    else CY_GNB_ACT(CY_ACT_LINEAR);
#undef CY_GNB_ACT
#undef CY_GNB
    CY_LAUNCH_CHECK();
    return 0;
}

// 16-byte accesses where every row of every operand starts on one
template <typename T>
bool rows16(const void* p, int ld) {
    return !p || (aligned_to(p, 16) && ld % Elem<T>::CH == 0);
}

template <typename T>
int forward_any(const void* x, int ldx, void* y, int ldy, const void* res, int ldres, int N, long HW, int C, int G,
                const float* gamma, const float* beta, float eps, int act, const DropRng& rng, float* stats, float* ws,
                int64_t ws_bytes, hipStream_t s) {
    constexpr int CH = Elem<T>::CH;
    if (!aligned_to(x, sizeof(T)) || !aligned_to(y, sizeof(T)) || !aligned_to(res, sizeof(T))) return CY_ERR_ARG;
    const bool vec = C % CH == 0 && rows16<T>(x, ldx) && rows16<T>(y, ldy) && rows16<T>(res, ldres);
    const Shape sh = make_shape(N, HW, C, G, vec ? CH : 1);
    if (ws_bytes < 4 * need_floats(sh)) return CY_ERR_ARG;
    if (vec) return forward<T, CH>((const T*)x, ldx, (T*)y, ldy, (const T*)res, ldres, sh, gamma, beta, eps, act, rng, stats, ws, s);
    return forward<T, 1>((const T*)x, ldx, (T*)y, ldy, (const T*)res, ldres, sh, gamma, beta, eps, act, rng, stats, ws, s);
}

template <typename T>
int backward_any(const void* x, int ldx, const void* dy, int lddy, void* dx, int lddx, void* resg, int ldrg, int res_accum, int N,
                 long HW, int C, int G, const float* gamma, const float* beta, const float* stats, int act, const DropRng& rng,
                 float* ggamma, float* gbeta, float gscale, int accumulate, float* ws, int64_t ws_bytes, hipStream_t s) {
    constexpr int CH = Elem<T>::CH;
    if (!aligned_to(x, sizeof(T)) || !aligned_to(dy, sizeof(T)) || !aligned_to(dx, sizeof(T)) || !aligned_to(resg, sizeof(T)))
        return CY_ERR_ARG;
    const bool vec = C % CH == 0 && rows16<T>(x, ldx) && rows16<T>(dy, lddy) && rows16<T>(dx, lddx) && rows16<T>(resg, ldrg);
    const Shape sh = make_shape(N, HW, C, G, vec ? CH : 1);
    if (ws_bytes < 4 * need_floats(sh)) return CY_ERR_ARG;
    if (vec)
        return backward<T, CH>((const T*)x, ldx, (const T*)dy, lddy, (T*)dx, lddx, (T*)resg, ldrg, res_accum, sh, gamma, beta, stats,
                               act, rng, ggamma, gbeta, gscale, accumulate, ws, s);
    return backward<T, 1>((const T*)x, ldx, (const T*)dy, lddy, (T*)dx, lddx, (T*)resg, ldrg, res_accum, sh, gamma, beta, stats, act,
                          rng, ggamma, gbeta, gscale, accumulate, ws, s);
}

}  // namespace

extern "C" int64_t cy_gn_workspace(int N, int64_t HW, int C, int groups, int dtype) {
    if (!sizes_ok(N, HW, C, groups, dtype)) return CY_ERR_ARG;
    if (N == 0 || HW == 0) return 16;
    int64_t most = need_floats(make_shape(N, (long)HW, C, groups, 1));       // (whichever access width a call's pointers allow)
    const int ch = dtype == CY_F32 ? 4 : 8;
    if (C % ch == 0) {
        const int64_t v = need_floats(make_shape(N, (long)HW, C, groups, ch));
        if (v > most) most = v;
    }
    return 4 * most;
}

extern "C" int cy_gn_act_fwd(const void* x, int ldx, void* y, int ldy, const void* res, int ldres, int N, int64_t HW, int C,
                             int groups, const float* gamma, const float* beta, float eps, int act, int dtype, float* stats, int q,
                             const int64_t* rng, int id, void* ws, int64_t ws_bytes, cy_stream_t s) {
    CY_ENTER();
    DropRng r;
    if (!sizes_ok(N, HW, C, groups, dtype) || ldx < C || ldy < C || (res && ldres < C) || !gamma || !beta || !(eps >= 0.f) ||
        act < CY_ACT_LINEAR || act > CY_ACT_MISH || !make_drop(q, rng, id, r))
        return CY_ERR_ARG;
    if (N == 0 || HW == 0) return 0;
    if (!x || !y || !ws || !aligned_to(ws, 8) || !aligned_to(stats, 8)) return CY_ERR_ARG;
#define CY_GNF(T) \
    return forward_any<T>(x, ldx, y, ldy, res, ldres, N, (long)HW, C, groups, gamma, beta, eps, act, r, stats, (float*)ws, ws_bytes, cy_s(s))
    if (dtype == CY_F16) CY_GNF(f16);
    if (dtype == CY_BF16) CY_GNF(bf16);
    CY_GNF(float);
#undef CY_GNF
}

extern "C" int cy_gn_act_bwd(const void* x, int ldx, const void* dy, int lddy, void* dx, int lddx, void* res_grad, int ldrg,
                             int res_accum, int N, int64_t HW, int C, int groups, const float* gamma, const float* beta,
                             const float* stats, int act, int dtype, float* ggamma, float* gbeta, float gscale, int accumulate,
                             int q, const int64_t* rng, int id, void* ws, int64_t ws_bytes, cy_stream_t s) {
    CY_ENTER();
    DropRng r;
    if (!sizes_ok(N, HW, C, groups, dtype) || ldx < C || lddy < C || lddx < C || (res_grad && ldrg < C) || !gamma || !beta ||
        act < CY_ACT_LINEAR || act > CY_ACT_MISH || !make_drop(q, rng, id, r))
        return CY_ERR_ARG;
    if (N == 0 || HW == 0) {
        if (accumulate || (!ggamma && !gbeta)) return 0;
        hipLaunchKernelGGL(gn_no_pixels_kernel, dim3((C + 255) / 256), dim3(256), 0, cy_s(s), ggamma, gbeta, C);
        CY_LAUNCH_CHECK();
        return 0;
    }
    if (!x || !dy || !dx || !stats || !ws || !aligned_to(ws, 8) || !aligned_to(stats, 8)) return CY_ERR_ARG;
#define CY_GNBW(T)                                                                                                             \
    return backward_any<T>(x, ldx, dy, lddy, dx, lddx, res_grad, ldrg, res_accum, N, (long)HW, C, groups, gamma, beta, stats, act, r, \
                           ggamma, gbeta, gscale, accumulate, (float*)ws, ws_bytes, cy_s(s))
    if (dtype == CY_F16) CY_GNBW(f16);
    if (dtype == CY_BF16) CY_GNBW(bf16);
    CY_GNBW(float);
#undef CY_GNBW
}
