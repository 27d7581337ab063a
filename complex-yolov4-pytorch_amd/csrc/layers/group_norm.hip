// Group normalisation + activation (+ dropout) (+ shortcut), channels last, forward and backward.
//
//   mean, var over one image's HW pixels and one group's Cg = C / G channels;  r = 1 / sqrt(var + eps)
//   z = gamma (x - mean) r + beta,   y = res + drop(act(z))
//   dz = drop(dy) act'(z),  xh = (x - mean) r,   dbeta = sum dz,  dgamma = sum dz xh
//   dx = r (gamma dz - S1 - xh S2),   S1, S2 = group means of gamma dz and gamma dz xh
//
// This file: the choice of kernels, the C entry points, and the general kernels -- three launches per direction: partial sums per
// (image, pixel range, column), a fold, the element pass -- for any row stride, alignment and channel count (16 x 304 x 304 x 64 f16
// backward 191 us in three launches, 171 in one and the parameter gradients'; 32 x 76 x 76 x 256 bf16 with a shortcut forward 68 and 64;
// 1 x 1216 x 1216 x 32 f16, which only they take, 64 forward and 97 backward).  The one-launch kernels are in gn_resident*.
// No floating-point atomics anywhere: a call's results do not depend on scheduling.
//
// A block works on one image n, one span of chunk columns and one range of pixels; thread = (row = t / width, chunk = t % width).
#include "gn_math.hpp"
#include "gn_resident.hpp"

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

// Pixels of this thread in batches of U: batch(first pixel of the thread, distance) while U are left, then the rest one at a time.  Inside a batch
// there is no branch, so that its loads stay in front of its arithmetic and are in flight together.
template <int U, class Batch, class Single>
__device__ __forceinline__ void each_pixel(const Where& w, Batch batch, Single single) {
    long p = w.p0 + w.row;
    for (; p + (long)(U - 1) * w.rows < w.p1; p += (long)U * w.rows) batch(p);
    for (; p < w.p1; p += w.rows) single(p);
}

// Statistics of a column: NACC = 1 -- a chunk lies in one group, one (mean, sum of squares) per thread; NACC = V -- one per channel.
// Every thread sums deviations from the FIRST value it reads: that value is one of the column's own, so the square of its distance
// to the mean is at most the column's sum of squares and the subtraction q - s^2 / n loses at most a factor of the (small) number
// of values a thread holds -- whatever the mean of the data.  Threads are merged by mean and centred sum of squares.
template <typename T, int V, int NACC>
__global__ void __launch_bounds__(256) gn_stats_kernel(const T* x, int ldx, Shape sh, float* part) {
    constexpr int U = 8;
    __shared__ float s_m[256 * NACC], s_q[256 * NACC], s_n[256];
    const Where w = where(sh);
    float K[NACC], s[NACC], q[NACC];
#pragma unroll
    for (int a = 0; a < NACC; ++a) K[a] = s[a] = q[a] = 0.f;
    int cnt = 0;
    if (w.on) {
        const T* src = x + (long)w.n * sh.HW * ldx + w.chunk * V;
        auto take = [&](const Raw<T, V>& in) {
            float f[V];
            in.get(f);
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
        };
        each_pixel<U>(
            w,
            [&](long p) {
                Raw<T, V> in[U];
#pragma unroll
                for (int u = 0; u < U; ++u) in[u].load(src + (p + u * w.rows) * ldx);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int u = 0; u < U; ++u) take(in[u]);
            },
            [&](long p) {
                Raw<T, V> in;
                in.load(src + p * ldx);
                take(in);
            });
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

// Sum over the block, the same in every thread
__device__ __forceinline__ double block_sum_d(double v, double* s4) {
    v = wave_sum_d(v);
    if ((threadIdx.x & 63) == 0) s4[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (s4[0] + s4[1]) + (s4[2] + s4[3]);
    __syncthreads();
    return v;
}

// One block per (image, group): the group's columns over all pixel ranges -> (mean, r).  Double, two passes over the partials
// (weighted mean, then centred sum of squares).
__global__ void __launch_bounds__(256) gn_fold_kernel(const float* part, Shape sh, int cols_per_group, int per_col, float eps,
                                                     float* stats) {
    __shared__ double s4[4];
    const long job = blockIdx.x;
    const int n = (int)(job / sh.G), g = (int)(job % sh.G);
    const int cols = cols_per_group * sh.G;
    const float2* src = reinterpret_cast<const float2*>(part) + (long)n * sh.nblk * cols + g * cols_per_group;
    const int E = sh.nblk * cols_per_group;
    double sum = 0.0;
#pragma unroll 4
    for (int i = threadIdx.x; i < E; i += 256) {
        const int blk = i / cols_per_group, k = i - blk * cols_per_group;
        const long px = blk == sh.nblk - 1 ? sh.HW - blk * sh.ppb : sh.ppb;
        sum += (double)px * (double)src[(long)blk * cols + k].x;
    }
    const double total = (double)sh.HW * cols_per_group;
    const double mean = block_sum_d(sum, s4) / total;
    double m2 = 0.0;
#pragma unroll 4
    for (int i = threadIdx.x; i < E; i += 256) {
        const int blk = i / cols_per_group, k = i - blk * cols_per_group;
        const long px = blk == sh.nblk - 1 ? sh.HW - blk * sh.ppb : sh.ppb;
        const float2 v = src[(long)blk * cols + k];
        const double d = (double)v.x - mean;
        m2 += (double)v.y + (double)px * per_col * d * d;
    }
    m2 = block_sum_d(m2, s4);
    if (threadIdx.x == 0) {
        stats[2 * job] = (float)mean;
        stats[2 * job + 1] = gn_rstd(m2 / (total * per_col), eps);
    }
}

template <typename T, int V, int ACT, bool DROP>
__global__ void __launch_bounds__(256) gn_apply_kernel(const T* x, int ldx, T* y, int ldy, const T* res, int ldres, Shape sh,
                                                      const float* stats, const float* gamma, const float* beta,
                                                      DropRng rng) {
    constexpr bool FAST = sizeof(T) == 2;
    constexpr int U = 4;
    const Where w = where(sh);
    if (!w.on) return;
    DropKey key;
    if constexpr (DROP) key = drop_key(rng);
    Norm<T, ACT> nm[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = w.chunk * V + i;
        nm[i].set(*reinterpret_cast<const float2*>(stats + 2 * ((long)w.n * sh.G + c / sh.Cg)), gamma[c], beta[c]);
    }
    const long img = (long)w.n * sh.HW;
    auto put = [&](long px, const Raw<T, V>& in, const Raw<T, V>& rin) {
        float f[V];
        in.get(f);
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = gn_act<ACT, FAST>(nm[i].z(f[i]));
        if constexpr (DROP) drop_apply<V>(key, rng.q, rng.scale, (unsigned long long)px * sh.C + w.chunk * V, f);
        if (res) {
            float r[V];
            rin.get(r);
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] += r[i];
        }
        store_v<T, V>(y + px * ldy + w.chunk * V, f);
    };
    each_pixel<U>(
        w,
        [&](long p) {
            Raw<T, V> in[U], rin[U];
#pragma unroll
            for (int u = 0; u < U; ++u) in[u].load(x + (img + p + u * w.rows) * ldx + w.chunk * V);
            if (res) {
#pragma unroll
                for (int u = 0; u < U; ++u) rin[u].load(res + (img + p + u * w.rows) * ldres + w.chunk * V);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < U; ++u) put(img + p + u * w.rows, in[u], rin[u]);
        },
        [&](long p) {
            Raw<T, V> in, rin;
            in.load(x + (img + p) * ldx + w.chunk * V);
            if (res) rin.load(res + (img + p) * ldres + w.chunk * V);
            put(img + p, in, rin);
        });
}

// Partial sums of dz and dz * xh per (image, pixel range, channel)
template <typename T, int V, int ACT, bool DROP>
__global__ void __launch_bounds__(256) gn_bwd_sums_kernel(const T* x, int ldx, const T* dy, int lddy, Shape sh, const float* stats,
                                                         const float* gamma, const float* beta, DropRng rng, float* part) {
    constexpr bool FAST = sizeof(T) == 2;
    constexpr int U = 4;
    __shared__ float red[256 * V * 2];
    const Where w = where(sh);
    float a[V], b[V];
#pragma unroll
    for (int i = 0; i < V; ++i) a[i] = b[i] = 0.f;
    if (w.on) {
        DropKey key;
        if constexpr (DROP) key = drop_key(rng);
        Norm<T, ACT> nm[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = w.chunk * V + i;
            nm[i].set(*reinterpret_cast<const float2*>(stats + 2 * ((long)w.n * sh.G + c / sh.Cg)), gamma[c], beta[c]);
        }
        const long img = (long)w.n * sh.HW;
        auto take = [&](long px, const Raw<T, V>& in, const Raw<T, V>& gin) {
            float f[V], g[V];
            in.get(f);
            gin.get(g);
            if constexpr (DROP) drop_apply<V>(key, rng.q, rng.scale, (unsigned long long)px * sh.C + w.chunk * V, g);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float dz = rounded(g[i] * gn_act_grad<ACT, FAST>(nm[i].z(f[i])));
                a[i] += dz;
                b[i] += dz * (f[i] - nm[i].mean);
            }
        };
        each_pixel<U>(
            w,
            [&](long p) {
                Raw<T, V> in[U], gin[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    in[u].load(x + (img + p + u * w.rows) * ldx + w.chunk * V);
                    gin[u].load(dy + (img + p + u * w.rows) * lddy + w.chunk * V);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int u = 0; u < U; ++u) take(img + p + u * w.rows, in[u], gin[u]);
            },
            [&](long p) {
                Raw<T, V> in, gin;
                in.load(x + (img + p) * ldx + w.chunk * V);
                gin.load(dy + (img + p) * lddy + w.chunk * V);
                take(img + p, in, gin);
            });
#pragma unroll
        for (int i = 0; i < V; ++i) b[i] *= nm[i].r;
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

// One block per (image, group): channel sums over the pixel ranges -> chan[n][c] = (sum dz, sum dz xh), and the group's S1, S2.
// P = threads side by side on channels (a power of two, at most 256); the other 256 / P take pixel ranges in turn.
__global__ void __launch_bounds__(256) gn_bwd_fold_kernel(const float* part, Shape sh, const float* gamma, float* chan, float* s12) {
    __shared__ double s_a[256], s_b[256], s4[4];
    const long job = blockIdx.x;
    const int t = threadIdx.x, n = (int)(job / sh.G), g = (int)(job % sh.G);
    const int up = pow2_up(sh.Cg), P = up < 256 ? up : 256;
    const float2* src = reinterpret_cast<const float2*>(part) + (long)n * sh.nblk * sh.C + (long)g * sh.Cg;
    double s1 = 0.0, s2 = 0.0;
    for (int c0 = 0; c0 < sh.Cg; c0 += P) {
        const int c = c0 + (t & (P - 1));
        double a = 0.0, b = 0.0;
        if (c < sh.Cg) {
#pragma unroll 4
            for (int k = t / P; k < sh.nblk; k += 256 / P) {
                const float2 v = src[(long)k * sh.C + c];
                a += (double)v.x;
                b += (double)v.y;
            }
        }
        s_a[t] = a;
        s_b[t] = b;
        __syncthreads();
        for (int h = 128; h >= P; h >>= 1) {
            if (t < h) {
                s_a[t] += s_a[t + h];
                s_b[t] += s_b[t + h];
            }
            __syncthreads();
        }
        if (c < sh.Cg && t < P) {
            const int cc = g * sh.Cg + c;
            chan[2 * ((long)n * sh.C + cc)] = (float)s_a[t];
            chan[2 * ((long)n * sh.C + cc) + 1] = (float)s_b[t];
            s1 += (double)gamma[cc] * s_a[t];
            s2 += (double)gamma[cc] * s_b[t];
        }
        __syncthreads();
    }
    s1 = block_sum_d(s1, s4);
    s2 = block_sum_d(s2, s4);
    if (t == 0) {
        const double m = (double)sh.HW * sh.Cg;
        s12[2 * job] = (float)(s1 / m);
        s12[2 * job + 1] = (float)(s2 / m);
    }
}

// Parameter gradients from the images' channel sums, in double: a block takes eight channels, 32 lanes take images in turn and are added
// in order.
__device__ __forceinline__ void param_grads(int first, int N, int C, const float* chan, float* ggamma, float* gbeta, float gscale,
                                            int accumulate) {
    __shared__ double s_a[32][9], s_b[32][9];
    const int k = threadIdx.x & 7, l = threadIdx.x >> 3, c = first + k;
    double a = 0.0, b = 0.0;
    if (c < C) {
#pragma unroll 4
        for (int n = l; n < N; n += 32) {
            const float2 v = *reinterpret_cast<const float2*>(chan + 2 * ((long)n * C + c));
            a += (double)v.x;
            b += (double)v.y;
        }
    }
    s_a[l][k] = a;
    s_b[l][k] = b;
    __syncthreads();
    if (l > 0 || c >= C) return;
    for (int i = 1; i < 32; ++i) {
        a += s_a[i][k];
        b += s_b[i][k];
    }
    if (gbeta) gbeta[c] = (accumulate ? gbeta[c] : 0.f) + gscale * (float)a;
    if (ggamma) ggamma[c] = (accumulate ? ggamma[c] : 0.f) + gscale * (float)b;
}

template <typename T, int V, int ACT, bool DROP>
__global__ void __launch_bounds__(256) gn_bwd_apply_kernel(const T* x, int ldx, const T* dy, int lddy, T* dx, int lddx, T* resg,
                                                          int ldrg, int res_accum, Shape sh, const float* stats,
                                                          const float* gamma, const float* beta, const float* chan,
                                                          const float* s12, float* ggamma, float* gbeta, float gscale,
                                                          int accumulate, DropRng rng) {
    constexpr bool FAST = sizeof(T) == 2;
    constexpr int U = 4;
    const long work = (long)sh.N * sh.nspan * sh.nblk;
    if (blockIdx.x >= work) return param_grads((int)(blockIdx.x - work) * 8, sh.N, sh.C, chan, ggamma, gbeta, gscale, accumulate);
    const Where w = where(sh);
    if (!w.on) return;
    DropKey key;
    if constexpr (DROP) key = drop_key(rng);
    Norm<T, ACT> nm[V];
    float2 k[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = w.chunk * V + i;
        const long j = 2 * ((long)w.n * sh.G + c / sh.Cg);
        nm[i].set(*reinterpret_cast<const float2*>(stats + j), gamma[c], beta[c]);
        k[i] = gn_k01(nm[i].r, s12[j], s12[j + 1]);
    }
    const long img = (long)w.n * sh.HW;
    auto put = [&](long px, const Raw<T, V>& in, const Raw<T, V>& gin) {
        float f[V], g[V];
        in.get(f);
        gin.get(g);
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
        for (int i = 0; i < V; ++i) f[i] = gn_dx(nm[i], k[i], f[i], rounded(g[i] * gn_act_grad<ACT, FAST>(nm[i].z(f[i]))));
        store_v<T, V>(dx + px * lddx + w.chunk * V, f);
    };
    each_pixel<U>(
        w,
        [&](long p) {
            Raw<T, V> in[U], gin[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                in[u].load(x + (img + p + u * w.rows) * ldx + w.chunk * V);
                gin[u].load(dy + (img + p + u * w.rows) * lddy + w.chunk * V);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < U; ++u) put(img + p + u * w.rows, in[u], gin[u]);
        },
        [&](long p) {
            Raw<T, V> in, gin;
            in.load(x + (img + p) * ldx + w.chunk * V);
            gin.load(dy + (img + p) * lddy + w.chunk * V);
            put(img + p, in, gin);
        });
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

constexpr int64_t MAX_BLOCKS = 1 << 24;      // a launch has fewer than 2^32 threads
bool grid_ok(const Shape& sh) {
    return (int64_t)sh.N * sh.nspan * sh.nblk + sh.C / 8 + 1 < MAX_BLOCKS && (int64_t)sh.N * sh.G < MAX_BLOCKS;
}

template <typename T, int V>
int forward(const T* x, int ldx, T* y, int ldy, const T* res, int ldres, const Shape& sh, const float* gamma, const float* beta,
            float eps, int act, const DropRng& rng, float* stats, float* ws, hipStream_t s) {
    if (!grid_ok(sh)) return CY_ERR_ARG;
    float* part = ws;
    if (!stats) stats = ws + 2 * (int64_t)sh.N * sh.nblk * sh.C;
    const dim3 grid((unsigned)((long)sh.N * sh.nspan * sh.nblk)), fgrid((unsigned)((long)sh.N * sh.G));
    const bool one = sh.Cg % V == 0;
    if (one) hipLaunchKernelGGL((gn_stats_kernel<T, V, 1>), grid, dim3(256), 0, s, x, ldx, sh, part);
    else hipLaunchKernelGGL((gn_stats_kernel<T, V, V>), grid, dim3(256), 0, s, x, ldx, sh, part);
    CY_LAUNCH_CHECK();
    hipLaunchKernelGGL(gn_fold_kernel, fgrid, dim3(256), 0, s, part, sh, one ? sh.Cg / V : sh.Cg, one ? V : 1, eps, stats);
    CY_LAUNCH_CHECK();
#define CY_GNA(A_, D_)                                                                                                         \
    hipLaunchKernelGGL((gn_apply_kernel<T, V, A_, D_>), grid, dim3(256), 0, s, x, ldx, y, ldy, res, ldres, sh, stats, gamma, beta, rng)
#define CY_GNA_ACT(A_)             \
    do {                           \
        if (rng.q) CY_GNA(A_, true); \
        else CY_GNA(A_, false);    \
    } while (0)
    if (act == CY_ACT_MISH) CY_GNA_ACT(CY_ACT_MISH);
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
    const dim3 grid((unsigned)((long)sh.N * sh.nspan * sh.nblk)), fgrid((unsigned)((long)sh.N * sh.G)),
        agrid(grid.x + (ggamma || gbeta ? (sh.C + 7) / 8 : 0));
#define CY_GNB(A_, D_)                                                                                                        \
    do {                                                                                                                      \
        hipLaunchKernelGGL((gn_bwd_sums_kernel<T, V, A_, D_>), grid, dim3(256), 0, s, x, ldx, dy, lddy, sh, stats, gamma, beta, \
                           rng, part);                                                                                   \
        CY_LAUNCH_CHECK();                                                                                                    \
        hipLaunchKernelGGL(gn_bwd_fold_kernel, fgrid, dim3(256), 0, s, part, sh, gamma, chan, s12);                            \
        CY_LAUNCH_CHECK();                                                                                                    \
        hipLaunchKernelGGL((gn_bwd_apply_kernel<T, V, A_, D_>), agrid, dim3(256), 0, s, x, ldx, dy, lddy, dx, lddx, resg, ldrg, \
                           res_accum, sh, stats, gamma, beta, chan, s12, ggamma, gbeta, gscale, accumulate, rng);              \
    } while (0)
#define CY_GNB_ACT(A_)             \
    do {                           \
        if (rng.q) CY_GNB(A_, true); \
        else CY_GNB(A_, false);    \
    } while (0)
    if (act == CY_ACT_MISH) CY_GNB_ACT(CY_ACT_MISH);
    else if (act == CY_ACT_LEAKY) CY_GNB_ACT(CY_ACT_LEAKY);
    else CY_GNB_ACT(CY_ACT_LINEAR);
#undef CY_GNB_ACT
#undef CY_GNB
    CY_LAUNCH_CHECK();
    return 0;
}

// ---- the one-launch kernels: which calls take them ---------------------------------------------------------------------------
// Test / tool switch (cy_gn_config), of the thread that sets it: a call of another thread keeps the kernels that its workspace was sized for
struct Config {
    int mode, polls, width, R;
};
constexpr int POLLS = 1024;      // about a millisecond
constexpr Config DEFAULTS = {1, POLLS, 0, 0};
thread_local Config t_cfg = DEFAULTS;

int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

// Columns of V elements that make about a 128-byte line
int columns(int V) { return V == 1 ? 64 : 8; }

// One shape of blocks: `width` columns, R chunks to a thread.  false: its blocks cannot meet.
bool plan_width(int N, long HW, int C, int G, int V, int width, int R, int polls, ResPlan& p) {
    const int Cg = C / G, gps = width * V / Cg;
    p.R = R;
    p.V = V;
    p.sh = ResShape{HW, N, C, G, Cg, width, C / V / width, gps, GN_TB / width, 0, 0, 0, polls};
    const long nb = (HW + (long)R * p.sh.rows - 1) / ((long)R * p.sh.rows), clusters = (long)N * p.sh.nspan;
    if (nb > 512 || clusters * nb >= MAX_BLOCKS) return false;      // (half of the blocks that fit on the chip)
    p.sh.nb = (int)nb;
    if (nb > 1) {
        if (nb * gps > GN_ONE_STEP) {      // two steps of about the same number of entries
            int sub = 1;
            while ((long)sub * sub < nb) ++sub;
            p.sh.sub = sub;
            p.sh.nsub = (int)((nb + sub - 1) / sub);
        }
        if (clusters > GN_MAX_CLUSTERS || clusters * (nb + p.sh.nsub) * gps > GN_MAX_PAIRS) return false;
    }
    return true;
}

// Blocks that hold all pixels of their columns have nobody to meet: three to four microseconds less, where there are few enough of them
// that a block's own time is what counts (f16, 8 chunks a thread unless said otherwise):
//   1 x 19 x 19 x 1024 forward: 4 columns, alone 6.8 us; 8 columns, two blocks to an image 10.6     64 images: 27.0 against 20.3
//   1 x 26 x 26 x 512: 2 columns 7.1; 8 columns 10.3      16 images: 4 columns, 16 chunks 8.9; 8 columns 12.5; 2 columns 16.6
//   1 x 13 x 13 x 1024 backward: 4 columns, 4 chunks 9.5; 8 columns 12.5      16 images: 8 columns, 8 chunks 11.3; 8 columns, two blocks 14.5
//   16 x 38 x 38 x 256 forward: 2 columns, 16 chunks (256 blocks) 19.5; 8 columns 12.4      4 images: 9.7 and 10.3
// With a compute unit for each: as many blocks as there are compute units for, of four columns and more, or of two (up to 128 blocks).  With
// more blocks than that: of four columns and more (backward, which reads twice as much: eight), the fewest first.
bool plan_alone(int N, long HW, int C, int G, int V, bool bwd, int unit, int polls, ResPlan& p) {
    const int cpr = C / V, most = gn_held(V, bwd), line = columns(V);
    long best = 0;
    for (int w = unit; w <= line && w <= cpr; w += unit) {
        if (w < (V == 1 ? 4 : 2) || cpr % w) continue;
        const long rows = GN_TB / w, blocks = (long)N * (cpr / w);
        const int R = HW <= most / 2 * rows ? most / 2 : most;
        if (HW > R * rows || (R == most && bwd && w < line / 2)) continue;
        if (blocks > (w < line / 2 ? 128 : 256) && w < (bwd ? line : line / 2)) continue;
        // (columns grow, blocks become fewer: the first of at most 256 wins, else the last)
        if (best && best <= 256) continue;
        if (!plan_width(N, HW, C, G, V, w, R, polls, p)) continue;
        best = blocks;
    }
    return best > 0;
}

// Columns of a block: the number nearest to eight (one 128-byte line a pixel) that cuts the row into equal spans of whole groups: narrow
// spans make small clusters, and a narrower one splits cache lines.  16 x 76 x 76 x 256 f16 forward: 4 columns 28.2 us, 8: 22.5, 16: 22.9,
// 32: 23.4; backward 48.0, 37.6, 38.6, 42.7; 16 x 38 x 38 x 512 f16 backward with 64: 28.4, 8: 23.8.
// Chunks of a thread: 16 (backward 8: x and the 32-bit dz), half of that where fewer than 512 blocks would be left for 256 compute units:
// 16 x 38 x 38 x 512 f16 forward (384 blocks at 16) 16.4 us with 16, 14.7 with 8; 16 x 76 x 76 x 256 f16 (768) 22.5 with 16, 27.1 with 8.
// Where half as many make the cluster too large, all of them: 1 x 608 x 608 x 32 f16 forward 4 columns, 16 chunks 23.2 us; three launches 31.3.
// A large image of a small batch, too many blocks at eight columns: not less than half a line unless that is the whole row, and half a line
// only while all blocks fit at a time (1024), else three launches (us: narrow, three launches):
//   1 x 1216 x 1216 x 32 f16 forward  1 column of 4   204  64      1 x 608 x 608 x 64 f16 forward   4 of 8,  722 blocks   35.5  43.4
//   1 x 1024 x 1024 x 32 f16 forward  2 of 4           80  50      1 x 400 x 400 x 64 f16 backward  4 of 8,  626 blocks   31.8  35.3
//   1 x  608 x  608 x 64 f16 backward 2 of 8          112  58      1 x 480 x 480 x 64 f32 backward  4 of 16, 1800 blocks  63.6  56.6
//   1 x  800 x  800 x 64 f32 backward 1 of 16         698 158      1 x 512 x 512 x 128 f16 backward 4 of 16, 2048 blocks  97.7  71.6
// Element by element (rows that do not start on 16 bytes): the same in 64 columns and twice, backward four times, as many elements as there
// would be chunks.  Up to 2048 blocks -- as many as fit at a time, about: 16 x 38 x 38 x 255 f32 forward (720 blocks) 21.6 us, three
// launches 30.8; 16 x 76 x 76 x 255 f16 (2900 blocks) 55 and 38.  Backward with less than half of that line: up to 1024 (1 x 608 x 608 x 30 f32,
// 10 columns, 1389 blocks 71.6 and 52.3; 1 x 304 x 304 x 30 f32, 15 columns, 680 blocks 23.8 and 28.8).
constexpr long AT_A_TIME = 1024;
bool plan_resident(int N, long HW, int C, int G, int V, bool bwd, ResPlan& p, const Config& cfg = t_cfg) {
    if (!cfg.mode || C % V) return false;
    const int Cg = C / G, unit = Cg / gcd(Cg, V);      // columns of the smallest span of whole groups and whole chunks
    const int cpr = C / V, units = cpr / unit, most = gn_held(V, bwd), line = columns(V);
    if (!cfg.width && !cfg.R && plan_alone(N, HW, C, G, V, bwd, unit, cfg.polls, p)) return true;
    int tried = 0;      // (columns already looked at, as a lower bound of the distance from eight)
    for (;;) {
        int width = 0, best = 0;
        for (int i = 1; i <= units && i * unit <= GN_TB; ++i) {
            if (units % i) continue;
            const int w = i * unit, far = w >= line ? 64 * w / line : 64 * line / w;      // 64 times the factor between the two
            const int key = far * 2 + (w < line);
            if (key > tried && (!width || key < best)) {
                width = w;
                best = key;
            }
        }
        if (!width) return false;
        tried = best;
        if (cfg.width && cfg.width % unit == 0 && cpr % cfg.width == 0 && cfg.width <= GN_TB) width = cfg.width;
        const bool part = width < cpr && !cfg.width;      // (of a pixel row)
        if (part && V > 1 && 2 * width < line) continue;
        int R = cfg.R ? cfg.R * most / 16 : most;
        if (!cfg.R) {
            const long ppb = (long)most * (GN_TB / width);
            if ((long)N * (cpr / width) * ((HW + ppb - 1) / ppb) < 512) R = most / 2;
        }
        bool fits = plan_width(N, HW, C, G, V, width, R, cfg.polls, p);
        if (!fits && V > 1 && !cfg.R && R < most) fits = plan_width(N, HW, C, G, V, width, most, cfg.polls, p);
        if (!fits && cfg.width) return false;
        const long blocks = (long)N * p.sh.nspan * p.sh.nb;
        if (!fits || (part && width < line && blocks > AT_A_TIME && (V > 1 || (bwd && 2 * width < line)))) continue;
        return V > 1 || cfg.width || blocks <= 2 * AT_A_TIME;
    }
}

int64_t part_bytes(const ResPlan& p) { return (int64_t)gn_param_slices((long)p.sh.N * p.sh.nb) * ((p.sh.C + 7) / 8) * 16 * 8; }

// bytes behind the part of a workspace that stays zero
int64_t resident_bytes(const ResPlan& p) {
    const int64_t clusters = (int64_t)p.sh.N * p.sh.nspan;
    return 8 * clusters * p.sh.gps + part_bytes(p) + 8 * (int64_t)p.sh.N * p.sh.nb * p.sh.C + 4 * clusters * p.sh.nb;
}

ResWork resident_work(const ResPlan& p, char* ws) {
    const int64_t clusters = (int64_t)p.sh.N * p.sh.nspan;
    ResWork w;
    w.counters = (unsigned*)ws;
    w.pairs = (unsigned long long*)(ws + GN_COUNTER_BYTES);
    w.fin = (unsigned long long*)(ws + GN_ZERO_BYTES);
    w.part = (double*)(w.fin + clusters * p.sh.gps);
    w.chan = (float*)((char*)w.part + part_bytes(p));
    w.list = (unsigned*)(w.chan + 2 * (int64_t)p.sh.N * p.sh.nb * p.sh.C);
    return w;
}

// 16-byte accesses where every row of every operand starts on one
template <typename T>
bool rows16(const void* p, int ld) {
    return !p || (aligned_to(p, 16) && ld % Elem<T>::CH == 0);
}

template <typename T>
int forward_any(const void* x, int ldx, void* y, int ldy, const void* res, int ldres, int N, long HW, int C, int G,
                const float* gamma, const float* beta, float eps, int act, const DropRng& rng, float* stats, char* ws,
                int64_t ws_bytes, hipStream_t s) {
    constexpr int CH = Elem<T>::CH;
    if (!aligned_to(x, sizeof(T)) || !aligned_to(y, sizeof(T)) || !aligned_to(res, sizeof(T))) return CY_ERR_ARG;
    const bool vec = C % CH == 0 && rows16<T>(x, ldx) && rows16<T>(y, ldy) && rows16<T>(res, ldres);
    ResPlan rp;
    if (plan_resident(N, HW, C, G, vec ? CH : 1, false, rp)) {
        if (ws_bytes < GN_ZERO_BYTES + resident_bytes(rp)) return CY_ERR_ARG;
        const auto call = sizeof(T) == 4 ? gn_resident_fwd_f32 : Elem<T>::DT == CY_F16 ? gn_resident_fwd_f16 : gn_resident_fwd_bf16;
        return call(rp, ResFwd{x, ldx, y, ldy, res, ldres, gamma, beta, eps, stats}, resident_work(rp, ws), act, rng, s);
    }
    const Shape sh = make_shape(N, HW, C, G, vec ? CH : 1);
    if (ws_bytes < GN_ZERO_BYTES + 4 * need_floats(sh)) return CY_ERR_ARG;
    float* fws = (float*)(ws + GN_ZERO_BYTES);
    if (vec) return forward<T, CH>((const T*)x, ldx, (T*)y, ldy, (const T*)res, ldres, sh, gamma, beta, eps, act, rng, stats, fws, s);
    return forward<T, 1>((const T*)x, ldx, (T*)y, ldy, (const T*)res, ldres, sh, gamma, beta, eps, act, rng, stats, fws, s);
}

template <typename T>
int backward_any(const void* x, int ldx, const void* dy, int lddy, void* dx, int lddx, void* resg, int ldrg, int res_accum, int N,
                 long HW, int C, int G, const float* gamma, const float* beta, const float* stats, int act, const DropRng& rng,
                 float* ggamma, float* gbeta, float gscale, int accumulate, char* ws, int64_t ws_bytes, hipStream_t s) {
    constexpr int CH = Elem<T>::CH;
    if (!aligned_to(x, sizeof(T)) || !aligned_to(dy, sizeof(T)) || !aligned_to(dx, sizeof(T)) || !aligned_to(resg, sizeof(T)))
        return CY_ERR_ARG;
    const bool vec = C % CH == 0 && rows16<T>(x, ldx) && rows16<T>(dy, lddy) && rows16<T>(dx, lddx) && rows16<T>(resg, ldrg);
    ResPlan rp;
    if (plan_resident(N, HW, C, G, vec ? CH : 1, true, rp)) {
        if (ws_bytes < GN_ZERO_BYTES + resident_bytes(rp)) return CY_ERR_ARG;
        const auto call = sizeof(T) == 4 ? gn_resident_bwd_f32 : Elem<T>::DT == CY_F16 ? gn_resident_bwd_f16 : gn_resident_bwd_bf16;
        return call(rp, ResBwd{x, ldx, dy, lddy, dx, lddx, resg, ldrg, res_accum, gamma, beta, stats, ggamma, gbeta, gscale, accumulate},
                    resident_work(rp, ws), act, rng, s);
    }
    const Shape sh = make_shape(N, HW, C, G, vec ? CH : 1);
    if (ws_bytes < GN_ZERO_BYTES + 4 * need_floats(sh)) return CY_ERR_ARG;
    float* fws = (float*)(ws + GN_ZERO_BYTES);
    if (vec)
        return backward<T, CH>((const T*)x, ldx, (const T*)dy, lddy, (T*)dx, lddx, (T*)resg, ldrg, res_accum, sh, gamma, beta, stats,
                               act, rng, ggamma, gbeta, gscale, accumulate, fws, s);
    return backward<T, 1>((const T*)x, ldx, (const T*)dy, lddy, (T*)dx, lddx, (T*)resg, ldrg, res_accum, sh, gamma, beta, stats, act,
                          rng, ggamma, gbeta, gscale, accumulate, fws, s);
}

}  // namespace

extern "C" int64_t cy_gn_workspace(int N, int64_t HW, int C, int groups, int dtype) {
    if (!sizes_ok(N, HW, C, groups, dtype)) return CY_ERR_ARG;
    if (N == 0 || HW == 0) return GN_ZERO_BYTES;
    const int ch = dtype == CY_F32 ? 4 : 8;
    int64_t most = 0;      // (whichever kernels a call's pointers allow)
    for (int V : {1, ch}) {
        if (C % V) continue;
        const int64_t v = 4 * need_floats(make_shape(N, (long)HW, C, groups, V));
        if (v > most) most = v;
        for (int bwd = 0; bwd < 2; ++bwd)
            for (const Config& cfg : {t_cfg, DEFAULTS}) {      // (a backward pass runs in a thread of its own)
                ResPlan p;
                if (plan_resident(N, (long)HW, C, groups, V, bwd != 0, p, cfg) && resident_bytes(p) > most) most = resident_bytes(p);
            }
    }
    return GN_ZERO_BYTES + most;
}

extern "C" int cy_gn_config(int mode, int polls, int width, int chunks) {
    if (mode < 0 || mode > 1 || polls < -1 || width < 0 || (chunks != 0 && chunks != 8 && chunks != 16)) return CY_ERR_ARG;
    t_cfg = Config{mode, polls < 0 ? POLLS : polls, width, chunks};
    return 0;
}

extern "C" int cy_gn_plan(int N, int64_t HW, int C, int groups, int dtype, int backward, int rows16, int* plan) {
    const int V = !rows16 ? 1 : dtype == CY_F32 ? 4 : 8;
    if (!sizes_ok(N, HW, C, groups, dtype) || N == 0 || HW == 0 || C % V || !plan) return CY_ERR_ARG;
    ResPlan p;
    if (plan_resident(N, (long)HW, C, groups, V, backward != 0, p)) {
        const int out[6] = {1, p.sh.width, p.R, p.sh.nspan, p.sh.nb, p.sh.nsub};
        for (int i = 0; i < 6; ++i) plan[i] = out[i];
    } else {
        const Shape sh = make_shape(N, (long)HW, C, groups, V);
        const int out[6] = {3, sh.width, 0, sh.nspan, sh.nblk, 0};
        for (int i = 0; i < 6; ++i) plan[i] = out[i];
    }
    return 0;
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
    return forward_any<T>(x, ldx, y, ldy, res, ldres, N, (long)HW, C, groups, gamma, beta, eps, act, r, stats, (char*)ws, ws_bytes, cy_s(s))
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
                           ggamma, gbeta, gscale, accumulate, (char*)ws, ws_bytes, cy_s(s))
    if (dtype == CY_F16) CY_GNBW(f16);
    if (dtype == CY_BF16) CY_GNBW(bf16);
    CY_GNBW(float);
#undef CY_GNBW
}
