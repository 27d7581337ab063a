// Backward group norm in one pass over x and dy (plus the fold of the parameter gradients).  See gn_resident.hpp for how the blocks of
// an image meet.  (A source per element type includes this: they are built side by side.)
#pragma once
#include "gn_math.hpp"
#include "gn_resident.hpp"

namespace {

struct SumAcc {
    struct Shape {};
    struct Sum {
        double u, v;
    };
    Sum s;
    __device__ SumAcc(const Shape&, int, int) : s{0.0, 0.0} {}
    __device__ __forceinline__ void add(int, float2 t) {
        s.u += (double)t.x;
        s.v += (double)t.y;
    }
    __device__ __forceinline__ Sum sum() const { return s; }
    static __device__ __forceinline__ void merge(Sum& a, const Sum& b) {
        a.u += b.u;
        a.v += b.v;
    }
    static __device__ __forceinline__ float2 out(const Sum& s) { return make_float2((float)s.u, (float)s.v); }
};

// R: chunks of V elements of x and of dy a thread holds.  ONE: a chunk lies in one group.  x stays as stored; dz = drop(dy) act'(z) is formed
// once and kept in 32 bits in dy's place -- the derivative is most of this kernel's arithmetic (an exponential and a reciprocal per
// element), and rounding dz to the storage type would put its error into the sums.  Forming dz again after the meeting instead, with dy
// as stored in the registers, leaves room for four waves a SIMD in place of three and is slower all the same, since blocks of one image
// compute at the same time: by 12 % on 16 x 304 x 304 x 64 f16, by 27 % on 16 x 76 x 76 x 256 bf16 with dropout.  14 chunks a thread and
// two waves: 4 % faster on the former, 9 % slower on the latter.
// Bound: memory while blocks load and store, the arithmetic and the meeting in between; 16 x 304 x 304 x 64 f16, mish: 171 us for 568 MB.
// With the shortcut's gradient added 60 us where it takes 39 without (16 x 76 x 76 x 256 bf16; 237 and 142 MB): its loads and stores follow one
// another in front of the sums.
template <typename T, int V, bool ONE, int ACT, bool DROP, int R>
__global__ void __launch_bounds__(GN_TB) gn_bwd_resident_kernel(ResBwd a, ResShape sh, ResWork wk, DropRng rng) {
    constexpr int H = V < 4 ? V : 4;      // channels at a time
    constexpr bool FAST = sizeof(T) == 2;
    __shared__ __attribute__((aligned(16))) float s_red[V > 1 ? 2 * GN_TB * V : 4 * GN_TB];
    extern __shared__ __attribute__((aligned(16))) float2 s_dyn[];
    float2 *s_pair = s_dyn, *s_stat = s_dyn + sh.gps, *s_gb = s_stat + sh.gps;
    SumAcc::Sum* s_acc = reinterpret_cast<SumAcc::Sum*>(s_red);      // (after the block's own sums)
    static_assert(sizeof(SumAcc::Sum) * GN_TB <= sizeof(s_red), "accumulators fit where the sums were");
    const ResWhere w = res_where<R>(sh);
    const long img = (long)w.n * sh.HW, pmax = sh.HW - 1;
    Raw<T, V> d[R], g[R];
    float dz[R][V];
    int cnt = (w.px - w.row + sh.rows - 1) / sh.rows;
    cnt = !w.on || cnt < 0 ? 0 : cnt;
    DropKey key;
    if constexpr (DROP) key = drop_key(rng);
    const int nch = sh.width * V, c0 = w.span * nch, cc = w.chunk * V, lc0 = cc - c0;
    {      // statistics, gamma and beta go to LDS.  They are asked for first: loads answer in order
        const float2* st = reinterpret_cast<const float2*>(a.stats) + (long)w.n * sh.G + w.span * sh.gps;
        const int t = threadIdx.x, ct = t < nch ? t : nch - 1, gt = t < sh.gps ? t : sh.gps - 1;
        const float2 gb = make_float2(a.gamma[c0 + ct], a.beta[c0 + ct]), s0 = st[gt];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int r = 0; r < R; ++r) {      // (beyond the image: its last pixel, dy cleared below)
            long p = w.p0 + w.row + r * sh.rows;
            p = img + (p < pmax ? p : pmax);
            d[r].load((const T*)a.x + p * a.ldx + cc);
            g[r].load((const T*)a.dy + p * a.lddy + cc);
        }
        // (nor is there a branch around the arithmetic: the loads would be moved into it, one behind the other, for 4 % more)
        __builtin_amdgcn_sched_barrier(0);
        s_gb[ct] = gb;
        s_stat[gt] = s0;
        for (int c = t + GN_TB; c < nch; c += GN_TB) s_gb[c] = make_float2(a.gamma[c0 + c], a.beta[c0 + c]);
        for (int i = t + GN_TB; i < sh.gps; i += GN_TB) s_stat[i] = st[i];
    }
    __syncthreads();
    if (a.resg) {      // the shortcut branch's gradient is dy itself
        T* rg = (T*)a.resg + (img + w.p0 + w.row) * a.ldrg + cc;
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (r < cnt) {
                T* at = rg + (long)r * sh.rows * a.ldrg;
                if (a.res_accum) {
                    float t[V], f[V];
                    g[r].get(t);
                    load_v<T, V>(at, f);
#pragma unroll
                    for (int i = 0; i < V; ++i) f[i] += t[i];
                    store_v<T, V>(at, f);
                } else {
                    g[r].store(at);
                }
            }
    }
    asm volatile("" : "+v"(cnt));      // (this and the ones below: what can be had again is not kept in registers)
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (r >= cnt) g[r].clear();
        if constexpr (DROP) drop_raw(key, rng.q, (unsigned long long)(img + w.p0 + w.row + r * sh.rows) * sh.C + cc, g[r]);
        g[r].pin();
    }
    // Four channels at a time: their constants are fetched from LDS, their four elements of a pixel hide each other's latency.
    auto grad = [&](float dy, float z) { return rounded((DROP ? dy * rng.scale : dy) * gn_act_grad<ACT, FAST>(z)); };
#pragma unroll
    for (int h = 0; h < V; h += H) {
        Norm<T, ACT> nm[H];
        float sa[H], sb[H];
#pragma unroll
        for (int i = 0; i < H; ++i) {
            const int c = lc0 + h + i;
            nm[i].set(s_stat[(ONE ? lc0 : c) / sh.Cg], s_gb[c].x, s_gb[c].y);
            sa[i] = sb[i] = 0.f;
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float f[H], t[H];
            d[r].template part<H>(h, f);
            g[r].template part<H>(h, t);
#pragma unroll
            for (int i = 0; i < H; ++i) {
                const float v = grad(t[i], nm[i].z(f[i]));
                dz[r][h + i] = v;
                sa[i] += v;
                sb[i] += v * (f[i] - nm[i].mean);      // (times r when the rows are folded)
            }
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < H; ++i) *reinterpret_cast<float2*>(s_red + (threadIdx.x * V + h + i) * 2) = make_float2(sa[i], sb[i]);
    }
    asm volatile("" : "+v"(cnt));
#pragma unroll
    for (int r = 0; r < R; ++r) d[r].pin();
    __syncthreads();
    // channels: a thread folds one channel's rows (neighbouring threads read neighbouring words), the sums go to the workspace for the
    // parameter gradients and, weighted with gamma, back into the first row
    float* chan = wk.chan + 2 * (((long)w.n * sh.nb + w.blk) * sh.C + c0);
    for (int c = threadIdx.x; c < nch; c += GN_TB) {
        float u = 0.f, v = 0.f;
#pragma unroll 8
        for (int r = 0; r < sh.rows; ++r) {
            const float2 t = *reinterpret_cast<const float2*>(s_red + 2 * (r * nch + c));
            u += t.x;
            v += t.y;
        }
        v *= s_stat[c / sh.Cg].y;
        *reinterpret_cast<float2*>(chan + 2 * c) = make_float2(u, v);
        const float gm = s_gb[c].x;
        *reinterpret_cast<float2*>(s_red + 2 * c) = make_float2(u * gm, v * gm);
    }
    __syncthreads();
    const double all = (double)sh.HW * sh.Cg;
    {
        const int L = lanes_for(sh.gps), l = threadIdx.x & (L - 1);
        for (int g = threadIdx.x / L; g < sh.gps; g += GN_TB / L) {
            float u = 0.f, v = 0.f;
            for (int c = l; c < sh.Cg; c += L) {
                const float2 t = *reinterpret_cast<const float2*>(s_red + 2 * (g * sh.Cg + c));
                u += t.x;
                v += t.y;
            }
            u = lanes_sum(u, L);
            v = lanes_sum(v, L);
            if (l == 0) s_pair[g] = sh.nb == 1 ? gn_k01(s_stat[g].y, (double)u / all, (double)v / all) : make_float2(u, v);
        }
    }
    __syncthreads();
    auto result = [&](int g, float2 v) { return gn_k01(s_stat[g].y, (double)v.x / all, (double)v.y / all); };
    auto keep = [](int, float2) {};
    bool ok = true;
    unsigned out = 0;
    if (sh.nb > 1) ok = cluster_meet<SumAcc>(sh, wk, w, SumAcc::Shape{}, s_pair, s_acc, &out, result, keep);
    if (ok) {
#pragma unroll
        for (int h = 0; h < V; h += H) {      // (dx takes x's place)
            Norm<T, ACT> nm[H];
            float2 k[H];
#pragma unroll
            for (int i = 0; i < H; ++i) {
                const int c = lc0 + h + i, j = (ONE ? lc0 : c) / sh.Cg;
                nm[i].set(s_stat[j], s_gb[c].x, s_gb[c].y);
                k[i] = s_pair[j];
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float f[H];
                d[r].template part<H>(h, f);
#pragma unroll
                for (int i = 0; i < H; ++i) f[i] = gn_dx(nm[i], k[i], f[i], dz[r][h + i]);
                d[r].template set_part<H>(h, f);
                __builtin_amdgcn_sched_barrier(0);
                if (h == V - H && r < cnt) d[r].store((T*)a.dx + (img + w.p0 + w.row + (long)r * sh.rows) * a.lddx + cc);
            }
        }
    }
    if (sh.nb == 1) return;
    cluster_leave<SumAcc>(sh, wk, w, SumAcc::Shape{}, s_acc, out, result, keep, [&](int blk, const unsigned long long* fin) {
        const long p0 = (long)blk * R * sh.rows, left = sh.HW - p0, px = left < (long)R * sh.rows ? left : (long)R * sh.rows;
        for (long e = threadIdx.x; e < px * sh.width; e += 64) {
            const long p = e / sh.width, pix = img + p0 + p;
            const int lc = (int)(e - p * sh.width), c = (w.span * sh.width + lc) * V;
            float f[V], t[V];
            load_v<T, V>((const T*)a.x + pix * a.ldx + c, f);
            load_v<T, V>((const T*)a.dy + pix * a.lddy + c, t);
            if constexpr (DROP) drop_apply<V>(key, rng.q, rng.scale, (unsigned long long)pix * sh.C + c, t);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int g = (lc * V + i) / sh.Cg;
                const float2 st = s_stat[g];
                Norm<T, ACT> one;
                one.set(st, a.gamma[c + i], a.beta[c + i]);
                f[i] = gn_dx(one, agent_load_pair(fin + g), f[i], rounded(t[i] * gn_act_grad<ACT, FAST>(one.z(f[i]))));
            }
            store_v<T, V>((T*)a.dx + pix * a.lddx + c, f);
        }
    });
}

// ggamma / gbeta from the blocks' channel sums chan[row][C][2], in double: eight channels by up to 128 row lanes, each lane's rows in
// order, then the lanes in order.  Many rows are cut into gridDim.y slices: the last of them to come adds the slices' sums in order (through
// the cache behind the XCDs, like the meetings; the counter is zero again afterwards).  5776 rows of 64 channels: 18 us in one slice, 6.6 in sixteen.
__global__ void __launch_bounds__(1024) gn_param_grad_kernel(const float* chan, long rows, int C, float* ggamma, float* gbeta,
                                                            float gscale, int accumulate, unsigned* counters, double* part) {
    __shared__ double s_a[128][9], s_b[128][9];
    __shared__ bool s_last;
    const int k = threadIdx.x & 7, c = blockIdx.x * 8 + k, l = threadIdx.x >> 3, lanes = blockDim.x >> 3, slices = gridDim.y;
    const long per = (rows + slices - 1) / slices, r1 = (blockIdx.y + 1) * per;
    double a = 0.0, b = 0.0;
    if (c < C) {
        const float2* src = reinterpret_cast<const float2*>(chan) + c;
#pragma unroll 8
        for (long r = blockIdx.y * per + l; r < (r1 < rows ? r1 : rows); r += lanes) {
            const float2 v = src[r * C];
            a += (double)v.x;
            b += (double)v.y;
        }
    }
    s_a[l][k] = a;
    s_b[l][k] = b;
    __syncthreads();
    for (int h = lanes >> 1; h > 0; h >>= 1) {
        if (l < h) {
            s_a[l][k] += s_a[l + h][k];
            s_b[l][k] += s_b[l + h][k];
        }
        __syncthreads();
    }
    if (slices > 1) {
        unsigned long long* mine = reinterpret_cast<unsigned long long*>(part) + (long)blockIdx.x * slices * 16;
        if (threadIdx.x < 16)
            __hip_atomic_store(mine + blockIdx.y * 16 + threadIdx.x, __double_as_longlong(l ? s_b[0][k] : s_a[0][k]), __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
        stores_done();
        __syncthreads();
        if (threadIdx.x == 0) {
            unsigned* cnt = counters + (long)GN_WORDS * blockIdx.x;
            s_last = agent_add(cnt, 1u) == (unsigned)slices - 1;
            if (s_last) agent_store(cnt, 0u);
        }
        __syncthreads();
        if (!s_last) return;
        for (int t = threadIdx.x; t < slices * 16; t += blockDim.x)      // (all at once: sixteen round trips would cost what the slices save)
            (l & 1 ? s_b : s_a)[t >> 4][k] = __longlong_as_double(__hip_atomic_load(mine + t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
        __syncthreads();
        if (l == 0)
            for (int i = 1; i < slices; ++i) {
                s_a[0][k] += s_a[i][k];
                s_b[0][k] += s_b[i][k];
            }
    }
    if (l == 0 && c < C) {
        if (gbeta) gbeta[c] = (accumulate ? gbeta[c] : 0.f) + gscale * (float)s_a[0][k];
        if (ggamma) ggamma[c] = (accumulate ? ggamma[c] : 0.f) + gscale * (float)s_b[0][k];
    }
}

template <typename T, int V, bool ONE, int ACT>
int launch(const ResPlan& p, const ResBwd& a, const ResWork& wk, const DropRng& rng, hipStream_t s) {
    constexpr int R = GN_HELD_BWD<V>;
    const dim3 grid((unsigned)((long)p.sh.N * p.sh.nspan * p.sh.nb));
    const size_t lds = sizeof(float2) * (2 * p.sh.gps + p.sh.width * V);
#define CY_R(D_, R_) hipLaunchKernelGGL((gn_bwd_resident_kernel<T, V, ONE, ACT, D_, R_>), grid, dim3(GN_TB), lds, s, a, p.sh, wk, rng)
    if (rng.q && p.R < R) CY_R(true, R / 2);
    else if (rng.q) CY_R(true, R);
    else if (p.R < R) CY_R(false, R / 2);
    else CY_R(false, R);
#undef CY_R
    CY_LAUNCH_CHECK();
    if (a.ggamma || a.gbeta) {
        const long rows = (long)p.sh.N * p.sh.nb;
        int lanes = 8;
        while (lanes < 128 && lanes < rows) lanes *= 2;
        const int blocks = (p.sh.C + 7) / 8, slices = blocks > GN_MAX_CLUSTERS ? 1 : gn_param_slices(rows);
        hipLaunchKernelGGL(gn_param_grad_kernel, dim3(blocks, slices), dim3(8 * lanes), 0, s, wk.chan, rows, p.sh.C, a.ggamma, a.gbeta, a.gscale,
                           a.accumulate, wk.counters, wk.part);
        CY_LAUNCH_CHECK();
    }
    return 0;
}

template <typename T, int V, bool ONE>
int launch_act(const ResPlan& p, const ResBwd& a, const ResWork& wk, int act, const DropRng& rng, hipStream_t s) {
    if (act == CY_ACT_MISH) return launch<T, V, ONE, CY_ACT_MISH>(p, a, wk, rng, s);
    if (act == CY_ACT_LEAKY) return launch<T, V, ONE, CY_ACT_LEAKY>(p, a, wk, rng, s);
    return launch<T, V, ONE, CY_ACT_LINEAR>(p, a, wk, rng, s);
}

template <typename T>
int launch_any(const ResPlan& p, const ResBwd& a, const ResWork& wk, int act, const DropRng& rng, hipStream_t s) {
    constexpr int CH = Elem<T>::CH;
    if (p.V == 1) return launch_act<T, 1, true>(p, a, wk, act, rng, s);
    if (p.sh.Cg % CH == 0) return launch_act<T, CH, true>(p, a, wk, act, rng, s);
    return launch_act<T, CH, false>(p, a, wk, act, rng, s);
}

}  // namespace
