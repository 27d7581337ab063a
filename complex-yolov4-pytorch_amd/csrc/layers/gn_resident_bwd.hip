// Backward group norm in one pass over x and dy (plus the fold of the parameter gradients).  See gn_resident.hpp for how the blocks of
// an image meet.
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

// R: 16-byte chunks of x and of dy a thread holds.  ONE: a chunk lies in one group.  x stays as stored; dz = drop(dy) act'(z) is formed once and kept in 32 bits -- the
// activation's derivative is most of this kernel's arithmetic (an exponential and a reciprocal per element), and rounding dz to the
// storage type would put its error into the sums.
template <typename T, bool ONE, int ACT, bool DROP, int R>
__global__ void __launch_bounds__(GN_TB) gn_bwd_resident_kernel(ResBwd a, ResShape sh, ResWork wk, DropRng rng) {
    constexpr int V = Elem<T>::CH;
    constexpr bool FAST = sizeof(T) == 2;
    __shared__ __attribute__((aligned(16))) float s_red[2 * GN_TB * V];
    __shared__ float2 s_pair[ONE ? GN_TB : GN_TB * V], s_stat[ONE ? GN_TB : GN_TB * V];
    SumAcc::Sum* s_acc = reinterpret_cast<SumAcc::Sum*>(s_red);      // (after the block's own sums)
    static_assert(sizeof(SumAcc::Sum) * GN_TB <= sizeof(s_red), "accumulators fit where the sums were");
    const ResWhere w = res_where<R>(sh);
    const long img = (long)w.n * sh.HW, pmax = sh.HW - 1;
    u32x4 d[R];
    float dz[R][V];
    Norm<T, ACT> nm[V];
    float sa[V], sb[V];
    int cnt = (w.px - w.row + sh.rows - 1) / sh.rows;
    cnt = !w.on || cnt < 0 ? 0 : cnt;
    DropKey key;
    if constexpr (DROP) key = drop_key(rng);
    const int cc = w.chunk * V;
    for (int g = threadIdx.x; g < sh.gps; g += GN_TB)
        s_stat[g] = *reinterpret_cast<const float2*>(a.stats + 2 * ((long)w.n * sh.G + w.span * sh.gps + g));
#pragma unroll
    for (int i = 0; i < V; ++i) sa[i] = sb[i] = 0.f;
    if (w.on) {
        u32x4 g[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {      // (beyond the image: its last pixel, left out below)
            long p = w.p0 + w.row + r * sh.rows;
            p = img + (p < pmax ? p : pmax);
            d[r] = *reinterpret_cast<const u32x4*>((const T*)a.x + p * a.ldx + cc);
            g[r] = *reinterpret_cast<const u32x4*>((const T*)a.dy + p * a.lddy + cc);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float2 st = *reinterpret_cast<const float2*>(a.stats + 2 * ((long)w.n * sh.G + (cc + (ONE ? 0 : i)) / sh.Cg));
            nm[i].set(st, a.gamma[cc + i], a.beta[cc + i]);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (r < cnt) {
                const long p = img + w.p0 + w.row + r * sh.rows;
                float f[V], t[V];
                chunk_to_f32<T>(d[r], f);
                chunk_to_f32<T>(g[r], t);
                if (a.resg) {      // the shortcut branch's gradient is dy itself
                    T* rg = (T*)a.resg + p * a.ldrg + cc;
                    if (a.res_accum) {
                        float o[V];
                        load_v<T, V>(rg, o);
#pragma unroll
                        for (int i = 0; i < V; ++i) o[i] += t[i];
                        store_v<T, V>(rg, o);
                    } else {
                        *reinterpret_cast<u32x4*>(rg) = g[r];
                    }
                }
                if constexpr (DROP) drop_apply<V>(key, rng.q, rng.scale, (unsigned long long)p * sh.C + cc, t);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float v = t[i] * gn_act_grad<ACT, FAST>(nm[i].z(f[i]));
                    dz[r][i] = v;
                    sa[i] += v;
                    sb[i] += v * (f[i] - nm[i].mean);      // (times r when the rows are folded)
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
        s_red[(threadIdx.x * V + i) * 2] = sa[i];
        s_red[(threadIdx.x * V + i) * 2 + 1] = sb[i];
    }
    __syncthreads();
    // channels: a thread folds one channel's rows (neighbouring threads read neighbouring words), the sums go to the workspace for the
    // parameter gradients and, weighted with gamma, back into the first row
    const int nch = sh.width * V;
    float* chan = wk.chan + 2 * (((long)w.n * sh.nb + w.blk) * sh.C + (long)w.span * nch);
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
        const float gm = a.gamma[w.span * nch + c];
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
    if (ok && cnt > 0) {
        float2 k[V];
#pragma unroll
        for (int i = 0; i < V; ++i) k[i] = s_pair[(cc - w.span * nch + (ONE ? 0 : i)) / sh.Cg];
        T* dx = (T*)a.dx + (img + w.p0 + w.row) * a.lddx + cc;
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (r < cnt) {
                float f[V];
                chunk_to_f32<T>(d[r], f);
#pragma unroll
                for (int i = 0; i < V; ++i) f[i] = gn_dx(nm[i], k[i], f[i], dz[r][i]);
                store_v<T, V>(dx + (long)r * sh.rows * a.lddx, f);
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
                f[i] = gn_dx(one, agent_load_pair(fin + g), f[i], t[i] * gn_act_grad<ACT, FAST>(one.z(f[i])));
            }
            store_v<T, V>((T*)a.dx + pix * a.lddx + c, f);
        }
    });
}

// ggamma / gbeta from the blocks' channel sums chan[row][C][2]: eight channels by 128 row lanes, each lane's rows in order, then the
// lanes in order; double.
__global__ void __launch_bounds__(1024) gn_param_grad_kernel(const float* chan, long rows, int C, float* ggamma, float* gbeta,
                                                            float gscale, int accumulate) {
    __shared__ double s_a[128][9], s_b[128][9];
    const int c = blockIdx.x * 8 + (threadIdx.x & 7), l = threadIdx.x >> 3;
    double a = 0.0, b = 0.0;
    if (c < C) {
        const float2* src = reinterpret_cast<const float2*>(chan) + c;
#pragma unroll 8
        for (long r = l; r < rows; r += 128) {
            const float2 v = src[r * C];
            a += (double)v.x;
            b += (double)v.y;
        }
    }
    s_a[l][threadIdx.x & 7] = a;
    s_b[l][threadIdx.x & 7] = b;
    __syncthreads();
    for (int h = 64; h > 0; h >>= 1) {
        if (l < h) {
            s_a[l][threadIdx.x & 7] += s_a[l + h][threadIdx.x & 7];
            s_b[l][threadIdx.x & 7] += s_b[l + h][threadIdx.x & 7];
        }
        __syncthreads();
    }
    if (l == 0 && c < C) {
        if (gbeta) gbeta[c] = (accumulate ? gbeta[c] : 0.f) + gscale * (float)s_a[0][threadIdx.x];
        if (ggamma) ggamma[c] = (accumulate ? ggamma[c] : 0.f) + gscale * (float)s_b[0][threadIdx.x];
    }
}

template <typename T, bool ONE, int ACT>
int launch(const ResPlan& p, const ResBwd& a, const ResWork& wk, const DropRng& rng, hipStream_t s) {
    const dim3 grid((unsigned)((long)p.sh.N * p.sh.nspan * p.sh.nb));
#define CY_R(D_, R_) hipLaunchKernelGGL((gn_bwd_resident_kernel<T, ONE, ACT, D_, R_>), grid, dim3(GN_TB), 0, s, a, p.sh, wk, rng)
    if (rng.q && p.R == 4) CY_R(true, 4);
    else if (rng.q) CY_R(true, 8);
    else if (p.R == 4) CY_R(false, 4);
    else CY_R(false, 8);
#undef CY_R
    CY_LAUNCH_CHECK();
    if (a.ggamma || a.gbeta) {
        hipLaunchKernelGGL(gn_param_grad_kernel, dim3((p.sh.C + 7) / 8), dim3(1024), 0, s, wk.chan, (long)p.sh.N * p.sh.nb, p.sh.C, a.ggamma,
                           a.gbeta, a.gscale, a.accumulate);
        CY_LAUNCH_CHECK();
    }
    return 0;
}

template <typename T>
int launch_any(const ResPlan& p, const ResBwd& a, const ResWork& wk, int act, const DropRng& rng, hipStream_t s) {
    if (p.sh.Cg % Elem<T>::CH == 0) {
        if (act == CY_ACT_MISH) return launch<T, true, CY_ACT_MISH>(p, a, wk, rng, s);
        if (act == CY_ACT_LEAKY) return launch<T, true, CY_ACT_LEAKY>(p, a, wk, rng, s);
        return launch<T, true, CY_ACT_LINEAR>(p, a, wk, rng, s);
    }
    if (act == CY_ACT_MISH) return launch<T, false, CY_ACT_MISH>(p, a, wk, rng, s);
    if (act == CY_ACT_LEAKY) return launch<T, false, CY_ACT_LEAKY>(p, a, wk, rng, s);
    return launch<T, false, CY_ACT_LINEAR>(p, a, wk, rng, s);
}

}  // namespace

int gn_resident_bwd(const ResPlan& p, const ResBwd& a, const ResWork& wk, int act, int dtype, const DropRng& rng, hipStream_t s) {
    if (dtype == CY_F16) return launch_any<f16>(p, a, wk, act, rng, s);
    if (dtype == CY_BF16) return launch_any<bf16>(p, a, wk, act, rng, s);
    return launch_any<float>(p, a, wk, act, rng, s);
}
