// Forward group norm in one launch: x is read once.  See gn_resident.hpp for how the blocks of an image meet.  (A source per
// element type includes this: they are built side by side.)
#pragma once
#include "gn_math.hpp"
#include "gn_resident.hpp"

namespace {

template <typename T, int V, int ACT>
__device__ __forceinline__ void finish(float* f, const Norm<T, ACT>* nm) {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = gn_act<ACT, sizeof(T) == 2>(nm[i].z(f[i]));
}

// (mean, centred sum of squares) of one group over entries of `per` blocks each, from block `first` on: a lane sums deviations of the
// means from its first entry's, weighted with the entries' pixels; lanes are merged by mean and sum of squares.
struct StatAcc {
    struct Shape {
        long HW, ppb;
        int Cg;
    };
    struct Sum {
        double n, mean, m2;
    };
    long left, unit;
    int Cg;
    double n, m0, s1, s2, m2;
    __device__ StatAcc(const Shape& s, int first, int per) : left(s.HW - first * s.ppb), unit(per * s.ppb), Cg(s.Cg), n(0.0), m0(0.0), s1(0.0), s2(0.0), m2(0.0) {}
    __device__ __forceinline__ void add(int i, float2 v) {
        const long rest = left - i * unit;
        const double wt = (double)(rest < unit ? rest : unit) * Cg;
        if (n == 0.0) m0 = (double)v.x;
        const double d = (double)v.x - m0;
        n += wt;
        s1 += wt * d;
        s2 += wt * d * d;
        m2 += (double)v.y;
    }
    __device__ __forceinline__ Sum sum() const {
        if (n == 0.0) return Sum{0.0, 0.0, 0.0};
        const double d = s1 / n, q = s2 - s1 * d;
        return Sum{n, m0 + d, m2 + (q > 0.0 ? q : 0.0)};
    }
    static __device__ __forceinline__ void merge(Sum& a, const Sum& b) {
        const double nt = a.n + b.n;
        if (b.n == 0.0) return;
        const double d = b.mean - a.mean, f = b.n / nt;
        a.mean += d * f;
        a.m2 += b.m2 + d * d * a.n * f;
        a.n = nt;
    }
    static __device__ __forceinline__ float2 out(const Sum& s) { return make_float2((float)s.mean, (float)s.m2); }
};

// R: chunks of V elements of x a thread holds.  A: sums a thread keeps (gn_sums).
// Bound: memory while blocks load and store (4 waves a SIMD hold 64 MB of x on the chip); a block's life on an idle chip is 7 us of loads,
// 1.5 of sums, 4 to 6 of meeting, 4 of activation and stores.  16 x 152 x 152 x 128 f16 leaky 40 us for 189 MB; 16 x 608 x 608 x 32 f16 mish
// 178 us for 757 MB (361 blocks an image: three images at a time).  48 chunks a thread, two waves: 57 and 220 where 16 took 53 and 209.
template <typename T, int V, int A, int ACT, bool DROP, int R>
__global__ void __launch_bounds__(GN_TB) gn_fwd_resident_kernel(ResFwd a, ResShape sh, ResWork wk, DropRng rng) {
    constexpr int PER = V / A;      // PER: channels of a chunk that share a sum
    constexpr size_t SUMS = sizeof(float) * 2 * GN_TB * A, ACCS = sizeof(StatAcc::Sum) * GN_TB;
    __shared__ __attribute__((aligned(16))) char s_buf[SUMS > ACCS ? SUMS : ACCS];
    __shared__ float s_n[GN_TB];
    extern __shared__ __attribute__((aligned(16))) float2 s_dyn[];
    float2 *s_pair = s_dyn, *s_gb = s_dyn + sh.gps;
    float *s_m = reinterpret_cast<float*>(s_buf), *s_q = s_m + GN_TB * A;
    StatAcc::Sum* s_acc = reinterpret_cast<StatAcc::Sum*>(s_buf);      // (after the block's own sums)
    const ResWhere w = res_where<R>(sh);
    const T* x = (const T*)a.x + (long)w.n * sh.HW * a.ldx;
    const long pmax = sh.HW - 1;
    Raw<T, V> d[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {      // (pixels beyond the image are read as its last one and left out below: no branch between the loads)
        long p = w.p0 + w.row + r * sh.rows;
        p = p < pmax ? p : pmax;
        d[r].load(x + p * a.ldx + w.chunk * V);
    }
    int cnt = (w.px - w.row + sh.rows - 1) / sh.rows;      // pixels of this thread
    cnt = !w.on || cnt < 0 ? 0 : cnt;
    // gamma and beta wait in LDS (in registers they would cost a wave of occupancy, fetched after the meeting a round trip)
    for (int c = threadIdx.x; c < sh.width * V; c += GN_TB)
        s_gb[c] = make_float2(a.gamma[w.span * sh.width * V + c], a.beta[w.span * sh.width * V + c]);
    // deviations from the thread's first value, as in gn_stats_kernel
    float K[A], s[A], q[A];
    {
        float f[V];
        d[0].get(f);
#pragma unroll
        for (int j = 0; j < A; ++j) {
            K[j] = cnt > 0 ? f[j * PER] : 0.f;
            s[j] = q[j] = 0.f;
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (r < cnt) {
            float f[V];
            d[r].get(f);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float t = f[i] - K[i / PER];
                s[i / PER] += t;
                q[i / PER] += t * t;
            }
        }
    const float n = (float)(cnt * PER), inv = n > 0.f ? 1.f / n : 0.f;
#pragma unroll
    for (int j = 0; j < A; ++j) {
        const float sm = s[j] * inv;
        s_m[threadIdx.x * A + j] = K[j] + sm;
        s_q[threadIdx.x * A + j] = q[j] - s[j] * sm;
    }
    if (threadIdx.x == w.row * sh.width) s_n[w.row] = n;
    __syncthreads();
    {      // the block's (mean, centred sum of squares) of every group: weighted mean first, then the squares about it.  The mean is summed as
           // distances from the first thread's: a weighted sum of the means themselves would be off by many 2^-24 of a large mean, and its
           // square, beside a small eps, is a variance that is not there (60000 in every place of a group: r = 240 for 316).
        const int per = gn_cols<V>(sh.Cg), rw = sh.width * A, E = sh.rows * per;
        const int L = lanes_for(sh.gps), l = threadIdx.x & (L - 1);
        const float total = 1.f / ((float)w.px * sh.Cg);
        for (int g = threadIdx.x / L; g < sh.gps; g += GN_TB / L) {
            const float first = s_m[g * per];
            float sum = 0.f, m2 = 0.f;
            for (int e = l; e < E; e += L) {
                const int r = per == 1 ? e : e / per;
                sum += s_n[r] * (s_m[r * rw + g * per + e - r * per] - first);
            }
            const float mean = first + lanes_sum(sum, L) * total;
            for (int e = l; e < E; e += L) {
                const int r = per == 1 ? e : e / per, at = r * rw + g * per + e - r * per;
                const float t = s_m[at] - mean;
                m2 += s_q[at] + s_n[r] * t * t;
            }
            m2 = lanes_sum(m2, L);
            if (l == 0) s_pair[g] = make_float2(mean, m2);
        }
    }
    __syncthreads();
    const int g0 = w.span * sh.gps;
    const double all = (double)sh.HW * sh.Cg;
    auto keep = [&](int g, float2 v) {
        if (a.stats) *reinterpret_cast<float2*>(a.stats + 2 * ((long)w.n * sh.G + g0 + g)) = v;
    };
    const StatAcc::Shape as{sh.HW, (long)R * sh.rows, sh.Cg};
    auto result = [&](int, float2 v) { return make_float2(v.x, gn_rstd((double)v.y / all, a.eps)); };
    bool ok = true;
    unsigned out = 0;
    if (sh.nb == 1) {
        for (int g = threadIdx.x; g < sh.gps; g += GN_TB) {
            const float2 o = result(g, s_pair[g]);
            s_pair[g] = o;
            keep(g, o);
        }
        __syncthreads();
    } else {
        ok = cluster_meet<StatAcc>(sh, wk, w, as, s_pair, s_acc, &out, result, keep);
    }
    DropKey key;
    if constexpr (DROP) key = drop_key(rng);
    if (ok && cnt > 0) {
        Norm<T, ACT> nm[V];
        const int c0 = w.chunk * V - w.span * sh.width * V;
#pragma unroll
        for (int i = 0; i < V; ++i) nm[i].set(s_pair[(c0 + i / PER * PER) / sh.Cg], s_gb[c0 + i].x, s_gb[c0 + i].y);
        const long px0 = (long)w.n * sh.HW + w.p0 + w.row;
        T* y = (T*)a.y + px0 * a.ldy + w.chunk * V;
        const T* res = (const T*)a.res + px0 * a.ldres + w.chunk * V;
        auto put = [&](int r, const Raw<T, V>* other) {
            float f[V];
            d[r].get(f);
            finish<T, V, ACT>(f, nm);
            if constexpr (DROP) drop_apply<V>(key, rng.q, rng.scale, (unsigned long long)(px0 + r * sh.rows) * sh.C + w.chunk * V, f);
            if (other) {
                float o[V];
                other->get(o);
#pragma unroll
                for (int i = 0; i < V; ++i) f[i] += o[i];
            }
            store_v<T, V>(y + (long)r * sh.rows * a.ldy, f);
            if constexpr (V == 1 && DROP) __builtin_amdgcn_sched_barrier(0);      // (registers: not every element's generator at once)
        };
        // B shortcut loads in flight (beyond the image: the thread's first pixel, not used).  All of them in front of the meeting, in as many
        // registers as x: 70 us where this takes 67 (32 x 76 x 76 x 256 bf16)
        if (a.res) {
            constexpr int B = V > 1 ? 2 : 8;
#pragma unroll
            for (int r0 = 0; r0 < R; r0 += B) {
                Raw<T, V> o[B];
#pragma unroll
                for (int k = 0; k < B; ++k) o[k].load(res + (long)(r0 + k < cnt ? r0 + k : 0) * sh.rows * a.ldres);
#pragma unroll
                for (int k = 0; k < B; ++k) o[k].pin();
#pragma unroll
                for (int k = 0; k < B; ++k)
                    if (r0 + k < cnt) put(r0 + k, o + k);
            }
        } else {
#pragma unroll
            for (int r = 0; r < R; ++r)
                if (r < cnt) put(r, nullptr);
        }
    }
    if (sh.nb == 1) return;
    cluster_leave<StatAcc>(sh, wk, w, as, s_acc, out, result, keep, [&](int blk, const unsigned long long* fin) {
        const long p0 = (long)blk * R * sh.rows, left = sh.HW - p0, px = left < (long)R * sh.rows ? left : (long)R * sh.rows;
        for (long e = threadIdx.x; e < px * sh.width; e += 64) {
            const long p = e / sh.width, pix = (long)w.n * sh.HW + p0 + p;
            const int lc = (int)(e - p * sh.width), c = (w.span * sh.width + lc) * V;
            float f[V];
            Norm<T, ACT> nm[V];
            load_v<T, V>((const T*)a.x + pix * a.ldx + c, f);
#pragma unroll
            for (int i = 0; i < V; ++i) nm[i].set(agent_load_pair(fin + (lc * V + i) / sh.Cg), a.gamma[c + i], a.beta[c + i]);
            finish<T, V, ACT>(f, nm);
            if constexpr (DROP) drop_apply<V>(key, rng.q, rng.scale, (unsigned long long)pix * sh.C + c, f);
            if (a.res) {
                float o[V];
                load_v<T, V>((const T*)a.res + pix * a.ldres + c, o);
#pragma unroll
                for (int i = 0; i < V; ++i) f[i] += o[i];
            }
            store_v<T, V>((T*)a.y + pix * a.ldy + c, f);
        }
    });
}

template <typename T, int V, int A>
int launch(const ResPlan& p, const ResFwd& a, const ResWork& wk, int act, const DropRng& rng, hipStream_t s) {
    constexpr int R = GN_HELD_FWD<V>;
    const dim3 grid((unsigned)((long)p.sh.N * p.sh.nspan * p.sh.nb));
    const size_t lds = sizeof(float2) * (p.sh.gps + p.sh.width * V);
#define CY_R(ACT_, D_, R_) hipLaunchKernelGGL((gn_fwd_resident_kernel<T, V, A, ACT_, D_, R_>), grid, dim3(GN_TB), lds, s, a, p.sh, wk, rng)
#define CY_ACT(ACT_)                                  \
    if (rng.q && p.R < R) CY_R(ACT_, true, R / 2);    \
    else if (rng.q) CY_R(ACT_, true, R);              \
    else if (p.R < R) CY_R(ACT_, false, R / 2);       \
    else CY_R(ACT_, false, R)
    if (act == CY_ACT_MISH) { CY_ACT(CY_ACT_MISH); }
    else if (act == CY_ACT_LEAKY) { CY_ACT(CY_ACT_LEAKY); }
    else { CY_ACT(CY_ACT_LINEAR); }
#undef CY_ACT
#undef CY_R
    CY_LAUNCH_CHECK();
    return 0;
}

template <typename T>
int launch_any(const ResPlan& p, const ResFwd& a, const ResWork& wk, int act, const DropRng& rng, hipStream_t s) {
    constexpr int CH = Elem<T>::CH;
    if (p.V == 1) return launch<T, 1, 1>(p, a, wk, act, rng, s);
    const int A = gn_sums<CH>(p.sh.Cg);
    if (A == 1) return launch<T, CH, 1>(p, a, wk, act, rng, s);
    if (A == 2) return launch<T, CH, 2>(p, a, wk, act, rng, s);
    if constexpr (CH == 8)
        if (A == 8) return launch<T, CH, 8>(p, a, wk, act, rng, s);
    return launch<T, CH, 4>(p, a, wk, act, rng, s);
}

}  // namespace
