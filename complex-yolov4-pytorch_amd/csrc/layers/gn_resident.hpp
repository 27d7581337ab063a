// One-launch group norm: what the forward and the backward kernel share.
//
// A CLUSTER of nb blocks owns one image and one span of whole groups; every block loads its pixels ONCE into registers, reduces them
// to one pair of floats per group, and needs the pairs of the other blocks before it can finish.  It writes its pairs into the
// workspace and reads everybody's there until none is missing: a word of all zero bits is a pair that is not there yet (a pair that
// would be is written with a negative zero).  Clusters with many pairs meet in two steps: the first block of every `sub` blocks
// collects theirs and writes the combined pair, everybody collects those.  Pairs are combined in double in an order that depends on
// the shape alone, so results do not depend on who came when.
//
// Why so: what a meeting costs is the number of memory round trips that follow one another, a few microseconds each beside 5 TB/s of
// traffic.  Two (one step) or four, against eight with a counter of arrivals, a flag and a result to fetch; counters and flag in one
// cache line made it five times worse (16 x 304 x 304 x 64 f16 forward, 181 blocks a cluster: 405 us; 120 us with the words apart).
//
// No wait is unbounded and none decides about the result.  A block that has looked `polls` times without seeing all pairs writes its
// number into the cluster's list and LEAVES, without having written any output; every block writes its pairs before it waits, so
// whoever leaves the cluster last finds them all there and finishes what is on the list from memory.  A cluster therefore ends
// whatever else runs on the GPU and however few of its blocks fit at a time; how large a cluster may be is a question of speed.
//
// Everything that blocks say to each other goes through agent-scope atomics (performed behind the XCDs' separate L2 caches).  A block
// counts itself out of the cluster when its own stores have been performed (vmcnt) and it has read what it needs; the last one out
// puts counters and pairs back to zero: a workspace starts zeroed and is left so.  (One that is not -- never zeroed, or two calls at once in it
// -- gives wrong results; the list's bounds are checked all the same, so that nothing outside the workspace is touched.)
#pragma once
#include "layer_common.hpp"

constexpr int GN_TB = 256;                   // threads of a block
constexpr int GN_MAX_CLUSTERS = 512;         // the start of every workspace: zero before and after each call
constexpr int GN_MAX_PAIRS = 384 * 1024;
// a cluster's counters, in cache lines of their own: the root (departures, length of the list) and GN_SUBS lines (departures of a
// sixteenth of the blocks each)
constexpr int GN_LINE = 32, GN_SUBS = 16, GN_WORDS = GN_LINE * (1 + GN_SUBS);
constexpr int64_t GN_COUNTER_BYTES = (int64_t)GN_MAX_CLUSTERS * GN_WORDS * 4;
constexpr int64_t GN_ZERO_BYTES = GN_COUNTER_BYTES + (int64_t)GN_MAX_PAIRS * 8;
// up to this many pairs (32 KB to read for every block) a cluster meets in one step: 361 blocks of 8 groups in two 0 to 5 % slower
constexpr int GN_ONE_STEP = 4096;

// Chunks of V elements a thread holds at most: forward x, backward x and the 32-bit dz (half as many are built, too)
template <int V>
constexpr int GN_HELD_FWD = V == 1 ? 32 : 16;
template <int V>
constexpr int GN_HELD_BWD = V == 1 ? 32 : 8;
static inline int gn_held(int V, bool bwd) { return V == 1 ? (bwd ? GN_HELD_BWD<1> : GN_HELD_FWD<1>) : bwd ? GN_HELD_BWD<8> : GN_HELD_FWD<8>; }

struct ResShape {
    long HW;
    int N, C, G, Cg;
    int width, nspan;      // chunk columns (V elements) of a span; spans per pixel row (width * nspan = C / V)
    int gps;               // groups of a span
    int rows, nb;          // pixels a block takes per step; blocks of a cluster
    int sub, nsub;         // two-step meeting: blocks that are combined first, how many such (0: one step)
    int polls;
};

struct ResWork {
    unsigned* counters;              // [cluster][GN_WORDS]
    unsigned long long* pairs;       // [cluster][nb + nsub][group of the span]
    unsigned long long* fin;         // [cluster][group of the span]: results, for the block that finishes the list
    unsigned* list;                  // [cluster][block]
    double* part;                    // backward: [channels / 8][slice][2][8], parameter gradients
    float* chan;                     // backward: [image][block][channel][2]
};

struct ResWhere {
    int cluster, n, span, blk, chunk, row;
    bool on;
    long p0;
    int px;                          // pixels of this block
};

template <int R>
__device__ __forceinline__ ResWhere res_where(const ResShape& sh) {
    ResWhere w;
    w.cluster = blockIdx.x / sh.nb;
    w.blk = blockIdx.x - w.cluster * sh.nb;
    w.n = w.cluster / sh.nspan;
    w.span = w.cluster - w.n * sh.nspan;
    w.row = threadIdx.x / sh.width;
    w.chunk = w.span * sh.width + threadIdx.x - w.row * sh.width;
    w.on = w.row < sh.rows;
    const long ppb = (long)R * sh.rows;
    w.p0 = w.blk * ppb;
    w.px = (int)(sh.HW - w.p0 < ppb ? sh.HW - w.p0 : ppb);
    return w;
}

__device__ __forceinline__ unsigned agent_load(const unsigned* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ unsigned agent_add(unsigned* p, unsigned v) {
    return __hip_atomic_fetch_add(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void agent_store(unsigned* p, unsigned v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 agent_load_pair(const unsigned long long* p) {
    return __builtin_bit_cast(float2, __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}
__device__ __forceinline__ void agent_store_pair(unsigned long long* p, float2 v) {
    __hip_atomic_store(p, __builtin_bit_cast(unsigned long long, v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// this thread's stores and atomics have been performed
__device__ __forceinline__ void stores_done() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }

__device__ __forceinline__ int pow2_up(int n) { return n <= 1 ? 1 : 1 << (32 - __clz(n - 1)); }

// lanes that share one of `jobs` reductions of a 256-thread block: a power of two, at most a wave
__device__ __forceinline__ int lanes_for(int jobs) {
    const int up = pow2_up(jobs);
    return up >= GN_TB ? 1 : (GN_TB / up > 64 ? 64 : GN_TB / up);
}
__device__ __forceinline__ double lanes_sum(double v, int L) {
    for (int o = 1; o < L; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
}
__device__ __forceinline__ float lanes_sum(float v, int L) {
    for (int o = 1; o < L; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
}

__device__ __forceinline__ void publish_pair(unsigned long long* p, float2 v) {
    unsigned long long u = __builtin_bit_cast(unsigned long long, v);
    __hip_atomic_store(p, u ? u : 0x80000000ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Collects `count` published entries of gps pairs each, from src on, and combines them group by group.  Lane (g, l) of P = 2^k >= gps
// columns and 256 / P rows takes the entries l, l + 256 / P, ... of group g (neighbouring lanes read neighbouring words, four in
// flight), the rows are folded in a tree through LDS: the order is a function of the shape.  `vt` lets one wave play all 256 lanes.
// Acc: the caller's combination -- a lane's running sums Acc(shape, first block, blocks per entry).add(entry number, pair), their Sum,
// and merge(Sum&, Sum), out(Sum) -> combined pair.
template <class Acc>
struct Gather {
    const ResShape& sh;
    const unsigned long long* src;
    int count, P, rows;
    __device__ Gather(const ResShape& s, const unsigned long long* from, int n) : sh(s), src(from), count(n) {
        P = pow2_up(s.gps);
        rows = P < GN_TB ? GN_TB / P : 1;
    }
    // lanes (columns of groups beyond 256 in turn: c0); false when this lane looked `polls` times in vain
    __device__ __forceinline__ bool lane(int vt, int c0, int polls, Acc& acc) const {
        const int g = c0 + (P < GN_TB ? vt & (P - 1) : vt), l = P < GN_TB ? vt / P : 0;
        bool ok = true;
        if (g >= sh.gps) return true;
        for (int i0 = l; i0 < count; i0 += 4 * rows) {
            unsigned long long u[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int i = i0 + k * rows;
                u[k] = __hip_atomic_load(src + (long)(i < count ? i : count - 1) * sh.gps + g, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int i = i0 + k * rows;
                if (i < count) {
                    while (!u[k] && polls > 0) {
                        --polls;
                        __builtin_amdgcn_s_sleep(4);
                        u[k] = __hip_atomic_load(src + (long)i * sh.gps + g, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    }
                    ok = ok && u[k];
                    acc.add(i, __builtin_bit_cast(float2, u[k]));
                }
            }
        }
        return ok;
    }
};

// all threads of the block: out(g, combined pair) by one thread per group; false: some pair was missing (out was not called)
template <class Acc, class Out>
__device__ __forceinline__ bool gather_block(const ResShape& sh, const unsigned long long* src, int count, int first, int per, int polls,
                                             const typename Acc::Shape& as, typename Acc::Sum* s_acc, Out out) {
    const Gather<Acc> ga(sh, src, count);
    const int t = threadIdx.x;
    // one lane waits for the last entry, which most often is the last to come; the others look when it is there
    if (t == 0)
        while (polls > 0 && !__hip_atomic_load(src + (long)count * sh.gps - 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) {
            --polls;
            __builtin_amdgcn_s_sleep(4);
        }
    __syncthreads();
    bool ok = true;
    for (int c0 = 0; c0 < sh.gps; c0 += GN_TB) {
        Acc acc(as, first, per);
        ok = __syncthreads_and(ga.lane(t, c0, polls, acc)) && ok;
        typename Acc::Sum sum = acc.sum();
        for (int h = ga.rows >> 1; h > 0; h >>= 1) {
            if (t / ga.P >= h && t / ga.P < 2 * h) s_acc[t] = sum;
            __syncthreads();
            if (t / ga.P < h) Acc::merge(sum, s_acc[t + h * ga.P]);
            __syncthreads();
        }
        const int g = c0 + t;
        if (ok && t < (ga.P < GN_TB ? ga.P : GN_TB) && g < sh.gps) out(g, Acc::out(sum));
    }
    return ok;
}

// the same by one wave, every pair being there
template <class Acc, class Out>
__device__ __forceinline__ void gather_wave(const ResShape& sh, const unsigned long long* src, int count, int first, int per,
                                            const typename Acc::Shape& as, typename Acc::Sum* s_acc, Out out) {
    const Gather<Acc> ga(sh, src, count);
    const int cols = ga.P < GN_TB ? ga.P : GN_TB;
    for (int c0 = 0; c0 < sh.gps; c0 += GN_TB) {
        for (int vt = threadIdx.x; vt < GN_TB; vt += 64) {
            Acc acc(as, first, per);
            ga.lane(vt, c0, 0, acc);
            s_acc[vt] = acc.sum();
        }
        for (int h = ga.rows >> 1; h > 0; h >>= 1) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            for (int vt = threadIdx.x; vt < h * ga.P; vt += 64) Acc::merge(s_acc[vt], s_acc[vt + h * ga.P]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        for (int t = threadIdx.x; t < cols; t += 64)
            if (c0 + t < sh.gps) out(c0 + t, Acc::out(s_acc[t]));
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// s_pair[g] (LDS, one pair per group of the span): the block's pairs in, the cluster's result finish(g, combined pair) out; keep(g,
// result) runs in one block.  s_acc: 256 Sums of LDS.  -> false: gave up (the block is on the list).  All threads of the block call it.
// *out (thread 0): what the counter said that this block has left through.
template <class Acc, class Finish, class Keep>
__device__ __forceinline__ bool cluster_meet(const ResShape& sh, const ResWork& wk, const ResWhere& w, const typename Acc::Shape& as,
                                             float2* s_pair, typename Acc::Sum* s_acc, unsigned* out, Finish finish, Keep keep) {
    unsigned* cnt = wk.counters + (long)GN_WORDS * w.cluster;
    unsigned long long* one = wk.pairs + (long)w.cluster * (sh.nb + sh.nsub) * sh.gps;
    unsigned long long* two = one + (long)sh.nb * sh.gps;
    for (int g = threadIdx.x; g < sh.gps; g += GN_TB) publish_pair(one + (long)w.blk * sh.gps + g, s_pair[g]);
    bool ok = true;
    if (sh.nsub && w.blk % sh.sub == 0) {
        const int count = sh.nb - w.blk < sh.sub ? sh.nb - w.blk : sh.sub;
        ok = gather_block<Acc>(sh, one + (long)w.blk * sh.gps, count, w.blk, 1, sh.polls, as, s_acc,
                               [&](int g, float2 v) { publish_pair(two + (long)(w.blk / sh.sub) * sh.gps + g, v); });
    }
    if (ok)
        ok = gather_block<Acc>(sh, sh.nsub ? two : one, sh.nsub ? sh.nsub : sh.nb, 0, sh.nsub ? sh.sub : 1, sh.polls, as, s_acc, [&](int g, float2 v) {
            const float2 r = finish(g, v);
            s_pair[g] = r;
            if (w.blk == 0) keep(g, r);
        });
    stores_done();
    __syncthreads();
    if (threadIdx.x == 0) {
        if (!ok) {
            const unsigned at = agent_add(cnt + 1, 1u);      // (in a workspace that was left as it should not be this may be any number)
            if (at < (unsigned)sh.nb) agent_store(wk.list + (long)w.cluster * sh.nb + at, (unsigned)w.blk);
            stores_done();
        }
        *out = agent_add(sh.nb <= GN_SUBS ? cnt : cnt + GN_LINE * (1 + w.blk % GN_SUBS), 1u);
    }
    return ok;
}

// The first wave of every block, at its end: the last one out of the cluster finishes the listed blocks -- rest(block, group -> result)
// by one wave -- and puts the counters and the pairs back.
template <class Acc, class Finish, class Keep, class Rest>
__device__ __forceinline__ void cluster_leave(const ResShape& sh, const ResWork& wk, const ResWhere& w, const typename Acc::Shape& as,
                                              typename Acc::Sum* s_acc, unsigned out, Finish finish, Keep keep, Rest rest) {
    if (threadIdx.x >= 64) return;
    unsigned* cnt = wk.counters + (long)GN_WORDS * w.cluster;
    unsigned last = 0, left = 0;
    if (threadIdx.x == 0) {
        if (sh.nb <= GN_SUBS) {
            last = out == (unsigned)sh.nb - 1;
        } else {
            const int mine = (sh.nb - w.blk % GN_SUBS + GN_SUBS - 1) / GN_SUBS;
            last = out == (unsigned)mine - 1 && agent_add(cnt, 1u) == GN_SUBS - 1;
        }
        if (last) left = agent_load(cnt + 1);
    }
    last = __builtin_amdgcn_readfirstlane(last);
    if (!last) return;
    left = __builtin_amdgcn_readfirstlane(left);
    unsigned long long* one = wk.pairs + (long)w.cluster * (sh.nb + sh.nsub) * sh.gps;
    unsigned long long* two = one + (long)sh.nb * sh.gps;
    const int t = threadIdx.x;
    if (left) {      // the same steps in the same order, by this wave alone (the block's other waves are past the meeting)
        unsigned long long* fin = wk.fin + (long)w.cluster * sh.gps;
        for (int b = 0; sh.nsub && b < sh.nb; b += sh.sub) {
            gather_wave<Acc>(sh, one + (long)b * sh.gps, sh.nb - b < sh.sub ? sh.nb - b : sh.sub, b, 1, as, s_acc,
                             [&](int g, float2 v) { publish_pair(two + (long)(b / sh.sub) * sh.gps + g, v); });
            stores_done();
        }
        gather_wave<Acc>(sh, sh.nsub ? two : one, sh.nsub ? sh.nsub : sh.nb, 0, sh.nsub ? sh.sub : 1, as, s_acc, [&](int g, float2 v) {
            const float2 r = finish(g, v);
            agent_store_pair(fin + g, r);
            keep(g, r);
        });
        stores_done();
        for (unsigned i = 0; i < left && i < (unsigned)sh.nb; ++i) {
            const unsigned blk = agent_load(wk.list + (long)w.cluster * sh.nb + i);
            if (blk < (unsigned)sh.nb) rest((int)blk, fin);
        }
    }
    for (int i = t; i < (sh.nb + sh.nsub) * sh.gps; i += 64) __hip_atomic_store(one + i, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (t <= GN_SUBS) {
        agent_store(cnt + GN_LINE * t, 0u);
        agent_store(cnt + GN_LINE * t + 1, 0u);
    }
}

// ---- host: launched from group_norm.hip ---------------------------------------------------------------------------------------
struct ResPlan {
    ResShape sh;
    int R, V;              // V: 16 bytes, or 1
};
struct ResFwd {
    const void* x; int ldx;
    void* y; int ldy;
    const void* res; int ldres;
    const float* gamma; const float* beta;
    float eps;
    float* stats;
};
struct ResBwd {
    const void* x; int ldx;
    const void* dy; int lddy;
    void* dx; int lddx;
    void* resg; int ldrg; int res_accum;
    const float* gamma; const float* beta; const float* stats;
    float* ggamma; float* gbeta;
    float gscale; int accumulate;
};
// backward: the parameter gradients' rows (one per image and block) are added in this many slices, of at least 256 rows
static inline int gn_param_slices(long rows) { return rows >= 16 * 256 ? 16 : rows < 512 ? 1 : (int)(rows / 256); }

#define CY_DECL(NAME_, ARGS_) int NAME_(const ResPlan& p, const ARGS_& a, const ResWork& wk, int act, const DropRng& rng, hipStream_t s)
CY_DECL(gn_resident_fwd_f16, ResFwd);
CY_DECL(gn_resident_fwd_bf16, ResFwd);
CY_DECL(gn_resident_fwd_f32, ResFwd);
CY_DECL(gn_resident_bwd_f16, ResBwd);
CY_DECL(gn_resident_bwd_bf16, ResBwd);
CY_DECL(gn_resident_bwd_f32, ResBwd);
#undef CY_DECL
