// Shared by the per-image layers (group norm, dropout): element access that does not need 16-byte rows, and the dropout generator.
#pragma once
#include "common.hpp"

// The value as it stands: keeps the conversion to 16 bits that follows from being merged into the multiply-add before it (one rounding
// instead of two, where the compiler finds it: two kernels' stored values would differ in their last bit).
__device__ __forceinline__ float rounded(float v) {
    asm("" : "+v"(v));
    return v;
}

// Sixteen bytes of output, not kept in the caches: they hold what is still to be read instead.  f16, inputs and outputs alternating:
// 16 x 152 x 152 x 128 forward 51.5 -> 40 us, 16 x 304 x 304 x 64 backward 187 -> 170; with a pass that reads the output at once 87.6 -> 83.4
// and 252 -> 239, and at no size from 1 x 19 x 19 x 1024 up slower, with or without the reader.
template <typename T>
__device__ __forceinline__ void store_past(T* p, u32x4 v) {
    __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(p));
}

// V consecutive elements as floats: V = Elem<T>::CH is one 16-byte access, V = 1 takes any stride and alignment
template <typename T, int V>
__device__ __forceinline__ void load_v(const T* p, float* f) {
    if constexpr (V == 1) f[0] = (float)*p;
    else chunk_to_f32<T>(*reinterpret_cast<const u32x4*>(p), f);
}
template <typename T, int V>
__device__ __forceinline__ void store_v(T* p, const float* f) {
    if constexpr (V == 1) *p = (T)f[0];
    else store_past(p, f32_to_chunk<T>(f));
}

// The same in two steps, so that several loads can be in flight before the first is looked at.  part / set_part: H (4, or all) elements
// from h on.  pin: what was computed from the value is not kept in registers beyond this point, it is computed again.
template <typename T, int V>
struct Raw {
    u32x4 v;
    __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const u32x4*>(p); }
    __device__ __forceinline__ void store(T* p) const { store_past(p, v); }
    __device__ __forceinline__ void get(float* f) const { chunk_to_f32<T>(v, f); }
    __device__ __forceinline__ void clear() { v = u32x4{0u, 0u, 0u, 0u}; }
    __device__ __forceinline__ void pin() { asm volatile("" : "+v"(v)); }
    template <int H>
    __device__ __forceinline__ void part(int h, float* f) const {
        float t[V];
        chunk_to_f32<T>(V == 8 ? u32x4{v[h / 2], v[h / 2 + 1], 0u, 0u} : v, t);
#pragma unroll
        for (int i = 0; i < H; ++i) f[i] = t[i];
    }
    template <int H>
    __device__ __forceinline__ void set_part(int h, const float* f) {
        float t[V] = {};
#pragma unroll
        for (int i = 0; i < H; ++i) t[i] = f[i];
        const u32x4 b = f32_to_chunk<T>(t);
        if constexpr (V == 8) v[h / 2] = b[0], v[h / 2 + 1] = b[1];
        else v = b;
    }
};
template <typename T>
struct Raw<T, 1> {
    T v;
    __device__ __forceinline__ void load(const T* p) { v = *p; }
    __device__ __forceinline__ void store(T* p) const { *p = v; }
    __device__ __forceinline__ void get(float* f) const { f[0] = (float)v; }
    __device__ __forceinline__ void clear() { v = (T)0.f; }
    __device__ __forceinline__ void pin() {
        if constexpr (sizeof(T) == 4) {
            asm volatile("" : "+v"(v));
        } else {
            unsigned u = __builtin_bit_cast(unsigned short, v);
            asm volatile("" : "+v"(u));
            v = __builtin_bit_cast(T, (unsigned short)u);
        }
    }
    template <int H>
    __device__ __forceinline__ void part(int, float* f) const { f[0] = (float)v; }
    template <int H>
    __device__ __forceinline__ void set_part(int, const float* f) { v = (T)f[0]; }
};

// ---- dropout generator ---------------------------------------------------------------------------------------------------
// Philox-4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011): a 128-bit counter goes
// through ten rounds of two 32 x 32 -> 64 bit products under a 64-bit key.  Here key = seed, counter = (block, step, layer id):
// nothing is stored between the passes, the backward pass asks for the same words again.  One 128-bit result serves EIGHT
// elements, a 16-bit half-word each: p is resolved to 2^-16 (the scale uses the resolved p, so the expectation is exact), and
// the ~120 issue slots of the ten rounds cost 15 per element where 32 bits each would cost 30 -- below what an element's
// 4 bytes of traffic leave room for at 16-bit storage.
struct DropRng {
    const int64_t* state;      // device: (seed, step)
    int q;                     // an element is dropped when its half-word is below q (0: no dropout, 65536: all)
    unsigned id;               // layer
    float scale;               // 65536 / (65536 - q)
};

struct DropKey {
    unsigned k0, k1, step, id;
};

__device__ __forceinline__ DropKey drop_key(const DropRng& r) {
    const unsigned long long seed = (unsigned long long)r.state[0], step = (unsigned long long)r.state[1];
    return DropKey{(unsigned)seed, (unsigned)(seed >> 32), (unsigned)step, r.id};
}

__device__ __forceinline__ u32x4 drop_words(const DropKey& key, unsigned long long block) {
    unsigned c0 = (unsigned)block, c1 = (unsigned)(block >> 32), c2 = key.step, c3 = key.id;
    unsigned k0 = key.k0, k1 = key.k1;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
        const unsigned n0 = (unsigned)(b >> 32) ^ c1 ^ k0, n2 = (unsigned)(a >> 32) ^ c3 ^ k1;
        c1 = (unsigned)b;
        c3 = (unsigned)a;
        c0 = n0;
        c2 = n2;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return u32x4{c0, c1, c2, c3};
}

__device__ __forceinline__ int drop_half(const u32x4& w, int j) { return (int)((w[j >> 1] >> (16 * (j & 1))) & 0xFFFFu); }

// the same for a j that is not a constant
__device__ __forceinline__ int drop_one(const u32x4& w, int j) {
    const unsigned lo = (j & 2) ? w[1] : w[0], hi = (j & 2) ? w[3] : w[2];
    const unsigned x = (j & 4) ? hi : lo;
    return (int)((j & 1) ? x >> 16 : x & 0xFFFFu);
}

// f[i] = kept ? f[i] * scale : 0 for the V elements from dense element index e on.  A selection, not a product: what is in a dropped
// place (a NaN too) does not come through.  e is a multiple of V.  V = 1 runs the ten rounds for one half-word of eight (group norm +
// dropout on 16 x 76 x 76 x 255 f16: forward 83 us, 39 without dropout).
template <int V>
__device__ __forceinline__ void drop_apply(const DropKey& key, int q, float scale, unsigned long long e, float* f) {
    const u32x4 w = drop_words(key, e >> 3);
    if constexpr (V == 8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = drop_half(w, i) >= q ? rounded(f[i] * scale) : 0.f;
    } else if constexpr (V == 4) {
        const bool up = (e >> 2) & 1;
        const u32x4 h = {up ? w[2] : w[0], up ? w[3] : w[1], 0u, 0u};
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = drop_half(h, i) >= q ? rounded(f[i] * scale) : 0.f;
    } else {
        f[0] = drop_one(w, (int)(e & 7)) >= q ? rounded(f[0] * scale) : 0.f;
    }
}

// The selection alone, on a chunk as it is stored: what is dropped becomes zero, what is kept is to be scaled.
template <typename T, int V>
__device__ __forceinline__ void drop_raw(const DropKey& key, int q, unsigned long long e, Raw<T, V>& x) {
    const u32x4 w = drop_words(key, e >> 3);
    if constexpr (V == 8) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            x.v[k] &= (drop_half(w, 2 * k) >= q ? 0xFFFFu : 0u) | (drop_half(w, 2 * k + 1) >= q ? 0xFFFF0000u : 0u);
    } else if constexpr (V == 4) {
        const bool up = (e >> 2) & 1;
        const u32x4 h = {up ? w[2] : w[0], up ? w[3] : w[1], 0u, 0u};
#pragma unroll
        for (int i = 0; i < 4; ++i) x.v[i] = drop_half(h, i) >= q ? x.v[i] : 0u;
    } else {
        if (drop_one(w, (int)(e & 7)) < q) x.clear();
    }
}

// host: drop probability in 65536ths -> generator arguments; false for arguments no kernel takes
static inline bool make_drop(int q, const int64_t* state, int id, DropRng& r) {
    if (q < 0 || q > 65536 || (q > 0 && !state)) return false;
    r.state = state;
    r.q = q;
    r.id = (unsigned)id;
    r.scale = q < 65536 ? 65536.f / (float)(65536 - q) : 0.f;
    return true;
}

static inline bool aligned_to(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }
