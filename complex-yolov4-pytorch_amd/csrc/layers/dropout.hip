// Dropout over a channels-last view, mask never stored:  y = kept ? x * 65536 / (65536 - q) : 0  (or added to what y holds).
// The gradient is the same map of dy, so one kernel serves both directions.  Bound in 16-byte accesses (V = CH): memory; the generator's ten
// rounds are spread over eight elements (f32: four) and stay below it.  16 x 304 x 304 x 64 bf16 63.5 us (378 MB, 6.0 TB/s), 16 x 76 x 76 x 256
// f32 28 us (189 MB, 6.7 TB/s).  Element by element (V = 1: rows that do not start on 16 bytes): the generator, all ten rounds for every
// element, and a division; 16 x 76 x 76 x 255 f16 71 us where 256 channels take 17.
#include "layer_common.hpp"

namespace {

template <typename T, int V, bool ACCUM>
__global__ void __launch_bounds__(256) dropout_kernel(const T* x, int ldx, T* y, int ldy, long M, int C, DropRng rng) {
    const DropKey key = drop_key(rng);
    const int cpr = C / V;
    const long total = M * cpr, step = (long)gridDim.x * 256;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += step) {
        const long p = i / cpr;
        const int c = (int)(i - p * cpr) * V;
        float f[V];
        load_v<T, V>(x + p * ldx + c, f);
        drop_apply<V>(key, rng.q, rng.scale, (unsigned long long)i * V, f);
        if (ACCUM) {
            float o[V];
            load_v<T, V>(y + p * ldy + c, o);
#pragma unroll
            for (int k = 0; k < V; ++k) f[k] += o[k];
        }
        store_v<T, V>(y + p * ldy + c, f);
    }
}

template <typename T>
int launch(const void* x, int ldx, void* y, int ldy, long M, int C, const DropRng& rng, int accumulate, hipStream_t s) {
    constexpr int CH = Elem<T>::CH;
    if (!aligned_to(x, sizeof(T)) || !aligned_to(y, sizeof(T))) return CY_ERR_ARG;
    const bool vec = C % CH == 0 && ldx % CH == 0 && ldy % CH == 0 && aligned_to(x, 16) && aligned_to(y, 16);
    const long total = M * (C / (vec ? CH : 1));
    const long want = (total + 255) / 256;
    const dim3 grid((unsigned)(want < 16384 ? want : 16384));
#define CY_DROP(V_, A_) hipLaunchKernelGGL((dropout_kernel<T, V_, A_>), grid, dim3(256), 0, s, (const T*)x, ldx, (T*)y, ldy, M, C, rng)
    if (vec && accumulate) CY_DROP(CH, true);
    else if (vec) CY_DROP(CH, false);
    else if (accumulate) CY_DROP(1, true);
    else CY_DROP(1, false);
#undef CY_DROP
    CY_LAUNCH_CHECK();
    return 0;
}

}  // namespace

extern "C" int cy_dropout(const void* x, int ldx, void* y, int ldy, int64_t M, int C, int q, const int64_t* rng, int id,
                          int accumulate, int dtype, cy_stream_t s) {
    CY_ENTER();
    DropRng r;
    if (M < 0 || C < 1 || ldx < C || ldy < C || !make_drop(q, rng, id, r) || !rng) return CY_ERR_ARG;
    if (dtype != CY_F16 && dtype != CY_BF16 && dtype != CY_F32) return CY_ERR_ARG;
    if (M == 0) return 0;
    if (!x || !y) return CY_ERR_ARG;
    if (dtype == CY_F16) return launch<f16>(x, ldx, y, ldy, (long)M, C, r, accumulate, cy_s(s));
    if (dtype == CY_BF16) return launch<bf16>(x, ldx, y, ldy, (long)M, C, r, accumulate, cy_s(s));
    return launch<float>(x, ldx, y, ldy, (long)M, C, r, accumulate, cy_s(s));
}
