#include "gn_resident_bwd.hpp"

int gn_resident_bwd_f32(const ResPlan& p, const ResBwd& a, const ResWork& wk, int act, const DropRng& rng, hipStream_t s) {
    return launch_any<float>(p, a, wk, act, rng, s);
}
