#include "gn_resident_bwd.hpp"

int gn_resident_bwd_f16(const ResPlan& p, const ResBwd& a, const ResWork& wk, int act, const DropRng& rng, hipStream_t s) {
    return launch_any<f16>(p, a, wk, act, rng, s);
}
