#include "gn_resident_fwd.hpp"

int gn_resident_fwd_f32(const ResPlan& p, const ResFwd& a, const ResWork& wk, int act, const DropRng& rng, hipStream_t s) {
    return launch_any<float>(p, a, wk, act, rng, s);
}
