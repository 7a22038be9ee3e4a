// rotary_plan.cpp -- frequencies of rotary positions (geo_b200_rotary_plan_init).
// Extended precision (64-bit significands on x86), so that hi + lo carries the
// frequency beyond float64 and the angle of a far position stays accurate.
#include <cmath>
#include <cstring>

#include "geo/geo_b200.h"

extern "C" geo_b200_status_t geo_b200_rotary_plan_init(geo_b200_rotary_plan_t *plan,
                                                       const geo_b200_rotary_config_t *config) {
    auto positive = [](double v) { return std::isfinite(v) && v > 0.0; };
    if (plan == nullptr || config == nullptr || config->layout > GEO_B200_ROTARY_HALF || config->rotary_dim < 2 ||
        config->rotary_dim > GEO_B200_ROTARY_MAX_DIM || config->rotary_dim % 2 != 0 || !positive(config->base) ||
        config->scaling > GEO_B200_ROTARY_SCALING_BANDED || !std::isfinite(config->amplitude))
        return GEO_B200_INVALID_ARGUMENT;
    const bool scaled = config->scaling != GEO_B200_ROTARY_SCALING_NONE;
    const bool banded = config->scaling == GEO_B200_ROTARY_SCALING_BANDED;
    if (scaled && !positive(config->factor)) return GEO_B200_INVALID_ARGUMENT;
    if (banded && (!positive(config->original_length) || !std::isfinite(config->low_rotations) ||
                   !std::isfinite(config->high_rotations) || !(config->low_rotations < config->high_rotations)))
        return GEO_B200_INVALID_ARGUMENT;

    const int d = (int)config->rotary_dim;
    const long double two_pi = 8.0L * std::atan(1.0L);
    const long double factor = scaled ? (long double)config->factor : 1.0L;
    long double base = config->base;
    if (config->scaling == GEO_B200_ROTARY_SCALING_BASE && d > 2)
        base *= std::pow(factor, (long double)d / (long double)(d - 2));
    geo_b200_rotary_plan_t p;
    std::memset(&p, 0, sizeof(p));
    for (int i = 0; i < d / 2; ++i) {
        long double f = std::pow(base, -2.0L * i / (long double)d);
        if (config->scaling == GEO_B200_ROTARY_SCALING_LINEAR) f /= factor;
        if (banded) {
            const long double low = config->low_rotations, high = config->high_rotations;
            const long double turns = (long double)config->original_length * f / two_pi;
            long double keep = (turns - low) / (high - low);
            keep = keep < 0.0L ? 0.0L : (keep > 1.0L ? 1.0L : keep);
            f = f * keep + f / factor * (1.0L - keep);
        }
        const long double turns = f / two_pi;
        p.turns[i] = (double)turns;
        p.turns_low[i] = (double)(turns - (long double)p.turns[i]);
        // A frequency whose quarter turns at the farthest position leave 53 bits is not an angle any more.
        if (!(std::fabs(p.turns[i]) <= 0x1p18)) return GEO_B200_INVALID_ARGUMENT;
    }
    p.abi_version = GEO_B200_ABI_VERSION;
    p.layout = config->layout;
    p.rotary_dim = config->rotary_dim;
    p.amplitude = config->amplitude;
    *plan = p;
    return GEO_B200_OK;
}
