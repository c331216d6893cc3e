// Host code: the angular frequencies of rotary positions (mako_rope_freqs), with the scalings used to run past the
// trained context.
#include "kernels.h"
#include "mako_attn.h"

#include <algorithm>
#include <cmath>

extern "C" int mako_rope_freqs(uint32_t rot, double theta, int scaling, double factor, double context, double low,
                               double high, double* freq)
{
    if (!freq)
        return mako::set_error(MAKO_EINVAL, "rope_freqs: null freq");
    if (!rot || rot % 2 || rot > 256 || (scaling == MAKO_ROPE_BASE && rot == 2))
        return mako::set_error(MAKO_EINVAL, "rope_freqs: %u rotated", rot);
    if (scaling < MAKO_ROPE_PLAIN || scaling > MAKO_ROPE_PARTS)
        return mako::set_error(MAKO_EINVAL, "rope_freqs: scaling %d", scaling);
    if (!(theta > 1.0) || !std::isfinite(theta))
        return mako::set_error(MAKO_EINVAL, "rope_freqs: theta %g", theta);
    if (scaling != MAKO_ROPE_PLAIN && (!(factor >= 1.0) || !std::isfinite(factor)))
        return mako::set_error(MAKO_EINVAL, "rope_freqs: factor %g", factor);
    if (scaling == MAKO_ROPE_PARTS && (!(context > 0.0) || !std::isfinite(context) || !(low >= 0.0) || !(high > low) ||
                                       !std::isfinite(high)))
        return mako::set_error(MAKO_EINVAL, "rope_freqs: context %g, low %g, high %g", context, low, high);
    const double kTwoPi = 6.283185307179586476925;
    if (scaling == MAKO_ROPE_BASE)  // the last pair, i = rot / 2 - 1, is slowed by exactly factor
        theta *= std::pow(factor, double(rot) / double(rot - 2));
    for (uint32_t i = 0; i < rot / 2; ++i) {
        double f = std::pow(theta, -2.0 * double(i) / double(rot));
        if (scaling == MAKO_ROPE_LINEAR)
            f /= factor;
        if (scaling == MAKO_ROPE_PARTS) {
            const double g = std::min(1.0, std::max(0.0, (context * f / kTwoPi - low) / (high - low)));
            f *= g + (1.0 - g) / factor;
        }
        freq[i] = f;
    }
    mako::clear_error();
    return MAKO_OK;
}
