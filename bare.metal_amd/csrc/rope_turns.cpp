/* SPDX-License-Identifier: MPL-2.0
 *
 * rope_turns.cpp — the table of the rotation's turns a position
 * (include/bm_paged.h), as fractions of 2^64: a position times it, mod 2^64,
 * is the fraction of a turn without any rounding but the table's own, 2^-64
 * of a turn a position.  Long double carries the 63 bits that are kept.
 */
#include "bm_paged.h"
#include "bmk.h"

#include <math.h>

extern "C" int bm_rope_turns(int rot, int scaling, double theta, double factor, double low, double high, double original,
                             uint64_t* turns, float* mscale) {
    const long double pi = 3.14159265358979323846264338327950288L;
    BMK_REQUIRE(rot >= 0 && rot % 2 == 0 && theta > 1 && theta < INFINITY && mscale && (turns || rot == 0) &&
                    scaling >= BM_TURNS_NONE && scaling <= BM_TURNS_YARN,
                "bm_rope_turns: bad rot %d, scaling %d or theta %g", rot, scaling, theta);
    if (scaling != BM_TURNS_NONE)
        BMK_REQUIRE(factor >= 1 && factor < INFINITY, "bm_rope_turns: bad factor %g", factor);
    if (scaling == BM_TURNS_LLAMA3 || scaling == BM_TURNS_YARN)
        BMK_REQUIRE(original > 0 && original < INFINITY && low > 0 && high > low && high < INFINITY,
                    "bm_rope_turns: bad low %g, high %g or original %g", low, high, original);
    long double first = 0, last = 0;
    *mscale = 1.0f;
    if (scaling == BM_TURNS_YARN) {
        const long double per = rot / (2 * logl(theta));
        first = fmaxl(floorl(per * logl(original / (2 * pi * high))), 0);
        last = fminl(ceill(per * logl(original / (2 * pi * low))), rot - 1);
        *mscale = (float)(0.1 * log(factor) + 1);
    }
    for (int i = 0; i < rot / 2; i++) {
        long double f = powl(theta, -2.0L * i / rot);
        long double slow = 0; /* the part that factor slows down */
        if (scaling == BM_TURNS_LINEAR) slow = 1;
        if (scaling == BM_TURNS_LLAMA3) slow = 1 - fminl(fmaxl((original * f / (2 * pi) - low) / (high - low), 0), 1);
        if (scaling == BM_TURNS_YARN) slow = fminl(fmaxl((i - first) / fmaxl(last - first, 0.001L), 0), 1);
        if (slow > 0) f = (1 - slow) * f + slow * f / factor;
        const long double t = f / (2 * pi);
        turns[i] = (uint64_t)rintl((t - floorl(t)) * 0x1p63L) << 1;
    }
    return 0;
}
