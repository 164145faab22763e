// rta_rotary.hpp -- the angle of a pair of values at a position, and the host checks of a rotation.
#pragma once
#include <math.h>

#include "rta_common.hpp"
#include "rta_host.hpp"

namespace rta {

struct RotaryArgs {
    const double* turns;   // [dims / 2]
    double amplitude;
    int dims;
};

// amplitude (cos, sin) of 2 pi position turns.  Only the product's distance from a whole number of turns counts: the
// rounded product says which one, and one fma takes it off the exact product, so far positions lose nothing (but for
// the conversion to fp64 past 2^53; the rounded product would be off by 2^-53 of the turns made).  Within half a quarter
// turn the power series, to theta^16 and theta^15: the first terms left out are 2e-18 and 5e-17.
__device__ __forceinline__ double2 turn_of(double position, double turns, double amplitude) {
    const double quarters = 4.0 * fma(position, turns, -rint(position * turns)), n = rint(quarters);
    const double x = (quarters - n) * 1.5707963267948966, z = x * x;   // pi / 2
    double s = -1.0 / 1307674368000.0, c = 1.0 / 20922789888000.0;     // 15!, 16!
    s = fma(s, z, 1.0 / 6227020800.0);
    c = fma(c, z, -1.0 / 87178291200.0);
    s = fma(s, z, -1.0 / 39916800.0);
    c = fma(c, z, 1.0 / 479001600.0);
    s = fma(s, z, 1.0 / 362880.0);
    c = fma(c, z, -1.0 / 3628800.0);
    s = fma(s, z, -1.0 / 5040.0);
    c = fma(c, z, 1.0 / 40320.0);
    s = fma(s, z, 1.0 / 120.0);
    c = fma(c, z, -1.0 / 720.0);
    s = fma(s, z, -1.0 / 6.0);
    c = fma(c, z, 1.0 / 24.0);
    c = fma(c, z, -0.5);
    s = fma(s * z, x, x);
    c = fma(c, z, 1.0);
    const uint32_t quadrant = to_int(n) & 3;
    const double a = quadrant & 1 ? s : c, b = quadrant & 1 ? c : s;
    return double2{quadrant == 1 || quadrant == 2 ? -amplitude * a : amplitude * a, quadrant & 2 ? -amplitude * b : amplitude * b};
}

// own c + other s, rounded to fp32 once; the same operations whichever kernel and layout calls it, so that they
// agree bit by bit.
__device__ __forceinline__ float turn_value(float own, float other, double c, double s) {
    return (float)fma((double)own, c, (double)other * s);
}
// A pair (x, y) turned.
__device__ __forceinline__ void turn_pair(float& x, float& y, double2 t) {
    const float a = x;
    x = turn_value(a, y, t.x, -t.y);
    y = turn_value(y, a, t.x, t.y);
}

namespace host {

inline int rotary_args(const rta_rotary* r, RotaryArgs* a) {
    if (!r || !r->turns) return RTA_ERR_NULL;
    if (r->head_dim <= 0 || r->dims <= 0 || r->dims % 2 || r->dims > r->head_dim) return RTA_ERR_SHAPE;
    if ((r->layout != RTA_ROTARY_NEIGHBOURS && r->layout != RTA_ROTARY_HALVES) || r->head_dim > 512 ||
        !(fabs(r->amplitude) < INFINITY))
        return RTA_ERR_RANGE;
    if (!aligned(r->turns, 8)) return RTA_ERR_ALIGN;
    *a = RotaryArgs{r->turns, r->amplitude, r->dims};
    return RTA_OK;
}

}  // namespace host
}  // namespace rta
