// rta_rotary.hip -- rotary positions: frequencies as trained or scaled for longer contexts, and rows of
// heads turned to their positions (gfx950).
#include "rta_rotary.hpp"

namespace rta {

struct RotateArgs {
    RotaryArgs r;
    const float* x;
    float* y;
    int64_t x_stride, y_stride;
    const int64_t* positions;
    int heads, head_dim;
    int units;       // threads of a head: dims / (2 V) with pairs, then its last values, 2 V each
    int per_block;   // heads of a workgroup
};

// Bound by the bytes: a value is read and written once.  A workgroup takes one row; a thread V pairs of each of
// its heads (V 4 where the pairs come in fours: 16-byte accesses), whose angles it computes once, kAtOnce heads on
// their way together (8192 rows of 40 heads, 64 of 128 dims: 60 us, 5.6 TB/s; one head after the other, and values
// that stay one by one: 144).
template <int V, int LAYOUT>
__global__ void __launch_bounds__(256) rotate_kernel(const RotateArgs a) {
    constexpr int kAtOnce = 4;
    const int row = blockIdx.x, at_once = 256 / a.units;
    const int h0 = threadIdx.x / a.units, unit = threadIdx.x - h0 * a.units;
    if (h0 >= at_once) return;
    const int half = a.r.dims / 2, j = unit * V;
    const bool turns = j < half;
    // its values: neighbours 2 V from 2 j on; halves V from j and V from j + half on; those that stay 2 V from 2 j
    // on (half is a multiple of V), as far as the head goes
    const bool split = LAYOUT == RTA_ROTARY_HALVES && turns;
    const int lo = split ? j : 2 * j, hi = split ? j + half : 2 * j + V;
    const int part = turns ? 2 * V : min(2 * V, a.head_dim - lo);   // (below 2 V: the last values of a head)
    const bool copies = a.x != a.y;
    if (!turns && !copies) return;
    const int first = blockIdx.y * a.per_block + h0, last = min((int)(blockIdx.y + 1) * a.per_block, a.heads);
    const float* x = a.x + row * a.x_stride;
    float* y = a.y + row * a.y_stride;
    typedef float vec_t __attribute__((ext_vector_type(V), aligned(4)));
    double2 t[V] = {};
    if (turns) {
        const double position = (double)a.positions[row];
#pragma unroll
        for (int e = 0; e < V; ++e) t[e] = turn_of(position, a.r.turns[j + e], a.r.amplitude);
    }
    if (part < 2 * V) {
        for (int h = first; h < last; h += at_once)
            for (int e = 0; e < part; ++e) y[(int64_t)h * a.head_dim + lo + e] = x[(int64_t)h * a.head_dim + lo + e];
        return;
    }
    for (int h = first; h < last; h += kAtOnce * at_once) {
        float v[kAtOnce][2 * V];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const float* src = x + (int64_t)min(h + i * at_once, last - 1) * a.head_dim;
            *reinterpret_cast<vec_t*>(v[i]) = *reinterpret_cast<const vec_t*>(src + lo);
            *reinterpret_cast<vec_t*>(v[i] + V) = *reinterpret_cast<const vec_t*>(src + hi);
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            if (h + i * at_once >= last) break;
            if (turns) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    if constexpr (LAYOUT == RTA_ROTARY_NEIGHBOURS) turn_pair(v[i][2 * e], v[i][2 * e + 1], t[e]);
                    else turn_pair(v[i][e], v[i][V + e], t[e]);
                }
            }
            float* dst = y + (int64_t)(h + i * at_once) * a.head_dim;
            *reinterpret_cast<vec_t*>(dst + lo) = *reinterpret_cast<const vec_t*>(v[i]);
            *reinterpret_cast<vec_t*>(dst + hi) = *reinterpret_cast<const vec_t*>(v[i] + V);
        }
    }
}

}  // namespace rta

using namespace rta;

extern "C" {

int rta_rotary_turns(int dims, double theta, int scaling, double factor, double original, double low, double high,
                     double* turns, double* amplitude) {
    if (!turns) return RTA_ERR_NULL;
    if (dims <= 0 || dims % 2) return RTA_ERR_SHAPE;
    const bool bounded = scaling == RTA_ROTARY_RAMP || scaling == RTA_ROTARY_BANDS;
    if (scaling < RTA_ROTARY_PLAIN || scaling > RTA_ROTARY_BANDS || !(theta > 0.0) || !(theta < INFINITY) ||
        (scaling != RTA_ROTARY_PLAIN && (!(factor > 0.0) || !(factor < INFINITY))) ||
        (bounded && (!(original > 0.0) || !(original < INFINITY) || !(low > 0.0) || !(high > low) || !(high < INFINITY))) ||
        (scaling == RTA_ROTARY_RAMP && !(theta > 1.0)))
        return RTA_ERR_RANGE;
    const int half = dims / 2;
    const double kTau = 6.283185307179586;
    if (scaling == RTA_ROTARY_BASE && half > 1) theta *= pow(factor, (double)half / (half - 1));
    double first = 0.0, last = 1.0;
    if (scaling == RTA_ROTARY_RAMP) {   // the pairs that make `high` and `low` turns over the original length
        const double per = half / log(theta);
        first = fmax(floor(per * log(original / (kTau * high))), 0.0);
        last = fmax(fmin(ceil(per * log(original / (kTau * low))), dims - 1.0), first + 0.001);
    }
    for (int j = 0; j < half; ++j) {
        double f = pow(theta, -(double)j / half);
        if (scaling == RTA_ROTARY_LINEAR) f /= factor;
        if (bounded) {   // the share of a frequency that stays
            const double at = scaling == RTA_ROTARY_RAMP ? 1.0 - fmin(fmax((j - first) / (last - first), 0.0), 1.0)
                                                         : fmin(fmax((original * f / kTau - low) / (high - low), 0.0), 1.0);
            f = (1.0 - at) * f / factor + at * f;
        }
        turns[j] = f / kTau;
    }
    if (amplitude) *amplitude = scaling == RTA_ROTARY_RAMP && factor > 1.0 ? 0.1 * log(factor) + 1.0 : 1.0;
    return RTA_OK;
}

int rta_rotate(const rta_rotary* rotary, const float* x, int64_t x_stride, int rows, int heads, const int64_t* positions,
               float* y, int64_t y_stride, rta_stream_t stream) {
    RotateArgs a{};
    const int rc = host::rotary_args(rotary, &a.r);
    if (rc) return rc;
    if (!x || !y || !positions) return RTA_ERR_NULL;
    const int hd = rotary->head_dim;
    if (rows <= 0 || heads <= 0 || x_stride < (int64_t)heads * hd || y_stride < (int64_t)heads * hd) return RTA_ERR_SHAPE;
    if (rows >= 1 << 24 || heads > 65535) return RTA_ERR_RANGE;
    if (!host::aligned(x, 4) || !host::aligned(y, 4) || !host::aligned(positions, 8)) return RTA_ERR_ALIGN;
    if (x == y && x_stride != y_stride && rows > 1) return RTA_ERR_RANGE;
    a.x = x;
    a.y = y;
    a.x_stride = x_stride;
    a.y_stride = y_stride;
    a.positions = positions;
    a.heads = heads;
    a.head_dim = hd;
    const int half = a.r.dims / 2, v = half % 4 ? 1 : 4;
    a.units = half / v + (hd - a.r.dims + 2 * v - 1) / (2 * v);   // 256 at most
    // every workgroup computes its row's angles: all heads in one where there are rows enough for the chip
    const int at_once = 256 / a.units, passes = (heads + at_once - 1) / at_once;
    a.per_block = (int64_t)rows * passes <= 2048 ? at_once : heads;
    const dim3 grid(rows, (heads + a.per_block - 1) / a.per_block), block(256);
    hipStream_t s = (hipStream_t)stream;
    auto go = [&](auto vv, auto layout) {
        hipLaunchKernelGGL((rotate_kernel<decltype(vv)::value, decltype(layout)::value>), grid, block, 0, s, a);
    };
    auto by_layout = [&](auto vv) {
        if (rotary->layout == RTA_ROTARY_NEIGHBOURS) go(vv, std::integral_constant<int, RTA_ROTARY_NEIGHBOURS>{});
        else go(vv, std::integral_constant<int, RTA_ROTARY_HALVES>{});
    };
    if (v == 4) by_layout(std::integral_constant<int, 4>{});
    else by_layout(std::integral_constant<int, 1>{});
    return hipGetLastError() == hipSuccess ? RTA_OK : RTA_ERR_LAUNCH;
}

}  // extern "C"
