// rta_sample.hip -- the next token of rows of logits: temperature, top-k, top-p, min-p and a given uniform
// number (gfx950).
//
// The order of a row's words is by logit, largest first, equals by index; every rule keeps the first so
// many of them, so all of them together keep the words up to one place in that order.  Two kernels:
//   1. a workgroup per chunk of kChunk words reads the logits once and leaves the chunk's maximum and, by
//      bins of 1/8 octave of weight below it, counts and sums of weights;
//   2. a workgroup per row joins the bins, finds each rule's bin, ranks the words of that bin alone (read
//      again, from the caches, into LDS) by a radix search, and draws.
// A weight is 2^(y - y of the largest), y = logit log2(e) / temperature in fp64, as a whole number of 2^-50
// (fewer bits where more words than kChunk are summed): sums of whole numbers do not depend on the order of
// their atomics, and those of equal logits are exact.  Words below 2^-47 of the largest count as none.
#include <limits.h>
#include <math.h>

#include "rta_common.hpp"
#include "rta_host.hpp"

namespace rta {

constexpr int kChunk = 8192, kChunkThreads = 512, kPerThread = kChunk / kChunkThreads;
constexpr int kBins = 384;         // 48 octaves; the last one holds everything below, and is not kept
constexpr int kBits = 50;          // kChunk weights of up to 2^50 stay below 2^64
constexpr int kRowThreads = 1024, kMostChunks = 2048;
constexpr int kList = 8192;        // words ranked in LDS
constexpr uint32_t kNoToken = 0xffffffffu;

struct ChunkHead {
    double top;       // floor(8 y) of the largest
    float max;
    uint32_t arg;     // its first word
    uint32_t bad;     // a NaN or +inf
    uint32_t pad[3];
};

struct SampleArgs {
    const float* logits;
    int64_t stride;
    int rows, vocab, nchunk;
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    const float* u;
    uint32_t* ids;
    float* probs;
    ChunkHead* head;    // [rows][nchunk]
    uint64_t* mass;     // [rows][nchunk][kBins]
    uint32_t* count;    // [rows][nchunk][kBins]
};

// log2(e) / temperature; a temperature that is not above 0 means the largest (no scale).
__device__ __forceinline__ double word_scale(const SampleArgs& a, int row) {
    const float t = a.temperature ? a.temperature[row] : 1.0f;
    return t > 0.0f ? 1.4426950408889634 / (double)t : -1.0;
}

// y of a logit, rounded by itself: in one fma with the difference from the largest's, equal logits would
// differ by the product's rounding.
__device__ __forceinline__ double scaled(float v, double scale) {
#pragma clang fp contract(off)
    return (double)v * scale;
}

// 2^t for t <= 0, by 2^n times the series of e^(f ln 2), |f| <= 1/2, to the 11th power: 6e-15 left out.
__device__ __forceinline__ double exp2_below(double t) {
    const double n = rint(t), f = (t - n) * 0.6931471805599453;
    double p = 1.0 / 39916800.0;
    p = fma(p, f, 1.0 / 3628800.0);
    p = fma(p, f, 1.0 / 362880.0);
    p = fma(p, f, 1.0 / 40320.0);
    p = fma(p, f, 1.0 / 5040.0);
    p = fma(p, f, 1.0 / 720.0);
    p = fma(p, f, 1.0 / 120.0);
    p = fma(p, f, 1.0 / 24.0);
    p = fma(p, f, 1.0 / 6.0);
    p = fma(p, f, 0.5);
    p = fma(p, f, 1.0);
    p = fma(p, f, 1.0);
    return ldexp(p, n < -1000.0 ? -1000 : (int)n);
}

// A weight of at most 1 as a whole number of 2^-bits, rounded to nearest (bits <= 51): the last bits of 2^52 + w 2^bits.
__device__ __forceinline__ uint64_t whole(double w, int bits) {
    return __builtin_bit_cast(uint64_t, ldexp(w, bits) + 4503599627370496.0) & 0xfffffffffffffull;
}

// Words in order as ascending 64-bit numbers: logit (largest first; -0 is 0), then index.
__device__ __forceinline__ uint64_t word_order(float x, uint32_t i) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    const uint32_t up = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (uint64_t)~up << 32 | i;
}
__device__ __forceinline__ float word_logit(uint64_t order) {
    const uint32_t up = ~(uint32_t)(order >> 32);
    return __builtin_bit_cast(float, up & 0x80000000u ? up & 0x7fffffffu : ~up);
}

typedef f4_t f4w_t __attribute__((aligned(4)));

// Four logits from word i on, -inf past the end.
__device__ __forceinline__ f4_t load_words(const float* __restrict__ x, int i, int vocab) {
    if (i + 4 <= vocab) return *reinterpret_cast<const f4w_t*>(x + i);
    f4_t v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = i + e < vocab ? x[i + e] : -INFINITY;
    return v;
}

// Bound by the logits' bytes, and for many rows by some 25 fp64 instructions a word beside them.
__global__ void __launch_bounds__(kChunkThreads) sample_chunk_kernel(const SampleArgs a) {
    __shared__ unsigned long long mass[kBins];
    __shared__ uint32_t count[kBins];
    __shared__ float wave_max[kChunkThreads / kWave];
    __shared__ uint32_t first, bad;
    const int row = blockIdx.x / a.nchunk, chunk = blockIdx.x - row * a.nchunk, tid = threadIdx.x;
    const float* x = a.logits + row * a.stride;
    f4_t v[kPerThread / 4];
#pragma unroll
    for (int j = 0; j < kPerThread / 4; ++j) v[j] = load_words(x, chunk * kChunk + 4 * (tid + kChunkThreads * j), a.vocab);
    for (int b = tid; b < kBins; b += kChunkThreads) {
        mass[b] = 0;
        count[b] = 0;
    }
    if (tid == 0) {
        first = kNoToken;
        bad = 0;
    }
    float m = -INFINITY;
    bool odd = false;
#pragma unroll
    for (int j = 0; j < kPerThread / 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            m = fmaxf(m, v[j][e]);
            odd |= !(v[j][e] < INFINITY);
        }
    m = wave_max_dpp(m);
    if ((tid & 63) == 0) wave_max[tid >> 6] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kChunkThreads / kWave; ++w) m = fmaxf(m, wave_max[w]);
    if (odd) bad = 1;
    uint32_t at = kNoToken;
#pragma unroll
    for (int j = kPerThread / 4 - 1; j >= 0; --j)
#pragma unroll
        for (int e = 3; e >= 0; --e)
            if (v[j][e] == m) at = chunk * kChunk + 4 * (tid + kChunkThreads * j) + e;
    if (at != kNoToken && m > -INFINITY) atomicMin(&first, at);
    const double scale = word_scale(a, row);
    const double ym = m > -INFINITY ? scaled(m, scale) : 0.0, top = floor(8.0 * ym);
    if (scale >= 0.0 && m < INFINITY) {
#pragma unroll
        for (int j = 0; j < kPerThread / 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (!(v[j][e] > -INFINITY)) continue;
                const double y = scaled(v[j][e], scale), below = top - floor(8.0 * y);
                if (!(below < kBins - 1)) continue;
                atomicAdd(&mass[(int)below], (unsigned long long)whole(exp2_below(y - ym), kBits));
                atomicAdd(&count[(int)below], 1u);
            }
    }
    __syncthreads();
    if (tid == 0) a.head[blockIdx.x] = ChunkHead{top, m, first, bad, {0, 0, 0}};
    if (scale < 0.0) return;
    for (int b = tid; b < kBins; b += kChunkThreads) {
        a.mass[(int64_t)blockIdx.x * kBins + b] = mass[b];
        a.count[(int64_t)blockIdx.x * kBins + b] = count[b];
    }
}

// Where the words that count end: those of the bins below `bin`, and of `bin` those up to `order`.
struct Cut {
    int bin;
    uint64_t order;
};
__device__ __forceinline__ Cut earlier(Cut a, Cut b) {
    return a.bin < b.bin || (a.bin == b.bin && a.order < b.order) ? a : b;
}

struct RowLds {
    unsigned long long list[kList];
    double chunk_mass[kMostChunks], chunk_scale[kMostChunks];
    unsigned long long chunk_part[kMostChunks];   // of it, the words of the cut's own bin
    int chunk_shift[kMostChunks];
    double mass[kBins], half_mass[kBins];     // of a bin, then of all up to it
    uint32_t count[kBins], half_count[kBins];
    unsigned long long digit_mass[256];
    uint32_t digit_count[256];
    unsigned long long lo, hi, sum, before_mass;
    uint32_t n, before_count, digit, found;
    double red[kRowThreads / kWave];
    float fred[kRowThreads / kWave];
};

// One row's search, by all threads of its workgroup.
struct RowSearch {
    const SampleArgs& a;
    RowLds& l;
    const float* x;
    double scale, ym, top;   // y of the largest and floor(8 y)
    int list_lo, list_hi;   // the bins whose words are in the list (none: lo > hi)
    int list_n;

    __device__ __forceinline__ double bin_of(float v) const { return top - floor(8.0 * scaled(v, scale)); }
    __device__ __forceinline__ double weight(float v) const { return exp2_below(scaled(v, scale) - ym); }
    __device__ __forceinline__ bool inside(uint64_t order, int bin, const Cut& c) const {
        return bin < c.bin || (bin == c.bin && order <= c.order);
    }

    // f(order, bin) of the row's words in bins lo .. hi, each by one thread, in any order.
    template <class F>
    __device__ __forceinline__ void scan(int lo, int hi, F&& f) const {
        // a range of logits that holds the bins', with room for the roundings: what is outside needs no fp64
        const double step = 8.0 * scale;
        const double first = (top - hi) / step, last = (top - lo + 1.0) / step;
        const bool wide = !(step > 0.0);
        const float from = wide ? -INFINITY : (float)(first - fabs(first) * 1e-6 - 1e-30);
        const float to = wide ? INFINITY : (float)(last + fabs(last) * 1e-6 + 1e-30);
        constexpr int kAtOnce = 4;
        for (int i = 4 * threadIdx.x; i < a.vocab; i += 4 * kAtOnce * kRowThreads) {
            f4_t v[kAtOnce];
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) v[j] = load_words(x, min(i + 4 * kRowThreads * j, a.vocab), a.vocab);
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float t = v[j][e];
                    if (t < from || t > to || t == -INFINITY) continue;
                    const double b = bin_of(t);
                    if (b >= lo && b <= hi) f(word_order(t, i + 4 * kRowThreads * j + e), (int)b);
                }
        }
    }
    // The same from the list where it has them.
    template <class F>
    __device__ __forceinline__ void each(int lo, int hi, F&& f) const {
        if (list_lo <= lo && hi <= list_hi) {
            for (int i = threadIdx.x; i < list_n; i += kRowThreads) {
                const uint64_t order = l.list[i];
                const int b = (int)bin_of(word_logit(order));
                if (b >= lo && b <= hi) f(order, b);
            }
        } else {
            scan(lo, hi, f);
        }
    }
    // Puts the words of bin b into the list, with all before it if they fit.
    __device__ void want(int b) {
        if (list_lo <= b && b <= list_hi) return;
        const uint32_t upto = l.count[b], own = upto - (b ? l.count[b - 1] : 0);
        if (own > kList) return;
        const int lo = upto <= kList ? 0 : b;
        __syncthreads();
        if (threadIdx.x == 0) l.n = 0;
        __syncthreads();
        scan(lo, b, [&](uint64_t order, int) {
            const uint32_t at = atomicAdd(&l.n, 1u);
            if (at < kList) l.list[at] = order;
        });
        __syncthreads();
        list_lo = lo;
        list_hi = b;
        list_n = min((int)l.n, kList);
    }

    // The first word, by key(order), of those of bins lo .. hi that keep(order, bin) takes at which, with the
    // words before it, there are `words` of them (by count), or their weights reach `target` 2^-bits; the last
    // one where none does.  before: weights of those in front.  Radix search, 8 bits a pass, over the bits in which
    // the keys differ.
    template <bool COUNT, class K, class P>
    __device__ uint64_t search(int lo, int hi, K&& key, P&& keep, uint32_t words, uint64_t target, int bits, uint64_t& before) {
        __syncthreads();
        if (threadIdx.x == 0) {
            l.lo = ~0ull;
            l.hi = 0;
        }
        __syncthreads();
        uint64_t least = ~0ull, most = 0;
        each(lo, hi, [&](uint64_t order, int b) {
            if (!keep(order, b)) return;
            const uint64_t k = key(order);
            least = k < least ? k : least;
            most = k > most ? k : most;
        });
        // (one atomic a wave: those of all lanes on one place would follow each other)
        for (int o = 32; o > 0; o >>= 1) {
            const uint64_t t = __shfl_xor((unsigned long long)least, o, kWave), u = __shfl_xor((unsigned long long)most, o, kWave);
            least = t < least ? t : least;
            most = u > most ? u : most;
        }
        if ((threadIdx.x & 63) == 0) {
            atomicMin(&l.lo, (unsigned long long)least);
            atomicMax(&l.hi, (unsigned long long)most);
        }
        __syncthreads();
        uint64_t value = l.lo;   // the bits that are known, and zeros
        const uint64_t differ = l.lo ^ l.hi;
        before = 0;
        uint32_t before_n = 0;
        if (!differ) return value;
        int end = 64 - __clzll((long long)differ);   // bits not known yet
        value = end == 64 ? 0 : value >> end << end;
        while (end > 0) {
            const int shift = end > 8 ? end - 8 : 0;
            const uint64_t known = end == 64 ? 0 : ~0ull << end;
            const uint32_t mask = (1u << (end - shift)) - 1;
            __syncthreads();
            if (threadIdx.x < 256) {
                l.digit_mass[threadIdx.x] = 0;
                l.digit_count[threadIdx.x] = 0;
            }
            __syncthreads();
            each(lo, hi, [&](uint64_t order, int b) {
                if (!keep(order, b)) return;
                const uint64_t k = key(order);
                if ((k & known) != value) return;
                const uint32_t d = (uint32_t)(k >> shift) & mask;
                atomicAdd(&l.digit_count[d], 1u);
                atomicAdd(&l.digit_mass[d], (unsigned long long)whole(weight(word_logit(order)), bits));
            });
            __syncthreads();
            if (threadIdx.x < kWave) {   // four digits a lane
                uint32_t c[4], cs = 0;
                uint64_t w[4], ws = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    c[e] = l.digit_count[4 * threadIdx.x + e];
                    w[e] = l.digit_mass[4 * threadIdx.x + e];
                    cs += c[e];
                    ws += w[e];
                }
                uint32_t ci = cs;
                uint64_t wi = ws;
                for (int o = 1; o < kWave; o <<= 1) {
                    const uint32_t t = __shfl_up(ci, o, kWave);
                    const uint64_t s = __shfl_up((unsigned long long)wi, o, kWave);
                    if ((int)threadIdx.x >= o) {
                        ci += t;
                        wi += s;
                    }
                }
                uint32_t cb = before_n + ci - cs;
                uint64_t wb = before + wi - ws;
                int hit = -1, last = -1;
                uint32_t hit_c = 0, last_c = 0;
                uint64_t hit_w = 0, last_w = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (c[e]) {
                        last = e;
                        last_c = cb;
                        last_w = wb;
                        if (hit < 0 && (COUNT ? cb + c[e] >= words : wb + w[e] >= target)) {
                            hit = e;
                            hit_c = cb;
                            hit_w = wb;
                        }
                    }
                    cb += c[e];
                    wb += w[e];
                }
                const uint64_t hits = __builtin_amdgcn_ballot_w64(hit >= 0), any = __builtin_amdgcn_ballot_w64(last >= 0);
                const int lane = hits ? __builtin_ctzll(hits) : 63 - __builtin_clzll(any);
                if ((int)threadIdx.x == lane) {
                    const bool h = hits != 0;
                    l.digit = 4 * lane + (h ? hit : last);
                    l.before_count = h ? hit_c : last_c;
                    l.before_mass = h ? hit_w : last_w;
                    l.found = c[h ? hit : last];
                }
            }
            __syncthreads();
            before = l.before_mass;
            before_n = l.before_count;
            value |= (uint64_t)l.digit << shift;
            end = shift;
            if (l.found == 1 && end > 0) {   // the one that is left
                const uint64_t rest = ~0ull << end;
                each(lo, hi, [&](uint64_t order, int b) {
                    if (!keep(order, b)) return;
                    const uint64_t k = key(order);
                    if ((k & rest) == value) l.lo = k;
                });
                __syncthreads();
                return l.lo;
            }
        }
        return value;
    }
};

// Sums of v over the workgroup's first kBins threads up to each of them (all threads call it).
template <class T>
__device__ __forceinline__ void scan_bins(T* v, T* wave_sum) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    T sum = t < kBins ? v[t] : T(0);
    for (int o = 1; o < kWave; o <<= 1) {
        const T add = __shfl_up(sum, o, kWave);
        if (lane >= o) sum += add;
    }
    if (lane == kWave - 1) wave_sum[wave] = sum;
    __syncthreads();
    T before = T(0);
    for (int w = 0; w < wave; ++w) before += wave_sum[w];
    if (t < kBins) v[t] = before + sum;
    __syncthreads();
}

__global__ void __launch_bounds__(kRowThreads) sample_row_kernel(const SampleArgs a) {
    __shared__ RowLds l;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const ChunkHead* head = a.head + (int64_t)row * a.nchunk;
    const double scale = word_scale(a, row);
    // the row's maximum, its first word and whether all is well
    float m = -INFINITY;
    bool bad = false;
    for (int c = tid; c < a.nchunk; c += kRowThreads) {
        m = fmaxf(m, head[c].max);
        bad |= head[c].bad != 0;
    }
    m = wave_max_dpp(m);
    if (lane == 0) l.fred[wave] = m;
    if (tid == 0) l.found = kNoToken;
    const bool any_bad = __syncthreads_or(bad);
#pragma unroll
    for (int w = 0; w < kRowThreads / kWave; ++w) m = fmaxf(m, l.fred[w]);
    if (any_bad || !(m > -INFINITY)) {
        if (tid == 0) {
            a.ids[row] = kNoToken;
            if (a.probs) a.probs[row] = 0.0f;
            raise_error(RTA_DEVERR_DETECTOR);
        }
        return;
    }
    if (scale < 0.0) {   // the largest
        for (int c = tid; c < a.nchunk; c += kRowThreads)
            if (head[c].max == m) atomicMin(&l.found, head[c].arg);
        __syncthreads();
        if (tid == 0) {
            a.ids[row] = l.found;
            if (a.probs) a.probs[row] = 1.0f;
        }
        return;
    }
    const double ym = scaled(m, scale), top = floor(8.0 * ym);
    RowSearch s{a, l, a.logits + row * a.stride, scale, ym, top, 1, 0, 0};
    // how far a chunk's bins and largest weight lie below the row's
    for (int c = tid; c < a.nchunk; c += kRowThreads) {
        const bool some = head[c].max > -INFINITY;
        const double down = top - head[c].top;
        l.chunk_shift[c] = some && down < kBins ? (int)down : kBins;
        l.chunk_scale[c] = some ? ldexp(s.weight(head[c].max), -kBits) : 0.0;
    }
    __syncthreads();
    // the row's bins: two threads each, every other chunk
    const uint64_t* cm = a.mass + (int64_t)row * a.nchunk * kBins;
    const uint32_t* cc = a.count + (int64_t)row * a.nchunk * kBins;
    if (tid < 2 * kBins) {
        const int half = tid >= kBins, b = tid - half * kBins;
        double w = 0.0;
        uint32_t n = 0;
        if (b < kBins - 1) {
#pragma unroll 4
            for (int c = half; c < a.nchunk; c += 2) {
                const int from = b - l.chunk_shift[c];
                const int64_t at = (int64_t)c * kBins + max(from, 0);
                const uint64_t cw = cm[at];
                const uint32_t cn = cc[at];
                if (from >= 0) {
                    w += (double)cw * l.chunk_scale[c];
                    n += cn;
                }
            }
        }
        (half ? l.half_mass : l.mass)[b] = w;
        (half ? l.half_count : l.count)[b] = n;
    }
    __syncthreads();
    if (tid < kBins) {
        l.mass[tid] += l.half_mass[tid];
        l.count[tid] += l.half_count[tid];
    }
    __syncthreads();
    scan_bins(l.mass, l.red);
    scan_bins(l.count, l.digit_count);
    // the first bin up to which pred holds (kBins - 1: none)
    auto first_bin = [&](auto pred) {
        __syncthreads();
        if (tid == 0) l.found = kBins - 1;
        __syncthreads();
        if (tid < kBins - 1 && pred(tid)) atomicMin(&l.found, (uint32_t)tid);
        __syncthreads();
        return (int)l.found;
    };
    // bits of a weight where so many are summed
    auto bits_for = [](uint32_t n) { return min(kBits, 62 - (32 - __clz((int)(n | 1u)))); };
    auto order_key = [](uint64_t order) { return order; };
    Cut cut{kBins - 2, ~0ull};
    double total = l.mass[kBins - 2];

    // top-k: the first k words
    const int k = a.top_k ? a.top_k[row] : 0;
    if (k > 0) {
        const int b = first_bin([&](int t) { return l.count[t] >= (uint32_t)k; });
        if (b < kBins - 1) {
            const uint32_t in_front = b ? l.count[b - 1] : 0;
            s.want(b);
            uint64_t before;
            const int bits = bits_for(l.count[b] - in_front);
            const uint64_t at =
                s.search<true>(b, b, order_key, [](uint64_t, int) { return true; }, (uint32_t)k - in_front, 0, bits, before);
            cut = Cut{b, at};
            total = (b ? l.mass[b - 1] : 0.0) + ldexp((double)before, -bits) + s.weight(word_logit(at));
        }
    }
    // top-p: the fewest of those that hold p of their weight
    const double p = a.top_p ? (double)a.top_p[row] : 1.0;
    if (p < 1.0) {
        const double goal = p * total;
        const int b = min(first_bin([&](int t) { return l.mass[t] >= goal; }), cut.bin);
        s.want(b);
        const double in_front = b ? l.mass[b - 1] : 0.0;
        const int bits = bits_for(l.count[b] - (b ? l.count[b - 1] : 0));
        const uint64_t target = goal > in_front ? (uint64_t)ceil(ldexp(goal - in_front, bits)) : 0;
        uint64_t before;
        const uint64_t at =
            s.search<false>(b, b, order_key, [&](uint64_t order, int bin) { return s.inside(order, bin, cut); }, 0, target, bits, before);
        cut = earlier(cut, Cut{b, at});
    }
    // min-p: those of at least min_p of the largest weight, the largest among them
    const double least = a.min_p ? (double)a.min_p[row] : 0.0;
    if (least > 0.0) {
        const double down = top - floor(8.0 * (ym + log2(fmin(least, 1.0))));
        if (down <= cut.bin) {
            const int b = (int)down;
            s.want(b);
            __syncthreads();
            if (tid == 0) l.hi = 0;
            __syncthreads();
            s.each(b, b, [&](uint64_t order, int) {
                if (s.weight(word_logit(order)) >= fmin(least, 1.0)) atomicMax(&l.hi, (unsigned long long)order);
            });
            __syncthreads();
            cut = earlier(cut, Cut{b, l.hi});
        }
    }
    if (least > 1.0) {   // the first of the order alone
        s.want(0);
        uint64_t before;
        cut = Cut{0, s.search<true>(0, 0, order_key, [](uint64_t, int) { return true; }, 1, 0, kBits - 11, before)};
    }

    // draw
    const float given = a.u[row];
    const double u = given > 0.0f ? fmin((double)given, 1.0) : 0.0;
    if (s.list_lo == 0 && cut.bin <= s.list_hi) {
        // every word that counts is in the list
        auto keep = [&](uint64_t order, int bin) { return s.inside(order, bin, cut); };
        __syncthreads();
        if (tid == 0) l.sum = 0;
        __syncthreads();
        uint64_t own = 0;
        s.each(0, cut.bin, [&](uint64_t order, int bin) {
            if (keep(order, bin)) own += whole(s.weight(word_logit(order)), kBits);
        });
        for (int o = 32; o > 0; o >>= 1) own += __shfl_xor((unsigned long long)own, o, kWave);
        if (lane == 0) atomicAdd(&l.sum, (unsigned long long)own);
        __syncthreads();
        const uint64_t sum = l.sum;
        const uint64_t goal = (uint64_t)fmin(u * (double)sum, 18446744073709549568.0);
        uint64_t before;
        const uint64_t id = s.search<false>(0, cut.bin, [](uint64_t order) { return order & 0xffffffffull; }, keep, 0,
                                            (goal < sum ? goal : sum - 1) + 1, kBits, before);
        if (tid == 0) {
            a.ids[row] = (uint32_t)id;
            if (a.probs) a.probs[row] = (float)(s.weight(s.x[id]) / ldexp((double)sum, -kBits));
        }
        return;
    }
    // what each chunk holds: its bins below the cut's, and the words of that bin one by one
    const bool whole_bin = cut.order == ~0ull;
    const int bins = cut.bin + (whole_bin ? 1 : 0);
    for (int c = wave; c < a.nchunk; c += kRowThreads / kWave) {
        const int n = bins - l.chunk_shift[c];
        double w = 0.0;
        for (int b = lane; b < n; b += kWave) w += (double)cm[(int64_t)c * kBins + b];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) w += __shfl_xor(w, o, kWave);
        if (lane == 0) l.chunk_mass[c] = w * l.chunk_scale[c];
    }
    if (!whole_bin) {
        for (int c = tid; c < a.nchunk; c += kRowThreads) l.chunk_part[c] = 0;
        __syncthreads();
        s.each(cut.bin, cut.bin, [&](uint64_t order, int) {
            if (order <= cut.order)
                atomicAdd(&l.chunk_part[(uint32_t)order / kChunk], (unsigned long long)whole(s.weight(word_logit(order)), kBits));
        });
        __syncthreads();
        for (int c = tid; c < a.nchunk; c += kRowThreads) l.chunk_mass[c] += ldexp((double)l.chunk_part[c], -kBits);
    }
    __syncthreads();
    // the chunk of the word: sums in the chunks' order, 64 at a time, by one wave
    if (wave == 0) {
        double sum = 0.0;
        for (int pass = 0; pass < 2; ++pass) {
            const double goal = u * sum;   // (the second time)
            double run = 0.0, base = 0.0;
            int at = -1, last = 0;
            double last_base = 0.0;
            for (int c0 = 0; c0 < a.nchunk; c0 += kWave) {
                const double w = c0 + lane < a.nchunk ? l.chunk_mass[c0 + lane] : 0.0;
                double upto = w;
                for (int o = 1; o < kWave; o <<= 1) {
                    const double t = __shfl_up(upto, o, kWave);
                    if (lane >= o) upto += t;
                }
                if (pass == 1) {
                    const uint64_t hit = __builtin_amdgcn_ballot_w64(w > 0.0 && run + upto > goal);
                    const uint64_t any = __builtin_amdgcn_ballot_w64(w > 0.0);
                    if (any) {
                        const int e = 63 - __builtin_clzll(any);
                        last = c0 + e;
                        last_base = run + __shfl(upto - w, e, kWave);
                    }
                    if (hit) {
                        const int e = __builtin_ctzll(hit);
                        at = c0 + e;
                        base = run + __shfl(upto - w, e, kWave);
                        break;
                    }
                }
                run += __shfl(upto, kWave - 1, kWave);
            }
            if (pass == 0) {
                sum = run;
            } else if (lane == 0) {
                l.found = at >= 0 ? at : last;
                l.red[0] = goal - (at >= 0 ? base : last_base);
                l.red[1] = sum;
            }
        }
    }
    __syncthreads();
    // the word of the chunk: a thread sums kChunk / kRowThreads of them that follow each other
    constexpr int kEach = kChunk / kRowThreads;
    const int first = (int)l.found * kChunk + kEach * tid;
    const double rest = l.red[0], sum = l.red[1];
    uint64_t w[kEach], own = 0;
#pragma unroll
    for (int j = 0; j < kEach; j += 4) {
        const f4_t v = load_words(s.x, min(first + j, a.vocab), a.vocab);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            w[j + e] = 0;
            if (v[e] > -INFINITY) {
                const double b = s.bin_of(v[e]);
                if (b < kBins - 1 && s.inside(word_order(v[e], first + j + e), (int)b, cut)) w[j + e] = whole(s.weight(v[e]), kBits);
            }
            own += w[j + e];
        }
    }
    uint64_t upto = own;
    for (int o = 1; o < kWave; o <<= 1) {
        const uint64_t t = __shfl_up((unsigned long long)upto, o, kWave);
        if (lane >= o) upto += t;
    }
    __syncthreads();
    unsigned long long* wave_sum = l.digit_mass;
    if (lane == kWave - 1) wave_sum[wave] = upto;
    if (tid == 0) {
        l.lo = ~0ull;   // the first word past the goal
        l.hi = 0;       // the last one with a weight, plus one
    }
    __syncthreads();
    for (int v = 0; v < wave; ++v) upto += wave_sum[v];
    const uint64_t goal = rest > 0.0 ? (uint64_t)ldexp(rest, kBits) : 0;
    uint64_t run = upto - own;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        run += w[j];
        if (w[j] && run > goal && run - w[j] <= goal) atomicMin(&l.lo, (unsigned long long)(first + j));
        if (w[j]) atomicMax(&l.hi, (unsigned long long)(first + j + 1));
    }
    __syncthreads();
    if (tid == 0) {
        const uint32_t id = l.lo != ~0ull ? (uint32_t)l.lo : (uint32_t)l.hi - 1;
        a.ids[row] = id;
        if (a.probs) a.probs[row] = (float)(s.weight(s.x[id]) / sum);
    }
}

static size_t sample_bytes(int64_t rows, int64_t nchunk) {
    return (size_t)(rows * nchunk) * (sizeof(ChunkHead) + kBins * 12);
}

}  // namespace rta

using namespace rta;

extern "C" {

size_t rta_sample_workspace_bytes(int rows, int vocab) {
    if (rows <= 0 || vocab <= 0 || vocab > kMostChunks * kChunk) return 0;
    return sample_bytes(rows, (vocab + kChunk - 1) / kChunk);
}

int rta_sample(const float* logits, int64_t stride, int rows, int vocab, const float* temperature, const int32_t* top_k,
               const float* top_p, const float* min_p, const float* u, uint32_t* ids, float* probs, void* workspace,
               size_t workspace_bytes, rta_stream_t stream) {
    if (!logits || !u || !ids) return RTA_ERR_NULL;
    if (rows <= 0 || vocab <= 0 || (stride < vocab && stride != 0)) return RTA_ERR_SHAPE;
    if (vocab > kMostChunks * kChunk) return RTA_ERR_RANGE;
    SampleArgs a{};
    a.nchunk = (vocab + kChunk - 1) / kChunk;
    if ((int64_t)rows * a.nchunk >= 1 << 22) return RTA_ERR_RANGE;   // (grids of fewer than 2^32 threads)
    if (!host::aligned(logits, 4) || !host::aligned(temperature, 4) || !host::aligned(top_k, 4) || !host::aligned(top_p, 4) ||
        !host::aligned(min_p, 4) || !host::aligned(u, 4) || !host::aligned(ids, 4) || !host::aligned(probs, 4))
        return RTA_ERR_ALIGN;
    if (!workspace || workspace_bytes < sample_bytes(rows, a.nchunk) || !host::aligned(workspace, 16)) return RTA_ERR_WORKSPACE;
    a.logits = logits;
    a.stride = stride;
    a.rows = rows;
    a.vocab = vocab;
    a.temperature = temperature;
    a.top_k = top_k;
    a.top_p = top_p;
    a.min_p = min_p;
    a.u = u;
    a.ids = ids;
    a.probs = probs;
    const int64_t chunks = (int64_t)rows * a.nchunk;
    a.head = static_cast<ChunkHead*>(workspace);
    a.mass = reinterpret_cast<uint64_t*>(a.head + chunks);
    a.count = reinterpret_cast<uint32_t*>(a.mass + chunks * kBins);
    hipStream_t s = (hipStream_t)stream;
    hipLaunchKernelGGL(sample_chunk_kernel, dim3(chunks), dim3(kChunkThreads), 0, s, a);
    hipLaunchKernelGGL(sample_row_kernel, dim3(rows), dim3(kRowThreads), 0, s, a);
    return hipGetLastError() == hipSuccess ? RTA_OK : RTA_ERR_LAUNCH;
}

}  // extern "C"
