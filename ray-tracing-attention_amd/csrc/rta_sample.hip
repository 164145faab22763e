// rta_sample.hip -- the next token of rows of logits: temperature, top-k, top-p, min-p and a given uniform
// number (gfx950).
//
// The order of a row's words is by logit, largest first, equals by index; every rule keeps the first so
// many of them, so all of them together keep the words up to one place in that order.  Two kernels:
//   1. a workgroup per chunk of kChunk words reads the logits once and leaves the chunk's maximum and, by
//      bins of 1/8 octave of weight below it, how many words lie in the bins up to each and their weights' sums,
//      and which words (of the first bins, as far as the rules may ask for them);
//   2. a workgroup per row joins the bins, finds each rule's bin, ranks the words of that bin (or of all bins up
//      to it) in LDS by a radix search, and draws.
// A weight is 2^t, t = (logit - the largest) log2(e) / temperature in fp64, as a whole number of 2^-50
// (of one bin's words, of its own weights: as many bits as their sum has room for): sums of whole numbers do not depend on the order of
// their atomics, and those of equal logits are exact.  Words below the last bin that is
// kept, 2^-47.875 to 2^-47.75 of the largest by where in its eighth of an octave that one lies, count as none.
#include <limits.h>
#include <math.h>

#include "rta_common.hpp"
#include "rta_host.hpp"

namespace rta {

constexpr int kChunk = 8192, kChunkThreads = 512, kPerThread = kChunk / kChunkThreads;
constexpr int kBins = 384;         // 48 octaves; the last one holds everything below, and is not kept
constexpr int kBits = 50;          // kChunk weights of up to 2^50 stay below 2^64
constexpr int kRowThreads = 512, kMostChunks = 512;
constexpr int kList = 8192;        // words ranked in LDS
// Words of all bins up to one that are ranked rather than that bin's alone: then the draw needs no sums over chunks,
// but more words are gathered and searched (256 flat rows, the slowest's time: with 8192 for it 60 us, so, and with the
// places looked up together, 43).
constexpr int kFromTop = 2048;
constexpr uint32_t kNoToken = 0xffffffffu;

struct ChunkHead {
    double top;       // the largest's eighth
    float max;
    uint32_t arg;     // its first word
    uint32_t bad;     // a NaN or +inf
    uint32_t pad[3];
};

// What kernel 1 leaves of a chunk.
struct Chunk {
    ChunkHead head;
    double mass[kBins];         // weights (in 2^-kBits) of all bins up to each, against the chunk's largest
    uint16_t upto[kBins];       // and their words
    alignas(16) uint16_t place[kChunk];   // words (from the chunk's first) by bins, in any order inside one
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
    Chunk* chunks;      // [rows][nchunk]
};

// log2(e) / temperature; a temperature that is not above 0 means the largest (no scale).  An infinite one: kAlike, by
// which every finite logit's weight is 1 (the largest difference times it is 7e-212), bins keep two signs apart (the
// smallest logit times it, 1e-295, is no zero), and -inf stays -inf.
constexpr double kAlike = 1e-250;
__device__ __forceinline__ double word_scale(const SampleArgs& a, int row) {
    const float t = a.temperature ? a.temperature[row] : 1.0f;
    return t > 0.0f ? fmax(1.4426950408889634 / (double)t, kAlike) : -1.0;
}

// t, the log2 of v's weight against the largest m's.  The difference is exact but for logits 2^29 apart in size, so t is
// off by 2^-51 of itself, however large logits and scale are (of two products the difference would be off by 2^-53 of
// these).  The product is rounded by itself: in one fma with what is subtracted from it, it would differ from place to place.
__device__ __forceinline__ double distance(float v, float m, double scale) {
#pragma clang fp contract(off)
    return ((double)v - (double)m) * scale;
}
// Which eighth of an octave a logit lies in: bins are these, counted from the largest's, the same ones in every chunk.
__device__ __forceinline__ double eighth(float v, double scale) { return floor((double)v * (8.0 * scale)); }

// Weights 2^t, t <= 0: 2^n times the series of e^(f ln 2), |f| <= 1/2, to the 9th power, whose 10th and 11th are spread over the
// lower ones by Chebyshev's polynomials (Lanczos: f^10 less its share of T10(2 f) is of 8th degree; its constant is left
// out, so that the largest weighs 1).  4.7e-14 of a weight is off, 2^-44; the series as it stands would be 9.5e-12 off.  It
// moves the border between two words by less than that of all weights (and a word's rounding to a whole number by
// 2^-51 of the largest), and u falls between where a border lies and where it ought to as often.  The coefficients are kept
// in scalar registers: as literals each took two moves to the vector registers a word.
struct Exp2 {
    static constexpr int kDegree = 9;
    double c[kDegree + 1];
    __device__ __forceinline__ Exp2() {
        double f = 1.0, a[kDegree + 3];
#pragma unroll
        for (int i = 0; i < kDegree + 3; ++i) {   // ln 2^i / i!
            a[i] = f;
            f *= 0.6931471805599453 / (i + 1);
        }
#pragma unroll
        for (int i = 0; i <= kDegree; ++i) c[i] = a[i];
        // T10(x) = 512 x^10 - 1280 x^8 + 1120 x^6 - 400 x^4 + 50 x^2 - 1, x = 2 f
        const double s = a[10] / (512.0 * 1024.0);
        c[8] += s * (1280 * 256);
        c[6] -= s * (1120 * 64);
        c[4] += s * (400 * 16);
        c[2] -= s * (50 * 4);
        // T11(x) = 1024 x^11 - 2816 x^9 + 2816 x^7 - 1232 x^5 + 220 x^3 - 11 x
        const double r = a[11] / (1024.0 * 2048.0);
        c[9] += r * (2816 * 512);
        c[7] -= r * (2816 * 128);
        c[5] += r * (1232 * 32);
        c[3] -= r * (220 * 8);
        c[1] += r * (11 * 2);
#pragma unroll
        for (int i = 2; i <= kDegree; ++i) asm("" : "+s"(c[i]));
    }
    // 2^(t + bits); 0 for t however low (of -inf NaN, which the chunks' kernel adds where nothing is read)
    __device__ __forceinline__ double operator()(double t, int bits = 0) const {
        const double n = rint(t), f = t - n;
        double p = c[kDegree];
#pragma unroll
        for (int i = kDegree - 1; i > 0; --i) p = fma(p, f, c[i]);
        return ldexp(fma(p, f, 1.0), (int)(to_int(n) + (uint32_t)bits));
    }
    // The same as a whole number, rounded to nearest (bits <= 51): the last bits of 2^52 + it, plus kOffset.
    static constexpr uint64_t kOffset = 0x4330000000000000ull;
    __device__ __forceinline__ uint64_t whole_offset(double t, int bits) const {
        return __builtin_bit_cast(uint64_t, (*this)(t, bits) + 4503599627370496.0);
    }
    __device__ __forceinline__ uint64_t whole(double t, int bits) const { return whole_offset(t, bits) - kOffset; }
};

// Floats in order as ascending numbers (-0 is 0), and back.
__device__ __forceinline__ uint32_t order_bits(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float bits_order(uint32_t up) {
    return __builtin_bit_cast(float, up & 0x80000000u ? up & 0x7fffffffu : ~up);
}
// Words in order as ascending 64-bit numbers: logit, largest first, then index.
__device__ __forceinline__ uint64_t word_order(float x, uint32_t i) { return (uint64_t)~order_bits(x) << 32 | i; }
__device__ __forceinline__ float word_logit(uint64_t order) { return bits_order(~(uint32_t)(order >> 32)); }

typedef f4_t f4w_t __attribute__((aligned(4)));

// Four logits from word i on, -inf past the end.
__device__ __forceinline__ f4_t load_words(const float* __restrict__ x, int i, int vocab) {
    if (i + 4 <= vocab) return *reinterpret_cast<const f4w_t*>(x + i);
    f4_t v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = i + e < vocab ? x[i + e] : -INFINITY;
    return v;
}

template <int CTRL, int ROWS, class T>
__device__ __forceinline__ T dpp_or_zero(T v) {
    if constexpr (sizeof(T) == 8) {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xf, false);
        const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, ROWS, 0xf, false);
        return __builtin_bit_cast(T, (uint64_t)hi << 32 | lo);
    } else {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
    }
}
// The sum over the wave's lanes up to each: steps inside its rows of 16 lanes, then the rows' last lanes.
template <class T>
__device__ __forceinline__ T wave_prefix(T v) {
    v += dpp_or_zero<0x111, 0xf>(v);
    v += dpp_or_zero<0x112, 0xf>(v);
    v += dpp_or_zero<0x114, 0xf>(v);
    v += dpp_or_zero<0x118, 0xf>(v);
    v += dpp_or_zero<0x142, 0xa>(v);
    v += dpp_or_zero<0x143, 0xc>(v);
    return v;
}
template <class T>
__device__ __forceinline__ T lane_of(T v, int lane) {   // (lane: the same for all)
    if constexpr (sizeof(T) == 8) {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)b, lane), hi = __builtin_amdgcn_readlane((int)(b >> 32), lane);
        return __builtin_bit_cast(T, (uint64_t)hi << 32 | lo);
    } else {
        return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
    }
}

// Bound by latency for a few rows (one: 6 us), for many by vector instructions, 25 a word and as many again for its place
// (256 rows of 151936 words by top-p: 62 us, on 73% of the cycles; 155 MB read and 78 of places written).
__global__ void __launch_bounds__(kChunkThreads) sample_chunk_kernel(const SampleArgs a) {
    constexpr int kWaves = kChunkThreads / kWave, kBinWaves = kBins / kWave;
    // (from the last bin on, a place a lane for words that do not count: no branches, and no lanes on one place)
    __shared__ unsigned long long mass[kBins + kWave], wave_mass[kWaves];
    __shared__ uint32_t count[kBins + kWave], wave_count[kWaves];
    __shared__ float wave_max[kWaves];
    __shared__ __align__(16) uint16_t place[kChunk];
    __shared__ uint32_t first, bins;
    const int row = blockIdx.x / a.nchunk, chunk = blockIdx.x - row * a.nchunk, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float* x = a.logits + row * a.stride;
    f4_t v[kPerThread / 4];
#pragma unroll
    for (int j = 0; j < kPerThread / 4; ++j) v[j] = load_words(x, chunk * kChunk + 4 * (tid + kChunkThreads * j), a.vocab);
    const double scale = word_scale(a, row);
    const int k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.0f, least = a.min_p ? a.min_p[row] : 0.0f;
    if (tid < kBins) {   // (what lies behind is never read)
        mass[tid] = 0;
        count[tid] = 0;
    }
    if (tid == 0) {
        first = kNoToken;
        bins = 0;
    }
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < kPerThread / 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) m = __builtin_elementwise_maximum(m, v[j][e]);   // (NaN stays)
    const uint64_t odd = __builtin_amdgcn_ballot_w64(!(m < INFINITY));
    m = odd ? NAN : wave_max_dpp(m);
    if (lane == 0) wave_max[wave] = m;
    __syncthreads();
    bool wrong = false;
    m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        wrong |= wave_max[w] != wave_max[w];
        m = fmaxf(m, wave_max[w]);
    }
    Chunk& out = a.chunks[blockIdx.x];
    const double top = m > -INFINITY ? eighth(m, scale) : 0.0;
    if (scale < 0.0 || wrong || !(m > -INFINITY)) {   // the largest is all that counts, if anything does
        uint32_t at = kNoToken;
#pragma unroll
        for (int j = kPerThread / 4 - 1; j >= 0; --j)
#pragma unroll
            for (int e = 3; e >= 0; --e)
                if (v[j][e] == m) at = chunk * kChunk + 4 * (tid + kChunkThreads * j) + e;
        if (at != kNoToken && m > -INFINITY) atomicMin(&first, at);
        __syncthreads();
        if (tid == 0) out.head = ChunkHead{top, m, first, wrong, {0, 0, 0}};
        return;   // (the row's kernel reads no bins of such a chunk)
    }
    const Exp2 exp2;
    uint32_t rank[kPerThread];   // bin and place inside it
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
        const float x = v[j >> 2][j & 3];
        const uint32_t b = min(to_int(top - eighth(x, scale)), (uint32_t)(kBins - 1 + lane));   // (-inf: the latter)
        atomicAdd(&mass[b], (unsigned long long)exp2.whole_offset(distance(x, m, scale), kBits));
        rank[j] = b << 16 | atomicAdd(&count[b], 1u);
    }
    __syncthreads();
    // sums over the bins up to each
    uint64_t ms = 0;
    uint32_t cs = 0;
    if (wave < kBinWaves) {
        cs = count[tid];
        ms = wave_prefix<uint64_t>(mass[tid] - cs * Exp2::kOffset);
        cs = wave_prefix<uint32_t>(cs);
        if (lane == kWave - 1) {
            wave_mass[wave] = ms;
            wave_count[wave] = cs;
        }
    }
    __syncthreads();
    if (wave < kBinWaves) {
        const uint32_t own = count[tid];
#pragma unroll
        for (int w = 0; w < kBinWaves; ++w)
            if (w < wave) {
                ms += wave_mass[w];
                cs += wave_count[w];
            }
        out.mass[tid] = (double)ms;
        out.upto[tid] = (uint16_t)cs;
        count[tid] = cs - own;   // words in front of the bin
        // the bins whose words the rules may ask for one by one: of a chunk's words the first k, and, if top-p does
        // not have to know what top-k keeps, those of min_p of its largest (and one bin more for the roundings)
        const float deep = least > 0.0f && !(k > 0 && p < 1.0f) ? 2.5f - 8.0f * log2f(fminf(least, 1.0f)) : (float)kBins;
        const bool ask = (k > 0 || p < 1.0f || least > 0.0f) && tid < kBins - 1 && tid <= deep && (k <= 0 || cs - own < (uint32_t)k);
        const int n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(ask));   // (the first so many)
        if (lane == 0 && n) atomicAdd(&bins, (uint32_t)n);
    }
    __syncthreads();
    const int asked = (int)bins;
    if (tid == 0) out.head = ChunkHead{top, m, 0, 0, {0, 0, 0}};
    if (!asked) return;
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
        const int b = (int)(rank[j] >> 16);
        if (b < asked) place[count[b] + (rank[j] & 0xffffu)] = (uint16_t)(4 * (tid + kChunkThreads * (j >> 2)) + (j & 3));
    }
    __syncthreads();
    const int stored = (int)count[asked];   // (the last bin, which is never asked for, has words in front too)
    for (int i = tid; i < (stored + 7) / 8; i += kChunkThreads)
        reinterpret_cast<uint4*>(out.place)[i] = reinterpret_cast<const uint4*>(place)[i];
}

struct RowLds {
    uint64_t list[kList], weight[kList];      // words in order, and their weights
    double chunk_mass[kMostChunks], chunk_scale[kMostChunks];
    unsigned long long chunk_part[kMostChunks];
    uint32_t chunk_end[kMostChunks];
    int chunk_from[kMostChunks];
    uint32_t wave_words[kRowThreads / kWave];
    int chunk_shift[kMostChunks];
    double mass[kBins];                       // of all bins up to each
    uint32_t count[kBins];
    // a pass fills one of them and clears the next: with three, a wave that still reads the last one is not disturbed
    unsigned long long digit_mass[3][256];
    uint32_t digit_count[3][256];
    double goal, sum;
    unsigned long long lo;
    float max[kRowThreads / kWave];
    uint32_t n, found;
    int least_bin;
    float edge;
};

// One row.  Bound by latency: some 20 steps between barriers, and a trip to the chunks' heads, to their bins, to the
// places of the words that are ranked, and to these (one row of 151936 words, every rule: 14.5 us; 256 by top-p, whose
// bins hold some 3000 words: 39).
__global__ void __launch_bounds__(kRowThreads) sample_row_kernel(const SampleArgs a) {
    __shared__ RowLds l;
    constexpr int kWaves = kRowThreads / kWave;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Chunk* chunks = a.chunks + (int64_t)row * a.nchunk;
    const float* x = a.logits + row * a.stride;
    const double scale = word_scale(a, row);
    const int k = a.top_k ? a.top_k[row] : 0;
    const double p = a.top_p ? (double)a.top_p[row] : 1.0, least = a.min_p ? (double)a.min_p[row] : 0.0;
    const float given = a.u[row];
    // the row's maximum, its first word and whether all is well
    float m = -INFINITY;
    bool wrong = false;
    for (int c = tid; c < a.nchunk; c += kRowThreads) {
        m = fmaxf(m, chunks[c].head.max);
        wrong |= chunks[c].head.bad != 0;
    }
    m = wave_max_dpp(m);
    if (__builtin_amdgcn_ballot_w64(wrong)) m = NAN;
    if (lane == 0) l.max[wave] = m;
    if (tid == 0) l.found = kNoToken;
    if (tid < 256) {
        l.digit_mass[0][tid] = 0;
        l.digit_count[0][tid] = 0;
    }
    __syncthreads();
    wrong = false;
    m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        wrong |= l.max[w] != l.max[w];
        m = fmaxf(m, l.max[w]);
    }
    if (wrong || !(m > -INFINITY)) {
        if (tid == 0) {
            a.ids[row] = kNoToken;
            if (a.probs) a.probs[row] = 0.0f;
            raise_error(RTA_DEVERR_DETECTOR);
        }
        return;
    }
    if (scale < 0.0) {   // the largest
        for (int c = tid; c < a.nchunk; c += kRowThreads)
            if (chunks[c].head.max == m) atomicMin(&l.found, chunks[c].head.arg);
        __syncthreads();
        if (tid == 0) {
            a.ids[row] = l.found;
            if (a.probs) a.probs[row] = 1.0f;
        }
        return;
    }
    const Exp2 exp2;
    const double top = eighth(m, scale);
    auto below = [&](float v) { return fmax(distance(v, m, scale), -1000.0); };   // log2 of a weight
    auto bin_of = [&](float v) { return top - eighth(v, scale); };
    // how far a chunk's bins and largest weight lie below the row's
    for (int c = tid; c < a.nchunk; c += kRowThreads) {
        const float cm = chunks[c].head.max;
        const bool some = cm > -INFINITY;
        const double down = top - chunks[c].head.top;
        l.chunk_shift[c] = some && down < kBins ? (int)down : kBins;
        l.chunk_scale[c] = some ? exp2(below(cm), -kBits) : 0.0;
    }
    __syncthreads();
    // what the row's bins up to each hold
    if (wave < kBins / kWave) {
        double w = 0.0;
        uint32_t n = 0;
        constexpr int kAtOnce = 24;   // on their way together: a trip takes over 1 us
        for (int c0 = 0; c0 < a.nchunk; c0 += kAtOnce) {
            // lane j: chunk c0 + j's (past the last one a shift that no bin reaches)
            const int cl = min(c0 + lane, a.nchunk - 1), shifts = c0 + lane < a.nchunk ? l.chunk_shift[cl] : kBins;
            const double scales = l.chunk_scale[cl];
            double cw[kAtOnce];
            uint16_t cn[kAtOnce];
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) {
                const Chunk& c = chunks[min(c0 + j, a.nchunk - 1)];
                const int at = max(tid - lane_of(shifts, j), 0);
                cw[j] = c.mass[at];
                cn[j] = c.upto[at];
            }
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) {
                const bool in = tid >= lane_of(shifts, j);
                w += in ? cw[j] * lane_of(scales, j) : 0.0;
                n += in ? cn[j] : 0;
            }
        }
        l.mass[tid] = w;
        l.count[tid] = n;
    } else if (wave == kWaves - 1) {
        // The smallest logit that weighs enough, by the weights' logarithms (of a min-p of 2^-37 the whole numbers would
        // leave 13 bits): of all floats from the lowest up to the largest, by their order, 64 of them tried at once.  What
        // it divides is then the same wherever it is asked, and the bin that it lies in is the last that matters (behind
        // it chunks need not have kept their words).
        double log = least > 0.0 ? log2(fmin(least, 1.0)) : -INFINITY;
        if (scale == kAlike) log = fmin(log, -1e-200);   // (below 0: a min-p of 1 keeps all finite logits too)
        const uint32_t lowest = order_bits(-3.4028234663852886e38f), span = order_bits(m) - lowest;
        uint32_t at = 0;                                 // those below it do not weigh enough
#pragma unroll 1
        for (int shift = 26; shift >= 0; shift = shift > 6 ? shift - 6 : shift ? 0 : -1) {
            const uint64_t tried = at + ((uint64_t)lane << shift);
            const bool enough = tried >= span || distance(bits_order(lowest + (uint32_t)tried), m, scale) >= log;
            const int n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(!enough));   // (the first so many)
            if (n) at += ((uint32_t)(n - 1) << shift) + 1;
        }
        if (lane == 0) {
            const double bin = bin_of(bits_order(lowest + at));
            l.edge = bits_order(lowest + at);
            l.least_bin = at && bin < kBins ? (int)bin : kBins;   // (all of them: no matter)
        }
    }
    __syncthreads();
    const int least_bin = l.least_bin;
    const float edge = l.edge;
    auto weighs_enough = [&](float v) { return v >= edge; };

    // The words that count are those up to last_order, all of bins up to last_bin, of it those that weigh enough
    // (whole_bin: all of that one's).  The list holds the words of bins list_lo .. list_hi (none: list_lo > list_hi).
    int last_bin = kBins - 2, list_lo = 1, list_hi = 0, list_n = 0, list_bits = kBits, part_bits = kBits;
    uint64_t last_order = ~0ull;
    bool whole_bin = true;
    double total = l.mass[kBins - 2];
    int buf = 0;   // the digits that are clear
    const double u = given > 0.0f ? fmin((double)given, 1.0) : 0.0;

    // top-k, top-p, and the draw from the list (or, where many words count, the sums of the last bin's by chunk).
    // One loop, and in it one loop of passes over the words, so that the code is there and fetched once.
    for (int rule = 0; rule < 3; ++rule) {
        uint32_t words = 0;   // the search: the first word up to which there are so many,
        double goal = 0.0;    // or weights of at least (the draw: more than) goal
        int b = last_bin;
        if (rule == 0) {
            if (!(k > 0) && !(least > 1.0)) continue;
            words = least > 1.0 ? 1 : (uint32_t)k;
        }
        if (rule == 1) {
            if (!(p < 1.0)) continue;
            goal = p * total;
        }
        if (rule < 2) {
            b = 0;   // the bins up to which there is not enough
#pragma unroll
            for (int j = 0; j < kBins / kWave; ++j) {
                const int t = lane + j * kWave;
                b += __builtin_popcountll(__builtin_amdgcn_ballot_w64(t < kBins - 1 && (rule == 0 ? l.count[t] < words : l.mass[t] < goal)));
            }
            if (rule == 0 && (b == kBins - 1 || (b > least_bin && !(p < 1.0)))) continue;   // (not so many, or no matter)
            if (rule == 1 && b > least_bin) continue;
            b = min(b, last_bin);
        } else {
            if (least_bin <= last_bin) {
                last_bin = b = (int)least_bin;
                whole_bin = false;
            }
            if (whole_bin) break;   // no word to be looked at by itself
        }
        // the words of bin b, with all before it if they fit
        const uint32_t upto = l.count[b], before_b = b ? l.count[b - 1] : 0;
        // Whole numbers of words of this bin alone keep as many bits as fit of the bin's own weights, which are at most
        // 2^-((b - 1) / 8) of the largest: 2^17 equal words at 2^-36 of it would have 8 bits of 2^-44.
        const int below_one = b > 0 ? (b - 1) / 8 : 0;
        bool listed = list_lo <= b && b <= list_hi;
        if (!listed) {
            const int lo = upto <= kFromTop ? 0 : b;
            list_n = (int)(lo ? upto - before_b : upto);
            listed = list_n <= kList;
            list_lo = listed ? lo : 1;
            list_hi = listed ? b : 0;
            list_bits = lo ? kBits + below_one : kBits;
            if (listed) {
                // where each chunk's words of these bins lie and go: thread c has chunk c
                uint32_t i0 = 0, own = 0;
                if (tid < a.nchunk) {
                    const int cb = b - l.chunk_shift[tid], cl = lo - l.chunk_shift[tid];
                    i0 = cl > 0 && cb >= 0 ? chunks[tid].upto[cl - 1] : 0;
                    own = cb >= 0 ? chunks[tid].upto[cb] - i0 : 0;
                }
                uint32_t to = wave_prefix<uint32_t>(own);
                __syncthreads();   // (their room may still be read)
                if (lane == kWave - 1) l.wave_words[wave] = to;
                __syncthreads();
                for (int w = 0; w < wave; ++w) to += l.wave_words[w];
                if (tid < a.nchunk) {
                    l.chunk_end[tid] = to;
                    l.chunk_from[tid] = (int)(i0 - (to - own));
                }
                __syncthreads();
                constexpr int kAtOnce = 8;
                const int first_step = 1 << (31 - __clz(a.nchunk));
                for (int i = tid; i < list_n; i += kAtOnce * kRowThreads) {
                    uint32_t id[kAtOnce];
                    float t[kAtOnce];
                    int c[kAtOnce] = {};   // the first chunk that ends behind the word
                    for (int step = first_step; step > 0; step >>= 1)
#pragma unroll
                        for (int j = 0; j < kAtOnce; ++j) {
                            const int mid = min(c[j] + step, a.nchunk);
                            if ((int)l.chunk_end[mid - 1] <= i + j * kRowThreads) c[j] = mid;
                        }
#pragma unroll
                    for (int j = 0; j < kAtOnce; ++j) {
                        c[j] = min(c[j], a.nchunk - 1);
                        id[j] = chunks[c[j]].place[(i + j * kRowThreads + l.chunk_from[c[j]]) & (kChunk - 1)];
                    }
#pragma unroll
                    for (int j = 0; j < kAtOnce; ++j) {
                        id[j] = min(c[j] * kChunk + (id[j] & (kChunk - 1)), (uint32_t)a.vocab - 1);
                        t[j] = x[id[j]];
                    }
#pragma unroll
                    for (int j = 0; j < kAtOnce; ++j)
                        if (i + j * kRowThreads < list_n) {
                            l.list[i + j * kRowThreads] = word_order(t[j], id[j]);
                            l.weight[i + j * kRowThreads] = exp2.whole(below(t[j]), list_bits);
                        }
                }
            }
            __syncthreads();
        }
        const bool draw = rule == 2 && list_lo == 0 && b <= list_hi;
        // what lies in front of the words that are searched
        double before = list_lo == 0 || !b ? 0.0 : l.mass[b - 1];
        uint32_t before_n = list_lo == 0 ? 0 : before_b;
        const int bits = min(kBits, 62 - (32 - __clz((int)(upto - before_b)))) + below_one;
        // a range of logits that holds bin b's, with room for the roundings
        const double step = 8.0 * scale, e0 = (top - b) / step, e1 = (top - b + 1.0) / step;
        const float from = (float)fmax(e0 - fabs(e0) * 1e-6 - 1e-30, -3.4028234663852886e38);
        const float to = list_lo != 0 ? fminf((float)(e1 + fabs(e1) * 1e-6 + 1e-30), m) : m;
        // Radix search over the keys (order, from the range's first on, or index), 8 bits a pass.  kDigits counts and
        // weighs the words of the value so far by their next 8, kOne takes the only word left, kGather puts a group
        // that fits into the list.  kParts: the last bin's words that count, by chunk.  Where a bin is too large for
        // the list, its words are met in the row.
        enum { kDigits, kOne, kGather, kParts };
        const uint64_t lowest = word_order(to, 0), highest = word_order(from, kNoToken);
        int mode = rule < 2 || draw ? kDigits : kParts;
        int end = draw ? 32 - __clz(a.vocab) : 64 - __clzll((long long)(highest - lowest));
        uint64_t known = end == 64 ? 0 : ~0ull << end, value = 0;
        bool opened = false;   // a draw's goal is known
        part_bits = kBits + below_one;   // (kParts' words are of this bin, and kChunk of a chunk at most)
        if (mode == kParts)
            for (int c = tid; c < a.nchunk; c += kRowThreads) l.chunk_part[c] = 0;
        if (mode == kParts) __syncthreads();
        for (;;) {
            const int shift = end > 8 ? end - 8 : 0, next = buf == 2 ? 0 : buf + 1;
            const uint32_t mask = (1u << (end - shift)) - 1;
            if (mode == kDigits && tid < 256) {
                l.digit_mass[next][tid] = 0;
                l.digit_count[next][tid] = 0;
            }
            auto visit = [&](uint64_t order, uint64_t w) {
                if (order > last_order || (rule == 2 && !weighs_enough(word_logit(order)))) return;
                const uint64_t key = draw ? order & 0xffffffffull : order - lowest;
                if (mode == kParts) {
                    atomicAdd(&l.chunk_part[(uint32_t)order / kChunk], (unsigned long long)w);
                } else if ((key & known) == value) {
                    if (mode == kDigits) {
                        const uint32_t d = (uint32_t)(key >> shift) & mask;
                        atomicAdd(&l.digit_count[buf][d], 1u);
                        atomicAdd(&l.digit_mass[buf][d], (unsigned long long)w);
                    } else if (mode == kOne) {
                        l.lo = key;
                    } else {
                        const uint32_t at = atomicAdd(&l.n, 1u);
                        l.list[at] = order;
                        l.weight[at] = exp2.whole(below(word_logit(order)), kBits + below_one);
                    }
                }
            };
            if (listed) {
                for (int i = tid; i < list_n; i += kRowThreads) visit(l.list[i], l.weight[i]);
            } else {
                for (int i = tid; i < a.vocab; i += 4 * kRowThreads) {
                    float t[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) t[j] = i + j * kRowThreads < a.vocab ? x[i + j * kRowThreads] : -INFINITY;
#pragma unroll 1
                    for (int j = 0; j < 4; ++j) {
                        const float v = j == 0 ? t[0] : j == 1 ? t[1] : j == 2 ? t[2] : t[3];
                        if (v < from || v > to || v == -INFINITY || bin_of(v) != b) continue;
                        visit(word_order(v, i + j * kRowThreads), exp2.whole(below(v), mode == kParts ? part_bits : bits));
                    }
                }
            }
            __syncthreads();
            if (mode == kParts) break;
            if (mode == kOne) {
                value = l.lo;
                break;
            }
            if (mode == kGather) {
                listed = true;
                list_n = (int)l.n;
                list_bits = kBits + below_one;
                mode = kDigits;
                continue;
            }
            // every wave by itself: four digits a lane
            uint32_t c[4], cs = 0;
            uint64_t w[4], ws = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                c[e] = l.digit_count[buf][4 * lane + e];
                w[e] = l.digit_mass[buf][4 * lane + e];
                cs += c[e];
                ws += w[e];
            }
            buf = next;
            uint32_t cb = wave_prefix<uint32_t>(cs);
            uint64_t wb = wave_prefix<uint64_t>(ws);
            const int at_bits = listed ? list_bits : bits;
            if (draw && !opened) {   // all weights have been seen
                total = ldexp((double)lane_of(wb, kWave - 1), -at_bits);
                goal = u * total;
                opened = true;
            }
            cb -= cs;
            wb -= ws;
            int hit = -1;
            uint32_t hit_n = 0, hit_c = 0;
            uint64_t hit_w = 0;
            bool met = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const double sum = before + ldexp((double)(wb + w[e]), -at_bits);
                if (c[e] && !met) {   // (none that meets it: the last)
                    met = rule == 0 ? before_n + cb + c[e] >= words : rule == 1 ? sum >= goal : sum > goal;
                    hit = e;
                    hit_n = cb;
                    hit_c = c[e];
                    hit_w = wb;
                }
                cb += c[e];
                wb += w[e];
            }
            const uint64_t hits = __builtin_amdgcn_ballot_w64(met), any = __builtin_amdgcn_ballot_w64(hit >= 0);
            const int at = hits ? __builtin_ctzll(hits) : 63 - __builtin_clzll(any | 1);
            before += ldexp((double)lane_of(hit_w, at), -at_bits);
            before_n += lane_of(hit_n, at);
            const uint32_t left = lane_of(hit_c, at);
            value |= (uint64_t)(uint32_t)(4 * at + lane_of(hit, at)) << shift;
            end = shift;
            if (end == 0) break;
            known = ~0ull << end;
            if (left == 1) mode = kOne;
            else if (!listed && left <= kList) mode = kGather;
            if (mode == kGather) {
                if (tid == 0) l.n = 0;
                __syncthreads();
            }
        }
        if (mode == kParts) break;
        if (draw) {
            const uint32_t id = (uint32_t)value;
            if (tid == 0) {
                a.ids[row] = id;
                if (a.probs) a.probs[row] = (float)(exp2(below(x[id])) / total);
            }
            return;
        }
        last_bin = b;
        last_order = value + lowest;
        whole_bin = false;
        total = before + exp2(below(word_logit(last_order)));
        __syncthreads();   // (l.lo has been read)
    }

    // Many words: what each chunk holds, its bins before the last and of that one what has been added up.
    const int bins = last_bin + (whole_bin ? 1 : 0);
    for (int c = tid; c < a.nchunk; c += kRowThreads) {
        const int n = bins - l.chunk_shift[c];
        l.chunk_mass[c] = (n > 0 ? chunks[c].mass[n - 1] * l.chunk_scale[c] : 0.0) +
                          (whole_bin ? 0.0 : ldexp((double)l.chunk_part[c], -part_bits));
    }
    __syncthreads();
    // the chunk of the word: sums in the chunks' order, 64 at a time, by one wave
    if (wave == 0) {
        double sum = 0.0;
        for (int pass = 0; pass < 2; ++pass) {
            const double goal = u * sum;   // (the second time)
            double run = 0.0, base = 0.0;
            int at = 0;
            for (int c0 = 0; c0 < a.nchunk; c0 += kWave) {
                const double w = c0 + lane < a.nchunk ? l.chunk_mass[c0 + lane] : 0.0;
                const double upto = wave_prefix<double>(w);
                const uint64_t any = __builtin_amdgcn_ballot_w64(w > 0.0);
                const uint64_t hit = pass ? __builtin_amdgcn_ballot_w64(w > 0.0 && run + upto > goal) : 0;
                if (any) {   // (none past the goal, by roundings or u = 1: the last that holds something)
                    const int e = hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(any);
                    at = c0 + e;
                    base = run + lane_of(upto - w, e);
                }
                if (hit) break;
                run += lane_of(upto, kWave - 1);
            }
            if (pass == 0) {
                sum = run;
            } else if (lane == 0) {
                l.found = at;
                l.goal = goal - base;
                l.sum = sum;
            }
        }
    }
    __syncthreads();
    // the word of the chunk: a thread sums kChunk / kRowThreads of them that follow each other
    constexpr int kEach = kChunk / kRowThreads;
    const int first = (int)l.found * kChunk + kEach * tid;
    const double rest = l.goal, sum = l.sum;
    uint64_t w[kEach], own = 0;
#pragma unroll
    for (int j = 0; j < kEach; j += 4) {
        const f4_t v = load_words(x, min(first + j, a.vocab), a.vocab);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            w[j + e] = 0;
            const double b = bin_of(v[e]);   // (-inf: none)
            if (b < kBins - 1 && word_order(v[e], first + j + e) <= last_order) {
                // (as in the sums, so the chunk that is drawn has a word)
                if (b < bins || (b == last_bin && weighs_enough(v[e]))) w[j + e] = exp2.whole(below(v[e]), kBits);
            }
            own += w[j + e];
        }
    }
    uint64_t upto = wave_prefix<uint64_t>(own);
    if (lane == kWave - 1) l.digit_mass[0][wave] = upto;
    if (tid == 0) l.lo = ~0ull;
    if (tid < kWaves) l.wave_words[tid] = 0;
    __syncthreads();
    for (int v = 0; v < wave; ++v) upto += l.digit_mass[0][v];
    const uint64_t goal = rest > 0.0 ? (uint64_t)ldexp(rest, kBits) : 0;
    uint64_t run = upto - own;
    uint32_t last = 0;   // the thread's last word with a weight, plus one
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        run += w[j];
        if (w[j]) last = first + j + 1;
        if (w[j] && run > goal && run - w[j] <= goal) l.lo = first + j;   // (one word's)
    }
    const uint64_t some = __builtin_amdgcn_ballot_w64(last > 0);
    if (some && lane == 63 - __builtin_clzll(some)) l.wave_words[wave] = last;
    __syncthreads();
    if (tid == 0) {
        uint32_t id = (uint32_t)l.lo;
        if (l.lo == ~0ull)   // none past the goal: the last one
            for (int v = 0; v < kWaves; ++v)
                if (l.wave_words[v]) id = l.wave_words[v] - 1;
        a.ids[row] = id;
        if (a.probs) a.probs[row] = (float)(exp2(below(x[id])) / sum);
    }
}

static size_t sample_bytes(int64_t rows, int64_t nchunk) {
    return (size_t)(rows * nchunk) * sizeof(Chunk);
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
    a.chunks = static_cast<Chunk*>(workspace);
    hipStream_t s = (hipStream_t)stream;
    hipLaunchKernelGGL(sample_chunk_kernel, dim3(chunks), dim3(kChunkThreads), 0, s, a);
    hipLaunchKernelGGL(sample_row_kernel, dim3(rows), dim3(kRowThreads), 0, s, a);
    return hipGetLastError() == hipSuccess ? RTA_OK : RTA_ERR_LAUNCH;
}

}  // extern "C"
