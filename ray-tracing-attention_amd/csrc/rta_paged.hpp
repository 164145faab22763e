// rta_paged.hpp -- what the kernels of attention over the paged history share: the arguments,
// what a row sees, and the matrix-core operands of its formats.
//
// The products run on v_mfma_f32_16x16x32 with the positions as rows:
//   S^T = K Q^T   A = K (row: position), B = Q^T (column: a query), and
//   O^T = V^T P^T A = V^T (row: dim),    B = P^T (column: the same query).
// Lane (i = lane % 16, u = lane / 16) of the result of the first holds positions 4u .. 4u + 3 of
// column i, which is where the second wants its B operand (k slots 8u ..) if its k axis is
// ordered  slot 8u + s  <->  position 4u + s (s < 4), 16 + 4u + s - 4 (else) of 32 positions;
// so weights never leave their lane, and V^T comes in that order from a transposing LDS read.
// On v_mfma_f32_32x32x16 (prompts) lane (i = lane % 32, u = lane / 32) holds positions 8h + 4u + e
// of 32, h = 0 .. 3, and the two products of 16 positions have their k axis in that order.
//
// fp32 queries and weights meet 16-bit values, so each is split into parts that are exact
// 16-bit numbers and whose products are added in fp32:
//   binary16 pages (and 8-bit codes, exact in binary16): two parts, 22 bits, of the value times a
//   power of two that puts its row's largest at 2^13 to 2^14.  Weights are cut off, not rounded:
//   the instruction that packs two of them cuts (queries, outside the loops, have their second part
//   rounded).  The second part ends at 2^-24, so values below 2^-16 of the largest have fewer
//   bits and those below 2^-38 none: weights of N positions lose N 2^-38 of their sum at most;
//   bfloat16 pages: three parts of 8 bits, 24 bits and no scale.
// Where few of a product's 16 columns are needed, two parts are neighbouring columns (query g in
// 2g and 2g + 1) and the third a second product into the same accumulator; else every part is a
// product of its own.  One rounding to 16 bits instead would cost
// 2^-12 (2^-9) of the result where fp32 results are wanted.
#pragma once
#include <math.h>

#include "rta_pages.hpp"

namespace rta {

typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
typedef float acc16_t __attribute__((ext_vector_type(16)));

struct PagedAttnArgs {
    PageArgs p;
    RowList l;
    const float* q;
    int64_t q_stride;
    const float* gate;
    float* out;
    float* m_out;
    float* z_out;
    int hq, group;      // group: q heads per kv head
    int max_rows, max_len, window, sinks;
    // work split: chunks of `chunk` visible positions; with nchunk > 1 every (row, q head, chunk)
    // leaves U[HD] in `part` and (m, z) in `mz`, both [row][hq][nchunk]
    int chunk, nchunk;
    int ntile;          // several rows per entry: tiles of (row, q head) columns, at most (0: one row
                        // per entry, a chunk counts along that row's own visible positions)
    float* part;
    float2* mz;
};

// What a row at position t sees: the first `head` positions and then those from `lo` on, `count`
// of them; the j-th is j for j < head, else j + lo - head.
struct Visible {
    int head, lo, count;
    __device__ __forceinline__ int position(int j) const { return j < head ? j : j + lo - head; }
};
__device__ __forceinline__ Visible visible(int t, int window, int sinks) {
    const int lo = window > 0 && t >= window ? t - window + 1 : 0;
    const int head = min(lo, sinks);
    return Visible{head, lo, head + t + 1 - lo};
}

// Row r's table row and what it sees (nothing for a bad one); false for a row that no entry
// lists or that is past max_rows.  err collects the error bits.
__device__ __forceinline__ bool resolve_row(const PagedAttnArgs& a, int r, const int32_t*& table, Visible& see,
                                            uint32_t& err) {
    int i, first, count;
    see = Visible{0, 0, 0};
    table = a.p.table;
    if (!row_entry(a.l, r, i, first, count)) return false;
    if (r - first >= a.max_rows) {
        err |= RTA_DEVERR_PAGES;
        return false;
    }
    const int s = list_seq(a.l.seqs, i);
    if ((unsigned)s >= (unsigned)a.p.max_seqs) {
        err |= RTA_DEVERR_PAGES;
        return true;
    }
    const int len = a.p.lengths[s], t = len - count + (r - first);
    table += (int64_t)s * a.p.max_pages;
    if (len > a.max_len || len < 0 || (t < 0 && (len > 0 || count > 1))) err |= RTA_DEVERR_PAGES;
    else if (t >= 0) see = visible(t, a.window, a.sinks);
    return true;
}

typedef f4_t f4u_t __attribute__((aligned(4)));   // at an address of a multiple of 4

// Sums of weights leave the kernels' loops 2^-kRoom times what they are against the maximum (weight 2^-kRoom
// for the largest score): a mean of finite values is finite, and their plain sum need not be.  20: 2^20 positions of
// the same weight with values at fp32's end, and values down to 2^-100 whose sums are normal numbers.
constexpr int kRoom = 20;
// The final values of (row, q head) at dims c .. c + 3 from U and Z (both 2^-kRoom times) and M (natural units).
__device__ __forceinline__ void write_result(const PagedAttnArgs& a, int64_t at, int hd, int c, f4_t u, float m,
                                             float z, uint32_t& err) {
    f4_t o = u * (z > 0.0f || z != z ? 1.0f / z : 0.0f);   // nothing seen: zeros
    const int64_t to = at * hd + c;
    if (a.gate) {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] *= detector_sigmoid(a.gate[to + e]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (!isfinite(o[e])) err |= RTA_DEVERR_DETECTOR;
    *reinterpret_cast<f4u_t*>(a.out + to) = o;
    if (c == 0) {
        if (a.m_out) a.m_out[at] = m;
        if (a.z_out) a.z_out[at] = ldexpf(z, kRoom);
    }
}

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// ---- operands by page format ----
template <int FMT> struct PageFmt;
template <> struct PageFmt<RTA_F16> {
    // element bytes; parts of a query or weight; products of a pair of operands with parts in columns
    static constexpr int kBytes = 2, kParts = 2, kOps = 1;
    static constexpr bool kScaled = false;       // scales beside the elements
};
template <> struct PageFmt<RTA_BF16> {
    static constexpr int kBytes = 2, kParts = 3, kOps = 2;
    static constexpr bool kScaled = false;
};
template <> struct PageFmt<RTA_Q8_ROW> {
    static constexpr int kBytes = 1, kParts = 2, kOps = 1;
    static constexpr bool kScaled = true;
};

template <int FMT>
__device__ __forceinline__ f4_t page_mfma(u4_t a, u4_t b, f4_t c) {
    if constexpr (FMT == RTA_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), c, 0, 0,
                                                       0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0,
                                                      0);
}
template <int FMT>
__device__ __forceinline__ acc16_t page_mfma(u4_t a, u4_t b, acc16_t c) {
    if constexpr (FMT == RTA_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), c, 0, 0,
                                                       0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0,
                                                      0);
}

// Registers 4h .. 4h + 3 of a product: four rows that follow each other.
__device__ __forceinline__ f4_t quad_of(f4_t c, int) { return c; }
__device__ __forceinline__ f4_t quad_of(acc16_t c, int h) { return f4_t{c[4 * h], c[4 * h + 1], c[4 * h + 2], c[4 * h + 3]}; }

// Four int8 codes as four binary16 (1024 + (c + 128) has the code in its last bits; minus 1152).
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
    const uint32_t x = w ^ 0x80808080u;
    const h2v_t off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2v_t, __builtin_amdgcn_perm(x, 0x64646464u, 0x00050004u)) + off);
    hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2v_t, __builtin_amdgcn_perm(x, 0x64646464u, 0x00070006u)) + off);
}

// The upper halves of two floats as one dword: bfloat16 cut off, not rounded.
__device__ __forceinline__ uint32_t upper_halves(float lo, float hi) {
    return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, hi), __builtin_bit_cast(uint32_t, lo), 0x07060302u);
}
__device__ __forceinline__ float cut(float v, uint32_t mask) {
    return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, v) & mask);
}

// Two floats as binary16, cut off or rounded to the nearest.
template <bool NEAREST>
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    if constexpr (NEAREST) return __builtin_bit_cast(uint32_t, h2v_t{(_Float16)lo, (_Float16)hi});
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(lo, hi));
}

// Part `part` (0, 1) of eight values as B operands (op 1, of bfloat16 only: the third part in
// part 0's columns).  Parts are cut off, not rounded, so that each remainder is exact; a value
// that is not finite stays so.
template <int FMT, bool NEAREST = false>
__device__ __forceinline__ void split_parts(const float v[8], int part, u4_t op[PageFmt<FMT>::kOps]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float x[2], y[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float w = v[2 * j + e], top = cut(w, FMT == RTA_BF16 ? 0xffff0000u : 0xffffe000u), r = w - top;
            x[e] = part ? r : NEAREST ? top : w;
            if constexpr (FMT == RTA_BF16) y[e] = part ? 0.0f : r - cut(r, 0xffff0000u);
        }
        if constexpr (FMT == RTA_BF16) {
            op[0][j] = upper_halves(x[0], x[1]);
            op[1][j] = upper_halves(y[0], y[1]);
        } else {
            op[0][j] = pack_half<NEAREST>(x[0], x[1]);
        }
    }
}

// Whether a piece of 2-byte elements holds an inf or a NaN: an exponent of ones carries into the
// half's top bit.
template <int FMT>
__device__ __forceinline__ bool piece_not_finite(u4_t x) {
    constexpr uint32_t kE = FMT == RTA_BF16 ? 0x7f807f80u : 0x7c007c00u, kOne = FMT == RTA_BF16 ? 0x00800080u : 0x04000400u;
    uint32_t hit = 0;
#pragma unroll
    for (int y = 0; y < 4; ++y) hit |= (x[y] & kE) + kOne;
    return (hit & 0x80008000u) != 0;
}

// Dims of element s of the 8 that lane segment u holds for product kb: 16-byte pieces of a row
// follow the segments, one piece per product (2-byte elements) or two products (codes).
template <int FMT>
__device__ __forceinline__ int operand_dim(int kb, int u) {
    if constexpr (FMT == RTA_Q8_ROW) return 64 * (kb >> 1) + 16 * u + 8 * (kb & 1);
    else return 32 * kb + 8 * u;
}

// Power-of-two exponent that brings values up to mx below 2^14 (for binary16 operands);
// zero or not finite: the lowest.
__device__ __forceinline__ int part_exponent(float mx) {
    int e = -110;
    if (mx > 0.0f && mx < INFINITY) (void)frexpf(mx, &e);
    return e < -110 ? -110 : e;
}

// An entry's rows as columns (row, q head of one kv head): column c is row c / group.
struct Entry {
    int base, count;    // its first row and how many it has
    int rows;           // of which this many are written
    int len;            // its sequence's positions, 0 for a bad one
    const int32_t* table;
};
// False for an entry without rows or with bad ones.  err collects the error bits.
__device__ __forceinline__ bool resolve_entry(const PagedAttnArgs& a, int entry, Entry& e, uint32_t& err) {
    if (!entry_rows(a.l, entry, e.base, e.count)) {
        err |= RTA_DEVERR_PAGES;
        return false;
    }
    if (!e.count) return false;
    e.rows = min(e.count, a.max_rows);
    if (e.count > a.max_rows) err |= RTA_DEVERR_PAGES;
    const int s = list_seq(a.l.seqs, entry);
    e.len = 0;
    e.table = a.p.table;
    if ((unsigned)s >= (unsigned)a.p.max_seqs) {
        err |= RTA_DEVERR_PAGES;
        return true;
    }
    const int len = a.p.lengths[s];
    e.table += (int64_t)s * a.p.max_pages;
    if (len < 0 || len > a.max_len) {
        err |= RTA_DEVERR_PAGES;
        return true;
    }
    e.len = len;
    if (len < e.count && (len > 0 || e.count > 1)) err |= RTA_DEVERR_PAGES;
    return true;
}

// What the columns [tile cols, (tile + 1) cols) of an entry of `count` rows and a sequence of `len` positions
// see, any of them; t0: the first one's position.
__device__ __forceinline__ Visible prompt_span(const PagedAttnArgs& a, int len, int count, int tile, int cols) {
    const int tok0 = (int)((int64_t)tile * cols / a.group);
    const int tok1 = min((int)(((int64_t)(tile + 1) * cols - 1) / a.group), count - 1);
    const int t0 = max(len - count + tok0, 0), t1 = len - count + tok1;
    if (t1 < 0) return Visible{0, 0, 0};
    const int lo = a.window > 0 && t0 >= a.window ? t0 - a.window + 1 : 0;
    const int head = min(lo, a.sinks);
    return Visible{head, lo, head + t1 + 1 - lo};
}

// Over 8-bit pages an operand of the second product is a weight times a value scale, the scales brought
// below 1 by the largest met so far (2^ve): one multiplication for all columns.  The parts end at
// 2^-24, so what a scale is below the largest is lost at that end, and the largest may have no
// weight, or be at a position that the column cannot see.  So in a tile with a scale below
// 2^(ve - kSpread) every column's operands and sums have a power of two of their own (Softmax::up).
// Relative error of a sum over 65536 positions whose scales are 2^-6, 2^-8 and 2^-12 of the largest: 1.4e-7
// (as at 2^0), 1.7e-7, 1.9e-6.  Scales of normal values differ by less than 2^3, ve's rounding
// included: their tiles pay for the comparison only (1 to 3.5% of a call); where every tile is spread, single
// rows of 32 sequences over 4000 positions take 74.8 us, else 72.9, a prompt of 4096 rows 406, else 339.
constexpr int kSpread = 6;
__device__ __forceinline__ bool far_below(float scale, int ve) {
    return scale != 0.0f && fabsf(scale) < ldexpf(1.0f, ve - kSpread);
}

// All parts of eight values as operands.
template <int FMT, bool NEAREST = false>
__device__ __forceinline__ void split_all(const float v[8], u4_t* op) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float a = v[2 * j], b = v[2 * j + 1];
        if constexpr (FMT == RTA_BF16) {
            const float ra = a - cut(a, 0xffff0000u), rb = b - cut(b, 0xffff0000u);
            op[0][j] = upper_halves(a, b);
            op[1][j] = upper_halves(ra, rb);
            op[2][j] = upper_halves(ra - cut(ra, 0xffff0000u), rb - cut(rb, 0xffff0000u));
        } else {
            // (one mixed fma per remainder; a multiplication by 1 in sight would become two instructions)
            float minus = -1.0f;
            asm("" : "+s"(minus));
            const h2v_t hi = __builtin_bit_cast(h2v_t, __builtin_amdgcn_cvt_pkrtz(a, b));
            op[0][j] = __builtin_bit_cast(uint32_t, hi);
            op[1][j] = pack_half<NEAREST>(fmaf((float)hi[0], minus, a), fmaf((float)hi[1], minus, b));
        }
    }
}

// A product under its mask: -inf is a masked one's from here on, so one that is seen becomes NaN (as does
// inf), which reaches the result.
__device__ __forceinline__ float seen_or_masked(float x, bool sees) { return sees ? fmaf(x, 0.0f, x) : -INFINITY; }

// Masks the products of 32 positions j0 .. of a list that the columns see between them (a lane
// holds positions 32 / N h + 4u + e of each column tile, h < N, e < 4): bit k of
// ok says whether position k counts, t_col is the lane's column's position, -1 at least.  What a
// column sees is one unsigned comparison of its distance (the first positions' window is all):
// booleans of their own would each take a pair of scalar registers.
template <int NC, int N>
__device__ __forceinline__ void mask_columns(f4_t (*x)[N], uint32_t ok, const Visible& see, int j0, int u,
                                             const int* t_col, int window, int sinks) {
    const uint32_t mine = ok >> (4 * u);
#pragma unroll
    for (int h = 0; h < N; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int p = see.position(j0 + 32 / N * h + 4 * u + e);
            const uint32_t reach = window == 0 || p < sinks ? 0x80000000u : (uint32_t)window;
            const int at = (mine >> (32 / N * h + e)) & 1u ? p : INT_MAX;   // no distance reaches it
#pragma unroll
            for (int c = 0; c < NC; ++c)
                x[c][h][e] = seen_or_masked(x[c][h][e], (uint32_t)(t_col[c] - at) < reach);
        }
}

// The online softmax of NC column tiles, a lane holding 4N positions of its column of each, N = 2
// (16 columns) or 4 (32 columns) (products x; score = x fac in log2 units, fac a power of two: so a
// score is its product exactly, and its distance from low is rounded once, however large both are).
// Weights are 2^(score - low), 2^kTop for the largest score when low was set; low follows the
// maximum only when weights would pass 2^(kTop + kSlack), 2^15 for binary16 parts, so the sums are
// not rescaled for every small step, and binary16 parts do not overflow.  kTop is as high as that
// allows: the second part ends at 2^-24, and over a long history most of the sum lies in weights far
// below the largest.  bfloat16 parts have fp32's exponents, and values may too: there the largest
// weight is 2^-kRoom from the start.
template <int NC, int N, int FMT>
struct Softmax {
    static constexpr float kTop = FMT == RTA_BF16 ? -kRoom : 14, kSlack = 1.0f;
    static constexpr bool SCALED = PageFmt<FMT>::kScaled;
    float m[NC], low[NC], z[NC];   // m: the largest product; z: of the lane's positions
    float lowest;                  // of the products in tiles that are seen whole: a -inf shows nowhere else
    int up[NC];                    // SCALED: the sums o and the tile's operands are 2^up times what they are else
    bool lifted;                   // some of them are not 0

    __device__ __forceinline__ void start() {
        lowest = INFINITY;
        lifted = false;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            m[c] = low[c] = -INFINITY;
            z[c] = 0.0f;
            up[c] = 0;
        }
    }
    // Over the lanes that hold a column.
    static __device__ __forceinline__ float column_max(float v) {
        if constexpr (N == 2) v = max_xor16(v);
        return max_xor32(v);
    }
    static __device__ __forceinline__ float column_sum(float v) {
        if constexpr (N == 2) v = add_xor16(v);
        return add_xor32(v);
    }
    __device__ __forceinline__ void watch(const f4_t (*x)[N], bool whole) {
        float t = lowest;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int j = 0; j < 4 * N; ++j) t = fminf(t, x[c][j >> 2][j & 3]);
        lowest = whole ? t : lowest;
    }
    // Takes in the maxima of x (masked positions -inf) and brings z and o to the new base; vshift:
    // the power of two by which o has to follow a value scale; spread (all lanes alike): the scales vf are
    // far apart, so each column's largest operand is brought to 2^14, but no sum past 2^100.
    template <class O, int DT>
    __device__ __forceinline__ void raise(const f4_t (*x)[N], const float* fac, int vshift, O (*o)[DT], bool spread,
                                          const f4_t* vf) {
        bool lift = vshift != 0 || spread || lifted;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float t = x[c][0][0];
#pragma unroll
            for (int j = 1; j < 4 * N; ++j) t = fmaxf(t, x[c][j >> 2][j & 3]);
            m[c] = fmaxf(m[c], column_max(t));
            lift = lift || fmaf(m[c], fac[c], -low[c]) > kTop + kSlack;
        }
        if (__builtin_amdgcn_ballot_w64(lift)) {
            lifted = spread;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const float top = m[c] * fac[c];
                float base = fmaxf(low[c], top - kTop);
                if (top - base > kTop + kSlack) base = top;   // (past 2^25, where floats are 4 apart)
                const float al = __builtin_amdgcn_exp2f(low[c] - (base == -INFINITY ? 0.0f : base));
                int by = vshift;
                z[c] *= al;
                low[c] = base;
                if constexpr (SCALED) {
                    by -= up[c];
                    up[c] = 0;
                    if (spread) {
                        float most = 0.0f, sum = 0.0f;
#pragma unroll
                        for (int j = 0; j < 4 * N; ++j)
                            most = fmaxf(most, fabsf(weight(c, x[c][j >> 2][j & 3], fac[c]) * vf[j >> 2][j & 3]));
#pragma unroll
                        for (int d = 0; d < DT; ++d)
#pragma unroll
                            for (int e = 0; e < (int)(sizeof(O) / 4); ++e) sum = fmaxf(sum, fabsf(o[c][d][e]));
                        up[c] = min(14 - part_exponent(column_max(most)),
                                    100 - by - part_exponent(column_max(sum) * al));
                        by += up[c];
                    }
                }
                const float f = ldexpf(al, by);
#pragma unroll
                for (int d = 0; d < DT; ++d) o[c][d] *= f;
            }
        }
    }
    __device__ __forceinline__ float weight(int c, float x, float fac) const {
        const float base = low[c] == -INFINITY ? 0.0f : low[c];   // (nothing seen yet: weights 0)
        return __builtin_amdgcn_exp2f(fmaf(x, fac, -base));
    }
    __device__ __forceinline__ void weights(int c, const f4_t* x, float fac, float w[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            w[j] = weight(c, x[j >> 2][j & 3], fac);
            z[c] += w[j];
        }
    }
    // A weight of 0 times a value that is not finite is not 0.  Where the columns do not all see a
    // tile whole, rows with such values (bad, bit 32 / N h + 4 u + e of a lane's position) are zeros in
    // the product, and the sums of the columns that do see one become NaN.
    __device__ __forceinline__ void poison(const f4_t (*s)[N], uint32_t bad, int u) {
        const uint32_t mine = bad >> (4 * u);
#pragma unroll
        for (int j = 0; j < 4 * N; ++j)
#pragma unroll
            for (int c = 0; c < NC; ++c)
                if (((mine >> (32 / N * (j >> 2) + (j & 3))) & 1u) && s[c][j >> 2][j & 3] != -INFINITY) z[c] = NAN;
    }
    // The maximum in log2 units, and what brings sums over weights to 2^-kRoom against it: back 2^kBack.
    static constexpr int kBack = -(int)kTop - kRoom;
    __device__ __forceinline__ void finish(int c, float fac, float& M, float& back) const {
        M = m[c] * fac;
        back = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(low[c] - M + kTop);
    }
    // A sum of o so, the value scales below 2^ve (one power of two at the end: parts of it may have none).
    __device__ __forceinline__ float settled(int c, float o, float back, int ve) const {
        return SCALED ? ldexpf(o * back, ve - up[c] + kBack) : o * ldexpf(back, kBack);
    }
};

}  // namespace rta
