// rta_paged_decode4.hpp -- attention of one row per sequence over 4-bit pages, up to four q heads a kv head.
//
// The work is cut as in paged_decode_kernel, but codes that become binary16 take 12 vector instructions for eight
// values, so vector instructions bind, not the history's bytes (in that kernel 456 of them a tile of 32 positions,
// on 75% of the cycles).  Four queries in two parts fill half of a product's 16 columns; here the other half
// takes them too, for other positions:
//   S^T: rows are positions i of the tile's first half (k slots 0 .. 15: 16 of their dims) and of its second
//   (slots 16 .. 31: the same dims); columns 0 .. 7 hold the queries in the first slots and zeros in the others,
//   columns 8 .. 15 the reverse.  So a lane has 4 scores, none twice, and one row's address and words to deal with.
//   O^T: the weights of columns 0 .. 7 lie in the slots of the first half's positions, zeros in the others.
// The two halves of the columns are summed as if they were rows of their own, and joined with the waves'.  368
// instructions a tile, on 70% of the cycles.  845 MB of 8 sequences: 164 us at least in a kernel trace (5.2 TB/s;
// paged_decode_kernel 196), where the median of 20 is 210; 180 untraced, with the merge (205).  88 MB of 32: 28.4, median 30.5.
#pragma once
#include "rta_paged_decode.hpp"

namespace rta {

template <int HD>
struct Decode4Lds {
    static constexpr int kPitch = 2 * HD + 16;                  // bytes of a V row
    static constexpr int kQ = 16 * HD;                          // Q^T operands, of both halves; then as many zeros
    static constexpr int kV = kDecTile * kPitch;                // per wave: V, at the end U
    static constexpr int kPer = 8;                              // queries, those of either half
    static constexpr int kTotal = 2 * kQ + kDecWaves * kV + kDecWaves * kPer * 8;   // and (m, z) per wave and query
    static_assert(kPer * HD * 4 <= kV, "U of a wave's queries fits its V rows");
    static constexpr int kPerSimd = HD == 64 ? 5 : HD == 128 ? 4 : 2;   // waves per SIMD, by registers
};

template <int HD>
__global__ void __launch_bounds__(64 * kDecWaves, (Decode4Lds<HD>::kPerSimd)) paged_decode4_kernel(const PagedAttnArgs a) {
    using L = Decode4Lds<HD>;
    constexpr int FMT = RTA_Q4_GROUP;
    constexpr int kRow = page_row_bytes(FMT, HD), kScaleRow = page_scale_bytes(FMT, HD);
    constexpr int kGroups = HD / 32, kG = kGroups < 4 ? kGroups : 4;   // groups of a row, and of a block of its dwords
    constexpr int kLoads = HD / 64;             // 16-byte pieces per lane and row: half a row
    constexpr int kDt = HD / 16;                // dim tiles of O^T
    __shared__ __align__(16) uint8_t lds[L::kTotal];
    const int lane = threadIdx.x & 63, i = lane & 15, u = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int set = u >> 1, half = u & 1;       // the lane's row is position 16 set + i of a tile; half of its dims
    const int kvh = blockIdx.x % a.p.kv_heads;
    const int r = (int)((blockIdx.x / a.p.kv_heads + blockIdx.z) % a.l.rows);   // (turned, as in paged_decode_kernel)
    uint32_t err = 0;
    Visible see;
    const int32_t* table;
    if (!resolve_row(a, r, table, see, err)) {
        if (blockIdx.x == 0 && blockIdx.z == 0 && bad_rows(a.l)) err |= RTA_DEVERR_PAGES;
        if (err) raise_error(err);
        return;
    }
    const int cols = a.group;                   // <= 4
    const int begin = blockIdx.z * a.chunk, end = see.count - begin > a.chunk ? begin + a.chunk : see.count;
    if (begin >= end && blockIdx.z > 0) return;

    uint8_t* vl = lds + 2 * L::kQ + wave * L::kV;
    const int64_t plane = (int64_t)a.p.kv_heads * a.p.page;   // rows of a page's keys
    const int64_t v_off = plane * kRow, head_row = (int64_t)kvh * a.p.page;
    const int ntile = (end - begin + kDecTile - 1) / kDecTile;

    const Q4Bits q4;
    f4_t o[1][kDt];
    Softmax<1, 1, FMT> sm;
    sm.start();
#pragma unroll
    for (int d = 0; d < kDt; ++d) o[0][d] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
    // the lane's position of tile t, clamped to the last visible one: its page's number and place
    struct Spot {
        int page, off;
    };
    auto spot = [&](int t, Spot& s) {
        const int j = min(begin + t * kDecTile + 16 * set + i, end - 1);
        const uint32_t p = (uint32_t)see.position(j), e = a.p.by_page.div(p);
        s.off = (int)(p - e * a.p.page);
        s.page = table[e];
    };
    u4_t k[kLoads], v[kLoads];          // dword (block, y, x) of them: dims 32 x + 16 half + 8 y .. of the block
    uint32_t kw[kGroups / 2], vw[kGroups / 2];
    uint32_t live = 0;                  // positions of the tile in k that count
    const uint8_t *row, *words;
    auto aim = [&](int t, const Spot& s) {   // where tile t's rows are, and which count
        const bool have = (unsigned)s.page < (unsigned)a.p.n_pages;
        const bool in = begin + t * kDecTile + 16 * set + i < end;
        if (in && !have) err |= RTA_DEVERR_PAGES;
        const uint8_t* page = a.p.pool + page_offset(a.p, have ? s.page : 0);
        const int64_t at = head_row + s.off;
        row = page + at * kRow + 8 * kG * half;
        words = page + 2 * v_off + at * kScaleRow;
        const uint64_t on = __builtin_amdgcn_ballot_w64(in && have);
        live = ((uint32_t)on & 0xffffu) | (uint32_t)(on >> 32) << 16;
    };
    auto load = [&](const uint8_t* from, const uint8_t* w, u4_t* x, uint32_t* xw) {
#pragma unroll
        for (int b = 0; b < kLoads; ++b)   // (blocks of 128 dims have two pieces of 16 bytes a lane, of 64 one)
            x[b] = *reinterpret_cast<const u4_t*>(from + 64 * (b * 4 / (2 * kG)) + 16 * (b % (kG / 2)));
#pragma unroll
        for (int b = 0; b < kGroups / 2; ++b) xw[b] = reinterpret_cast<const uint32_t*>(w)[b];
    };
    auto load_kv = [&] {
        load(row, words, k, kw);
        load(row + v_off, words + plane * kScaleRow, v, vw);
    };
    // f(group, y, dword, words of the group's pair), the groups in order
    auto each = [&](const u4_t* x, const uint32_t* xw, auto&& f) {
#pragma unroll
        for (int g = 0; g < kGroups; g += 2) {
            const Q4Words two(xw[g / 2]);
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const int at = (g + e) / kG * 2 * kG + y * kG + (g + e) % kG;
                    const uint32_t w = x[at >> 2][at & 3];
                    f(g + e, y, e ? q4_to_half<1>(w, two, q4) : q4_to_half<0>(w, two, q4));
                }
        }
    };

    // the first tile's rows are on their way while q is prepared
    Spot next;
    if (wave < ntile) {
        spot(wave, next);
        aim(wave, next);
        load_kv();
        spot(wave + kDecWaves, next);   // clamped past the end
    }

    // q as B operands: entry (product, column & 7, half) has the dims that this half of a row feeds to the product
    const int part = i & 1, query = (i & 7) >> 1;
    const float kScale = kLog2e / sqrtf((float)HD);
    const float* q = a.q + r * a.q_stride + ((int64_t)kvh * a.group + min(query, cols - 1)) * HD;
    float mx = 0.0f;
#pragma unroll
    for (int j = 0; j < HD / 4; ++j) mx = fmaxf(mx, fabsf(q[u * (HD / 4) + j]));
    const int qe = part_exponent(max_xor32(max_xor16(mx)) * kScale);
    const float fac[1] = {ldexpf(1.0f, qe - 14)};   // score in log2 units = product * fac
    if (threadIdx.x < HD) {
        const int product = threadIdx.x >> 4, g = product >> 1, y = product & 1, of = (threadIdx.x >> 3) & 1;
        const float sg = ldexpf(kScale, 14 - qe);
        float x[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) x[s] = q[32 * g + 16 * of + 8 * y + s] * sg;
        u4_t op[1];
        split_parts<FMT, true>(x, part, op);
        *reinterpret_cast<u4_t*>(lds + threadIdx.x * 16) = op[0];
        *reinterpret_cast<u4_t*>(lds + L::kQ + threadIdx.x * 16) = u4_t{0, 0, 0, 0};
    }
    const uint8_t* ql = lds + (i >> 3 == set ? 0 : L::kQ) + ((i & 7) + 8 * half) * 16;
    const int mine = 16 * (i >> 3) + 4 * u;     // the lane's scores: positions mine .. mine + 3
    __syncthreads();

    for (int t = wave; t < ntile; t += kDecWaves) {
        const uint32_t now = live;
        const bool more = t + kDecWaves < ntile, whole = now == 0xffffffffu;
        // A position that does not count: zeros (scales of 0), keys too.  Its scores are masked, but a row of the product
        // holds a second position, which meets its values times zeros: NaN from what lies there without a page.
        if (!whole) {
            const bool on = (now >> (16 * set + i)) & 1u;
#pragma unroll
            for (int x = 0; x < kGroups / 2; ++x) {
                kw[x] = on ? kw[x] : 0u;
                vw[x] = on ? vw[x] : 0u;
            }
        }
        f4_t s[2] = {f4_t{0.0f, 0.0f, 0.0f, 0.0f}, f4_t{0.0f, 0.0f, 0.0f, 0.0f}};   // (neighbours go into different sums)
        each(k, kw, [&](int g, int y, u4_t ka) {
            s[y] = page_mfma<FMT>(ka, *reinterpret_cast<const u4_t*>(ql + (2 * g + y) * 256), s[y]);
        });
        // V into LDS, then the next tile's rows
        uint8_t* dst = vl + (16 * set + i) * L::kPitch + 32 * half;
        each(v, vw, [&](int g, int y, u4_t x) { *reinterpret_cast<u4_t*>(dst + 64 * g + 16 * y) = x; });
        if (more) {
            aim(t + kDecWaves, next);
            load_kv();
            spot(t + 2 * kDecWaves, next);
        }
        // Both parts of a score; the two columns have to come to the same weights bit by bit (paged_decode_kernel).
        f4_t x[1][1] = {{s[0] + s[1]}};
#pragma unroll
        for (int e = 0; e < 4; ++e) x[0][0][e] += dpp_mov<0xB1>(x[0][0][e]);
        sm.watch(x, whole);
        if (!whole) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[0][0][e] = seen_or_masked(x[0][0][e], (now >> (mine + e)) & 1u);
        }
        sm.raise(x, fac, 0, o, false, static_cast<const f4_t*>(nullptr));
        float w[8] = {};
        sm.weights(0, x[0], fac[0], w);
        u4_t op[1];
        split_parts<FMT>(w, part, op);
        const bool first = i < 8;
        const u4_t pb = {first ? op[0][0] : 0u, first ? op[0][1] : 0u, first ? 0u : op[0][0], first ? 0u : op[0][1]};
#pragma unroll
        for (int d = 0; d < kDt; ++d) {
            const uint8_t* src = vl + (4 * u + (i >> 2)) * L::kPitch + 32 * d + 8 * (i & 3);
            const s4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t*)src);
            const s4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t*)(src + 16 * L::kPitch));
            const uint2 l2 = __builtin_bit_cast(uint2, lo), h2 = __builtin_bit_cast(uint2, hi);
            o[0][d] = page_mfma<FMT>(u4_t{l2.x, l2.y, h2.x, h2.y}, pb, o[0][d]);
        }
    }
    if (sm.lowest == -INFINITY) err |= RTA_DEVERR_DETECTOR;   // (larger ones and NaN reach the results)

    // join: U per query of either half and dim in the wave's own LDS, then over waves and halves
    float2* mzl = reinterpret_cast<float2*>(lds + 2 * L::kQ + kDecWaves * L::kV);
    float M, back;
    sm.finish(0, fac[0], M, back);
    const float zz = sm.column_sum(sm.z[0]) * ldexpf(back, sm.kBack);
    if (lane < 16 && part == 0) mzl[wave * L::kPer + (i >> 1)] = float2{M, zz};
    float* ul = reinterpret_cast<float*>(vl) + (i >> 1) * HD;
#pragma unroll
    for (int d = 0; d < kDt; ++d) {
        f4_t x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = sm.settled(0, o[0][d][e] + dpp_mov<0xB1>(o[0][d][e]), back, 0);
        if (part == 0) *reinterpret_cast<f4_t*>(ul + 16 * d + 4 * u) = x;
    }
    __syncthreads();
    for (int at = threadIdx.x; at < cols * (HD / 4); at += 64 * kDecWaves) {
        const int j = at / (HD / 4), dim = 4 * (at - j * (HD / 4));
        float2 mz[2 * kDecWaves];
        float top = -INFINITY, Z = 0.0f;
#pragma unroll
        for (int w = 0; w < 2 * kDecWaves; ++w) {
            mz[w] = mzl[w * 4 + j];   // wave w / 2, half w % 2
            top = fmaxf(top, mz[w].x);
        }
        const float base = top == -INFINITY ? 0.0f : top;
        f4_t U = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < 2 * kDecWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(mz[w].x - base);
            Z += mz[w].y * f;
            U += *reinterpret_cast<const f4_t*>(lds + 2 * L::kQ + (w >> 1) * L::kV + ((4 * (w & 1) + j) * HD + dim) * 4) * f;
        }
        const int64_t row_head = (int64_t)r * a.hq + (int64_t)kvh * a.group + j;
        if (a.nchunk == 1) {
            write_result(a, row_head, HD, dim, U, top * kLn2, Z, err);
        } else {
            const int64_t rec = row_head * a.nchunk + blockIdx.z;
            *reinterpret_cast<f4_t*>(a.part + rec * HD + dim) = U;
            if (dim == 0) a.mz[rec] = float2{top, Z};
        }
    }
    if (blockIdx.x == 0 && blockIdx.z == 0 && bad_rows(a.l)) err |= RTA_DEVERR_PAGES;
    if (err) raise_error(err);
}

}  // namespace rta
