// rta_paged_decode.hpp -- attention of one row per sequence over its pages.
//
// Bound by the history's bytes: every visible key and value is read once per kv head (for more
// than 8 NC q heads per kv head once per group of those).  A workgroup of 4 waves takes one
// (row, kv head, chunk of visible positions); a wave takes every fourth tile of 32 positions and
// works alone until the end, so the waves of a compute unit (12 of them for 128-wide heads) drift apart
// and cover each other's waits:
//   lane (i, u) loads piece u of the rows of positions i and 16 + i, keys straight as the A
//   operand, values into LDS (32 rows, 16 bytes of padding each: the 16 rows that a transposing
//   read touches then fall on every bank exactly twice) and back transposed;
//   the next tile's keys go out as soon as the scores have been formed, its values as soon as
//   these are in LDS, its pages' numbers a tile earlier.
// The chunk's four (m, z, U) are joined in LDS, those of a row's chunks by paged_merge_kernel.
#pragma once
#include "rta_paged.hpp"

namespace rta {

typedef short s4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4_t lds_s4_t;

constexpr int kDecWaves = 4, kDecTile = 32;

template <int FMT, int HD, int NC, bool MULTI>
struct DecLds {
    static constexpr int kPitch = 2 * HD + 16;                                  // bytes of a V row
    static constexpr int kOps = MULTI ? PageFmt<FMT>::kParts : PageFmt<FMT>::kOps;
    static constexpr int kQ = NC * kOps * (HD / 32) * 64 * 16;                  // Q^T operands, of all waves
    static constexpr int kV = kDecTile * kPitch;                                // per wave: V, at the end U
    static constexpr int kS = PageFmt<FMT>::kScaled ? 2 * kDecTile * 4 : 0;     // per wave: the tile's scales
    static constexpr int kWave = kV + kS;
    static constexpr int kPer = MULTI ? 16 : 8;                                 // queries of a column tile
    static constexpr int kHeads = kPer * NC;
    static constexpr int kTotal = kQ + kDecWaves * kWave + kDecWaves * kPer * 8;   // and (m, z) per wave and head
    static_assert(kPer * HD * 4 <= kV, "U of a wave's queries fits its V rows");
    // waves per SIMD, by registers: 168 hold keys, values and sums of 128-wide heads
    static constexpr int kPerSimd =
        HD == 64 ? (NC == 1 && !MULTI ? 4 : NC == 1 ? 3 : 2) : HD == 128 ? (NC == 1 && !MULTI ? 3 : 2) : 1;
};

template <int FMT, int HD, int NC, bool MULTI>
__global__ void __launch_bounds__(64 * kDecWaves, (DecLds<FMT, HD, NC, MULTI>::kPerSimd)) paged_decode_kernel(const PagedAttnArgs a) {
    using L = DecLds<FMT, HD, NC, MULTI>;
    constexpr int kOps = L::kOps, kPer = L::kPer;
    constexpr int kRow = page_row_bytes(FMT, HD), kScaleRow = page_scale_bytes(FMT, HD);
    constexpr bool kQ4 = FMT == RTA_Q4_GROUP;
    constexpr int kKb = HD / 32;                // products per 16 positions
    constexpr int kPiece = kRow < 64 ? kRow / 4 : 16;    // bytes that a lane loads at once
    constexpr int kLoads = kRow / (4 * kPiece);          // pieces per lane and row
    constexpr int kWords = HD / 64;             // pairs of RTA_Q4_GROUP's words of a row
    constexpr int kDt = HD / 16;                // dim tiles of O^T
    constexpr bool kScaled = PageFmt<FMT>::kScaled;
    __shared__ __align__(16) uint8_t lds[L::kTotal];
    const int lane = threadIdx.x & 63, i = lane & 15, u = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Workgroups go round the 8 XCDs in order.  Heads first and rows turned by the chunk keep a long
    // row's chunks on all of them (rows first: 32 rows of 256 to 8192 bf16 positions 124 us, so 65)
    const int groups = MULTI ? 1 : (a.group + L::kHeads - 1) / L::kHeads;   // column groups of a kv head
    const int per_row = a.p.kv_heads * groups, y = blockIdx.x % per_row;
    const int turned = (int)((blockIdx.x / per_row + blockIdx.z) % (MULTI ? a.l.n : a.l.rows));
    const int kvh = MULTI ? y : y / groups, g0 = (y - kvh * groups) * L::kHeads;
    uint32_t err = 0;
    Visible see;
    const int32_t* table;
    // columns g0 .. g0 + cols - 1 of the entry: (row, head) pairs (MULTI), or the row's heads
    int row0 = turned, cols, t0 = 0;   // t0: the position of the entry's first row
    if constexpr (MULTI) {
        Entry en;
        const bool ok = resolve_entry(a, turned, en, err);
        if (kvh > 0) err &= ~RTA_DEVERR_PAGES;   // told once
        if (!ok) {
            if (err && threadIdx.x == 0) raise_error(err);
            return;
        }
        cols = en.rows * a.group;                // <= kHeads: max_rows bounds them
        row0 = en.base;
        table = en.table;
        t0 = en.len - en.count;
        see = en.len ? prompt_span(a, en.len, en.count, 0, L::kHeads) : Visible{0, 0, 0};
    } else {
        if (!resolve_row(a, turned, table, see, err)) {
            if (blockIdx.x == 0 && blockIdx.z == 0 && bad_rows(a.l)) err |= RTA_DEVERR_PAGES;
            if (err) raise_error(err);
            return;
        }
        cols = min(a.group - g0, L::kHeads);
    }
    const int begin = blockIdx.z * a.chunk, end = see.count - begin > a.chunk ? begin + a.chunk : see.count;
    // row and q head of column c (< cols)
    auto column = [&](int c, int& row, int& head) {
        const int at = g0 + c, tok = MULTI ? at / a.group : 0;
        row = row0 + tok;
        head = kvh * a.group + at - tok * a.group;
    };
    if (begin >= end && blockIdx.z > 0) {
        // (m, z) for paged_merge_kernel, which takes the chunks of a single row from its length instead
        // (ragged batches leave many empty: 72 us with them written for 32 of 256 to 8192, without 67.5)
        for (int c = threadIdx.x; MULTI && c < cols; c += 64 * kDecWaves) {
            int row, head;
            column(c, row, head);
            a.mz[((int64_t)row * a.hq + head) * a.nchunk + blockIdx.z] = float2{-INFINITY, 0.0f};
        }
        return;
    }

    uint8_t* vl = lds + L::kQ + wave * L::kWave;
    float* sl = reinterpret_cast<float*>(vl + L::kV);
    const int64_t plane = (int64_t)a.p.kv_heads * a.p.page;   // rows of a page's keys
    const int64_t v_off = plane * kRow, head_row = (int64_t)kvh * a.p.page, head_off = head_row * kRow;
    const int ntile = (end - begin + kDecTile - 1) / kDecTile;

    const Q4Bits q4;
    f4_t o[NC][kDt];
    Softmax<NC, 2, FMT> sm;
    sm.start();
    int ve = -110;   // exponent of the largest value scale so far
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        for (int d = 0; d < kDt; ++d) o[c][d] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // position i + 16 h of tile t: its page's number and place, clamped to the last visible one
    struct Spot {
        int page[2], off[2];
    };
    auto spot = [&](int t, Spot& s) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int j = min(begin + t * kDecTile + 16 * h + i, end - 1);
            const uint32_t p = (uint32_t)see.position(j), e = a.p.by_page.div(p);
            s.off[h] = (int)(p - e * a.p.page);
            s.page[h] = table[e];
        }
    };
    using Piece = std::conditional_t<kPiece == 16, u4_t, u2_t>;
    Piece k[2][kLoads], v[2][kLoads];
    float ks[2], vs[2];
    uint32_t kw[2][kWords], vw[2][kWords];
    uint32_t live = 0;   // positions of the tile in k that count
    const uint8_t* row[2];
    const uint8_t* srow[2];
    auto aim = [&](int t, const Spot& s) {   // where tile t's rows are, and which count
        uint32_t ok[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const bool have = (unsigned)s.page[h] < (unsigned)a.p.n_pages;
            const bool in = begin + t * kDecTile + 16 * h + i < end;
            if (in && !have) err |= RTA_DEVERR_PAGES;
            const uint8_t* page = a.p.pool + page_offset(a.p, have ? s.page[h] : 0);
            row[h] = page + head_off + (uint32_t)(s.off[h] * kRow + kPiece * u);
            srow[h] = page + 2 * v_off + (head_row + s.off[h]) * kScaleRow;
            ok[h] = (uint32_t)__builtin_amdgcn_ballot_w64(in && have) & 0xffffu;
        }
        live = ok[0] | ok[1] << 16;
    };
    auto load_k = [&] {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int x = 0; x < kLoads; ++x) k[h][x] = *reinterpret_cast<const Piece*>(row[h] + 4 * kPiece * x);
            if constexpr (kScaled) {
                ks[h] = *reinterpret_cast<const float*>(srow[h]);
                vs[h] = *reinterpret_cast<const float*>(srow[h] + plane * kScaleRow);
            }
            if constexpr (kQ4) {
#pragma unroll
                for (int x = 0; x < kWords; ++x) {
                    kw[h][x] = reinterpret_cast<const uint32_t*>(srow[h])[x];
                    vw[h][x] = reinterpret_cast<const uint32_t*>(srow[h] + plane * kScaleRow)[x];
                }
            }
        }
    };
    auto load_v = [&] {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int x = 0; x < kLoads; ++x) v[h][x] = *reinterpret_cast<const Piece*>(row[h] + v_off + 4 * kPiece * x);
    };

    // the first tile's rows are on their way while q is prepared
    Spot next;
    if (wave < ntile) {
        spot(wave, next);
        aim(wave, next);
        load_k();
        load_v();
        spot(wave + kDecWaves, next);   // clamped past the end
    }

    // q as B operands, one wave per quarter of the products.  Every wave finds the queries' largest
    // |q| (the power of two of binary16 operands).
    const int part = MULTI ? 0 : i & 1, query = MULTI ? i : i >> 1;   // lane's column of a column tile
    int t_col[NC];
    float fac[NC];   // score in log2 units = product * fac, a power of two; q takes log2 e / sqrt(HD) with it
    int qe[NC];
    const float kScale = kLog2e / sqrtf((float)HD);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        int row, head;
        column(min(kPer * c + query, cols - 1), row, head);
        t_col[c] = max(t0 + row - row0, -1);
        const float* q = a.q + row * a.q_stride + (int64_t)head * HD;
        qe[c] = 14;
        if constexpr (FMT != RTA_BF16) {
            float mx = 0.0f;
#pragma unroll
            for (int j = 0; j < HD / 4; ++j) mx = fmaxf(mx, fabsf(q[u * (HD / 4) + j]));
            qe[c] = part_exponent(max_xor32(max_xor16(mx)) * kScale);
        }
        fac[c] = ldexpf(1.0f, qe[c] - 14);
        for (int kb = wave; kb < kKb; kb += kDecWaves) {
            float v[8];
            const float sg = ldexpf(kScale, 14 - qe[c]);
#pragma unroll
            for (int s = 0; s < 8; ++s) v[s] = q[operand_dim<FMT>(kb, u) + s] * sg;
            u4_t op[kOps];
            if constexpr (MULTI) split_all<FMT, true>(v, op);
            else split_parts<FMT, true>(v, part, op);
#pragma unroll
            for (int o = 0; o < kOps; ++o)
                *reinterpret_cast<u4_t*>(lds + (((c * kOps + o) * kKb + kb) * 64 + lane) * 16) = op[o];
        }
    }
    int t_first = 0, t_last = 0;   // the columns' first and last positions
    if constexpr (MULTI) {
        t_first = t0;
        t_last = t0 + (cols - 1) / a.group;
    }
    __syncthreads();

    for (int t = wave; t < ntile; t += kDecWaves) {
        const uint32_t now = live;
        const bool more = t + kDecWaves < ntile;
        // every column sees the whole tile
        bool whole = now == 0xffffffffu;
        if constexpr (MULTI)
            whole = whole && see.position(begin + t * kDecTile + kDecTile - 1) <= t_first &&
                    (a.window == 0 || see.position(begin + t * kDecTile) > t_last - a.window);
        // scores of positions 4u + e (h = 0) and 16 + 4u + e (h = 1) in column i
        f4_t s[NC][2];
#pragma unroll
        for (int c = 0; c < NC; ++c) s[c][0] = s[c][1] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
        Q4Words kg[2] = {Q4Words(0), Q4Words(0)};   // of the products' pair of groups
#pragma unroll
        for (int kb = 0; kb < kKb; ++kb) {
            u4_t ka[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if constexpr (FMT == RTA_Q8_ROW) {
                    const int x = kb >> 1, b = 2 * (kb & 1);
                    uint32_t w[4];
                    codes_to_half(k[h][x][b], w[0], w[1]);
                    codes_to_half(k[h][x][b + 1], w[2], w[3]);
                    ka[h] = u4_t{w[0], w[1], w[2], w[3]};
                } else if constexpr (kQ4) {   // dword kb of a piece: dims 32 kb + 8 u ..
                    if (kb & 1) {
                        ka[h] = q4_to_half<1>(k[h][kb >> 2][kb & 3], kg[h], q4);
                    } else {
                        kg[h] = Q4Words(kw[h][kb >> 1]);
                        ka[h] = q4_to_half<0>(k[h][kb >> 2][kb & 3], kg[h], q4);
                    }
                } else {
                    ka[h] = k[h][kb];
                }
            }
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int op = 0; op < kOps; ++op) {
                    const u4_t qb = *reinterpret_cast<const u4_t*>(lds + (((c * kOps + op) * kKb + kb) * 64 + lane) * 16);
                    s[c][0] = page_mfma<FMT>(ka[0], qb, s[c][0]);
                    s[c][1] = page_mfma<FMT>(ka[1], qb, s[c][1]);
                }
        }
        // the tile's scales, from the lane of a position to the lanes that score it
        f4_t kf[2], vf[2];
        float mine[2];      // the value scales of the lane's positions that count, as far as they are finite
        int largest = 0;    // and the exponent of the tile's largest
        if constexpr (kScaled) {
#pragma unroll
            for (int h = 0; h < 2; ++h) mine[h] = ((now >> (16 * h + i)) & 1u) && fabsf(vs[h]) < INFINITY ? vs[h] : 0.0f;
            // (the four rows of 16 lanes hold the same positions)
            largest = __builtin_amdgcn_readfirstlane(part_exponent(group_max(fmaxf(fabsf(mine[0]), fabsf(mine[1])), 16)));
            if (u == 0) {
                sl[i] = ks[0];
                sl[16 + i] = ks[1];
                sl[32 + i] = vs[0];
                sl[48 + i] = vs[1];
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                kf[h] = *reinterpret_cast<const f4_t*>(sl + 16 * h + 4 * u);
                vf[h] = *reinterpret_cast<const f4_t*>(sl + 32 + 16 * h + 4 * u);
            }
        }
        uint32_t bad = 0;
        if (MULTI && !whole) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                bool hit = false;
                if constexpr (kScaled) {   // (the scale as its position's lanes hold it)
                    hit = !(fabsf(sl[32 + 16 * h + i]) < INFINITY);
#pragma unroll
                    for (int e = 0; e < 4; ++e) vf[h][e] = fabsf(vf[h][e]) < INFINITY ? vf[h][e] : 0.0f;
                } else if constexpr (kQ4) {
#pragma unroll
                    for (int x = 0; x < kWords; ++x)
                        if (q4_not_finite(vw[h][x])) {   // (a scale of 0: zeros)
                            vw[h][x] = 0;
                            hit = true;
                        }
                } else {
#pragma unroll
                    for (int x = 0; x < kLoads; ++x)
                        if (piece_not_finite<FMT>(v[h][x])) {
                            v[h][x] = u4_t{0, 0, 0, 0};
                            hit = true;
                        }
                }
                uint64_t rows = __builtin_amdgcn_ballot_w64(hit);   // bit 16 u + i: a piece of row i
                rows |= rows >> 32;
                bad |= (uint32_t)((rows | rows >> 16) & 0xffffu) << (16 * h);
            }
            bad &= now;
        }
        // V into LDS (rows that do not count as zeros), then the next tile's rows
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (now != 0xffffffffu) {   // uniform: the last tile, or one with a page missing
                const bool on = (now >> (16 * h + i)) & 1u;
#pragma unroll
                for (int x = 0; x < (kQ4 ? 0 : kLoads); ++x) v[h][x] = on ? v[h][x] : (Piece)(0u);
                if constexpr (kQ4) {   // a scale of 0
#pragma unroll
                    for (int x = 0; x < kWords; ++x) vw[h][x] = on ? vw[h][x] : 0u;
                }
                if constexpr (kScaled) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) vf[h][e] = (now >> (16 * h + 4 * u + e)) & 1u ? vf[h][e] : 0.0f;
                }
            }
            uint8_t* dst = vl + (16 * h + i) * L::kPitch;
            if constexpr (kQ4) {
#pragma unroll
                for (int x = 0; x < kKb; x += 2) {
                    const Q4Words g(vw[h][x >> 1]);
                    *reinterpret_cast<u4_t*>(dst + 64 * x + 16 * u) = q4_to_half<0>(v[h][x >> 2][x & 3], g, q4);
                    *reinterpret_cast<u4_t*>(dst + 64 * x + 64 + 16 * u) = q4_to_half<1>(v[h][x >> 2][(x & 3) + 1], g, q4);
                }
            }
#pragma unroll
            for (int x = 0; x < (kQ4 ? 0 : kLoads); ++x) {
                if constexpr (FMT == RTA_Q8_ROW) {
                    uint32_t w[8];
#pragma unroll
                    for (int y = 0; y < 4; ++y) codes_to_half(v[h][x][y], w[2 * y], w[2 * y + 1]);
                    *reinterpret_cast<u4_t*>(dst + 128 * x + 32 * u) = u4_t{w[0], w[1], w[2], w[3]};
                    *reinterpret_cast<u4_t*>(dst + 128 * x + 32 * u + 16) = u4_t{w[4], w[5], w[6], w[7]};
                } else if constexpr (!kQ4) {
                    *reinterpret_cast<u4_t*>(dst + 64 * x + 16 * u) = v[h][x];
                }
            }
        }
        if (more) {
            aim(t + kDecWaves, next);
            load_k();
            load_v();
            spot(t + 2 * kDecWaves, next);
        }
        // Both parts of a score.  The two columns have to come to the same weights bit by bit, since
        // one takes its upper part and the other the rest: so their sum comes first (behind a
        // product it could be contracted, to one rounding here and another there).
        if constexpr (!MULTI) {
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int j = 0; j < 8; ++j) s[c][j >> 2][j & 3] += dpp_mov<0xB1>(s[c][j >> 2][j & 3]);
        }
        int ve_new = ve;
        bool spread = false;
        if constexpr (kScaled) {   // value scales below 2^0
            ve_new = max(ve, largest);
            spread = __builtin_amdgcn_ballot_w64(far_below(mine[0], ve_new) || far_below(mine[1], ve_new)) != 0;
            const float down = ldexpf(1.0f, -ve_new);
            vf[0] *= down;
            vf[1] *= down;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                s[c][0] *= kf[0];
                s[c][1] *= kf[1];
            }
        }
        sm.watch(s, whole);
        if (!whole) {
            if constexpr (MULTI) {
                mask_columns<NC>(s, now, see, begin + t * kDecTile, u, t_col, a.window, a.sinks);
                if (bad) sm.poison(s, bad, u);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const bool on = (now >> (16 * (j >> 2) + 4 * u + (j & 3))) & 1u;
#pragma unroll
                    for (int c = 0; c < NC; ++c) s[c][j >> 2][j & 3] = seen_or_masked(s[c][j >> 2][j & 3], on);
                }
            }
        }
        sm.raise(s, fac, kScaled ? ve - ve_new : 0, o, spread, vf);
        ve = ve_new;
        u4_t pb[NC][kOps];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float w[8];
            sm.weights(c, s[c], fac[c], w);
            if constexpr (kScaled) {
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] *= vf[j >> 2][j & 3];
                if (spread) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) w[j] = ldexpf(w[j], sm.up[c]);
                }
            }
            if constexpr (MULTI) split_all<FMT>(w, pb[c]);
            else split_parts<FMT>(w, part, pb[c]);
        }
#pragma unroll
        for (int d = 0; d < kDt; ++d) {
            const uint8_t* src = vl + (4 * u + (i >> 2)) * L::kPitch + 32 * d + 8 * (i & 3);
            const s4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t*)src);
            const s4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t*)(src + 16 * L::kPitch));
            const uint2 l2 = __builtin_bit_cast(uint2, lo), h2 = __builtin_bit_cast(uint2, hi);
            const u4_t va = {l2.x, l2.y, h2.x, h2.y};
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int op = 0; op < kOps; ++op) o[c][d] = page_mfma<FMT>(va, pb[c][op], o[c][d]);
        }
    }
    if (sm.lowest == -INFINITY) err |= RTA_DEVERR_DETECTOR;   // (larger ones and NaN reach the results)

    // join: U per query and dim in the wave's own LDS, then over the waves
    float2* mzl = reinterpret_cast<float2*>(lds + L::kQ + kDecWaves * L::kWave);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        float M, back;
        sm.finish(c, fac[c], M, back);
        const float zz = sm.column_sum(sm.z[c]) * ldexpf(back, sm.kBack);
        if (lane < 16 && part == 0) mzl[wave * kPer + query] = float2{M, zz};
        float* ul = reinterpret_cast<float*>(vl) + query * HD;
#pragma unroll
        for (int d = 0; d < kDt; ++d) {
            f4_t x;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                x[e] = sm.settled(c, MULTI ? o[c][d][e] : o[c][d][e] + dpp_mov<0xB1>(o[c][d][e]), back, ve);
            if (part == 0) *reinterpret_cast<f4_t*>(ul + 16 * d + 4 * u) = x;
        }
        __syncthreads();
        for (int at = threadIdx.x; at < min(kPer, cols - kPer * c) * (HD / 4); at += 64 * kDecWaves) {
            const int j = at / (HD / 4), dim = 4 * (at - j * (HD / 4));
            float2 mz[kDecWaves];
            float M = -INFINITY, Z = 0.0f;
#pragma unroll
            for (int w = 0; w < kDecWaves; ++w) {
                mz[w] = mzl[w * kPer + j];
                M = fmaxf(M, mz[w].x);
            }
            const float base = M == -INFINITY ? 0.0f : M;
            f4_t U = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < kDecWaves; ++w) {
                const float f = __builtin_amdgcn_exp2f(mz[w].x - base);
                Z += mz[w].y * f;
                U += reinterpret_cast<const f4_t*>(lds + L::kQ + w * L::kWave)[at] * f;
            }
            int row, head;
            column(kPer * c + j, row, head);
            const int64_t row_head = (int64_t)row * a.hq + head;
            if (a.nchunk == 1) {
                write_result(a, row_head, HD, dim, U, M * kLn2, Z, err);
            } else {
                const int64_t rec = row_head * a.nchunk + blockIdx.z;
                *reinterpret_cast<f4_t*>(a.part + rec * HD + dim) = U;
                if (dim == 0) a.mz[rec] = float2{M, Z};
            }
        }
        if (c + 1 < NC) __syncthreads();
    }
    // (at the end: ahead of the first loads it took single rows of 32 sequences over 4000 positions 2% longer)
    if (!MULTI && blockIdx.x == 0 && blockIdx.z == 0 && bad_rows(a.l)) err |= RTA_DEVERR_PAGES;
    if (err) raise_error(err);
}

}  // namespace rta
