// rta_paged_prompt.hpp -- causal attention of several rows per sequence over its pages.
//
// Bound by the matrix cores and, beside them, by vector instructions: 4 hq HD operations per
// (row, position), twice that with q and the weights in two binary16 parts, three times in three
// bfloat16 parts (rta_paged.hpp), and about 200 vector instructions per 32 x 32 scores, of which
// two waves of a SIMD hide some.  4096 rows of 32 heads over 4096 bf16 positions: 348 to 360 us, three
// parts at the rate of a large library product 350; the matrix cores are busy 45% of it (binary16
// pages 311 to 320 us, 38%; 8-bit ones 345 to 351, 32%).
// The columns of a kv head's products are its (row, q head) pairs, so the heads that share keys
// share their loads and no group size leaves columns empty.  A workgroup of 4 waves takes 128 (wide
// heads: 64) columns and the positions that any of them sees, in tiles staged in LDS by all of it
// (two buffers, one barrier per tile); each wave keeps its q operands, running maxima and sums, and
// O^T in registers.  A tile that every column of a wave sees whole takes no masks, one that no
// column sees is skipped.  The last rows, which see most, come first; kv heads go over the XCDs, so
// that one L2 serves all rows of a head.  With few workgroups the positions are cut into chunks as
// well, joined by paged_merge_kernel.
#pragma once
#include "rta_paged_decode.hpp"

namespace rta {

template <int FMT, int HD>
struct PromptLds {
    static constexpr int kTile = HD > 64 ? 32 : 64;    // positions per tile
    // a wave's columns are NQ tiles of kWide (32: half the matrix instructions and one column per lane,
    // 64-wide heads 111 -> 97 us, 128-wide 163 -> 153; with bfloat16's third part, which comes from
    // LDS between them, 348 -> 378 us)
    static constexpr int kWide = HD == 256 || FMT == RTA_BF16 ? 16 : 32;
    static constexpr int kNQ = HD == 256 ? 1 : 32 / kWide;
    static constexpr int kCols = 4 * kWide * kNQ;      // columns of a workgroup
    // Bytes of a row: 16 of padding spread the rows of a key operand over the banks, and the 16 rows
    // that a transposing read of values touches, 32 bytes each; 8 rows of 64 bytes need 64.
    static constexpr int kPitch = 2 * HD + 16, kPitchV = 2 * HD + (kWide == 32 ? 64 : 16);
    static constexpr int kKeys = kTile * kPitch, kRows = kKeys + kTile * kPitchV;
    static constexpr int kScales = PageFmt<FMT>::kScaled ? 2 * kTile * 4 : 0;
    static constexpr int kBuf = kRows + kScales + kTile * 4;   // and which rows count
    static constexpr int kThird = FMT == RTA_BF16 ? kNQ * kWide * HD * 2 : 0;   // per wave: q's third part
    static constexpr int kTotal = 2 * kBuf + 4 * kThird;
};

template <int FMT, int HD>
__global__ void __launch_bounds__(256, (PromptLds<FMT, HD>::kTotal > 80 << 10 ? 1 : 2)) paged_prompt_kernel(const PagedAttnArgs a) {
    using L = PromptLds<FMT, HD>;
    constexpr int kParts = PageFmt<FMT>::kParts, kRow = page_row_bytes(FMT, HD);
    constexpr bool kQ4 = FMT == RTA_Q4_GROUP;
    // products: kDims dims of kWide positions, kH of them for 32 positions, then kWide dims of
    // 32 / kP positions; kKg and kDg of them have their operands read ahead
    constexpr int W = L::kWide, NQ = L::kNQ, kDims = 512 / W, kH = 32 / W, kP = W / 16, N = W / 8;
    constexpr int kKb = HD / kDims, kDt = HD / W, kKg = kKb * kH < 8 ? kKb : 8 / kH;
    constexpr int kDg = kDt < 4 ? kDt : 4, kDn = kP * kDt / kDg;   // V^T: kDn groups of kDg operands
    using Acc = std::conditional_t<W == 32, acc16_t, f4_t>;
    constexpr int kQuads = sizeof(Acc) / 16;
    // (RTA_Q4_GROUP: a dword, which becomes 16 bytes, so as many threads a row as with 2-byte elements)
    using Piece = std::conditional_t<kQ4, uint32_t, u4_t>;
    constexpr int kPieces = kRow / (int)sizeof(Piece), kStep = 256 / kPieces, kPass = L::kTile / kStep;
    constexpr bool kScaled = PageFmt<FMT>::kScaled;
    __shared__ __align__(16) uint8_t lds[L::kTotal];
    const int tid = threadIdx.x, lane = tid & 63, i = lane & (W - 1), u = lane / W;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hkv = a.p.kv_heads;
    const int kvh = blockIdx.x % hkv, rest = blockIdx.x / hkv;
    const int entry = rest % a.l.n, tile = a.ntile - 1 - rest / a.l.n;
    uint32_t err = 0;
    Entry en;
    const bool ok = resolve_entry(a, entry, en, err);
    if (tile > 0) err &= ~RTA_DEVERR_PAGES;   // the first tile tells
    if (!ok) {
        if (err && tid == 0) raise_error(err);
        return;
    }
    if ((int64_t)tile * L::kCols >= (int64_t)en.rows * a.group) return;
    const int base = en.base, count = en.count, live_rows = en.rows, len = en.len;
    const int32_t* table = en.table;
    const Visible see = len ? prompt_span(a, len, count, tile, L::kCols) : Visible{0, 0, 0};
    const int begin = blockIdx.z * a.chunk, end = see.count - begin > a.chunk ? begin + a.chunk : see.count;
    if (begin >= end && blockIdx.z > 0) {   // for paged_merge_kernel, which reads every chunk's
        const int64_t col = (int64_t)tile * L::kCols + tid;
        if (tid < L::kCols && col < (int64_t)live_rows * a.group) {
            const int64_t tok = col / a.group, at = (base + tok) * a.hq + (int64_t)kvh * a.group + (col - tok * a.group);
            a.mz[at * a.nchunk + blockIdx.z] = float2{-INFINITY, 0.0f};
        }
        return;
    }
    const int nt = (end - begin + L::kTile - 1) / L::kTile;

    // staging: thread -> piece of a row; its rows of a tile are kStep apart
    const int64_t plane = (int64_t)hkv * a.p.page, v_off = plane * kRow;
    const int64_t head_row = (int64_t)kvh * a.p.page, head_off = head_row * kRow;
    const int piece = tid % kPieces, row0 = tid / kPieces;
    const int dim = q4_dim(HD, piece);   // RTA_Q4_GROUP: the piece's first dim
    struct Spot {
        int page[kPass], off[kPass];
    };
    auto spot = [&](int t, Spot& sp) {
#pragma unroll
        for (int k = 0; k < kPass; ++k) {
            const int j = min(begin + t * L::kTile + row0 + k * kStep, end - 1);
            const uint32_t p = (uint32_t)see.position(j), e = a.p.by_page.div(p);
            sp.off[k] = (int)(p - e * a.p.page);
            sp.page[k] = table[e];
        }
    };
    Piece kr[kPass], vr[kPass];
    float ksr[kPass], vsr[kPass];
    uint32_t kw[kPass], vw[kPass];
    uint32_t okr = 0;
    auto load = [&](int t, const Spot& sp) {
        okr = 0;
#pragma unroll
        for (int k = 0; k < kPass; ++k) {
            const bool have = (unsigned)sp.page[k] < (unsigned)a.p.n_pages;
            const bool in = begin + t * L::kTile + row0 + k * kStep < end;
            if (in && !have) err |= RTA_DEVERR_PAGES;
            if (in && have) okr |= 1u << k;
            const uint8_t* page = a.p.pool + page_offset(a.p, have ? sp.page[k] : 0);
            const uint8_t* src = page + head_off + (uint32_t)(sp.off[k] * kRow + (int)sizeof(Piece) * piece);
            kr[k] = *reinterpret_cast<const Piece*>(src);
            vr[k] = *reinterpret_cast<const Piece*>(src + v_off);
            if constexpr (kQ4) {
                const uint16_t* w = reinterpret_cast<const uint16_t*>(page + 2 * v_off) + (head_row + sp.off[k]) * (HD / 32) + (dim >> 5);
                kw[k] = w[0];
                vw[k] = w[plane * (HD / 32)];
            }
            if constexpr (kScaled) {
                const float* f = reinterpret_cast<const float*>(page + 2 * v_off) + head_row + sp.off[k];
                ksr[k] = f[0];
                vsr[k] = f[plane];
            }
        }
    };
    const Q4Bits q4;
    auto put = [&](uint8_t* dst, Piece x, uint32_t word) {   // one piece as 2-byte elements
        if constexpr (kQ4) {
            *reinterpret_cast<u4_t*>(dst + 2 * dim) = q4_to_half<0>(x, Q4Words(word), q4);
        } else if constexpr (FMT == RTA_Q8_ROW) {
            uint32_t w[8];
#pragma unroll
            for (int y = 0; y < 4; ++y) codes_to_half(x[y], w[2 * y], w[2 * y + 1]);
            *reinterpret_cast<u4_t*>(dst + 32 * piece) = u4_t{w[0], w[1], w[2], w[3]};
            *reinterpret_cast<u4_t*>(dst + 32 * piece + 16) = u4_t{w[4], w[5], w[6], w[7]};
        } else {
            *reinterpret_cast<u4_t*>(dst + 16 * piece) = x;
        }
    };
    // the rows' first and last positions: tiles that all of them see whole need no care for values
    // that are not finite
    const int lo = len - count + tile * L::kCols / a.group;
    const int hi = len - count + min((tile + 1) * L::kCols - 1, live_rows * a.group - 1) / a.group;
    auto store = [&](int t, uint8_t* buf) {
        // rows that do not count are zeros: a weight of 0 times what lies there must be 0
        if (__builtin_amdgcn_ballot_w64(okr != (1u << kPass) - 1)) {   // the last tile, or a page missing
#pragma unroll
            for (int k = 0; k < kPass; ++k)
                if (!((okr >> k) & 1u)) {
                    kr[k] = vr[k] = (Piece)(0u);
                    if constexpr (kQ4) kw[k] = vw[k] = 0;   // (scales)
                    if constexpr (kScaled) ksr[k] = vsr[k] = 0.0f;
                }
        }
        uint32_t bad = 0;
        const int j0 = begin + t * L::kTile;
        if (see.position(min(j0 + L::kTile, end) - 1) > lo || (a.window && see.position(j0) <= hi - a.window)) {
#pragma unroll
            for (int k = 0; k < kPass; ++k) {
                if constexpr (kScaled) {
                    if (!(fabsf(vsr[k]) < INFINITY)) {
                        vsr[k] = 0.0f;
                        bad |= 1u << k;
                    }
                } else {   // a row's threads are of one wave
                    constexpr uint64_t kLanes = kPieces == 32 ? 0xffffffffull : (1ull << kPieces) - 1;
                    bool hit;
                    if constexpr (kQ4) hit = q4_not_finite(vw[k]);
                    else hit = piece_not_finite<FMT>(vr[k]);
                    if (hit) {
                        vr[k] = (Piece)(0u);
                        if constexpr (kQ4) vw[k] = 0;
                    }
                    if (__builtin_amdgcn_ballot_w64(hit) & (kLanes << (lane & ~(kPieces - 1)))) bad |= 1u << k;
                }
            }
        }
#pragma unroll
        for (int k = 0; k < kPass; ++k) {
            const int row = row0 + k * kStep;
            put(buf + row * L::kPitch, kr[k], kw[k]);
            put(buf + L::kKeys + row * L::kPitchV, vr[k], vw[k]);
            if (piece == 0) {
                if constexpr (kScaled) {
                    float* f = reinterpret_cast<float*>(buf + L::kRows);
                    f[row] = ksr[k];
                    f[L::kTile + row] = vsr[k];
                }
                reinterpret_cast<uint32_t*>(buf + L::kRows + L::kScales)[row] = ((okr >> k) & 1u) | ((bad >> k) & 1u) << 1;
            }
        }
    };
    Spot next;
    if (nt > 0) {
        spot(0, next);
        load(0, next);
        spot(1, next);
    }

    // the lane's columns: (row, head) pairs, their positions and q operands
    const int col0 = tile * L::kCols + wave * W * NQ, cols = live_rows * a.group;
    const bool on = col0 < cols;   // uniform: this wave has columns
    int t_col[NQ];
    u4_t qb[NQ][kKb][2];   // (the third part of bfloat16 lies in LDS: its registers would leave none for operands)
    u4_t* third = reinterpret_cast<u4_t*>(lds + 2 * L::kBuf + wave * L::kThird) + lane;
    float fac[NQ];
    const float kScale = kLog2e / sqrtf((float)HD);   // (into q: then a score is its product times a power of two)
    auto column = [&](int c, int& tok, int& head) {   // past the last one: the last
        const int col = min(col0 + W * c + i, cols - 1);
        tok = col / a.group;
        head = kvh * a.group + col - tok * a.group;
    };
#pragma unroll
    for (int c = 0; c < NQ; ++c) {
        int tok, head;
        column(c, tok, head);
        t_col[c] = max(len - count + tok, -1);
        const float* q = a.q + (int64_t)(base + tok) * a.q_stride + (int64_t)head * HD;
        float v[kKb][8], mx = 0.0f;
#pragma unroll
        for (int kb = 0; kb < kKb; ++kb)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[kb][e] = q[kDims * kb + 8 * u + e];
                mx = fmaxf(mx, fabsf(v[kb][e]));
            }
        int qe = 14;
        if constexpr (FMT != RTA_BF16) qe = part_exponent(Softmax<NQ, N, FMT>::column_max(mx) * kScale);
        const float sg = ldexpf(kScale, 14 - qe);
        fac[c] = ldexpf(1.0f, qe - 14);
#pragma unroll
        for (int kb = 0; kb < kKb; ++kb) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[kb][e] *= sg;
            u4_t part[kParts];
            split_all<FMT, true>(v[kb], part);
            qb[c][kb][0] = part[0];
            qb[c][kb][1] = part[1];
            if constexpr (kParts == 3) third[(c * kKb + kb) * 64] = part[2];
        }
    }
    // the wave's first and last positions
    const int t_lo = len - count + col0 / a.group;
    const int t_hi = len - count + min(col0 + W * NQ - 1, cols - 1) / a.group;

    Acc o[NQ][kDt];
    Softmax<NQ, N, FMT> sm;
    sm.start();
    int ve = -110;
#pragma unroll
    for (int c = 0; c < NQ; ++c)
#pragma unroll
        for (int d = 0; d < kDt; ++d)
#pragma unroll
            for (int e = 0; e < 4 * kQuads; ++e) o[c][d][e] = 0.0f;
    if (nt > 0) store(0, lds);
    __syncthreads();

    for (int t = 0; t < nt; ++t) {
        const uint8_t* buf = lds + (t & 1) * L::kBuf;
        if (t + 1 < nt) {
            load(t + 1, next);
            spot(t + 2, next);
        }
        const int j0 = begin + t * L::kTile, j1 = min(j0 + L::kTile, end) - 1;
        const int p0 = see.position(j0), p1 = see.position(j1);
        if (on && p0 <= t_hi) {
            uint32_t row_state = reinterpret_cast<const uint32_t*>(buf + L::kRows + L::kScales)[lane & (L::kTile - 1)];
            if (L::kTile < 64 && lane >= L::kTile) row_state = 0;
            const uint64_t okm = __builtin_amdgcn_ballot_w64(row_state != 0), badm = __builtin_amdgcn_ballot_w64(row_state > 1);
            const bool whole = okm == (L::kTile == 64 ? ~0ull : 0xffffffffull) && badm == 0 && p1 <= t_lo &&
                               (a.window == 0 || p0 > t_hi - a.window);
            const float* sc = reinterpret_cast<const float*>(buf + L::kRows);
            float wscale = 1.0f;
            int ve_new = ve;
            bool spread = false;
            if constexpr (kScaled) {   // value scales below 2^0
                const float mx = lane < L::kTile ? fabsf(sc[L::kTile + lane]) : 0.0f;
                ve_new = max(ve, __builtin_amdgcn_readfirstlane(part_exponent(wave_max_dpp(mx))));
                spread = __builtin_amdgcn_ballot_w64(far_below(mx, ve_new)) != 0;
                wscale = ldexpf(1.0f, -ve_new);
            }
#pragma unroll
            for (int sub = 0; sub < L::kTile / 32; ++sub) {
                // S^T of 32 positions
                Acc st[NQ][kH];
#pragma unroll
                for (int c = 0; c < NQ; ++c)
#pragma unroll
                    for (int h = 0; h < kH; ++h)
#pragma unroll
                        for (int e = 0; e < 4 * kQuads; ++e) st[c][h][e] = 0.0f;
#pragma unroll
                for (int k0 = 0; k0 < kKb; k0 += kKg) {
                    u4_t ka[kKg][kH];   // all on their way before the first product
#pragma unroll
                    for (int k = 0; k < kKg; ++k)
#pragma unroll
                        for (int h = 0; h < kH; ++h)
                            ka[k][h] = *reinterpret_cast<const u4_t*>(buf + (32 * sub + W * h + i) * L::kPitch +
                                                                      2 * kDims * (k0 + k) + 16 * u);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int k = 0; k < kKg; ++k)
#pragma unroll
                        for (int p = 0; p < kParts; ++p)   // neighbours go into different accumulators
#pragma unroll
                            for (int c = 0; c < NQ; ++c) {
                                const u4_t q = p < 2 ? qb[c][k0 + k][p & 1] : third[(c * kKb + k0 + k) * 64];
#pragma unroll
                                for (int h = 0; h < kH; ++h) st[c][h] = page_mfma<FMT>(ka[k][h], q, st[c][h]);
                            }
                }
                // the first of V^T's operands, ready when the weights are
                const uint8_t* vb = buf + L::kKeys + (32 * sub + 4 * u + ((lane & 15) >> 2)) * L::kPitchV +
                                    32 * (i >> 4) + 8 * (lane & 3);
                u4_t va[2][kDg];
                auto load_va = [&](int n) {   // group n: dim tiles d0 .. of positions 32 / kP h ..
                    const int h = n * kDg / kDt, d0 = n * kDg % kDt;
#pragma unroll
                    for (int d = 0; d < kDg; ++d) {
                        const uint8_t* src = vb + 2 * W * (d0 + d) + 16 * h * L::kPitchV;
                        const s4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t*)src);
                        const s4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t*)(src + 16 / kP * L::kPitchV));
                        const uint2 l2 = __builtin_bit_cast(uint2, lo), h2 = __builtin_bit_cast(uint2, hi);
                        va[n & 1][d] = u4_t{l2.x, l2.y, h2.x, h2.y};
                    }
                };
                load_va(0);
                __builtin_amdgcn_sched_barrier(0);
                f4_t x[NQ][N], vf[N];   // positions 32 / N h + 4 u + e
#pragma unroll
                for (int c = 0; c < NQ; ++c)
#pragma unroll
                    for (int h = 0; h < N; ++h) x[c][h] = quad_of(st[c][h / kQuads], h % kQuads);
                if constexpr (kScaled) {
#pragma unroll
                    for (int h = 0; h < N; ++h) {
                        const float* at = sc + 32 * sub + 32 / N * h + 4 * u;
                        const f4_t kf = *reinterpret_cast<const f4_t*>(at);
                        vf[h] = *reinterpret_cast<const f4_t*>(at + L::kTile) * wscale;
#pragma unroll
                        for (int c = 0; c < NQ; ++c) x[c][h] *= kf;
                    }
                }
                sm.watch(x, whole);
                if (!whole) {
                    mask_columns<NQ>(x, (uint32_t)(okm >> (32 * sub)), see, j0 + 32 * sub, u, t_col, a.window, a.sinks);
                    if (badm) sm.poison(x, (uint32_t)(badm >> (32 * sub)), u);
                }
                sm.raise(x, fac, kScaled ? ve - ve_new : 0, o, spread, vf);
                ve = ve_new;
                if constexpr (kScaled) {
                    static_assert(NQ == 1, "the value scales take on one column's power of two");
                    if (spread) {
                        const float by = ldexpf(1.0f, sm.up[0]);
#pragma unroll
                        for (int h = 0; h < N; ++h) vf[h] *= by;
                    }
                }
                // O^T += V^T P^T
                u4_t pb[NQ][kP][kParts];
#pragma unroll
                for (int n = 0; n < kDn; ++n) {
                    const int h = n * kDg / kDt, d0 = n * kDg % kDt;
#pragma unroll
                    for (int c = 0; c < NQ && d0 == 0; ++c) {
                        float w[8];
                        sm.weights(c, x[c] + 2 * h, fac[c], w);
                        if constexpr (kScaled) {
#pragma unroll
                            for (int e = 0; e < 8; ++e) w[e] *= vf[2 * h + (e >> 2)][e & 3];
                        }
                        split_all<FMT>(w, pb[c][h]);
                    }
                    if (n + 1 < kDn) {
                        load_va(n + 1);
                        if constexpr (kP == 1) __builtin_amdgcn_sched_barrier(0);
                    }
#pragma unroll
                    for (int p = 0; p < kParts; ++p)
#pragma unroll
                        for (int d = 0; d < kDg; ++d)
#pragma unroll
                            for (int c = 0; c < NQ; ++c)
                                o[c][d0 + d] = page_mfma<FMT>(va[n & 1][d], pb[c][h][p], o[c][d0 + d]);
                }
            }
        }
        if (t + 1 < nt) store(t + 1, lds + ((t + 1) & 1) * L::kBuf);
        __syncthreads();
    }

    if (sm.lowest == -INFINITY) err |= RTA_DEVERR_DETECTOR;   // (larger ones and NaN reach the results)
#pragma unroll
    for (int c = 0; c < NQ; ++c) {
        float M, back;
        sm.finish(c, fac[c], M, back);
        const float Z = sm.column_sum(sm.z[c]) * ldexpf(back, sm.kBack);
        if (col0 + W * c + i >= cols) continue;
        int tok, head;
        column(c, tok, head);
        const int64_t at = (int64_t)(base + tok) * a.hq + head, rec = at * a.nchunk + blockIdx.z;
        if (a.nchunk > 1 && u == 0) a.mz[rec] = float2{M, Z};
#pragma unroll
        for (int d = 0; d < kDt; ++d)
#pragma unroll
            for (int h = 0; h < kQuads; ++h) {
                const int dim = W * d + 8 * h + 4 * u;
                f4_t U = quad_of(o[c][d], h);
#pragma unroll
                for (int e = 0; e < 4; ++e) U[e] = sm.settled(c, U[e], back, ve);
                if (a.nchunk > 1) *reinterpret_cast<f4_t*>(a.part + rec * HD + dim) = U;
                else write_result(a, at, HD, dim, U, M * kLn2, Z, err);
            }
    }
    if (err) raise_error(err);
}

// Joins the chunks of a (row, q head): M = max m, o = sum U e^(m - M) / sum z e^(m - M).  HD / 4
// lanes of 4 dims by the rest of 256 threads over the chunks.  Bound by latency: a trip for the
// (m, z), beside the search for the row's entry, and one for the U of the chunks that see something.
// (Of several rows per entry every chunk has its (m, z); found from the row's length, which chunks
// there are took the kernel 9.5 us after 16 x 5 rows of 9 chunks, so 5.7.)
template <int HD>
__global__ void __launch_bounds__(256) paged_merge_kernel(const PagedAttnArgs a) {
    constexpr int kLanes = HD / 4, kRows = 256 / kLanes;
    __shared__ f4_t us[kRows][kLanes];
    __shared__ float red[4], zred[4];
    const int r = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
    const int64_t at = (int64_t)r * a.hq + h;
    const float2* mz = a.mz + at * a.nchunk;
    float m = tid < a.nchunk ? mz[tid].x : -INFINITY;
    int n = a.nchunk;
    uint32_t err = 0;   // the chunks have reported what is wrong
    if (a.ntile) {
        int i, first, count;
        if (!row_entry(a.l, r, i, first, count) || r - first >= a.max_rows) return;
    } else {
        Visible see;
        const int32_t* table;
        if (!resolve_row(a, r, table, see, err)) return;
        n = (int)(((int64_t)see.count + a.chunk - 1) / a.chunk);
        if (tid >= n) m = -INFINITY;
    }
    err = 0;
    for (int c = tid + 256; c < n; c += 256) m = fmaxf(m, mz[c].x);
    m = wave_max_dpp(m);
    if ((tid & 63) == 0) red[tid >> 6] = m;
    __syncthreads();
    const float M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), base = M == -INFINITY ? 0.0f : M;
    const int d = tid % kLanes, k = tid / kLanes;
    f4_t u = {0.0f, 0.0f, 0.0f, 0.0f};
    float z = 0.0f;
    for (int c = k; c < n; c += kRows) {
        const float2 t = mz[c];
        if (t.y == 0.0f) continue;   // sees nothing; its U may not be there
        const float f = __builtin_amdgcn_exp2f(t.x - base);
        z += t.y * f;
        u += *reinterpret_cast<const f4_t*>(a.part + (at * a.nchunk + c) * HD + 4 * d) * f;
    }
    us[k][d] = u;
    // lanes of one row hold the same z: one of them counts
    const float zw = wave_sum_dpp(d == 0 ? z : 0.0f);
    if ((tid & 63) == 0) zred[tid >> 6] = zw;
    __syncthreads();
    if (tid >= kLanes) return;
    const float Z = (zred[0] + zred[1]) + (zred[2] + zred[3]);
    f4_t U = us[0][tid];
#pragma unroll
    for (int j = 1; j < kRows; ++j) U += us[j][tid];
    write_result(a, at, HD, 4 * tid, U, M * kLn2, Z, err);
    if (err) raise_error(err);
}

}  // namespace rta
