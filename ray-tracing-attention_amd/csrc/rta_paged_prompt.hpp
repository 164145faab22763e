// rta_paged_prompt.hpp -- causal attention of several rows per sequence over its pages.
//
// Bound by the matrix cores: 4 hq HD operations per (row, position), twice that with q and the
// weights in two binary16 parts, three times in three bfloat16 parts (rta_paged.hpp).  The columns
// of a kv head's products are its (row, q head) pairs, so the heads that share keys share their
// loads and no group size leaves columns empty.  A workgroup of 4 waves takes 4 x 16 NQ columns
// and the positions that any of them sees, in tiles staged in LDS by all of it (two buffers, one
// barrier per tile; a row's 16 bytes of padding keep the operand reads off each other's banks);
// each wave keeps its q operands, running maxima and sums, and O^T in registers.  A tile that
// every column of a wave sees whole takes no masks, one that no column sees is skipped.
// The last rows, which see most, come first; kv heads go over the XCDs, so that one L2 serves
// all rows of a head.  With few workgroups the positions are cut into chunks as well, joined by
// paged_merge_kernel.
#pragma once
#include "rta_paged_decode.hpp"

namespace rta {

template <int FMT, int HD>
struct PromptLds {
    static constexpr int kNQ = HD == 256 ? 1 : 2;      // column tiles of a wave
    static constexpr int kTile = HD > 64 ? 32 : 64;    // positions per tile
    static constexpr int kCols = 64 * kNQ;             // columns of a workgroup
    static constexpr int kPitch = 2 * HD + 16;
    static constexpr int kRows = 2 * kTile * kPitch;   // keys, then values
    static constexpr int kScales = PageFmt<FMT>::kScaled ? 2 * kTile * 4 : 0;
    static constexpr int kBuf = kRows + kScales + kTile * 4;   // and which rows count
    static constexpr int kThird = FMT == RTA_BF16 ? kNQ * (HD / 32) * 1024 : 0;   // per wave: q's third part
    static constexpr int kTotal = 2 * kBuf + 4 * kThird;
};

template <int FMT, int HD>
__global__ void __launch_bounds__(256, (PromptLds<FMT, HD>::kTotal > 80 << 10 ? 1 : 2)) paged_prompt_kernel(const PagedAttnArgs a) {
    using L = PromptLds<FMT, HD>;
    constexpr int kParts = PageFmt<FMT>::kParts, kB = PageFmt<FMT>::kBytes, NQ = L::kNQ;
    constexpr int kKb = HD / 32, kDt = HD / 16;
    constexpr int kKg = kKb < 4 ? kKb : 4, kDg = 4;   // operands read ahead
    constexpr int kPieces = HD * kB / 16, kStep = 256 / kPieces, kPass = L::kTile / kStep;
    constexpr bool kScaled = PageFmt<FMT>::kScaled;
    __shared__ __align__(16) uint8_t lds[L::kTotal];
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 15, u = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hkv = a.p.kv_heads;
    const int kvh = blockIdx.x % hkv, rest = blockIdx.x / hkv;
    const int entry = rest % a.l.n, tile = a.ntile - 1 - rest / a.l.n;
    uint32_t err = 0;
    Entry en;
    if (!resolve_entry(a, entry, en, err)) return;
    if (tile > 0) err &= ~RTA_DEVERR_PAGES;   // the first tile tells
    if ((int64_t)tile * L::kCols >= (int64_t)en.rows * a.group) return;
    const int base = en.base, count = en.count, live_rows = en.rows, len = en.len;
    const int32_t* table = en.table;
    const Visible see = len ? prompt_span(a, len, count, tile, L::kCols) : Visible{0, 0, 0};
    const int begin = blockIdx.z * a.chunk, end = see.count - begin > a.chunk ? begin + a.chunk : see.count;
    if (begin >= end && blockIdx.z > 0) return;
    const int nt = (end - begin + L::kTile - 1) / L::kTile;

    // staging: thread -> piece of a row; its rows of a tile are kStep apart
    const int64_t plane = (int64_t)hkv * a.p.page, v_off = plane * HD * kB;
    const int64_t head_row = (int64_t)kvh * a.p.page, head_off = head_row * HD * kB;
    const int piece = tid % kPieces, row0 = tid / kPieces;
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
    u4_t kr[kPass], vr[kPass];
    float ksr[kPass], vsr[kPass];
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
            const uint8_t* src = page + head_off + (uint32_t)(sp.off[k] * (HD * kB) + 16 * piece);
            kr[k] = *reinterpret_cast<const u4_t*>(src);
            vr[k] = *reinterpret_cast<const u4_t*>(src + v_off);
            if constexpr (kScaled) {
                const float* f = reinterpret_cast<const float*>(page + 2 * v_off) + head_row + sp.off[k];
                ksr[k] = f[0];
                vsr[k] = f[plane];
            }
        }
    };
    auto put = [&](uint8_t* dst, u4_t x) {   // one piece as 2-byte elements
        if constexpr (FMT == RTA_Q8_ROW) {
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
                    kr[k] = vr[k] = u4_t{0, 0, 0, 0};
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
                    constexpr uint64_t kRow = kPieces == 32 ? 0xffffffffull : (1ull << kPieces) - 1;
                    const bool hit = piece_not_finite<FMT>(vr[k]);
                    if (hit) vr[k] = u4_t{0, 0, 0, 0};
                    if (__builtin_amdgcn_ballot_w64(hit) & (kRow << (lane & ~(kPieces - 1)))) bad |= 1u << k;
                }
            }
        }
#pragma unroll
        for (int k = 0; k < kPass; ++k) {
            const int row = row0 + k * kStep;
            put(buf + row * L::kPitch, kr[k]);
            put(buf + (L::kTile + row) * L::kPitch, vr[k]);
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
    const int col0 = tile * L::kCols + wave * 16 * NQ, cols = live_rows * a.group;
    const bool on = col0 < cols;   // uniform: this wave has columns
    int t_col[NQ];
    u4_t qb[NQ][kKb][2];   // (the third part of bfloat16 lies in LDS: 96 registers would leave none for operands)
    u4_t* third = reinterpret_cast<u4_t*>(lds + 2 * L::kBuf + wave * L::kThird) + lane;
    float fac[NQ];
#pragma unroll
    for (int c = 0; c < NQ; ++c) {
        const int col = min(col0 + 16 * c + i, cols - 1), tok = col / a.group, g = col - tok * a.group;
        t_col[c] = max(len - count + tok, -1);
        const float* q = a.q + (int64_t)(base + tok) * a.q_stride + ((int64_t)kvh * a.group + g) * HD;
        float v[kKb][8], mx = 0.0f;
#pragma unroll
        for (int kb = 0; kb < kKb; ++kb)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[kb][e] = q[32 * kb + 8 * u + e];
                mx = fmaxf(mx, fabsf(v[kb][e]));
            }
        int qe = 14;
        if constexpr (FMT != RTA_BF16) qe = part_exponent(max_xor32(max_xor16(mx)));
        const float sg = ldexpf(1.0f, 14 - qe);
        fac[c] = ldexpf(kLog2e / sqrtf((float)HD), qe - 14);
#pragma unroll
        for (int kb = 0; kb < kKb; ++kb) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[kb][e] *= sg;
            u4_t part[kParts];
            split_all<FMT>(v[kb], part);
            qb[c][kb][0] = part[0];
            qb[c][kb][1] = part[1];
            if constexpr (kParts == 3) third[(c * kKb + kb) * 64] = part[2];
        }
    }
    // the wave's first and last positions
    const int t_lo = len - count + col0 / a.group;
    const int t_hi = len - count + min(col0 + 16 * NQ - 1, cols - 1) / a.group;

    f4_t o[NQ][kDt];
    Softmax<NQ> sm;
    sm.start();
    int ve = -110;
#pragma unroll
    for (int c = 0; c < NQ; ++c) {
        for (int d = 0; d < kDt; ++d) o[c][d] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
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
            if constexpr (kScaled) {   // value scales below 2^0
                const float mx = lane < L::kTile ? fabsf(sc[L::kTile + lane]) : 0.0f;
                ve_new = max(ve, part_exponent(wave_max_dpp(mx)));
                wscale = ldexpf(1.0f, -ve_new);
            }
#pragma unroll
            for (int sub = 0; sub < L::kTile / 32; ++sub) {
                // S^T of 32 positions
                f4_t x[NQ][2];
#pragma unroll
                for (int c = 0; c < NQ; ++c) x[c][0] = x[c][1] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int k0 = 0; k0 < kKb; k0 += kKg) {
                    u4_t ka[kKg][2];   // all on their way before the first product
#pragma unroll
                    for (int k = 0; k < kKg; ++k)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            ka[k][h] = *reinterpret_cast<const u4_t*>(buf + (32 * sub + 16 * h + i) * L::kPitch +
                                                                      64 * (k0 + k) + 16 * u);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int k = 0; k < kKg; ++k)
#pragma unroll
                        for (int p = 0; p < kParts; ++p)   // neighbours go into different accumulators
#pragma unroll
                            for (int c = 0; c < NQ; ++c) {
                                const u4_t q = p < 2 ? qb[c][k0 + k][p & 1] : third[(c * kKb + k0 + k) * 64];
#pragma unroll
                                for (int h = 0; h < 2; ++h) x[c][h] = page_mfma<FMT>(ka[k][h], q, x[c][h]);
                            }
                }
                // the first of V^T's operands, ready when the weights are
                const uint8_t* vb = buf + (L::kTile + 32 * sub + 4 * u + (i >> 2)) * L::kPitch + 8 * (i & 3);
                u4_t va[2][kDg];
                auto load_va = [&](int d0) {
#pragma unroll
                    for (int d = 0; d < kDg; ++d) {
                        const uint8_t* src = vb + 32 * (d0 + d);
                        const s4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t*)src);
                        const s4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t*)(src + 16 * L::kPitch));
                        const uint2 l2 = __builtin_bit_cast(uint2, lo), h2 = __builtin_bit_cast(uint2, hi);
                        va[(d0 / kDg) & 1][d] = u4_t{l2.x, l2.y, h2.x, h2.y};
                    }
                };
                load_va(0);
                __builtin_amdgcn_sched_barrier(0);
                f4_t vf[2];
                if constexpr (kScaled) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const f4_t kf = *reinterpret_cast<const f4_t*>(sc + 32 * sub + 16 * h + 4 * u);
                        vf[h] = *reinterpret_cast<const f4_t*>(sc + L::kTile + 32 * sub + 16 * h + 4 * u) * wscale;
#pragma unroll
                        for (int c = 0; c < NQ; ++c) x[c][h] *= kf;
                    }
                }
                sm.watch(x);
                if (!whole) {
                    mask_columns<NQ>(x, (uint32_t)(okm >> (32 * sub)), see, j0 + 32 * sub, u, t_col, a.window, a.sinks);
                    if (badm) sm.poison(x, (uint32_t)(badm >> (32 * sub)), u);
                }
                sm.template raise<kDt>(x, fac, kScaled ? ve - ve_new : 0, o);
                u4_t pb[NQ][kParts];
#pragma unroll
                for (int c = 0; c < NQ; ++c) {
                    float w[8];
                    sm.weights(c, x[c], fac[c], w);
                    if constexpr (kScaled) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) w[j] *= vf[j >> 2][j & 3];
                    }
                    split_all<FMT>(w, pb[c]);
                }
                ve = ve_new;
                // O^T += V^T P^T
#pragma unroll
                for (int d0 = 0; d0 < kDt; d0 += kDg) {
                    if (d0 + kDg < kDt) {
                        load_va(d0 + kDg);
                        __builtin_amdgcn_sched_barrier(0);
                    }
#pragma unroll
                    for (int p = 0; p < kParts; ++p)
#pragma unroll
                        for (int d = 0; d < kDg; ++d)
#pragma unroll
                            for (int c = 0; c < NQ; ++c) o[c][d0 + d] = page_mfma<FMT>(va[(d0 / kDg) & 1][d], pb[c][p], o[c][d0 + d]);
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
        const float Z = add_xor32(add_xor16(sm.z[c])) * back, unscale = kScaled ? ldexpf(back, ve) : back;
        const int col = col0 + 16 * c + i;
        if (col >= cols) continue;
        const int tok = col / a.group, g = col - tok * a.group;
        const int64_t at = (int64_t)(base + tok) * a.hq + (int64_t)kvh * a.group + g;
        if (a.nchunk > 1) {
            const int64_t rec = at * a.nchunk + blockIdx.z;
#pragma unroll
            for (int d = 0; d < kDt; ++d)
                *reinterpret_cast<f4_t*>(a.part + rec * HD + 16 * d + 4 * u) = o[c][d] * unscale;
            if (u == 0) a.mz[rec] = float2{M, Z};
            continue;
        }
#pragma unroll
        for (int d = 0; d < kDt; ++d) write_result(a, at, HD, 16 * d + 4 * u, o[c][d] * unscale, M * kLn2, Z, err);
    }
    if (err) raise_error(err);
}

// Joins the chunks of a (row, q head): M = max m, o = sum U e^(m - M) / sum z e^(m - M).  HD / 4
// lanes of 4 dims by the rest of 256 threads over the chunks.  Bound by latency: the lengths, the
// (m, z) of the chunks and their U, each one trip.
template <int HD>
__global__ void __launch_bounds__(256) paged_merge_kernel(const PagedAttnArgs a) {
    constexpr int kLanes = HD / 4, kRows = 256 / kLanes;
    __shared__ f4_t us[kRows][kLanes];
    __shared__ float red[4], zred[4];
    const int r = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
    uint32_t err = 0;
    Visible see;
    const int32_t* table;
    if (!resolve_row(a, r, table, see, err)) return;   // the chunks have reported what is wrong
    err = 0;
    const int64_t at = (int64_t)r * a.hq + h;
    int span = see.count;
    if (a.cols) {   // the chunks of the row's column tile
        int i, first, count;
        row_entry(a.l, r, i, first, count);
        const int s = list_seq(a.l.seqs, i);   // bad ones see nothing
        if (span) {
            const int tile = (int)(((int64_t)(r - first) * a.group + h % a.group) / a.cols);
            span = prompt_span(a, a.p.lengths[s], count, tile, a.cols).count;
        }
    }
    const int n = (int)(((int64_t)span + a.chunk - 1) / a.chunk);
    const float2* mz = a.mz + at * a.nchunk;
    float m = -INFINITY;
    for (int c = tid; c < n; c += 256) m = fmaxf(m, mz[c].x);
    m = wave_max_dpp(m);
    if ((tid & 63) == 0) red[tid >> 6] = m;
    __syncthreads();
    const float M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), base = M == -INFINITY ? 0.0f : M;
    const int d = tid % kLanes, k = tid / kLanes;
    f4_t u = {0.0f, 0.0f, 0.0f, 0.0f};
    float z = 0.0f;
    for (int c = k; c < n; c += kRows) {
        const float2 t = mz[c];
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
