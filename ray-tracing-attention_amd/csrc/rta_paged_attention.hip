// rta_paged_attention.hip -- causal attention of new rows over the paged history, with a sliding
// window and first positions that stay visible (gfx950).
#include "rta_paged_decode4.hpp"
#include "rta_paged_prompt.hpp"

namespace rta {

// How a call with one row per sequence is cut: chunks of a multiple of 128 positions (a tile for
// each of 4 waves), so many that the chip has about kDecGroups workgroups to hand out if every
// row sees the most it may.  Chunks of 128 are for calls that run in one go on the chip's two
// workgroups per compute unit (wide heads: one), where every further tile of a wave adds its
// latency (us, chunks of 128 / 256 / 512: one sequence of 1000 positions 9.4 / 11.9 / 17.0); past
// that a workgroup's start costs more (one of 16000: 25.2 / 22.1 / 21.6; 32 of 1000, 8-bit: 27.3 /
// 23.4 / 22.4), and larger ones yet balance ragged rows worse (32 of 256 to 8192: 512 70, 1024 75).
constexpr int kDecGroups = 4096;
struct Cut {
    int chunk, nchunk;
};
// Over 4-bit pages a chunk's bytes are a quarter, so its start, the merge and the second launch weigh more.  Up to 512
// positions, and up to 1024 where the rows alone fill the chip's four workgroups per compute unit, are not cut at all (us in
// one chunk / in several: 32 rows of 300 8.0 / 11.1, of 500 9.2 / 12.5, 128 of 300 15.3 / 25, of 600 21.6 / 31.3, one of
// 300 7.7 / 8.5, of 500 8.9 / 8.4, and 4 less of the host's); calls that do not run in one go have chunks of 512 at least
// (512 / 256: one of 16000 13.5 / 15.8, 32 of 1000 16.7 / 17.5), and a single sequence, which no other can be longer than,
// one round of them (one of 100000 37, so 44; 32 of 256 to 8192 would take 34.9, so 32.4).
static Cut decode_cut(int64_t rows, int heads, int hd, int64_t most, bool q4 = false, int at_least = 128) {
    if (q4 && (most <= 512 || (most <= 1024 && rows * heads >= 1024))) return Cut{1024, 1};
    const int64_t want = (rows * heads * most / (q4 && rows == 1 ? 1024 : kDecGroups) + 127) / 128 * 128;
    const int64_t some = rows * heads * ((most + 127) / 128) <= (hd == 256 ? 256 : 512) ? 128 : q4 ? 512 : 256;
    const int64_t least = some < at_least ? at_least : some;
    const int64_t chunk = want < least ? least : want < 1 << 30 ? want : 1 << 30;
    return Cut{(int)chunk, (int)((most + chunk - 1) / chunk)};
}
// Up to 32 (row, q head) columns of a kv head (wide heads: 16) are few: the kernel of single rows
// takes them in one group, bound by the history's bytes, where the other kernel's 128 columns would
// stay mostly empty (us, this / the other: 16 sequences of 4 rows over 4000 bf16 positions, 4 q
// heads per kv head 60 / 91, 8 rows 76 / 97; one of 12 rows over 8000, in two groups 31 / 27).
// Their workgroups start and end with more work, so fewer are asked for, as for 4 rows an entry (5
// rows of 16 sequences over 500 to 16384 8-bit positions 73.5; as for 2, 3, 6 and 8: 81, 76, 97, 123;
// the one set of lengths and rows that this was measured on).
static bool few_rows(int64_t max_rows, int group, int hd) { return max_rows * group <= (hd == 256 ? 16 : 32); }
// With several rows: column tiles enough for two workgroups per compute unit stand alone, fewer
// are cut into chunks of positions (a multiple of 64, 256 at least).
constexpr int kPromptGroups = 1024;
static int few_cols(int cols) { return cols <= 16 ? 16 : 32; }
static int prompt_cols(int hd) { return hd == 256 ? 64 : 128; }
static Cut prompt_cut(int64_t tiles, int64_t most) {
    if (2 * tiles >= kPromptGroups) return Cut{INT_MAX, 1};
    int64_t chunk = (tiles * most / kPromptGroups + 63) / 64 * 64;
    chunk = chunk < 256 ? 256 : chunk < 1 << 30 ? chunk : 1 << 30;
    return Cut{(int)chunk, (int)((most + chunk - 1) / chunk)};
}
// Workgroups per row: kv heads times the groups of up to 8 (16) q heads that share one.
static int decode_nc(int group, int hd) { return group > 8 && hd < 256 ? 2 : 1; }
static int decode_heads(int kv_heads, int group, int hd) {
    const int per = 8 * decode_nc(group, hd);
    return kv_heads * ((group + per - 1) / per);
}
static int64_t most_visible(int64_t max_len, int window, int sinks) {
    return window > 0 && max_len - window > sinks ? (int64_t)window + sinks : max_len;
}
static int64_t bound_len(const rta_pages* p, int max_len) {
    const int64_t most = (int64_t)p->max_pages * p->page;
    return max_len > 0 && max_len < most ? max_len : most;
}
// The cut of a call, and its column tiles per entry (0: one row per entry).
static Cut cut_of(const rta_pages* p, int hq, int rows, int n, bool several, int max_rows, int max_len, int window,
                  int sinks, int* ntile) {
    const int group = hq / p->kv_heads;
    const int64_t len = bound_len(p, max_len);
    *ntile = 0;
    if (!several)
        return decode_cut(rows, decode_heads(p->kv_heads, group, p->head_dim), p->head_dim,
                          most_visible(len, window, sinks), p->fmt == RTA_Q4_GROUP);
    const bool few = few_rows(max_rows, group, p->head_dim);
    const int cols = few ? few_cols(max_rows * group) : prompt_cols(p->head_dim);
    *ntile = (int)(((int64_t)max_rows * group + cols - 1) / cols);
    // (a column tile sees from its first row's window on)
    int64_t most = len;
    if (window > 0) {
        const int64_t span = (int64_t)window + cols / group + 1;
        most = most_visible(len, (int)(span < INT_MAX ? span : INT_MAX), sinks);
    }
    // (4-bit pages, us so / as the others: 16 sequences of 5 rows over 500 to 16384 positions 58 / 84, 4 of 8 over 4000
    // 23 / 27, one of 4 over 30000 25 / 32, 32 of 4 over 300 8 / 11; 24 of 5 through a window of 4096 25.5 / 25.4)
    if (few && p->fmt == RTA_Q4_GROUP) return decode_cut(2 * (int64_t)n, p->kv_heads, p->head_dim, most, true, 512);
    if (few) return decode_cut(4 * (int64_t)n, p->kv_heads, p->head_dim, most);
    return prompt_cut((int64_t)*ntile * n * p->kv_heads, most);
}
static bool grid_fits(const rta_pages* p, int hq, int rows, int n, int max_rows) {
    const int64_t group = hq / p->kv_heads, most = host::kMostGroups, tiles = (max_rows * group + 63) / 64;
    return (int64_t)rows * p->kv_heads * group <= INT_MAX &&
           rows * (int64_t)decode_heads(p->kv_heads, (int)group, p->head_dim) <= most &&
           (max_rows == 1 || tiles <= most / ((int64_t)n * p->kv_heads));
}
static size_t split_bytes(int64_t rows, int hq, int hd, int nchunk) {
    if (nchunk <= 1) return 0;
    return ((size_t)rows * hq * nchunk * (hd + 2) * 4 + 15) / 16 * 16;
}

}  // namespace rta

using namespace rta;

extern "C" {

size_t rta_paged_attention_workspace_bytes(const rta_pages* pages, int hq, int rows, int n, int max_rows, int max_len,
                                           int window, int sinks) {
    PageArgs p;
    if (host::pages_args(pages, -1, &p) || hq <= 0 || hq % pages->kv_heads || rows <= 0 || n <= 0 || max_rows <= 0 ||
        max_len < 0 || window < 0 || sinks < 0)
        return 0;
    int ntile;
    const Cut cut = cut_of(pages, hq, rows, n, max_rows > 1, max_rows, max_len, window, sinks, &ntile);
    return split_bytes(rows, hq, pages->head_dim, cut.nchunk);
}

int rta_paged_attention(const rta_pages* pages, int layer, const float* q, int64_t q_stride, int rows, int hq,
                        const int32_t* seqs, const int32_t* cu_rows, int n, int max_rows, int max_len, int window,
                        int sinks, const float* gate, float* out, float* m_out, float* z_out, void* workspace,
                        size_t workspace_bytes, rta_stream_t stream) {
    PagedAttnArgs a{};
    if (layer < 0) return RTA_ERR_RANGE;
    int rc = host::pages_args(pages, layer, &a.p);
    if (rc) return rc;
    if (!q || !out) return RTA_ERR_NULL;
    rc = host::rows_args(rows, seqs, cu_rows, n, &a.l);
    if (rc) return rc;
    if (hq <= 0 || hq % pages->kv_heads || q_stride < (int64_t)hq * pages->head_dim || max_rows <= 0 ||
        max_rows > rows || max_len < 0 || (!cu_rows && max_rows != 1))
        return RTA_ERR_SHAPE;
    if (window < 0 || sinks < 0 || hq > 65535 || !grid_fits(pages, hq, rows, n, max_rows)) return RTA_ERR_RANGE;
    if (!host::aligned(q, 4) || !host::aligned(gate, 4) || !host::aligned(out, 4) || !host::aligned(m_out, 4) ||
        !host::aligned(z_out, 4))
        return RTA_ERR_ALIGN;
    const size_t need = rta_paged_attention_workspace_bytes(pages, hq, rows, n, max_rows, max_len, window, sinks);
    if (need && (!workspace || workspace_bytes < need || !host::aligned(workspace, 16))) return RTA_ERR_WORKSPACE;
    hipStream_t s = (hipStream_t)stream;
    a.q = q;
    a.q_stride = q_stride;
    a.gate = gate;
    a.out = out;
    a.m_out = m_out;
    a.z_out = z_out;
    a.hq = hq;
    a.group = hq / pages->kv_heads;
    a.max_rows = max_rows;
    a.max_len = (int)bound_len(pages, max_len);
    a.window = window;
    a.sinks = sinks;
    auto launch = [&](auto fmt) {
        constexpr int F = decltype(fmt)::value;
        auto go = [&](auto hdim) {
            constexpr int HD = decltype(hdim)::value;
            int ntile;
            const Cut cut = cut_of(pages, hq, rows, n, max_rows > 1, max_rows, max_len, window, sinks, &ntile);
            a.chunk = cut.chunk;
            a.nchunk = cut.nchunk;
            a.part = static_cast<float*>(workspace);
            a.mz = reinterpret_cast<float2*>(a.part + (size_t)rows * hq * cut.nchunk * HD);
            a.ntile = ntile;
            if (ntile && few_rows(max_rows, a.group, HD)) {   // one group of columns
                const dim3 grid(n * pages->kv_heads, 1, cut.nchunk), block(64 * kDecWaves);
                if (few_cols(max_rows * a.group) == 16) hipLaunchKernelGGL((paged_decode_kernel<F, HD, 1, true>), grid, block, 0, s, a);
                else if constexpr (HD < 256) hipLaunchKernelGGL((paged_decode_kernel<F, HD, 2, true>), grid, block, 0, s, a);
            } else if (ntile) {
                hipLaunchKernelGGL((paged_prompt_kernel<F, HD>), dim3(ntile * n * pages->kv_heads, 1, cut.nchunk),
                                   dim3(256), 0, s, a);
            } else {
                const dim3 grid(rows * decode_heads(pages->kv_heads, a.group, HD), 1, cut.nchunk), block(64 * kDecWaves);
                // (us, this / the other kernel: 8 sequences of 60000 to 131072 178 / 205, 32 of 256 to 8192 32.6 / 37)
                if (F == RTA_Q4_GROUP && a.group <= 4)
                    hipLaunchKernelGGL((paged_decode4_kernel<HD>), grid, block, 0, s, a);
                else if (decode_nc(a.group, HD) == 1)
                    hipLaunchKernelGGL((paged_decode_kernel<F, HD, 1, false>), grid, block, 0, s, a);
                else if constexpr (HD < 256) hipLaunchKernelGGL((paged_decode_kernel<F, HD, 2, false>), grid, block, 0, s, a);
            }
            if (cut.nchunk > 1) hipLaunchKernelGGL((paged_merge_kernel<HD>), dim3(rows, hq), dim3(256), 0, s, a);
        };
        if (pages->head_dim == 64) go(std::integral_constant<int, 64>{});
        else if (pages->head_dim == 128) go(std::integral_constant<int, 128>{});
        else go(std::integral_constant<int, 256>{});
    };
    if (pages->fmt == RTA_F16) launch(std::integral_constant<int, RTA_F16>{});
    else if (pages->fmt == RTA_BF16) launch(std::integral_constant<int, RTA_BF16>{});
    else if (pages->fmt == RTA_Q8_ROW) launch(std::integral_constant<int, RTA_Q8_ROW>{});
    else launch(std::integral_constant<int, RTA_Q4_GROUP>{});
    return hipGetLastError() == hipSuccess ? RTA_OK : RTA_ERR_LAUNCH;
}

}  // extern "C"
