// rta_paged_attention.hip -- causal attention of new rows over the paged history, with a sliding
// window and first positions that stay visible (gfx950).
#include "rta_paged_decode.hpp"

namespace rta {

template <int FMT>
__device__ __forceinline__ float element(const uint8_t* page, int64_t i) {
    if constexpr (FMT == RTA_F16) return (float)reinterpret_cast<const _Float16*>(page)[i];
    else if constexpr (FMT == RTA_BF16)
        return __builtin_bit_cast(float, (uint32_t)reinterpret_cast<const uint16_t*>(page)[i] << 16);
    else return (float)reinterpret_cast<const int8_t*>(page)[i];
}

// A workgroup per (row, q head); each of its 4 waves takes every fourth visible position with an
// online softmax, lane l holding dims l, l + 64, ..; the waves are joined at the end.
template <int FMT, int HD>
__global__ void __launch_bounds__(256) paged_attention_kernel(const PagedAttnArgs a) {
    constexpr int kPer = HD / 64;
    __shared__ float u_s[4][HD], m_s[4], z_s[4];
    const int r = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int i, first, count;
    if (!row_entry(a.l, r, i, first, count)) return;
    if (r - first >= a.max_rows) {
        if (threadIdx.x == 0 && h == 0) raise_error(RTA_DEVERR_PAGES);
        return;
    }
    const int s = list_seq(a.l.seqs, i);
    int n = 0;
    uint32_t err = 0;
    Visible see{0, 0, 0};
    const int32_t* row = nullptr;
    if ((unsigned)s < (unsigned)a.p.max_seqs) {
        const int len = a.p.lengths[s], t = len - count + (r - first);
        row = a.p.table + (int64_t)s * a.p.max_pages;
        if (len > a.max_len || len < 0 || (t < 0 && len > 0) || (len == 0 && count > 1)) err = RTA_DEVERR_PAGES;
        else if (t >= 0) see = visible(t, a.window, a.sinks);
    } else {
        err = RTA_DEVERR_PAGES;
    }
    n = see.count;
    const int kvh = h / a.group;
    const float* q = a.q + r * a.q_stride + (int64_t)h * HD;
    float qv[kPer], u[kPer], m = -INFINITY, z = 0.0f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        qv[j] = q[lane + 64 * j];
        u[j] = 0.0f;
    }
    const float scale = 1.0f / sqrtf((float)HD);
    const int64_t plane = (int64_t)a.p.kv_heads * a.p.page;   // rows of the key half of a page
    for (int j = wave; j < n; j += 4) {
        const int p = see.position(j), e = (int)a.p.by_page.div((uint32_t)p), off = p - e * a.p.page;
        const int pg = page_of(a.p, row, e);
        if (pg < 0) {
            err = RTA_DEVERR_PAGES;
            continue;
        }
        const uint8_t* page = a.p.pool + pg * a.p.page_bytes;
        const int64_t kr = (int64_t)kvh * a.p.page + off, vr = plane + kr;
        float d = 0.0f;
#pragma unroll
        for (int c = 0; c < kPer; ++c) d += qv[c] * element<FMT>(page, kr * HD + lane + 64 * c);
        float sc = wave_sum_dpp(d) * scale, vs = 1.0f;
        if constexpr (FMT == RTA_Q8_ROW) {
            const float* f = reinterpret_cast<const float*>(page + 2 * plane * HD);
            sc *= f[kr];
            vs = f[vr];
        }
        if (!isfinite(sc)) err |= RTA_DEVERR_DETECTOR;
        const float mn = fmaxf(m, sc), al = expf(m - mn), w = expf(sc - mn);
        z = z * al + w;
#pragma unroll
        for (int c = 0; c < kPer; ++c) u[c] = u[c] * al + w * vs * element<FMT>(page, vr * HD + lane + 64 * c);
        m = mn;
    }
    if (lane == 0) {
        m_s[wave] = m;
        z_s[wave] = z;
    }
#pragma unroll
    for (int c = 0; c < kPer; ++c) u_s[wave][lane + 64 * c] = u[c];
    __syncthreads();
    float M = fmaxf(fmaxf(m_s[0], m_s[1]), fmaxf(m_s[2], m_s[3]));
    const float base = M == -INFINITY ? 0.0f : M;
    float Z = 0.0f, f[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        f[w] = expf(m_s[w] - base);
        Z += z_s[w] * f[w];
    }
    const int64_t at = (int64_t)r * a.hq + h;
    if (threadIdx.x < HD) {
        const int c = threadIdx.x;
        float o = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) o += u_s[w][c] * f[w];
        o = Z > 0.0f || Z != Z ? o / Z : 0.0f;
        if (a.gate) o *= detector_sigmoid(a.gate[at * HD + c]);
        if (!isfinite(o)) err |= RTA_DEVERR_DETECTOR;
        a.out[at * HD + c] = o;
        if (c == 0 && a.m_out) a.m_out[at] = M;
        if (c == 0 && a.z_out) a.z_out[at] = Z;
    }
    if (err) raise_error(err);
}

// How a call with one row per sequence is cut: chunks of a multiple of 128 positions (a tile for
// each of 4 waves), so many that the chip has about kDecGroups workgroups to hand out if every
// row sees the most it may.
constexpr int kDecGroups = 4096;
struct Cut {
    int chunk, nchunk;
};
static Cut decode_cut(int rows, int heads, int64_t most) {
    const int64_t want = (rows * (int64_t)heads * most / kDecGroups + 127) / 128 * 128;
    const int64_t chunk = want < 128 ? 128 : want < 1 << 30 ? want : 1 << 30;
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
    (void)n;
    if (host::pages_args(pages, -1, &p) || hq <= 0 || hq % pages->kv_heads || rows <= 0 || max_rows <= 0 ||
        max_len < 0 || window < 0 || sinks < 0)
        return 0;
    if (max_rows > 1) return 0;
    const int group = hq / pages->kv_heads;
    const Cut cut = decode_cut(rows, decode_heads(pages->kv_heads, group, pages->head_dim),
                               most_visible(bound_len(pages, max_len), window, sinks));
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
        max_rows > rows || max_len < 0)
        return RTA_ERR_SHAPE;
    if (window < 0 || sinks < 0 || hq > 65535) return RTA_ERR_RANGE;
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
            if (max_rows > 1) {
                hipLaunchKernelGGL((paged_attention_kernel<F, HD>), dim3(rows, hq), dim3(256), 0, s, a);
                return;
            }
            const int heads = decode_heads(pages->kv_heads, a.group, HD);
            const Cut cut = decode_cut(rows, heads, most_visible(a.max_len, window, sinks));
            a.chunk = cut.chunk;
            a.nchunk = cut.nchunk;
            a.part = static_cast<float*>(workspace);
            a.mz = reinterpret_cast<float2*>(a.part + (size_t)rows * hq * cut.nchunk * HD);
            const dim3 grid(rows * heads, 1, cut.nchunk), block(64 * kDecWaves);
            if constexpr (HD < 256) {
                if (decode_nc(a.group, HD) == 2) hipLaunchKernelGGL((paged_decode_kernel<F, HD, 2>), grid, block, 0, s, a);
                else hipLaunchKernelGGL((paged_decode_kernel<F, HD, 1>), grid, block, 0, s, a);
            } else {
                hipLaunchKernelGGL((paged_decode_kernel<F, HD, 1>), grid, block, 0, s, a);
            }
            if (cut.nchunk > 1) hipLaunchKernelGGL((paged_merge_kernel<HD>), dim3(rows, hq), dim3(256), 0, s, a);
        };
        if (pages->head_dim == 64) go(std::integral_constant<int, 64>{});
        else if (pages->head_dim == 128) go(std::integral_constant<int, 128>{});
        else go(std::integral_constant<int, 256>{});
    };
    if (pages->fmt == RTA_F16) launch(std::integral_constant<int, RTA_F16>{});
    else if (pages->fmt == RTA_BF16) launch(std::integral_constant<int, RTA_BF16>{});
    else launch(std::integral_constant<int, RTA_Q8_ROW>{});
    return hipGetLastError() == hipSuccess ? RTA_OK : RTA_ERR_LAUNCH;
}

}  // extern "C"
