// rta_pages.hpp -- the paged history as its kernels see it: where a position's keys and values
// lie, which sequence and position a row belongs to, and the host checks of the descriptor.
#pragma once
#include <limits.h>

#include "rta_common.hpp"
#include "rta_host.hpp"

namespace rta {

// p / d for 0 <= p < 2^31 and 1 <= d <= 65536 as (p m) >> (31 + l), m = floor(2^(31 + l) / d) + 1,
// l = ceil(log2 d): the error p (m d - 2^(31 + l)) / (d 2^(31 + l)) stays below 1 / d because
// m d - 2^(31 + l) <= d <= 2^l.  (2 p m) >> 32 >> l: one multiplication and two shifts.
struct FastDiv {
    uint32_t d = 1, m = 0, l = 0;
    FastDiv() = default;
    explicit FastDiv(uint32_t v) : d(v) {
        while ((1ull << l) < v) ++l;
        m = (uint32_t)((1ull << (31 + l)) / v + 1);
    }
    __device__ __forceinline__ uint32_t div(uint32_t p) const { return __umulhi(2 * p, m) >> l; }
};

struct PageArgs {
    uint8_t* pool;         // one layer
    int32_t* table;
    int32_t* lengths;
    int32_t* refs;
    int64_t page_bytes;
    int64_t layer_bytes;   // n_pages pages
    int layers, n_pages, max_seqs, max_pages, page, kv_heads;
    FastDiv by_page;
};

// Bytes of one position's elements of one head, and of its scales behind a page's elements.
constexpr int page_row_bytes(int fmt, int hd) { return fmt == RTA_Q8_ROW ? hd : fmt == RTA_Q4_GROUP ? hd / 2 : 2 * hd; }
constexpr int page_scale_bytes(int fmt, int hd) { return fmt == RTA_Q8_ROW ? 4 : fmt == RTA_Q4_GROUP ? hd / 16 : 0; }

// RTA_Q4_GROUP: a group's word is a scale (binary16 of six significant bits) with the zero point in its last
// four bits.  Scale * (code - zero) and scale * (16 + code) then have 11 bits at most and are exact in
// binary16 up to a scale of 2112 (31 of which end at 65504).
constexpr uint32_t kQ4Scale = 0xffe0u;
constexpr uint16_t kQ4NaN = 0x7fe0u;
constexpr float kQ4Most = 2112.0f;
// Which of a row's dwords holds dims d .. d + 7 (d % 8 = 0).  Blocks of up to 128 dims; dword
// (u, g) of a block is dims 32 g + 8 u .. of it, so that a 16-byte piece u holds, of every group, the 8 dims
// that lane segment u feeds to the matrix cores.  Dim 2 j + b of a dword: bits 16 b + 4 j .. + 3.
__device__ __forceinline__ int q4_dword(int hd, int d) {
    const int groups = hd < 128 ? 2 : 4, g = (d >> 5) & (groups - 1), u = (d >> 3) & 3;
    return (d >> 7) * 16 + u * groups + g;
}
// Its first dim.
__device__ __forceinline__ int q4_dim(int hd, int dword) {
    const int groups = hd < 128 ? 2 : 4, g = dword & (groups - 1), u = dword / groups & 3;
    return (dword >> 4) * 128 + 32 * g + 8 * u;
}

// A row list: entry of row r, and how many rows it has.
struct RowList {
    const int32_t* seqs;
    const int32_t* cu;
    int rows, n;
};

__device__ __forceinline__ int list_seq(const int32_t* seqs, int i) { return seqs ? seqs[i] : i; }

// Entry i's first row and its row count; false unless they lie in order within the rows.
__device__ __forceinline__ bool entry_rows(const RowList& l, int i, int& first, int& count) {
    first = l.cu[i];
    const int last = l.cu[i + 1];
    count = last - first;
    return first >= 0 && first <= last && last <= l.rows;
}

// Entry i with cu[i] <= r < cu[i + 1], its first row and its row count; false for a row outside
// every entry or of one that entry_rows refuses.  Every lane of a wave may ask for another row.
__device__ __forceinline__ bool row_entry(const RowList& l, int r, int& i, int& first, int& count) {
    if (!l.cu) {
        i = first = r;
        count = 1;
        return r < l.n;
    }
    int lo = 0, hi = l.n;   // the last i with cu[i] <= r, cu[0] being below all
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (l.cu[mid] <= r) lo = mid;
        else hi = mid;
    }
    i = lo;
    return entry_rows(l, lo, first, count) && r >= first && r - first < count;
}

// Whether an entry's rows are refused, over a whole list: for one workgroup of a kernel that goes by rows,
// where an entry may have none to find it by.
__device__ __forceinline__ bool bad_rows(const RowList& l) {
    bool bad = false;
    int first, count;
#pragma unroll 4
    for (int i = threadIdx.x; l.cu && i < l.n; i += blockDim.x) bad |= !entry_rows(l, i, first, count);
    return bad;
}

// Byte offset of page pg of a layer: page sizes are multiples of 128 below 2^38.
__device__ __forceinline__ uint64_t page_offset(const PageArgs& a, int pg) {
    return ((uint64_t)(uint32_t)pg * (uint32_t)(a.page_bytes >> 7)) << 7;
}

// Page of position p of a sequence's table row, -1 where there is none.
__device__ __forceinline__ int page_of(const PageArgs& a, const int32_t* __restrict__ row, uint32_t e) {
    const int p = row[e];
    return (unsigned)p < (unsigned)a.n_pages ? p : -1;
}

// A table entry that is neither a page of the pool nor -1.
__device__ __forceinline__ bool bad_page(const PageArgs& a, int p) { return p < -1 || p >= a.n_pages; }
// A length that the table cannot hold.
__device__ __forceinline__ bool bad_length(const PageArgs& a, int len) {
    return len < 0 || len > (int)((int64_t)a.max_pages * a.page);   // (<= INT_MAX)
}

namespace host {

inline bool page_format(int fmt) {
    return fmt == RTA_F16 || fmt == RTA_BF16 || fmt == RTA_Q8_ROW || fmt == RTA_Q4_GROUP;
}

inline int64_t page_bytes(int fmt, int kv_heads, int head_dim, int page) {
    if (!page_format(fmt) || kv_heads <= 0 || kv_heads > 1024 || page <= 0 || page > 65536 ||
        (head_dim != 64 && head_dim != 128 && head_dim != 256))
        return -1;
    const int64_t n = 2ll * kv_heads * page * (page_row_bytes(fmt, head_dim) + page_scale_bytes(fmt, head_dim));
    return (n + 127) / 128 * 128;
}

// The descriptor's checks and its device form (layer: -1 for the calls on every layer).
inline int pages_args(const rta_pages* p, int layer, PageArgs* a) {
    if (!p || !p->pool || !p->table || !p->lengths || !p->refs) return RTA_ERR_NULL;
    if (!page_format(p->fmt)) return RTA_ERR_FORMAT;
    if (p->kv_heads <= 0 || p->page <= 0 || p->layers <= 0 || p->n_pages <= 0 || p->max_seqs <= 0 || p->max_pages <= 0)
        return RTA_ERR_SHAPE;
    const int64_t bytes = page_bytes(p->fmt, p->kv_heads, p->head_dim, p->page);
    if (bytes < 0 || p->n_pages > 1 << 20 || (int64_t)p->max_pages * p->page > INT_MAX || layer < -1 ||
        layer >= p->layers)
        return RTA_ERR_RANGE;
    if (!aligned(p->pool, 16) || !aligned(p->table, 4) || !aligned(p->lengths, 4) || !aligned(p->refs, 4))
        return RTA_ERR_ALIGN;
    a->page_bytes = bytes;
    a->layer_bytes = bytes * p->n_pages;
    a->pool = static_cast<uint8_t*>(p->pool) + (layer > 0 ? layer : 0) * a->layer_bytes;
    a->table = p->table;
    a->lengths = p->lengths;
    a->refs = p->refs;
    a->layers = p->layers;
    a->n_pages = p->n_pages;
    a->max_seqs = p->max_seqs;
    a->max_pages = p->max_pages;
    a->page = p->page;
    a->kv_heads = p->kv_heads;
    a->by_page = FastDiv((uint32_t)p->page);
    return RTA_OK;
}

// Workgroups of 256 threads in one grid dimension: below 2^32 threads.
constexpr int kMostGroups = (1 << 24) - 1;

inline int rows_args(int rows, const int32_t* seqs, const int32_t* cu, int n, RowList* l) {
    if (rows <= 0 || n <= 0 || (!cu && rows != n)) return RTA_ERR_SHAPE;
    if (rows > kMostGroups) return RTA_ERR_RANGE;
    if (!aligned(seqs, 4) || !aligned(cu, 4)) return RTA_ERR_ALIGN;
    *l = RowList{seqs, cu, rows, n};
    return RTA_OK;
}

}  // namespace host
}  // namespace rta
