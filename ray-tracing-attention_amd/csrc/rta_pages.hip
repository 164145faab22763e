// rta_pages.hip -- the paged history's book (pages handed out, shared, freed and closed up on
// the device) and the rows written into its pages and read back (gfx950).
//
// The book is a table of page numbers per sequence, the lengths and a reference count per page;
// a page with count 0 is free, and the lowest free pages are handed out first, so every result
// follows from the arguments alone (no order of atomics, no free list to keep).
#include <math.h>

#include "rta_pages.hpp"

namespace rta {

constexpr int kPlanThreads = 1024;   // the plan kernels' one workgroup
constexpr int kPlanWaves = kPlanThreads / kWave;

// Sums over a workgroup of kPlanThreads: the exclusive prefix of v, and the total in `total`.
__device__ __forceinline__ int block_scan(int v, int* red, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int s = v;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const int t = __shfl_up(s, o, kWave);
        if (lane >= o) s += t;
    }
    __syncthreads();   // red of the scan before has been read
    if (lane == kWave - 1) red[wave] = s;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) {
        const int t = red[w];
        if (w < wave) before += t;
        all += t;
    }
    total = all;
    return before + s - v;
}

__device__ __forceinline__ int load_agent(const int32_t* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void store_agent(int32_t* p, int v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Workspace of rta_pages_extend and rta_pages_compact, in int32.
struct PlanWs {
    int32_t* owner;     // [max_seqs] the first list entry of a sequence
    int32_t* begin;     // [n] an entry's first page in `list`, -1: left undone
    int32_t* kind;      // [n] what its last page needs: 0 nothing, 1 a copy, 2 a page (a hole)
    int32_t* src;       // [max(n, n_pages)] pages to copy, and where to
    int32_t* dst;
    int32_t* list;      // [n_pages] free pages in order
    int32_t* holders;   // [n_pages] listed sequences that share a page
    int32_t* keeper;    // [n_pages] the last of them
    int32_t* map;       // [n_pages] where a page goes (itself, if it stays), -1: it is free
    int32_t* count;     // pairs in src / dst
};

static size_t plan_ints(const rta_pages* p, int64_t n) {
    const int64_t pairs = n > p->n_pages ? n : p->n_pages;
    return (size_t)(p->max_seqs + 2 * n + 2 * pairs + 4 * (int64_t)p->n_pages + 4);
}
static PlanWs plan_ws(void* ws, const PageArgs& a, int n) {
    const int64_t pairs = n > a.n_pages ? n : a.n_pages;
    PlanWs w;
    int32_t* p = static_cast<int32_t*>(ws);
    w.count = p;
    w.owner = p + 4;
    w.begin = w.owner + a.max_seqs;
    w.kind = w.begin + n;
    w.src = w.kind + n;
    w.dst = w.src + pairs;
    w.list = w.dst + pairs;
    w.holders = w.list + a.n_pages;
    w.keeper = w.holders + a.n_pages;
    w.map = w.keeper + a.n_pages;
    return w;
}

// What entry i of an extend wants: its sequence, length, new length, pages without the last
// page's copy, and the last page where it is partly filled and the sequence grows.
struct Want {
    int seq, len, add, fresh, tail;   // tail: -2 none, -1 a hole, else the page
};
__device__ __forceinline__ bool want_of(const PageArgs& a, const int32_t* seqs, const int32_t* add, int i, Want& w) {
    w.seq = list_seq(seqs, i);
    w.add = add ? add[i] : 1;
    w.len = w.fresh = 0;
    w.tail = -2;
    if ((unsigned)w.seq >= (unsigned)a.max_seqs || w.add < 0) return false;
    w.len = a.lengths[w.seq];
    if (w.len < 0 || (int64_t)w.len + w.add > (int64_t)a.max_pages * a.page) return false;
    const int last = w.len + w.add;   // <= max_pages page <= INT_MAX
    auto pages = [&](int n) { return n ? (int)a.by_page.div((uint32_t)n - 1) + 1 : 0; };
    w.fresh = pages(last) - pages(w.len);
    const int e = (int)a.by_page.div((uint32_t)w.len);
    if (w.add > 0 && w.len - e * a.page > 0) {
        w.tail = a.table[(int64_t)w.seq * a.max_pages + e];
        if (bad_page(a, w.tail)) return false;
    }
    return true;
}

// One workgroup plans an extend: claims (a sequence listed twice keeps its first entry), the
// shared last pages, how many pages each entry needs, the free pages, and who gets which.
// Bound by latency: a few dependent trips through L2 and a read of refs up to the last page handed
// out.  What an entry wants is found once and kept in LDS (the first 1024 of them: the rest is
// found again where it is needed; 16 entries and 4096 pages 10.0 us so, 5 times each).
__global__ void __launch_bounds__(kPlanThreads) extend_plan_kernel(const PageArgs a, const int32_t* __restrict__ seqs,
                                                                   const int32_t* __restrict__ add, int n, PlanWs ws) {
    __shared__ int red[kPlanWaves];
    __shared__ int s_pairs;
    __shared__ Want kept[kPlanThreads];
    __shared__ uint8_t kept_ok[kPlanThreads];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    bool bad = false;
    if (tid == 0) s_pairs = 0;
    for (int i = tid; i < n; i += kPlanThreads) {
        Want w;
        const bool ok = want_of(a, seqs, add, i, w);
        if ((unsigned)w.seq < (unsigned)a.max_seqs) store_agent(ws.owner + w.seq, INT_MAX);
        if (i < kPlanThreads) {
            kept[i] = w;
            kept_ok[i] = ok;
        }
    }
    auto entry = [&](int i, Want& w) {
        if (i >= kPlanThreads) return want_of(a, seqs, add, i, w);
        w = kept[i];
        return kept_ok[i] != 0;
    };
    __syncthreads();
    for (int i = tid; i < n; i += kPlanThreads) {
        Want w;
        const bool ok = entry(i, w);
        if ((unsigned)w.seq < (unsigned)a.max_seqs) atomicMin(ws.owner + w.seq, i);
        if (ok && w.tail >= 0) {
            store_agent(ws.holders + w.tail, 0);
            store_agent(ws.keeper + w.tail, -1);
        }
    }
    __syncthreads();
    // entry i wants something and is its sequence's first
    auto mine = [&](int i, Want& w) { return entry(i, w) && load_agent(ws.owner + w.seq) == i; };
    for (int i = tid; i < n; i += kPlanThreads) {
        Want w;
        const bool ok = mine(i, w);
        if (i < kPlanThreads) kept_ok[i] = ok;   // (settled: mine() finds the same below)
        if (ok && w.tail >= 0 && a.refs[w.tail] > 1) {
            atomicAdd(ws.holders + w.tail, 1);
            atomicMax(ws.keeper + w.tail, i);
        }
    }
    __syncthreads();
    // pages wanted up to each entry, left in begin[i] as the exclusive prefix
    int64_t upto = 0;
    for (int base = 0; base < n; base += kPlanThreads) {
        const int i = base + tid;
        int need = 0, kind = 0;
        Want w;
        bool ok = i < n && (i < kPlanThreads ? entry(i, w) : mine(i, w));
        if (i < n && !ok) bad = true;
        if (ok) {
            if (w.tail == -1) {
                kind = 2;
            } else if (w.tail >= 0) {
                const int refs = a.refs[w.tail];
                if (refs > 1 && !(load_agent(ws.holders + w.tail) == refs && load_agent(ws.keeper + w.tail) == i)) kind = 1;
            }
            need = w.fresh + (kind ? 1 : 0);
        }
        int total;
        // (more than the pool holds is one page more than that: 1024 such wants stay below 2^31)
        need = min(need, a.n_pages + 1);
        const int before = block_scan(need, red, total);
        if (i < n) {
            const int64_t b = upto + before;
            const bool fits = ok && b + need <= a.n_pages;
            if (ok && !fits) bad = true;
            ws.begin[i] = fits ? (int)b : -1;
            ws.kind[i] = kind;
        }
        upto += total;
    }
    const int wanted = upto < a.n_pages ? (int)upto : a.n_pages;
    // the lowest free pages, as many as wanted: 16 a thread and turn
    constexpr int kPer = 16;
    int found = 0;
    for (int base = 0; base < a.n_pages && found < wanted; base += kPer * kPlanThreads) {
        uint32_t mask = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int at = base + kPer * tid + j;
            mask |= (at < a.n_pages && a.refs[min(at, a.n_pages - 1)] == 0 ? 1u : 0u) << j;
        }
        int total;
        int at = found + block_scan(__popc(mask), red, total);
        for (; mask; mask &= mask - 1) {
            if (at < wanted) ws.list[at] = base + kPer * tid + __ffs(mask) - 1;
            ++at;
        }
        found += total;
    }
    __syncthreads();   // list, begin, kind are the workgroup's to read
    // hand out: a wave per entry
    for (int i = wave; i < n; i += kPlanWaves) {
        const int begin = ws.begin[i];
        if (begin < 0) continue;
        Want w;
        entry(i, w);
        const int kind = ws.kind[i], need = w.fresh + (kind ? 1 : 0);
        if (begin + need > found) {
            bad = true;
            continue;
        }
        int32_t* row = a.table + (int64_t)w.seq * a.max_pages;
        const int e0 = w.len ? (int)a.by_page.div((uint32_t)w.len - 1) + 1 : 0;
        for (int j = lane; j < w.fresh; j += kWave) {
            const int page = ws.list[begin + (kind ? 1 : 0) + j];
            row[e0 + j] = page;
            a.refs[page] = 1;
        }
        if (lane == 0) {
            if (kind) {
                const int page = ws.list[begin];
                row[a.by_page.div((uint32_t)w.len)] = page;
                a.refs[page] = 1;
                if (kind == 1) {
                    atomicSub(a.refs + w.tail, 1);
                    const int k = atomicAdd(&s_pairs, 1);
                    ws.src[k] = w.tail;
                    ws.dst[k] = page;
                }
            }
            a.lengths[w.seq] = w.len + w.add;
        }
    }
    if (bad) raise_error(RTA_DEVERR_PAGES);
    __syncthreads();
    if (tid == 0) *ws.count = s_pairs;
}

// ------------------------------------------------------------------ page copies ----
// Page src[k] to dst[k] of every layer, k < *count: pieces of 256 x 16 bytes handed out over the grid.
__device__ __forceinline__ void copy_pages(const PageArgs& a, const int32_t* src, const int32_t* dst, int pairs) {
    const int64_t words = a.page_bytes / 16;
    const int64_t pieces = (words + 255) / 256, items = pieces * a.layers * pairs;
    for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
        const int64_t piece = it % pieces, rest = it / pieces;
        const int layer = (int)(rest % a.layers), k = (int)(rest / a.layers);
        const int64_t w = piece * 256 + threadIdx.x;
        uint8_t* base = a.pool + layer * a.layer_bytes;
        if (w < words)
            reinterpret_cast<uint4*>(base + dst[k] * a.page_bytes)[w] =
                reinterpret_cast<const uint4*>(base + src[k] * a.page_bytes)[w];
    }
}

__global__ void __launch_bounds__(256) pages_copy_kernel(const PageArgs a, const int32_t* src, const int32_t* dst,
                                                         const int32_t* count) {
    copy_pages(a, src, dst, *count);
}

// ------------------------------------------------------------------ fork, free ----
// Whether an entry before i lists value s (read by the whole workgroup).
__device__ __forceinline__ bool listed_before(const int32_t* list, int i, int s) {
    bool hit = false;
    for (int j = threadIdx.x; j < i; j += blockDim.x) hit |= list_seq(list, j) == s;
    return __syncthreads_or(hit);
}

// A workgroup per entry.  No entry writes what another reads: a destination is empty, listed
// once and no source, so the sources' rows stand still.
__global__ void __launch_bounds__(256) pages_fork_kernel(const PageArgs a, const int32_t* __restrict__ src,
                                                         const int32_t* __restrict__ dst, int n) {
    const int i = blockIdx.x, s = src[i], d = dst[i];
    bool ok = (unsigned)s < (unsigned)a.max_seqs && (unsigned)d < (unsigned)a.max_seqs;
    ok = !listed_before(dst, i, d) && ok;
    ok = !listed_before(src, n, d) && ok;
    const int len = ok ? a.lengths[s] : 0;
    ok = ok && !bad_length(a, len) && a.lengths[d] == 0;
    const int pages = ok && len ? (int)a.by_page.div((uint32_t)len - 1) + 1 : 0;
    const int32_t* from = a.table + (int64_t)s * a.max_pages;
    int32_t* to = a.table + (int64_t)d * a.max_pages;
    bool bad = false;
    for (int e = threadIdx.x; e < pages; e += 256) bad = bad || bad_page(a, from[e]);
    if (__syncthreads_or(bad) || !ok) {   // (and every thread has read lengths[d])
        if (threadIdx.x == 0) raise_error(RTA_DEVERR_PAGES);
        return;
    }
    for (int e = threadIdx.x; e < pages; e += 256) {
        const int p = from[e];
        to[e] = p;
        if (p >= 0) atomicAdd(a.refs + p, 1);
    }
    if (threadIdx.x == 0) a.lengths[d] = len;
}

__global__ void __launch_bounds__(256) pages_free_kernel(const PageArgs a, const int32_t* __restrict__ seqs,
                                                         const int32_t* __restrict__ first,
                                                         const int32_t* __restrict__ last) {
    const int i = blockIdx.x, s = list_seq(seqs, i);
    bool ok = (unsigned)s < (unsigned)a.max_seqs;
    if (seqs) ok = !listed_before(seqs, i, s) && ok;
    const int lo = first ? first[i] : 0, len = ok ? a.lengths[s] : 0, hi = last ? last[i] : len;
    ok = ok && lo >= 0 && !bad_length(a, len);
    const int pages = ok && len ? (int)a.by_page.div((uint32_t)len - 1) + 1 : 0;
    int32_t* row = a.table + (int64_t)s * a.max_pages;
    // the first page that begins at or past lo, and how many from there end at hi
    const int e0 = ok ? (int)a.by_page.div((uint32_t)lo) + (lo % a.page ? 1 : 0) : 0;
    const int e1 = !ok ? 0 : hi >= len ? pages : hi > 0 ? (int)a.by_page.div((uint32_t)hi) : 0;
    bool bad = false;
    for (int e = e0 + (int)threadIdx.x; e < e1; e += 256) bad = bad || bad_page(a, row[e]);
    if (__syncthreads_or(bad) || !ok) {   // (and every thread has read lengths[s])
        if (threadIdx.x == 0) raise_error(RTA_DEVERR_PAGES);
        return;
    }
    for (int e = e0 + (int)threadIdx.x; e < e1; e += 256) {
        const int p = row[e];
        row[e] = -1;
        if (p >= 0) atomicSub(a.refs + p, 1);
    }
    if (threadIdx.x == 0 && hi >= len && lo < len) a.lengths[s] = lo;
}

__global__ void __launch_bounds__(256) pages_init_kernel(const PageArgs a) {
    const int64_t step = (int64_t)gridDim.x * 256, at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t entries = (int64_t)a.max_seqs * a.max_pages;
    for (int64_t i = at; i < entries; i += step) a.table[i] = -1;
    for (int64_t i = at; i < a.max_seqs; i += step) a.lengths[i] = 0;
    for (int64_t i = at; i < a.n_pages; i += step) a.refs[i] = 0;
}

// ------------------------------------------------------------------ compact ----
// One workgroup: the number U of used pages, the holes below it and the used pages past it, both
// in order (they are equally many), and where every page goes.
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const PageArgs a, PlanWs ws, int32_t* used_out) {
    __shared__ int red[kPlanWaves];
    const int tid = threadIdx.x;
    int used = 0;
    for (int i = tid; i < a.n_pages; i += kPlanThreads) used += a.refs[i] > 0;
    int total;
    block_scan(used, red, total);
    const int U = total;
    int holes = 0, movers = 0;
    for (int base = 0; base < a.n_pages; base += kPlanThreads) {
        const int i = base + tid;
        const bool in = i < a.n_pages, use = in && a.refs[i] > 0;
        const bool hole = in && !use && i < U, mover = use && i >= U;
        int k;
        int at = holes + block_scan(hole, red, k);
        if (hole) ws.dst[at] = i;
        holes += k;
        at = movers + block_scan(mover, red, k);
        if (mover) ws.src[at] = i;
        movers += k;
        if (in && !mover) ws.map[i] = use ? i : -1;
    }
    __syncthreads();
    for (int k = tid; k < movers; k += kPlanThreads) ws.map[ws.src[k]] = ws.dst[k];
    if (tid == 0) {
        *ws.count = movers;
        if (used_out) *used_out = U;
    }
}

__global__ void __launch_bounds__(256) compact_kernel(const PageArgs a, PlanWs ws) {
    const int pairs = ws.count[0];
    if (!pairs) return;
    const int64_t step = (int64_t)gridDim.x * 256, at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    for (int64_t k = at; k < pairs; k += step) {
        a.refs[ws.dst[k]] = a.refs[ws.src[k]];
        a.refs[ws.src[k]] = 0;
    }
    const int64_t entries = (int64_t)a.max_seqs * a.max_pages;
    bool bad = false;
    for (int64_t e = at; e < entries; e += step) {
        const int p = a.table[e];
        if (p == -1) continue;
        const int to = (unsigned)p < (unsigned)a.n_pages ? ws.map[p] : -1;
        if (to < 0) bad = true;   // (left as it is: a page that the counts call free)
        else if (to != p) a.table[e] = to;
    }
    if (bad) raise_error(RTA_DEVERR_PAGES);
    copy_pages(a, ws.src, ws.dst, pairs);
}

// ------------------------------------------------------------------ rows in, rows out ----
template <int FMT> struct Element;
template <> struct Element<RTA_F16> { using T = uint16_t; };
template <> struct Element<RTA_BF16> { using T = uint16_t; };
template <> struct Element<RTA_Q8_ROW> { using T = int8_t; };

// fp32 to bfloat16, nearest even; a NaN keeps its upper bits and stays one.
__device__ __forceinline__ uint16_t bf16_bits(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    if ((b & 0x7fffffffu) > 0x7f800000u) return (uint16_t)(b >> 16) | 0x40u;
    return (uint16_t)((b + 0x7fffu + ((b >> 16) & 1u)) >> 16);
}

// Where head h's row of position p lies: its element index inside the page and the page's bytes.
__device__ __forceinline__ uint8_t* row_page(const PageArgs& a, const RowList& l, int r, int& off, bool& listed) {
    int i, first, count;
    listed = row_entry(l, r, i, first, count);
    if (!listed) return nullptr;
    const int s = list_seq(l.seqs, i);
    if ((unsigned)s >= (unsigned)a.max_seqs) return nullptr;
    const int64_t pos = (int64_t)a.lengths[s] - count + (r - first);
    if (pos < 0 || pos >= (int64_t)a.max_pages * a.page) return nullptr;
    const int e = (int)a.by_page.div((uint32_t)pos);
    off = (int)pos - e * a.page;
    const int page = page_of(a, a.table + (int64_t)s * a.max_pages, e);
    return page < 0 ? nullptr : a.pool + page * a.page_bytes;
}

// A workgroup per row and 2048 of its 2 kv_heads hd values: 8 values a thread.
template <int FMT, int HD>
__device__ __forceinline__ void append_row(const PageArgs& a, const RowList& l, const float* __restrict__ k,
                                           int64_t k_stride, const float* __restrict__ v, int64_t v_stride) {
    const int r = blockIdx.x;
    int off = 0;
    bool listed;
    uint8_t* page = row_page(a, l, r, off, listed);
    if (!page) {
        if (listed && threadIdx.x == 0 && blockIdx.y == 0) raise_error(RTA_DEVERR_PAGES);
        return;
    }
    constexpr int kPer = HD / 8;   // threads per head
    const int c = blockIdx.y * 256 + threadIdx.x, which_h = c / kPer, d = 8 * (c % kPer);
    if (which_h >= 2 * a.kv_heads) return;   // whole heads: kPer divides 64
    const int which = which_h >= a.kv_heads, h = which_h - which * a.kv_heads;
    const float* x = (which ? v + r * v_stride : k + r * k_stride) + h * HD + d;
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = x[j];
    const int64_t row = (int64_t)which_h * a.page + off;
    if constexpr (FMT == RTA_Q8_ROW) {
        float m = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fabsf(f[j]) < INFINITY ? fmaxf(m, fabsf(f[j])) : INFINITY;   // NaN too
        m = group_max(m, kPer);
        const float scale = m * (1.0f / 127.0f), den = scale > 0.0f ? scale : 1.0f;
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            // (a subnormal scale may be rounded down by more than the half step of code 127; an
            // infinite one makes every value of the head 0 inf = NaN)
            const float code = scale < INFINITY ? fminf(fmaxf(rintf(f[j] / den), -127.0f), 127.0f) : 0.0f;
            w[j >> 2] |= ((uint32_t)(int)code & 255u) << (8 * (j & 3));
        }
        *reinterpret_cast<uint2*>(page + row * HD + d) = uint2{w[0], w[1]};
        if (d == 0) reinterpret_cast<float*>(page + (int64_t)2 * a.kv_heads * a.page * HD)[row] = scale;
    } else {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint16_t lo, hi;
            if constexpr (FMT == RTA_F16) {
                lo = __builtin_bit_cast(uint16_t, (_Float16)f[2 * j]);
                hi = __builtin_bit_cast(uint16_t, (_Float16)f[2 * j + 1]);
            } else {
                lo = bf16_bits(f[2 * j]);
                hi = bf16_bits(f[2 * j + 1]);
            }
            w[j] = lo | (uint32_t)hi << 16;
        }
        *reinterpret_cast<uint4*>(page + (row * HD + d) * 2) = uint4{w[0], w[1], w[2], w[3]};
    }
}

template <int FMT, int HD>
__global__ void __launch_bounds__(256) append_kernel(const PageArgs a, const RowList l, const float* __restrict__ k,
                                                     int64_t k_stride, const float* __restrict__ v,
                                                     int64_t v_stride) {
    append_row<FMT, HD>(a, l, k, k_stride, v, v_stride);
    if (blockIdx.x == 0 && blockIdx.y == 0 && bad_rows(l)) raise_error(RTA_DEVERR_PAGES);
}

template <int FMT, int HD>
__device__ __forceinline__ void read_row(const PageArgs& a, const RowList& l, float* __restrict__ k, int64_t k_stride,
                                         float* __restrict__ v, int64_t v_stride) {
    const int r = blockIdx.x;
    int off = 0;
    bool listed;
    const uint8_t* page = row_page(a, l, r, off, listed);
    if (!listed) return;
    if (!page && threadIdx.x == 0 && blockIdx.y == 0) raise_error(RTA_DEVERR_PAGES);
    constexpr int kPer = HD / 8;
    const int c = blockIdx.y * 256 + threadIdx.x, which_h = c / kPer, d = 8 * (c % kPer);
    if (which_h >= 2 * a.kv_heads) return;
    const int which = which_h >= a.kv_heads, h = which_h - which * a.kv_heads;
    float* x = which ? v : k;
    if (!x) return;
    x += r * (which ? v_stride : k_stride) + h * HD + d;
    float f[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (page) {
        const int64_t row = (int64_t)which_h * a.page + off;
        if constexpr (FMT == RTA_Q8_ROW) {
            const uint2 w = *reinterpret_cast<const uint2*>(page + row * HD + d);
            const float scale = reinterpret_cast<const float*>(page + (int64_t)2 * a.kv_heads * a.page * HD)[row];
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = (float)(int8_t)((j < 4 ? w.x : w.y) >> (8 * (j & 3))) * scale;
        } else {
            const uint4 w = *reinterpret_cast<const uint4*>(page + (row * HD + d) * 2);
            const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if constexpr (FMT == RTA_F16) f[j] = j & 1 ? half_hi(u[j >> 1]) : half_lo(u[j >> 1]);
                else f[j] = __builtin_bit_cast(float, j & 1 ? u[j >> 1] & 0xffff0000u : u[j >> 1] << 16);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = f[j];
}

template <int FMT, int HD>
__global__ void __launch_bounds__(256) page_read_kernel(const PageArgs a, const RowList l, float* __restrict__ k,
                                                        int64_t k_stride, float* __restrict__ v, int64_t v_stride) {
    read_row<FMT, HD>(a, l, k, k_stride, v, v_stride);
    if (blockIdx.x == 0 && blockIdx.y == 0 && bad_rows(l)) raise_error(RTA_DEVERR_PAGES);
}

// f(std::integral_constant<int, FMT>, std::integral_constant<int, HD>) of a checked descriptor.
template <class F>
static void with_page_format(const rta_pages* p, F&& f) {
    auto by_hd = [&](auto fmt) {
        if (p->head_dim == 64) f(fmt, std::integral_constant<int, 64>{});
        else if (p->head_dim == 128) f(fmt, std::integral_constant<int, 128>{});
        else f(fmt, std::integral_constant<int, 256>{});
    };
    if (p->fmt == RTA_F16) by_hd(std::integral_constant<int, RTA_F16>{});
    else if (p->fmt == RTA_BF16) by_hd(std::integral_constant<int, RTA_BF16>{});
    else by_hd(std::integral_constant<int, RTA_Q8_ROW>{});
}

static int launched() { return hipGetLastError() == hipSuccess ? RTA_OK : RTA_ERR_LAUNCH; }

// Workgroups of a copy of up to `pages` pages of every layer, 4 KB each, 8 per compute unit at most.
static unsigned copy_grid(const PageArgs& a, int64_t pages) {
    const int64_t items = (a.page_bytes / 16 + 255) / 256 * a.layers * pages;
    return (unsigned)(items < 2048 ? items : 2048);
}

}  // namespace rta

using namespace rta;

extern "C" {

int64_t rta_page_bytes(int fmt, int kv_heads, int head_dim, int page) {
    return host::page_bytes(fmt, kv_heads, head_dim, page);
}

int rta_pages_init(const rta_pages* pages, rta_stream_t stream) {
    PageArgs a;
    const int rc = host::pages_args(pages, -1, &a);
    if (rc) return rc;
    hipLaunchKernelGGL(pages_init_kernel, dim3(512), dim3(256), 0, (hipStream_t)stream, a);
    return launched();
}

size_t rta_pages_workspace_bytes(const rta_pages* pages, int n) {
    PageArgs a;
    if (host::pages_args(pages, -1, &a) || n <= 0) return 0;
    return (plan_ints(pages, n) * 4 + 15) / 16 * 16;
}

int rta_pages_extend(const rta_pages* pages, const int32_t* seqs, const int32_t* add, int n, void* workspace,
                     size_t workspace_bytes, rta_stream_t stream) {
    PageArgs a;
    const int rc = host::pages_args(pages, -1, &a);
    if (rc) return rc;
    if (n <= 0) return RTA_ERR_SHAPE;
    if (!host::aligned(seqs, 4) || !host::aligned(add, 4)) return RTA_ERR_ALIGN;
    if (!workspace || workspace_bytes < rta_pages_workspace_bytes(pages, n) || !host::aligned(workspace, 16))
        return RTA_ERR_WORKSPACE;
    const PlanWs ws = plan_ws(workspace, a, n);
    hipStream_t s = (hipStream_t)stream;
    hipLaunchKernelGGL(extend_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, a, seqs, add, n, ws);
    hipLaunchKernelGGL(pages_copy_kernel, dim3(copy_grid(a, n)), dim3(256), 0, s, a, ws.src, ws.dst, ws.count);
    return launched();
}

int rta_pages_fork(const rta_pages* pages, const int32_t* src, const int32_t* dst, int n, rta_stream_t stream) {
    PageArgs a;
    const int rc = host::pages_args(pages, -1, &a);
    if (rc) return rc;
    if (!src || !dst) return RTA_ERR_NULL;
    if (n <= 0) return RTA_ERR_SHAPE;
    if (n > host::kMostGroups) return RTA_ERR_RANGE;
    if (!host::aligned(src, 4) || !host::aligned(dst, 4)) return RTA_ERR_ALIGN;
    hipLaunchKernelGGL(pages_fork_kernel, dim3(n), dim3(256), 0, (hipStream_t)stream, a, src, dst, n);
    return launched();
}

int rta_pages_free(const rta_pages* pages, const int32_t* seqs, const int32_t* first, const int32_t* last, int n,
                   rta_stream_t stream) {
    PageArgs a;
    const int rc = host::pages_args(pages, -1, &a);
    if (rc) return rc;
    if (n <= 0) return RTA_ERR_SHAPE;
    if (n > host::kMostGroups) return RTA_ERR_RANGE;
    if (!host::aligned(seqs, 4) || !host::aligned(first, 4) || !host::aligned(last, 4)) return RTA_ERR_ALIGN;
    hipLaunchKernelGGL(pages_free_kernel, dim3(n), dim3(256), 0, (hipStream_t)stream, a, seqs, first, last);
    return launched();
}

int rta_pages_compact(const rta_pages* pages, int32_t* used, void* workspace, size_t workspace_bytes,
                      rta_stream_t stream) {
    PageArgs a;
    const int rc = host::pages_args(pages, -1, &a);
    if (rc) return rc;
    if (!host::aligned(used, 4)) return RTA_ERR_ALIGN;
    if (!workspace || workspace_bytes < rta_pages_workspace_bytes(pages, 1) || !host::aligned(workspace, 16))
        return RTA_ERR_WORKSPACE;
    const PlanWs ws = plan_ws(workspace, a, 1);
    hipStream_t s = (hipStream_t)stream;
    hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, a, ws, used);
    hipLaunchKernelGGL(compact_kernel, dim3(2048), dim3(256), 0, s, a, ws);
    return launched();
}

int rta_paged_append(const rta_pages* pages, int layer, const float* k, int64_t k_stride, const float* v,
                     int64_t v_stride, int rows, const int32_t* seqs, const int32_t* cu_rows, int n,
                     rta_stream_t stream) {
    PageArgs a;
    if (layer < 0) return RTA_ERR_RANGE;
    int rc = host::pages_args(pages, layer, &a);
    if (rc) return rc;
    if (!k || !v) return RTA_ERR_NULL;
    RowList l;
    rc = host::rows_args(rows, seqs, cu_rows, n, &l);
    if (rc) return rc;
    const int width = pages->kv_heads * pages->head_dim;
    if (k_stride < width || v_stride < width) return RTA_ERR_SHAPE;
    if (!host::aligned(k, 4) || !host::aligned(v, 4)) return RTA_ERR_ALIGN;
    with_page_format(pages, [&](auto fmt, auto hd) {
        hipLaunchKernelGGL((append_kernel<decltype(fmt)::value, decltype(hd)::value>),
                           dim3(rows, (2 * width + 2047) / 2048), dim3(256), 0, (hipStream_t)stream, a, l, k, k_stride,
                           v, v_stride);
    });
    return launched();
}

int rta_paged_read(const rta_pages* pages, int layer, int rows, const int32_t* seqs, const int32_t* cu_rows, int n,
                   float* k, int64_t k_stride, float* v, int64_t v_stride, rta_stream_t stream) {
    PageArgs a;
    if (layer < 0) return RTA_ERR_RANGE;
    int rc = host::pages_args(pages, layer, &a);
    if (rc) return rc;
    if (!k && !v) return RTA_ERR_NULL;
    RowList l;
    rc = host::rows_args(rows, seqs, cu_rows, n, &l);
    if (rc) return rc;
    const int width = pages->kv_heads * pages->head_dim;
    if ((k && k_stride < width) || (v && v_stride < width)) return RTA_ERR_SHAPE;
    if (!host::aligned(k, 4) || !host::aligned(v, 4)) return RTA_ERR_ALIGN;
    with_page_format(pages, [&](auto fmt, auto hd) {
        hipLaunchKernelGGL((page_read_kernel<decltype(fmt)::value, decltype(hd)::value>),
                           dim3(rows, (2 * width + 2047) / 2048), dim3(256), 0, (hipStream_t)stream, a, l, k, k_stride,
                           v, v_stride);
    });
    return launched();
}

}  // extern "C"
