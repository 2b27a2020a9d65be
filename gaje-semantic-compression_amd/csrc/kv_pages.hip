// Bookkeeping and copies of a paged KV cache (gaje_hip_kv_update, _compact, _append).
//
// Update.  Slot d takes slot source[d]'s pages as they were; kept positions
// n = min(len, len + add).  With G positions a page, pages 0 .. n/G - 1 are kept
// whole and shared; page n/G, if n % G > 0, is kept in part, and a slot may go on
// writing it only if no other slot refers to it: it stays with the lowest slot
// that keeps part of it when nobody keeps it whole, all others get a copy.  New
// pages are the lowest free ones, handed out in slot order.  All of it is counts,
// minima and prefix sums of integers, so the order of the atomics does not show.
// One workgroup does that in one launch (a grid the counting, where the table is large); a
// second one writes the new arrays and copies pages.
//
// Bound by the launches and by one workgroup's passes over table and counts for the
// bookkeeping, by HBM for the copies.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "common.h"
#include "device_util.h"
#include "serve.h"

namespace gaje {
namespace {

constexpr int PLAN_THREADS = 1024, PLAN_WAVES = PLAN_THREADS / WAVE;

// Workspace of a plan: [0] copies, [1] status bits so far; per page the slots that keep it
// (then: its new count), the lowest slot that keeps part of it, and the list of free pages
// (compact: where a page goes); per slot what it becomes, where its new pages start in the
// list, its copy's place or -1; the copies' pages.
struct PlanWorkspace {
    int32_t *n_copy, *bad;
    int32_t *count, *owner, *list;           // [n_pages]
    int32_t *from, *size, *whole, *first, *place;  // [n_seq]; whole: pages kept whole and flags
    int32_t *src, *dst;                      // copies
    int64_t bytes;
};
// In `whole`: one more page is kept in part; the slot's status bits 1 and 2.
constexpr int PART = 1 << 30, SLOT_ERROR = 28, KEPT = (1 << 28) - 1;
PlanWorkspace plan_workspace(void *base, const gaje_hip_kv_pages &c) {
    PlanWorkspace w{};
    int64_t off = 0;
    auto take = [&](int64_t n) {
        int32_t *p = (int32_t *)((char *)base + off);
        off += (n * 4 + 255) / 256 * 256;
        return p;
    };
    const int64_t copies = std::max(c.n_seq, c.n_pages);
    w.n_copy = take(2);
    w.bad = w.n_copy + 1;
    w.count = take(c.n_pages);
    w.owner = take(c.n_pages);
    w.list = take(c.n_pages);
    w.from = take(c.n_seq);
    w.size = take(c.n_seq);
    w.whole = take(c.n_seq);
    w.first = take(c.n_seq);
    w.place = take(c.n_seq);
    w.src = take(copies);
    w.dst = take(copies);
    w.bytes = off;
    return w;
}

// Values that other waves of the workgroup changed with atomics are read past the
// wave's own L1.
__device__ __forceinline__ int ld_shared(const int32_t *p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void st_shared(int32_t *p, int v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Sums stop at a value past every pool size: more pages than that are missing, however many.
constexpr int SUM_CAP = 1 << 28;
__device__ __forceinline__ int add_cap(int a, int b) { return min(a + b, SUM_CAP); }

// Exclusive prefix sums of two counts over the workgroup, with the totals; red:
// one int2 per wave.  Every thread calls it.
__device__ int2 scan2(int a, int b, int2 *red, int2 &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int2 v = make_int2(a, b);
#pragma unroll
    for (int o = 1; o < WAVE; o <<= 1) {
        const int x = __shfl_up(v.x, o, WAVE), y = __shfl_up(v.y, o, WAVE);
        if (lane >= o) v.x = add_cap(v.x, x), v.y = add_cap(v.y, y);
    }
    if (lane == WAVE - 1) red[wave] = v;
    __syncthreads();
    int2 before = make_int2(0, 0);
    total = make_int2(0, 0);
    for (int w = 0; w < PLAN_WAVES; ++w) {
        const int2 r = red[w];
        if (w < wave) before.x = add_cap(before.x, r.x), before.y = add_cap(before.y, r.y);
        total.x = add_cap(total.x, r.x), total.y = add_cap(total.y, r.y);
    }
    __syncthreads();
    return make_int2(before.x + v.x - a, before.y + v.y - b);
}

// The steps of an update, each by threads t, t + n, ... of one workgroup or of a grid.
struct UpdateArgs {
    gaje_hip_kv_pages c;
    const int32_t *source, *add;
    int32_t *new_table, *new_len, *new_ref, *status;
    PlanWorkspace w;
    int32_t shift;
};

// What every slot becomes; no references yet.
__device__ __forceinline__ void update_begin(const UpdateArgs &a, int64_t t, int64_t n) {
    const gaje_hip_kv_pages &c = a.c;
    for (int64_t p = t; p < c.n_pages; p += n) {
        st_shared(a.w.count + p, 0);
        st_shared(a.w.owner + p, INT32_MAX);
    }
    if (t == 0) st_shared(a.w.bad, 0);
    const int64_t most = c.max_pages << a.shift;
    for (int64_t d = t; d < c.n_seq; d += n) {
        int src = a.source ? a.source[d] : (int)d, err = 0;
        const int64_t more = a.add ? a.add[d] : 0;
        if (src < -1 || src >= c.n_seq) err = 1, src = -1;
        const int64_t base = src < 0 ? 0 : min(max((int64_t)c.len[src], (int64_t)0), most);
        int64_t size = base + more;
        if (size < 0 || size > most) err |= 2, size = 0;
        const int64_t kept = min(base, size);
        a.w.from[d] = src;
        a.w.size[d] = (int32_t)size;
        a.w.whole[d] = (int32_t)(kept >> a.shift) | (kept & (((int64_t)1 << a.shift) - 1) ? PART : 0) | err << SLOT_ERROR;
    }
}

// e / width, in 32 bits where all entries fit.
__device__ __forceinline__ int slot_of_entry(int64_t e, uint32_t width, bool narrow) {
    return narrow ? (int)((uint32_t)e / width) : (int)(e / width);
}

// References to every kept page: four table entries of a thread in flight.
__device__ __forceinline__ void update_count(const UpdateArgs &a, int64_t t, int64_t n) {
    const gaje_hip_kv_pages &c = a.c;
    const uint32_t width = (uint32_t)c.max_pages;
    const int64_t all = c.n_seq * c.max_pages;
    const bool narrow = all <= UINT32_MAX;
    int err = 0;
    for (int64_t e0 = t; e0 < all; e0 += 4 * n) {
        int id[4], d[4];
        bool in[4], part[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t e = e0 + u * n;
            d[u] = e < all ? slot_of_entry(e, width, narrow) : 0;
            const int i = e < all ? (int)(e - (int64_t)d[u] * width) : 0, whole = a.w.whole[d[u]], src = a.w.from[d[u]];
            part[u] = i == (whole & KEPT);
            in[u] = e < all && (i < (whole & KEPT) || (part[u] && (whole & PART)));
            id[u] = c.table[in[u] ? (int64_t)src * width + i : 0];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (!in[u]) continue;
            if (id[u] < 0 || id[u] >= c.n_pages) err = 8;
            else if (!part[u]) atomicAdd(a.w.count + id[u], 1);
            else atomicMin(a.w.owner + id[u], d[u]);
        }
    }
    if (err) atomicOr(a.w.bad, err);
}

// The new pages that each slot needs and where they start, its copy; the lowest free pages;
// the status.  By one workgroup.
__device__ __forceinline__ void update_plan(const UpdateArgs &a, int2 *red, int *bad_lds) {
    const gaje_hip_kv_pages &c = a.c;
    const PlanWorkspace &w = a.w;
    const int tid = threadIdx.x;
    const int64_t mask = ((int64_t)1 << a.shift) - 1;
    if (tid == 0) *bad_lds = ld_shared(w.bad);
    __syncthreads();
    int bad = 0;
    for (int64_t d = tid; d < c.n_seq; d += PLAN_THREADS) bad |= w.whole[d] >> SLOT_ERROR & 3;
    if (bad) atomicOr(bad_lds, bad);
    __syncthreads();
    bad = *bad_lds;
    int64_t need = 0, copies = 0, found = 0;
    if (!bad) {
        for (int64_t d0 = 0; d0 < c.n_seq; d0 += PLAN_THREADS) {
            const int64_t d = d0 + tid;
            int fresh = 0, copy = 0;
            if (d < c.n_seq) {
                const int whole = w.whole[d];
                bool keep = false;
                if (whole & PART) {
                    const int id = c.table[(int64_t)w.from[d] * c.max_pages + (whole & KEPT)];
                    keep = ld_shared(w.count + id) == 0 && ld_shared(w.owner + id) == d;
                    copy = !keep;
                }
                fresh = (int)((w.size[d] + mask) >> a.shift) - (whole & KEPT) - keep;
            }
            int2 total;
            const int2 at = scan2(fresh, copy, red, total);
            if (d < c.n_seq) {
                w.first[d] = (int32_t)(need + at.x);
                w.place[d] = copy ? (int32_t)(copies + at.y) : -1;
            }
            need += total.x;
            copies += total.y;
        }
        // (eight pages a thread and turn: the scans, not the counts, take the time)
        for (int64_t p0 = 0; p0 < c.n_pages && found < need; p0 += 8 * PLAN_THREADS) {
            const int64_t p = p0 + 8 * tid;
            uint32_t free = 0;
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (p + u < c.n_pages && c.ref[p + u] <= 0) free |= 1u << u;
            int2 total;
            int at = (int)min(found, need) + scan2(__popc(free), 0, red, total).x;
            for (; free && at < need; free &= free - 1) w.list[at++] = (int32_t)(p + __builtin_ctz(free));
            found += total.x;
        }
        if (found < need) bad = 4;
    }
    if (tid == 0) {
        a.status[0] = bad;
        w.n_copy[0] = bad ? 0 : (int32_t)copies;
        w.bad[0] = bad;
    }
    __syncthreads();
    if (bad) return;
    // the counts of new pages and of pages that stay with one slot
    for (int64_t i = tid; i < need; i += PLAN_THREADS) st_shared(w.count + w.list[i], 1);
    for (int64_t d = tid; d < c.n_seq; d += PLAN_THREADS) {
        const int whole = w.whole[d];
        if (whole & PART) {
            const int id = c.table[(int64_t)w.from[d] * c.max_pages + (whole & KEPT)];
            if (w.place[d] < 0) st_shared(w.count + id, 1);
            else w.src[w.place[d]] = id, w.dst[w.place[d]] = w.list[w.first[d]];
        }
    }
}

__global__ __launch_bounds__(256) void kv_begin_kernel(UpdateArgs a) {
    update_begin(a, (int64_t)blockIdx.x * 256 + threadIdx.x, (int64_t)gridDim.x * 256);
}
__global__ __launch_bounds__(256) void kv_count_kernel(UpdateArgs a) {
    update_count(a, (int64_t)blockIdx.x * 256 + threadIdx.x, (int64_t)gridDim.x * 256);
}
// ALL: the whole plan by one workgroup, else what follows the two above.
template <bool ALL>
__global__ __launch_bounds__(PLAN_THREADS) void kv_plan_kernel(UpdateArgs a) {
    __shared__ int2 red[PLAN_WAVES];
    __shared__ int bad;
    if constexpr (ALL) {
        update_begin(a, threadIdx.x, PLAN_THREADS);
        __syncthreads();
        update_count(a, threadIdx.x, PLAN_THREADS);
        __syncthreads();
    }
    update_plan(a, red, &bad);
}

// n_copy pages of every layer, K and V: one (copy, layer, pool) per workgroup and
// turn, 16 bytes per lane.
__device__ __forceinline__ void copy_pages(const gaje_hip_kv_pages &c, const int32_t *n_copy, const int32_t *src, const int32_t *dst,
                                           int64_t page_bytes) {
    const int64_t per = c.n_layer * 2, n = n_copy[0] * per;
    for (int64_t i = blockIdx.x; i < n; i += gridDim.x) {
        const int64_t copy = i / per, layer = i % per >> 1;
        char *pool = (char *)(i & 1 ? c.v : c.k) + layer * c.n_pages * page_bytes;
        const char *from = pool + src[copy] * page_bytes;
        char *to = pool + dst[copy] * page_bytes;
        // four pieces of a thread in flight
        for (int64_t b = threadIdx.x * 16; b < page_bytes; b += 4 * 256 * 16) {
            vu4 x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) x[u] = *(const vu4 *)(from + min(b + u * 4096, page_bytes - 16));
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (b + u * 4096 < page_bytes) *(vu4 *)(to + b + u * 4096) = x[u];
        }
    }
}
// The new arrays, or the old ones where the plan failed, and the copies.
__global__ __launch_bounds__(256) void kv_write_kernel(UpdateArgs a, int64_t page_bytes) {
    const gaje_hip_kv_pages &c = a.c;
    const PlanWorkspace &w = a.w;
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x, n = (int64_t)gridDim.x * 256, all = c.n_seq * c.max_pages;
    const bool bad = w.bad[0] != 0, narrow = all <= UINT32_MAX;
    const uint32_t width = (uint32_t)c.max_pages;
    for (int64_t e = t; e < all; e += n) {
        if (bad) {
            a.new_table[e] = c.table[e];
            continue;
        }
        const int d = slot_of_entry(e, width, narrow), i = (int)(e - (int64_t)d * width);
        const int whole = w.whole[d], held = (whole & KEPT) + ((whole & PART) && w.place[d] < 0 ? 1 : 0);
        const int pages = (int)((w.size[d] + ((int64_t)1 << a.shift) - 1) >> a.shift);
        a.new_table[e] = i < held ? c.table[(int64_t)w.from[d] * width + i] : i < pages ? w.list[w.first[d] + i - held] : -1;
    }
    for (int64_t d = t; d < c.n_seq; d += n) a.new_len[d] = bad ? c.len[d] : w.size[d];
    for (int64_t p = t; p < c.n_pages; p += n) a.new_ref[p] = bad ? c.ref[p] : w.count[p];
    copy_pages(c, w.n_copy, w.src, w.dst, page_bytes);
}

int64_t page_bytes(const gaje_hip_kv_pages &c) {
    return (int64_t)c.page * c.n_head_kv * c.head_dim * (c.dtype == GAJE_DTYPE_F32 ? 4 : 2);
}

// ---- compact ----
// The i-th page in use at L or above moves into the i-th free one below L.
__global__ __launch_bounds__(PLAN_THREADS) void kv_compact_plan_kernel(gaje_hip_kv_pages c, int32_t *new_ref,
                                                                       int32_t *n_live, PlanWorkspace w) {
    __shared__ int2 red[PLAN_WAVES];
    const int tid = threadIdx.x;
    int mine = 0;
    for (int64_t p = tid; p < c.n_pages; p += PLAN_THREADS) mine += c.ref[p] > 0;
    int2 total;
    scan2(mine, 0, red, total);
    const int64_t live = total.x;
    int64_t holes = 0, moved = 0;
    for (int64_t p0 = 0; p0 < c.n_pages; p0 += PLAN_THREADS) {
        const int64_t p = p0 + tid;
        const bool used = p < c.n_pages && c.ref[p] > 0;
        const bool hole = p < live && !used, move = p >= live && used;
        const int2 at = scan2(hole, move, red, total);
        if (hole) w.dst[holes + at.x] = (int32_t)p;
        if (move) w.src[moved + at.y] = (int32_t)p;
        if (p < c.n_pages) {
            w.list[p] = (int32_t)p;
            new_ref[p] = p < live && used ? c.ref[p] : 0;
        }
        holes += total.x;
        moved += total.y;
    }
    __syncthreads();
    for (int64_t i = tid; i < moved; i += PLAN_THREADS) {
        const int from = w.src[i], to = w.dst[i];
        w.list[from] = to;
        new_ref[to] = c.ref[from];
    }
    if (tid == 0) n_live[0] = (int32_t)live, w.n_copy[0] = (int32_t)moved;
}

// The renamed entries, and the moves.
__global__ __launch_bounds__(256) void kv_move_kernel(gaje_hip_kv_pages c, int32_t *new_table, PlanWorkspace w, int64_t page_bytes) {
    const int64_t n = c.n_seq * c.max_pages;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int id = c.table[i];
        new_table[i] = id >= 0 && id < c.n_pages ? w.list[id] : -1;
    }
    copy_pages(c, w.n_copy, w.src, w.dst, page_bytes);
}

// ---- append ----
// The sequence of row t, the last s with off[s] <= t (-1: none), by the whole wave: 64
// offsets a step.
__device__ __forceinline__ int seq_of_row(const int32_t *off, int n_seq, int64_t t) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = n_seq + 1;  // the offsets lo .. lo + n - 1 hold the last one <= t
    while (n > 0) {
        const int step = (n + WAVE - 1) / WAVE, i = lane * step;
        const int count = __popcll(__ballot(i < n && off[lo + i] <= t));
        if (count == 0) return -1;
        lo += (count - 1) * step;
        n = min(step, n - (count - 1) * step);
        if (step == 1) break;
    }
    return lo < n_seq ? lo : -1;
}

template <typename S, typename D>
__device__ __forceinline__ void copy8(const S *from, D *to) {
    if constexpr (sizeof(S) == sizeof(D)) {
#pragma unroll
        for (int b = 0; b < (int)sizeof(S) * 8; b += 16) *(vu4 *)((char *)to + b) = *(const vu4 *)((const char *)from + b);
    } else {
        const vf4 a = *(const vf4 *)from, b = *(const vf4 *)(from + 4);
        union { D e[8]; vu4 q; } u;
#pragma unroll
        for (int i = 0; i < 4; ++i) u.e[i] = (D)a[i], u.e[4 + i] = (D)b[i];
        *(vu4 *)to = u.q;
    }
}

// One wave per row and pool, eight elements per lane and turn.  Bound by HBM: 12 prompts' rows
// of 8 x 128, f32 into f16, 158 MB in 25 us.
template <typename S, typename D>
__global__ __launch_bounds__(256) void kv_append_kernel(gaje_hip_kv_pages c, int64_t layer, const S *k, int64_t ldk,
                                                        const S *v, int64_t ldv, const int32_t *seq_off, int64_t T,
                                                        int shift) {
    const int lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), t = item >> 1;
    if (t >= T) return;
    const int64_t s = seq_of_row(seq_off, (int)c.n_seq, t);
    if (s < 0) return;
    const int64_t len = min(max((int64_t)c.len[s], (int64_t)0), c.max_pages << shift);
    const int64_t pos = len - seq_off[s + 1] + t;
    if (pos < 0 || pos >= len) return;
    const int64_t id = c.table[s * c.max_pages + (pos >> shift)];
    if (id < 0 || id >= c.n_pages) return;
    const int64_t width = (int64_t)c.n_head_kv * c.head_dim;
    const int64_t row = ((layer * c.n_pages + id) << shift) + (pos & (((int64_t)1 << shift) - 1));
    const S *from = item & 1 ? v + t * ldv : k + t * ldk;
    D *to = (D *)(item & 1 ? c.v : c.k) + row * width;
    for (int64_t e = lane * 8; e < width; e += WAVE * 8) copy8(from + e, to + e);
}

}  // namespace

int64_t kv_update_workspace(const gaje_hip_kv_pages &c) { return plan_workspace(nullptr, c).bytes; }

int launch_kv_update(const gaje_hip_kv_pages &c, const int32_t *source, const int32_t *add, int32_t *new_table,
                     int32_t *new_len, int32_t *new_ref, int32_t *status, void *workspace, hipStream_t s) {
    const UpdateArgs a{c, source, add, new_table, new_len, new_ref, status, plan_workspace(workspace, c),
                       __builtin_ctz((unsigned)c.page)};
    const int64_t all = c.n_seq * c.max_pages, work = std::max(all, c.n_pages);
    // A workgroup by itself spares two launches, and takes 1.4 us per 1000 entries longer (with
    // the copies): 16 slots of 65 entries 13.9 us against 16.4, 256 slots of 46 entries 30.3
    // against 21.8, of 127 entries 56.4 against 21.4.
    if (work <= 6144) {
        kv_plan_kernel<true><<<1, PLAN_THREADS, 0, s>>>(a);
    } else {
        const unsigned grid = (unsigned)std::min<int64_t>((work + 1023) / 1024, 2048);
        kv_begin_kernel<<<grid, 256, 0, s>>>(a);
        kv_count_kernel<<<grid, 256, 0, s>>>(a);
        kv_plan_kernel<false><<<1, PLAN_THREADS, 0, s>>>(a);
    }
    GAJE_HIP_CHECK(hipGetLastError());
    const int64_t items = std::max(std::min(c.n_seq, c.n_pages) * c.n_layer * 2, (work + 255) / 256);
    kv_write_kernel<<<(unsigned)std::min<int64_t>(items, 1024), 256, 0, s>>>(a, page_bytes(c));
    GAJE_HIP_CHECK(hipGetLastError());
    return GAJE_OK;
}

int launch_kv_compact(const gaje_hip_kv_pages &c, int32_t *new_table, int32_t *new_ref, int32_t *n_live,
                      void *workspace, hipStream_t s) {
    const PlanWorkspace w = plan_workspace(workspace, c);
    kv_compact_plan_kernel<<<1, PLAN_THREADS, 0, s>>>(c, new_ref, n_live, w);
    GAJE_HIP_CHECK(hipGetLastError());
    const int64_t items = std::max(c.n_pages * c.n_layer * 2, (c.n_seq * c.max_pages + 255) / 256);
    kv_move_kernel<<<(unsigned)std::min<int64_t>(items, 4096), 256, 0, s>>>(c, new_table, w, page_bytes(c));
    GAJE_HIP_CHECK(hipGetLastError());
    return GAJE_OK;
}

int launch_kv_append(const gaje_hip_kv_pages &c, int64_t layer, int source_dtype, const void *k, int64_t ldk,
                     const void *v, int64_t ldv, const int32_t *seq_off, int64_t T, hipStream_t s) {
    const unsigned grid = (unsigned)((2 * T + 3) / 4);
    const int shift = __builtin_ctz((unsigned)c.page);
#define GAJE_APPEND(S, D) kv_append_kernel<S, D><<<grid, 256, 0, s>>>(c, layer, (const S *)k, ldk, (const S *)v, ldv, seq_off, T, shift)
    if (source_dtype == c.dtype) {
        if (c.dtype == GAJE_DTYPE_F32) GAJE_APPEND(float, float);
        else GAJE_APPEND(uint16_t, uint16_t);
    } else if (c.dtype == GAJE_DTYPE_F16) {
        GAJE_APPEND(float, _Float16);
    } else {
        GAJE_APPEND(float, __bf16);
    }
#undef GAJE_APPEND
    GAJE_HIP_CHECK(hipGetLastError());
    return GAJE_OK;
}

}  // namespace gaje
