// Bookkeeping and copies of a paged KV cache (gaje_hip_kv_update, _compact, _append).
//
// Update.  Slot d takes slot source[d]'s pages as they were; kept positions
// n = min(len, len + add).  With G positions a page, pages 0 .. n/G - 1 are kept
// whole and shared; page n/G, if n % G > 0, is kept in part, and a slot may go on
// writing it only if no other slot refers to it: it stays with the lowest slot
// that keeps part of it when nobody keeps it whole, all others get a copy.  New
// pages are the lowest free ones, handed out in slot order.  All of it is counts,
// minima and prefix sums of integers, so the order of the atomics does not show.
// One workgroup does that in one launch; a second launch copies pages.
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

// Workspace of a plan: [0] copies, then per page counts, owners and the list of
// free pages (compact: the pages to move and where), per slot the new page of a
// copy and its source.
struct PlanWorkspace {
    int32_t *n_copy, *count, *owner, *list, *src, *dst;
    int64_t bytes;
};
PlanWorkspace plan_workspace(void *base, const gaje_hip_kv_pages &c) {
    PlanWorkspace w{};
    int64_t off = 0;
    auto take = [&](int64_t n) {
        int32_t *p = (int32_t *)((char *)base + off);
        off += (n * 4 + 255) / 256 * 256;
        return p;
    };
    const int64_t copies = std::max(c.n_seq, c.n_pages);
    w.n_copy = take(1);
    w.count = take(c.n_pages);
    w.owner = take(c.n_pages);
    w.list = take(c.n_pages);
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

struct Slot {
    int64_t src;         // the slot it comes from, -1: empty
    int64_t base, size;  // positions before and after
    int64_t whole;       // pages kept whole
    bool part;           // page `whole` is kept in part
    int bad;             // status bits
};

__device__ Slot slot_of(const gaje_hip_kv_pages &c, const int32_t *source, const int32_t *add, int64_t d, int shift) {
    Slot s;
    s.bad = 0;
    s.src = source ? source[d] : d;
    if (s.src < -1 || s.src >= c.n_seq) s.bad = 1, s.src = -1;
    const int64_t most = c.max_pages << shift;
    s.base = s.src < 0 ? 0 : min(max((int64_t)c.len[s.src], (int64_t)0), most);
    s.size = s.base + (add ? add[d] : 0);
    if (s.size < 0 || s.size > most) s.bad |= 2, s.size = 0;
    const int64_t kept = min(s.base, s.size);
    s.whole = kept >> shift;
    s.part = (kept & (((int64_t)1 << shift) - 1)) != 0;
    return s;
}

__global__ __launch_bounds__(PLAN_THREADS) void kv_plan_kernel(gaje_hip_kv_pages c, const int32_t *source,
                                                              const int32_t *add, int32_t *new_table,
                                                              int32_t *new_len, int32_t *new_ref, int32_t *status,
                                                              PlanWorkspace w, int shift) {
    __shared__ int2 red[PLAN_WAVES];
    __shared__ int bad;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t mask = ((int64_t)1 << shift) - 1;
    if (tid == 0) bad = 0;
    for (int64_t p = tid; p < c.n_pages; p += PLAN_THREADS) {
        st_shared(w.count + p, 0);
        st_shared(w.owner + p, INT32_MAX);
    }
    __syncthreads();
    // references to every kept page
    for (int64_t d = wave; d < c.n_seq; d += PLAN_WAVES) {
        const Slot s = slot_of(c, source, add, d, shift);
        int err = s.bad;
        const int32_t *row = c.table + (s.src < 0 ? 0 : s.src) * c.max_pages;
        for (int64_t i = lane; i < s.whole + s.part; i += WAVE) {
            const int id = row[i];
            if (id < 0 || id >= c.n_pages) err |= 8;
            else if (i < s.whole) atomicAdd(w.count + id, 1);
            else atomicMin(w.owner + id, (int)d);
        }
        if (err) atomicOr(&bad, err);
    }
    __syncthreads();
    // slots in order: the new pages each needs and where they start; the copies
    int64_t need = 0, copies = 0;
    if (!bad)
        for (int64_t d0 = 0; d0 < c.n_seq; d0 += PLAN_THREADS) {
            const int64_t d = d0 + tid;
            int n = 0, copy = 0;
            if (d < c.n_seq) {
                const Slot s = slot_of(c, source, add, d, shift);
                bool keep = false;
                if (s.part) {
                    const int id = c.table[s.src * c.max_pages + s.whole];
                    keep = ld_shared(w.count + id) == 0 && ld_shared(w.owner + id) == d;
                }
                copy = s.part && !keep;
                n = (int)(((s.size + mask) >> shift) - s.whole - (s.part && keep));
            }
            int2 total;
            const int2 at = scan2(n, copy, red, total);
            if (d < c.n_seq) {
                // where this slot's new pages start, and its copy's place or -1
                new_len[d] = (int32_t)(need + at.x);
                w.dst[d] = copy ? (int32_t)(copies + at.y) : -1;
            }
            need += total.x;
            copies += total.y;
        }
    // the lowest free pages, as many as are needed
    int64_t found = 0;
    if (!bad)
        for (int64_t p0 = 0; p0 < c.n_pages && found < need; p0 += PLAN_THREADS) {
            const int64_t p = p0 + tid;
            const int free = p < c.n_pages && c.ref[p] <= 0;
            int2 total;
            const int2 at = scan2(free, 0, red, total);
            if (free && found + at.x < need) w.list[found + at.x] = (int32_t)p;
            found += total.x;
        }
    __syncthreads();
    if (tid == 0) {
        if (!bad && found < need) bad = 4;
        status[0] = bad;
        w.n_copy[0] = bad ? 0 : (int32_t)copies;
    }
    __syncthreads();
    if (bad) {
        for (int64_t i = tid; i < c.n_seq * c.max_pages; i += PLAN_THREADS) new_table[i] = c.table[i];
        for (int64_t i = tid; i < c.n_seq; i += PLAN_THREADS) new_len[i] = c.len[i];
        for (int64_t i = tid; i < c.n_pages; i += PLAN_THREADS) new_ref[i] = c.ref[i];
        return;
    }
    for (int64_t i = tid; i < c.n_pages; i += PLAN_THREADS) new_ref[i] = ld_shared(w.count + i);
    __syncthreads();
    for (int64_t d = wave; d < c.n_seq; d += PLAN_WAVES) {
        const Slot s = slot_of(c, source, add, d, shift);
        const int64_t first = new_len[d], place = w.dst[d], pages = (s.size + mask) >> shift;
        const int64_t held = s.whole + (s.part && place < 0);
        const int32_t *row = c.table + (s.src < 0 ? 0 : s.src) * c.max_pages;
        for (int64_t i = lane; i < c.max_pages; i += WAVE) {
            int id = -1;
            if (i < held) id = row[i];
            else if (i < pages) id = w.list[first + i - held];
            new_table[d * c.max_pages + i] = id;
            // pages kept whole have their count; a page of one slot only has 1
            if (id >= 0 && i >= s.whole) new_ref[id] = 1;
            if (place >= 0 && i == s.whole) w.src[place] = row[i], w.owner[place] = id;
        }
    }
    __syncthreads();
    for (int64_t d = tid; d < c.n_seq; d += PLAN_THREADS) new_len[d] = (int32_t)slot_of(c, source, add, d, shift).size;
}

// n_copy pages of every layer, K and V: one (copy, layer, pool) per workgroup and
// turn, 16 bytes per lane.
__global__ __launch_bounds__(256) void kv_copy_kernel(gaje_hip_kv_pages c, const int32_t *n_copy, const int32_t *src,
                                                      const int32_t *dst, int64_t page_bytes) {
    const int64_t per = c.n_layer * 2, n = n_copy[0] * per;
    for (int64_t i = blockIdx.x; i < n; i += gridDim.x) {
        const int64_t copy = i / per, layer = i % per >> 1;
        char *pool = (char *)(i & 1 ? c.v : c.k) + layer * c.n_pages * page_bytes;
        const char *from = pool + src[copy] * page_bytes;
        char *to = pool + dst[copy] * page_bytes;
        for (int64_t b = threadIdx.x * 16; b < page_bytes; b += 256 * 16) *(vu4 *)(to + b) = *(const vu4 *)(from + b);
    }
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

__global__ __launch_bounds__(256) void kv_rename_kernel(gaje_hip_kv_pages c, int32_t *new_table, const int32_t *to) {
    const int64_t n = c.n_seq * c.max_pages;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int id = c.table[i];
        new_table[i] = id >= 0 && id < c.n_pages ? to[id] : -1;
    }
}

// ---- append ----
// The sequence of row t: the last s with seq_off[s] <= t, or -1 outside all.
__device__ __forceinline__ int64_t seq_of(const int32_t *off, int64_t n_seq, int64_t t) {
    int64_t lo = 0, hi = n_seq;  // off[lo] <= t < off[hi] once found
    if (t < off[0] || t >= off[n_seq]) return -1;
    while (hi - lo > 1) {
        const int64_t mid = (lo + hi) >> 1;
        if (off[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
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

// One wave per row and pool, eight elements per lane and turn.
template <typename S, typename D>
__global__ __launch_bounds__(256) void kv_append_kernel(gaje_hip_kv_pages c, int64_t layer, const S *k, int64_t ldk,
                                                        const S *v, int64_t ldv, const int32_t *seq_off, int64_t T,
                                                        int shift) {
    const int lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), t = item >> 1;
    if (t >= T) return;
    const int64_t s = seq_of(seq_off, c.n_seq, t);
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
    const PlanWorkspace w = plan_workspace(workspace, c);
    kv_plan_kernel<<<1, PLAN_THREADS, 0, s>>>(c, source, add, new_table, new_len, new_ref, status, w,
                                              __builtin_ctz((unsigned)c.page));
    GAJE_HIP_CHECK(hipGetLastError());
    const int64_t items = c.n_seq * c.n_layer * 2;
    kv_copy_kernel<<<(unsigned)std::min<int64_t>(items, 2048), 256, 0, s>>>(c, w.n_copy, w.src, w.owner, page_bytes(c));
    GAJE_HIP_CHECK(hipGetLastError());
    return GAJE_OK;
}

int launch_kv_compact(const gaje_hip_kv_pages &c, int32_t *new_table, int32_t *new_ref, int32_t *n_live,
                      void *workspace, hipStream_t s) {
    const PlanWorkspace w = plan_workspace(workspace, c);
    kv_compact_plan_kernel<<<1, PLAN_THREADS, 0, s>>>(c, new_ref, n_live, w);
    GAJE_HIP_CHECK(hipGetLastError());
    kv_rename_kernel<<<(unsigned)std::min<int64_t>((c.n_seq * c.max_pages + 255) / 256, 1024), 256, 0, s>>>(c, new_table,
                                                                                                            w.list);
    GAJE_HIP_CHECK(hipGetLastError());
    const int64_t items = c.n_pages * c.n_layer * 2;
    kv_copy_kernel<<<(unsigned)std::min<int64_t>(items, 4096), 256, 0, s>>>(c, w.n_copy, w.src, w.dst, page_bytes(c));
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
