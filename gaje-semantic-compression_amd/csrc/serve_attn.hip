// Softmax attention of many sequences: causal over packed prompts, over the pages of
// a KV cache, and over a prefix that all sequences share.
//
// Row t of sequence s with n rows sees keys 0 .. len - n + (t - first row) of its
// len keys.  Over those, with c = scale * log2(e):
//   m = max_j s_j,  o = sum_j 2^(c (s_j - m)) v_j / sum_j 2^(c (s_j - m)),
// s_j = q . k_j, all in f32, in one pass over the keys: m is a running base, and what
// was summed is rescaled when it moves.
//
// Three forms over the same rows and keys: attend_tile (16-bit types, 128 rows a
// workgroup), attend_tile64 (64 rows; short prompts, and f32 on the bf16 matrix
// instructions) and attend_few (up to 16 rows, the keys split over the waves).  The keys of a
// tile are cut into parts where there are few tiles; attn_join_kernel joins what they leave.
// Measured, as launched in a graph:
//   attend_tile    one prompt of 8190, 32/8 heads of 128, f16: 620 us, 890 TFLOP/s
//   attend_tile64  4 f32 prompts of 970 to 1930, 12/2 heads of 128: 258 us, 143 TFLOP/s (f32
//                  products of a library: 154)
//   attend_few     512 sequences of 1000 keys, 12/2 heads of 128, bf16: 97 us, 5.4 TB/s
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "common.h"
#include "device_util.h"
#include "serve.h"

namespace gaje {
namespace {

constexpr float LOG2E = 1.44269504088896340736f;
// a factor of 2^8 between weights, in scores (finite for every scale)
__device__ __forceinline__ float slack_of(float c) { return fminf(8.0f / c, 1e30f); }

typedef float vf16 __attribute__((ext_vector_type(16)));
typedef _Float16 vh8 __attribute__((ext_vector_type(8)));
typedef __bf16 vb8 __attribute__((ext_vector_type(8)));

// What a row outside the sequence, a padded dimension and a page outside the pool
// read: loads are redirected here instead of being skipped.
__device__ const vu4 zero_piece[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
typedef const __attribute__((address_space(1))) vu4 *gvu4;
__device__ __forceinline__ gvu4 piece(const void *p, bool ok) { return ok ? (gvu4)(uintptr_t)p : (gvu4)(uintptr_t)zero_piece; }

// 16 x 16 and 32 x 32 products of 16-bit operands, eight of a lane's at a time.
template <typename T>
__device__ __forceinline__ vf4 mfma16(vu4 a, vu4 b, vf4 c) {
    if constexpr (std::is_same<T, _Float16>::value)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(vh8, a), __builtin_bit_cast(vh8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(vb8, a), __builtin_bit_cast(vb8, b), c, 0, 0, 0);
}
template <typename T>
__device__ __forceinline__ vf16 mfma32(vu4 a, vu4 b, vf16 c) {
    if constexpr (std::is_same<T, _Float16>::value)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(vh8, a), __builtin_bit_cast(vh8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(vb8, a), __builtin_bit_cast(vb8, b), c, 0, 0, 0);
}

// Prefix sums (and running maxima of values >= 0) over the wave, by cross-lane moves
// within the VALU.
template <int CTRL, int ROWS>
__device__ __forceinline__ int lane_move(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false); }
__device__ __forceinline__ int wave_scan(int v) {
    v += lane_move<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8: within 16 lanes
    v += lane_move<0x112, 0xf>(v);
    v += lane_move<0x114, 0xf>(v);
    v += lane_move<0x118, 0xf>(v);
    v += lane_move<0x142, 0xa>(v);  // row_bcast 15 into rows 1 and 3, 31 into rows 2 and 3
    v += lane_move<0x143, 0xc>(v);
    return v;
}
__device__ __forceinline__ int wave_most(int v) {
    v = max(v, lane_move<0x111, 0xf>(v));
    v = max(v, lane_move<0x112, 0xf>(v));
    v = max(v, lane_move<0x114, 0xf>(v));
    v = max(v, lane_move<0x118, 0xf>(v));
    v = max(v, lane_move<0x142, 0xa>(v));
    v = max(v, lane_move<0x143, 0xc>(v));
    return __builtin_amdgcn_readlane(v, WAVE - 1);
}

// The rows of one sequence and its keys.
struct Seq {
    int row0, rows;  // its rows of q and out
    int len;         // its keys
    int id;
};

__device__ __forceinline__ int cached(const ServeAttnParams &p, int len) { return min(max(len, 0), (int)(p.max_pages << p.page_shift)); }

__device__ __forceinline__ Seq seq_at(const ServeAttnParams &p, int s) {
    Seq q{s, 1, 0, s};
    const int len = p.table ? p.len[s] : 0;  // (all loads before the first use)
    if (p.seq_off) {
        const int a = p.seq_off[s], b = p.seq_off[s + 1];
        q.row0 = min(max(a, 0), (int)p.T);
        q.rows = max(min(b, (int)p.T) - q.row0, 0);
    }
    q.len = p.table ? cached(p, len) : q.rows;
    return q;
}

// The row of k and v that holds a sequence's position, -1 where its page is outside
// the pool.
__device__ __forceinline__ int64_t slot_at(const ServeAttnParams &p, const Seq &q, int64_t pos) {
    if (!p.table) return (int64_t)q.row0 + pos;
    const int32_t *row = pos < p.prefix_len && p.prefix_table ? p.prefix_table : p.table + (int64_t)q.id * p.max_pages;
    const int64_t id = row[pos >> p.page_shift];
    if (id < 0 || id >= p.n_pages) return -1;
    return (id << p.page_shift) + (pos & (((int64_t)1 << p.page_shift) - 1));
}

// One (row, head) by one wave, key by key: 64 scores at a time, one per lane, then
// the values of the keys that are seen and of no other, so that a NaN or an infinity
// in a key or value reaches only the rows that see it.  Lane l holds dimensions
// l, l + 64, ...
template <typename T>
__device__ void attend_row(const ServeAttnParams &p, const Seq &q, int64_t t, int h, int64_t k0, int64_t k1, float &m_out,
                           float &l_out, float (&o)[4]) {
    const int lane = threadIdx.x & 63, hd = p.head_dim, g = h / (p.n_head / p.n_head_kv);
    const T *Q = (const T *)p.q + t * p.ldq + (int64_t)h * hd;
    const T *K = (const T *)p.k + (int64_t)g * hd, *V = (const T *)p.v + (int64_t)g * hd;
    const float c = p.scale * LOG2E;
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = 0.0f;
    for (int64_t j0 = k0; j0 < k1; j0 += WAVE) {
        const int n = (int)min(k1 - j0, (int64_t)WAVE);
        float s = -INFINITY;
        int64_t slot = -1;
        if (lane < n) {
            slot = slot_at(p, q, j0 + lane);
            s = 0.0f;
            if (slot >= 0) {
                const T *kr = K + slot * p.ldk;
                for (int d = 0; d < hd; ++d) s = fmaf((float)Q[d], (float)kr[d], s);
            }
        }
        const float mt = fmaxf(m, wave_max(s)), base = mt == -INFINITY ? 0.0f : mt * c;
        const float e = lane < n ? __builtin_amdgcn_exp2f(fmaf(s, c, -base)) : 0.0f;
        const float shrink = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(fmaf(m, c, -base));
        l = fmaf(l, shrink, wave_sum(e));
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] *= shrink;
        for (int j = 0; j < n; ++j) {
            const float w = __shfl(e, j, WAVE);
            const int64_t sj = __shfl(slot, j, WAVE);
            if (sj < 0) continue;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (lane + 64 * i < hd) o[i] = fmaf(w, (float)V[sj * p.ldv + lane + 64 * i], o[i]);
        }
        m = mt;
    }
    m_out = m;
    l_out = l;
}

// ---- tiles ----
// A workgroup of four waves takes a tile of up to 128 query rows of one K/V head: the
// rows of a sequence are its (token, query head of the group) pairs, so that the heads
// that share K and V read them together.  Wave w holds rows 32 w .. 32 w + 31, one per
// lane pair (lane, lane + 32), and walks the keys in tiles of BN:
//   S^T = K Q^T   A = 32 keys, B = 32 queries: lane l has query l % 32 and, per 32 keys,
//                 keys 8 (i / 4) + 4 (l / 32) + i % 4 in registers i < 16
//   O^T = V^T P^T the same registers, rounded to the type, are the B operand as they
//                 stand if the keys of V^T's operand come in that order
// so a row's maximum, sum and rescaling stay within two lanes, and the weights never
// leave their registers.  K and V are staged in LDS in operand order (V transposed on
// the way, 8 keys x 8 dimensions per thread with v_perm), so that every operand is one
// conflict-free 16-byte read; two buffers, one barrier per tile, the next tile's global
// loads in flight during a tile's products.
// Bound by the matrix and vector units in turn (46% and 48% of the cycles at 8190 rows, 32
// heads of 128: one exponential per 2 * 128 products), which two waves of a SIMD seldom overlap.
template <typename T, int HD>
struct TileCfg {
    static_assert(sizeof(T) == 2, "f32 has tiles of its own");
    static constexpr int BN = 8192 / HD;               // keys per tile
    static constexpr int PCS = HD / 8;                 // 16-byte pieces per row
    static constexpr int NT = HD / 32;                 // 32-dimension blocks of O^T
    static constexpr int KROW = 32 * 16 + 16;          // bytes of 32 keys' pieces in LDS, 4 banks on
    static constexpr int KT = BN / 32 * PCS * KROW, VT = BN * HD * 2;
    static constexpr int LDS = 2 * (KT + VT);
    static constexpr int STEPS = HD / 16;              // of the scores' operands
};

struct TilePlan {
    int64_t items;   // bound on the (tile, part) pairs of a K/V head
    int32_t bm;      // rows of a tile
    int32_t splits;  // parts that the keys of a tile have at most
    int32_t part0;   // first partial result, -1: every tile has one part, the whole result
    int32_t alone;   // no other plan's parts join these: a single part is the whole result
    int32_t least;   // keys a part has at least
    int32_t key0;    // the first key (few rows only)
    int32_t blocks;  // log2 of the (tile, part, K/V head) triples wanted
    int32_t size;    // keys per part, 0: from the sequences' lengths, on the device
};
constexpr int PART_UNIT = 128;  // parts are whole multiples of it

// Keys per part where `total` units of keys over all tiles and K/V heads are to make about
// 2^blocks parts and the longest tile `splits` (a power of two) at most.
__host__ __device__ __forceinline__ int part_size(int64_t total, int longest, int splits, int least, int blocks) {
    const int64_t even = ((total >> blocks) + 1) * PART_UNIT;
    const int floor = longest / splits + 1;
    const int size = even > (1 << 30) ? 1 << 30 : (int)even;
    return ((size < floor ? floor : size) < least ? least : (size < floor ? (floor + PART_UNIT - 1) / PART_UNIT * PART_UNIT : size));
}

// One past the last key that a tile's rows see.
template <bool PREFIX>
__device__ __forceinline__ int tile_end(const ServeAttnParams &p, const Seq &q, int tile, int bm, int group) {
    if constexpr (PREFIX) return (int)p.prefix_len;
    const uint32_t last = (uint32_t)min((int64_t)q.rows * group, (int64_t)(tile + 1) * bm) - 1;
    return max(q.len - q.rows + (int)(last / (uint32_t)group) + 1, 0);
}

// What a workgroup does: part `part` of a tile's keys, `size` keys each.
struct Item {
    Seq q;
    int g, tile, part, size;  // g: the K/V head
};

// The item of a workgroup.  A sequence has ceil(rows group / bm) tiles, the ones over the
// longest contexts first, and as many parts as its longest tile needs (a workgroup past a
// shorter tile's end has nothing to do).  Every wave looks at all sequences, 64 at a time:
// once for the part size, if the keys are cut at all, once for its item.
// LONG_FIRST: of up to 64 sequences together, the items over the longest contexts first (an
// item takes up to 70 us, and one begun last ends last: 24 prompts of up to 2000 tokens, 12 heads
// of 128, bf16, 153 -> 150 us).
template <bool PREFIX, bool LONG_FIRST>
__device__ __forceinline__ bool find_item(const ServeAttnParams &p, const TilePlan &plan, int block, int group, Item &it) {
    if constexpr (PREFIX) {
        const int keys = plan.splits * p.n_head_kv, at = block % keys;
        it.q = Seq{0, 0, 0, 0};
        it.g = at % p.n_head_kv;
        it.part = at / p.n_head_kv;
        it.tile = block / keys;
        it.size = plan.size;
        return true;
    }
    const int b = block / p.n_head_kv;
    it.g = block % p.n_head_kv;
    const int lane = threadIdx.x & 63, from = plan.key0 & ~31, n_seq = (int)p.n_seq, shift = __builtin_ctz(plan.bm);
    Seq q;
    int tiles, cut;  // of sequence s0 + lane; cut: keys to cut into parts
    auto look = [&](int s0) {
        q = seq_at(p, min(s0 + lane, n_seq - 1));
        if (s0 + lane >= n_seq) q.rows = 0;
        tiles = (int)(((int64_t)q.rows * group + plan.bm - 1) >> shift);
        cut = max(q.len - from, 0);
    };
    int size = plan.size;
    if (size == 0) {
        int64_t total = 0;
        int longest = 0;
        for (int s0 = 0; s0 < n_seq; s0 += WAVE) {
            look(s0);
            // (a causal prompt's tiles see half of its own rows on average; units of 128 keys)
            const int units = tiles ? max(cut - q.rows / 2, cut / 2) / PART_UNIT + 1 : 0;
            total += __builtin_amdgcn_readlane(wave_scan(tiles * units), WAVE - 1);
            longest = max(longest, wave_most(tiles ? cut : 0));
        }
        size = part_size(total * p.n_head_kv, longest, plan.splits, plan.least, plan.blocks);
    }
    int base = 0, begin = 0;
    if (plan.splits == 1 && n_seq > 4 * WAVE) {
        // Of many sequences the eight that hold the item are found first, eight per lane (4096 of 200
        // cached keys, one token each, 12/2 heads of 128, bf16: 561 -> 400 us).
        constexpr int RUN = 8;
        for (; begin < n_seq; begin += WAVE * RUN) {
            const int left = n_seq - begin, first = min(lane * RUN, left);
            int at[RUN + 1], sum = 0;
#pragma unroll
            for (int i = 0; i <= RUN; ++i) {
                const int s = min(first + i, left);
                at[i] = p.seq_off ? min(max(p.seq_off[begin + s], 0), (int)p.T) : s;
            }
#pragma unroll
            for (int i = 0; i < RUN; ++i) sum += (int)(((int64_t)max(at[i + 1] - at[i], 0) * group + plan.bm - 1) >> shift);
            const int incl = wave_scan(sum);
            const uint64_t past = __ballot(base + incl > b);
            if (past) {
                const int l = __builtin_ctzll(past);
                base += __builtin_amdgcn_readlane(incl - sum, l);
                begin += l * RUN;
                break;
            }
            base += __builtin_amdgcn_readlane(incl, WAVE - 1);
        }
    }
    for (int s0 = begin; s0 < n_seq; s0 += WAVE) {
        if (plan.size || n_seq > WAVE) look(s0);
        const int parts = plan.splits == 1 ? 1 : (int)((uint32_t)max(cut - 1, 0) / (uint32_t)size) + 1;
        const int cnt = tiles * parts, incl = wave_scan(cnt), total = __builtin_amdgcn_readlane(incl, WAVE - 1);
        if (b < base + total) {
            int l, left;  // the sequence's lane, and its items after this one
            if (LONG_FIRST && n_seq <= WAVE) {
                // the largest depth with more than b items at it or deeper
                int after = 0, most = wave_most(cnt);
                left = 0;
                while (most - left > 1) {
                    const int mid = (left + most) >> 1;
                    const int deeper = __builtin_amdgcn_readlane(wave_scan(max(cnt - mid, 0)), WAVE - 1);
                    if (deeper > b) left = mid;
                    else most = mid, after = deeper;
                }
                const uint64_t there = __ballot(cnt > left);
                const int rank = __popcll(there & (((uint64_t)1 << lane) - 1));
                l = __builtin_ctzll(__ballot(cnt > left && rank == b - after));
            } else {
                l = __builtin_ctzll(__ballot(base + incl > b));
                left = base + __builtin_amdgcn_readlane(incl, l) - 1 - b;
            }
            const int n = __builtin_amdgcn_readlane(parts, l);
            it.q.row0 = __builtin_amdgcn_readlane(q.row0, l);
            it.q.rows = __builtin_amdgcn_readlane(q.rows, l);
            it.q.len = __builtin_amdgcn_readlane(q.len, l);
            it.q.id = s0 + l;
            it.tile = (int)((uint32_t)left / (uint32_t)n);
            it.part = n - 1 - (left - it.tile * n);
            it.size = size;
            return true;
        }
        base += total;
    }
    return false;
}

// Query row r of a tile's sequence (or, over a shared prefix, of all sequences): its
// row of q and out, its head, the last key it sees (-1: none).
struct Row {
    int64_t t;
    int lim, head;
    bool valid;
};
template <bool PREFIX>
__device__ __forceinline__ Row row_at(const ServeAttnParams &p, const Seq &q, int r, int group, int g) {
    Row w;
    const int tok = (int)((uint32_t)r / (uint32_t)group);
    w.head = g * group + (r - tok * group);
    if constexpr (PREFIX) {
        w.valid = tok < p.n_seq;
        w.t = w.valid ? tok : 0;
        w.lim = min(cached(p, p.len[w.t]), (int)p.prefix_len) - 1;
    } else {
        w.valid = tok < q.rows;
        w.t = q.row0 + (w.valid ? tok : 0);
        w.lim = min(q.len - q.rows + tok, q.len - 1);
    }
    if (!w.valid) w.lim = -1;
    return w;
}

// What the join needs to know of a row, from the first part of its own keys: how many parts
// those have; 0: the result is whole; negative: it sees no key.
__device__ __forceinline__ void tell_parts(const ServeAttnParams &p, const TilePlan &plan, const Item &it, const Row &row, int keys, bool whole) {
    if (plan.part0 < 0 || it.part > 0 || !row.valid) return;
    const int n = whole ? 0 : max((keys - 1) / it.size + 1, 1);
    p.parts[row.t * p.n_head + row.head] = row.lim >= 0 ? n : -n;
}

template <typename T>
__device__ __forceinline__ void store_row(const ServeAttnParams &p, int64_t t, int head, int part, bool whole, bool seen, float m,
                                          float l, const float (&o)[4]) {
    const int lane = threadIdx.x & 63, hd = p.head_dim;
    if (whole) {
        T *out = (T *)p.out + t * p.ldo + (int64_t)head * hd;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (lane + 64 * i < hd) out[lane + 64 * i] = (T)(seen ? o[i] / l : 0.0f);
    } else {
        const int64_t at = ((int64_t)part * p.T + t) * p.n_head + head;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (lane + 64 * i < hd) p.part_o[at * hd + lane + 64 * i] = o[i];
        if (lane == 0) p.part_ml[at] = make_float2(m, l);
    }
}

template <typename T, int HD, bool PREFIX>
__device__ __forceinline__ void attend_tile(const ServeAttnParams &p, const TilePlan &plan, int block, char *lds) {
    using C = TileCfg<T, HD>;
    constexpr int BM = 128, BN = C::BN, NB = BN / 32;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int half = lane >> 5, l32 = lane & 31;
    const int group = p.n_head / p.n_head_kv, hd = p.head_dim;
    Item it;
    if (!find_item<PREFIX, true>(p, plan, block, group, it)) return;
    const Seq q = it.q;
    const int g = it.g, tile = it.tile;
    const int kend = tile_end<PREFIX>(p, q, tile, BM, group);
    const bool whole = plan.part0 < 0 || (plan.alone && it.size >= kend);
    const int part = plan.part0 + it.part, kb0 = min(it.part * it.size, kend), kb1 = min(kb0 + it.size, kend);
    if (it.part > 0 && kb0 >= kb1) return;
    // This thread's unit: 8 rows x one piece, of K for the first two waves, of V for the others;
    // rows set * 8 + i, or V's in the order of the weights' registers, in two groups of four.
    const bool is_v = wave >= 2;
    const int unit = tid & 127, pc = unit % C::PCS, set = unit / C::PCS;
    int rows_at[2];
#pragma unroll
    for (int a = 0; a < 2; ++a) rows_at[a] = is_v ? (set >> 1) * 16 + (set & 1) * 4 + 8 * a : set * 8 + 4 * a;
    // (a padded dimension's thread reads zeros with a step of 0)
    const bool in = pc * 8 < hd;
    const char *const base = in ? (const char *)((const T *)(is_v ? p.v : p.k) + (int64_t)g * hd) + pc * 16 : (const char *)zero_piece;
    const uint32_t ld = in ? (uint32_t)(is_v ? p.ldv : p.ldk) * sizeof(T) : 0;
    vu4 rg[8];
    int ids[2];
    const int32_t *const pages = PREFIX ? p.prefix_table : p.table + (int64_t)q.id * p.max_pages;
    const int page_mask = (1 << p.page_shift) - 1;
    auto load_ids = [&](int k0) {
        if (!p.table) return;
#pragma unroll
        for (int a = 0; a < 2; ++a) ids[a] = pages[min(k0 + rows_at[a], kb1 - 1) >> p.page_shift];
    };
    auto load_tile = [&](int k0) {
        const char *at[2];
        bool held[2] = {true, true};
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            if (p.table) {
                held[a] = (uint32_t)ids[a] < (uint32_t)p.n_pages;
                at[a] = base + (uint32_t)((k0 + rows_at[a]) & page_mask) * ld + (uint64_t)(uint32_t)ids[a] * (ld << p.page_shift);
            } else {
                at[a] = base + (int64_t)(q.row0 + k0) * ld + (uint32_t)rows_at[a] * ld;
            }
        }
        if (k0 + BN <= kb1 && __all(held[0] & held[1])) {
#pragma unroll
            for (int i = 0; i < 8; ++i) rg[i] = *(gvu4)(uintptr_t)(at[i >> 2] + (i & 3) * ld);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                rg[i] = *piece(at[i >> 2] + (i & 3) * ld, (k0 + rows_at[i >> 2] + (i & 3) < kb1) & held[i >> 2]);
        }
    };
    char *const Kw = lds + ((set >> 2) * C::PCS + pc) * C::KROW + (set & 3) * 128;
    char *const Vw = lds + 2 * C::KT + (set >> 1) * C::NT * 1024 + (set & 1) * 512 + pc * 16;
    auto store_tile = [&](int buf) {
        if (!is_v) {
#pragma unroll
            for (int i = 0; i < 8; ++i) *(vu4 *)(Kw + buf * C::KT + i * 16) = rg[i];
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                vu4 w;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    w[k] = __builtin_amdgcn_perm(rg[2 * k + 1][e >> 1], rg[2 * k][e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
                *(vu4 *)(Vw + buf * C::VT + (e % C::NT) * 1024 + (e / C::NT) * C::PCS * 16) = w;
            }
        }
    };

    if (kb0 < kb1) {
        load_ids(kb0);
        load_tile(kb0);
        load_ids(kb0 + BN);
    }
    const Row row = row_at<PREFIX>(p, q, tile * BM + wave * 32 + l32, group, g);
    if (!PREFIX && half == 0) tell_parts(p, plan, it, row, kend, whole);
    // this wave's rows: the largest and the smallest last key
    int lim_hi = row.lim, lim_lo = row.valid ? row.lim : INT32_MAX;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        lim_hi = max(lim_hi, __shfl_xor(lim_hi, o, WAVE));
        lim_lo = min(lim_lo, __shfl_xor(lim_lo, o, WAVE));
    }
    lim_hi = __builtin_amdgcn_readfirstlane(lim_hi), lim_lo = __builtin_amdgcn_readfirstlane(lim_lo);

    // queries: B operand, piece 2 j + half of the row
    vu4 qf[C::STEPS];
    {
        const T *Q = (const T *)p.q + row.t * p.ldq + (int64_t)row.head * hd;
#pragma unroll
        for (int j = 0; j < C::STEPS; ++j) {
            const int e = (2 * j + half) * 8;
            qf[j] = *piece(Q + e, row.valid && e < hd);
        }
    }

    const float c = p.scale * LOG2E;
    // The weights' base m follows the maximum only where that is past it by a factor of
    // 2^8: they stay below 2^8, and O is seldom rescaled.
    const float slack = slack_of(c);
    float m = -INFINITY, l = 0.0f;
    vf16 o[C::NT];
#pragma unroll
    for (int t = 0; t < C::NT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;

    if (kb0 < kb1) store_tile(0);
    // The queries are waited for here: in the loop that wait, repeated, would be one for the
    // next tile's rows.
#pragma unroll
    for (int j = 0; j < C::STEPS; ++j) asm volatile("" : "+v"(qf[j]));
    __syncthreads();
    const char *const Kr = lds + half * C::KROW + l32 * 16;
    const char *const Vr = lds + 2 * C::KT + lane * 16;
    int buf = 0;
    for (int k0 = kb0; k0 < kb1; k0 += BN, buf ^= 1) {
        const bool more = k0 + BN < kb1;
        if (more) {
            load_tile(k0 + BN);
            load_ids(k0 + 2 * BN);
        }
        if (k0 <= lim_hi) {
            const char *Kl = Kr + buf * C::KT, *Vl = Vr + buf * C::VT;
            vf16 s[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[b][i] = 0.0f;
            // (blocks in turn: no product waits for the one before it)
#pragma unroll
            for (int j = 0; j < C::STEPS; ++j)
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const vu4 kf = *(const vu4 *)(Kl + (b * C::PCS + 2 * j) * C::KROW);
                    s[b] = mfma32<T>(kf, qf[j], s[b]);
                }
            if (k0 + BN - 1 > lim_lo) {
                int lim = row.lim - k0 - 4 * half;
                asm volatile("" : "+v"(lim));  // (keeps this a branch: most tiles are seen whole)
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (b * 32 + 8 * (i >> 2) + (i & 3) > lim) s[b][i] = -INFINITY;
            }
            float mt = s[0][0];
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) mt = fmaxf(mt, s[b][i]);
            mt = fmaxf(mt, __shfl_xor(mt, 32, WAVE));
            if (__any(mt > m + slack)) {
                const float to = fmaxf(mt, m);
                const float shrink = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - to) * c);
                l *= shrink;
#pragma unroll
                for (int t = 0; t < C::NT; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[t][i] *= shrink;
                m = to;
            }
            const float base = m == -INFINITY ? 0.0f : m * c;
            float sum = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    s[b][i] = __builtin_amdgcn_exp2f(fmaf(s[b][i], c, -base));
                    sum += s[b][i];
                }
            l += sum;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
#pragma unroll
                for (int st = 0; st < 2; ++st) {
                    // (rounded to the type, to nearest even: as far off as the result's own rounding)
                    union { T e[8]; vu4 u; } w;
#pragma unroll
                    for (int i = 0; i < 8; ++i) w.e[i] = (T)s[b][8 * st + i];
#pragma unroll
                    for (int t = 0; t < C::NT; ++t)
                        o[t] = mfma32<T>(*(const vu4 *)(Vl + ((b * 2 + st) * C::NT + t) * 1024), w.u, o[t]);
                }
            }
        }
        if (more) store_tile(buf ^ 1);
        __syncthreads();
    }
    l += __shfl_xor(l, 32, WAVE);

    // A row with a result that is no number: keys it does not see may be to blame (0 times
    // NaN), so it is computed again key by key.
    float odd = l * 0.0f;
#pragma unroll
    for (int t = 0; t < C::NT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) odd = fmaf(o[t][i], 0.0f, odd);
    odd += __shfl_xor(odd, 32, WAVE);
    const bool again = row.valid && row.lim >= kb0 && odd != 0.0f;
    if (odd != 0.0f && !again) {  // (the row sees none of these keys)
#pragma unroll
        for (int t = 0; t < C::NT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;
    }
    uint32_t todo = (uint32_t)__ballot(again);

    // Registers x, x + LANE_PCS, .. hold eight neighbouring dimensions, piece p of the row.  The
    // wave's rows go through LDS (the loop is done with it), so that its stores write whole rows:
    // 64 prompts of 21 tokens, 48 heads of 128, 19.3 -> 12.6 us, 24 prompts of up to 2000, 12 heads,
    // 147 -> 132, partial results over a prefix of 16000 28.2 -> 26.0.
    constexpr int SPAN = C::NT >= 8 ? 1 : 8 / C::NT, LANE_PCS = 16 / SPAN, PER = 8 / SPAN;  // PER dimensions from each of SPAN registers
    const float inv = !whole ? 1.0f : row.lim >= 0 ? 1.0f / l : 0.0f;
    const int64_t at = ((int64_t)part * p.T + row.t) * p.n_head + row.head;
    const uint64_t to = whole ? (uint64_t)(uintptr_t)((T *)p.out + row.t * p.ldo + (int64_t)row.head * hd) : (uint64_t)(uintptr_t)(p.part_o + at * hd);
    const uint32_t fine = (uint32_t)__ballot(row.valid && !again);
    char *const rows_lds = lds + wave * 32 * (HD == 256 ? 512 : HD * 4);
    // WORDS: 16-byte pieces of 8 dimensions (1 of the type, 2 of f32); x0, n: the lane's pieces
    auto put = [&](auto words, int x0, auto n_of) {
        constexpr int WORDS = decltype(words)::value, N = decltype(n_of)::value, ROW = N * 2 * WORDS;  // 16-byte pieces of a row here
#pragma unroll
        for (int x = 0; x < N; ++x) {
            float e[8];
#pragma unroll
            for (int z = 0; z < SPAN; ++z)
#pragma unroll
                for (int k = 0; k < PER; ++k) e[z * PER + k] = o[k][x0 + x + z * LANE_PCS] * inv;
            const int pc0 = 8 * (x >> 2) + 4 * half + (x & 3);
            vu4 v[WORDS];
            if constexpr (WORDS == 2) {
                __builtin_memcpy(v, e, 32);
            } else {
                T y[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) y[k] = (T)e[k];
                __builtin_memcpy(v, y, 16);
            }
#pragma unroll
            for (int h = 0; h < WORDS; ++h) *(vu4 *)(rows_lds + (l32 * ROW + ((pc0 * WORDS + h) ^ (l32 & (ROW - 1) & 15))) * 16) = v[h];
        }
#pragma unroll
        for (int x = 0; x < ROW / 2; ++x) {  // 64 / ROW rows of a store
            const int r = x * (64 / ROW) + lane / ROW, w = lane % ROW, d = (x0 * 2 + w / WORDS) * 8;
            const uint32_t lo = __shfl((uint32_t)to, r, WAVE), hi = __shfl((uint32_t)(to >> 32), r, WAVE);
            const vu4 v = *(const vu4 *)(rows_lds + (r * ROW + (w ^ (r & (ROW - 1) & 15))) * 16);
            if ((fine >> r & 1) && d < hd) *(vu4 *)((char *)(uintptr_t)((uint64_t)hi << 32 | lo) + x0 * 2 * WORDS * 16 + w * 16) = v;
        }
    };
    using std::integral_constant;
    if (whole) {
        put(integral_constant<int, 1>{}, 0, integral_constant<int, LANE_PCS>{});
    } else {
        constexpr int N = HD == 256 ? LANE_PCS / 2 : LANE_PCS;
#pragma unroll
        for (int x0 = 0; x0 < LANE_PCS; x0 += N) put(integral_constant<int, 2>{}, x0, integral_constant<int, N>{});
        if (row.valid && !again && half == 0) p.part_ml[at] = make_float2(m, l);
    }
    while (todo) {
        const int n = __builtin_ctz(todo);
        todo &= todo - 1;
        const Row w = row_at<PREFIX>(p, q, tile * BM + wave * 32 + n, group, g);
        const Seq qs = PREFIX ? seq_at(p, (int)w.t) : q;
        float mr, lr, orow[4];
        attend_row<T>(p, qs, w.t, w.head, kb0, min(kb1, w.lim + 1), mr, lr, orow);
        store_row<T>(p, w.t, w.head, part, whole, true, mr, lr, orow);
    }
}

// ---- tiles of 64 rows ----
// A workgroup takes 64 rows of one K/V head, 16 a wave, and the keys 32 at a time:
// S^T = K Q^T and O^T = V^T P^T in 16 x 16 blocks, lanes as in the few-row form.  K and V are
// staged in operand order, V transposed; one buffer, so that several workgroups of a CU fill
// each other's waits.
// 16-bit types: where tiles of 128 rows are too few to fill the chip.
// f32: on the bf16 matrix instructions.  x = x0 + x1 + x2, each the next 8 bits of the
// mantissa (cut, so that the three parts are exactly x), and x y summed from x0 y0, x0 y1,
// x1 y0, x1 y1, x0 y2, x2 y0: what is left out is below 2^-22 of |x y|, about f32's own
// rounding over a few products (measured against 64 bits: 4.2e-7 where f32 products give
// 5.4e-7).  Six products at 16 times the rate of the f32 matrix instructions; an infinity's
// parts are no numbers, and its rows are computed again.  K and V are split on the way into
// LDS, 48 KB for 128 dimensions.
template <typename T, int HD>
struct Tile64Cfg {
    static constexpr bool F32 = sizeof(T) == 4;
    using Op = std::conditional_t<F32, __bf16, T>;     // type of the products
    static constexpr int PL = F32 ? 3 : 1, PRODUCTS = F32 ? 6 : 1;  // planes of an operand, products of two
    static constexpr int BM = 64, BN = 32, PCS = HD / 8, STEPS = HD / 32, VT = HD / 16;
    static constexpr int VD = HD / 64;                 // dimensions of V per thread
    static constexpr int VW = F32 ? VD : (VD + 1) / 2; // dwords of them
    static constexpr int KU = BN * PCS / 256;          // rows x 8 dimensions of K per thread
    static constexpr int KL = F32 ? 2 : 1;             // loads of those
    static constexpr int KCH = 16 * 16 + 16;           // bytes of 16 keys' pieces, 4 banks on
    static constexpr int KP = 2 * PCS * KCH, VP = VT * 1024;  // bytes of a plane
    static constexpr int LDS = PL * (KP + VP);
};

// The three parts of a and b, packed: a in the low halves.
__device__ __forceinline__ void split3(float a, float b, uint32_t (&w)[3]) {
    float x = a, y = b;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const uint32_t u = __float_as_uint(x), v = __float_as_uint(y);
        w[i] = __builtin_amdgcn_perm(v, u, 0x07060302u);
        if (i < 2) x -= __uint_as_float(u & 0xffff0000u), y -= __uint_as_float(v & 0xffff0000u);
    }
}
// the products, the smallest first
constexpr int SPLIT_A[6] = {2, 1, 0, 1, 0, 0}, SPLIT_B[6] = {0, 1, 2, 0, 1, 0};
template <typename T, int HD, bool PREFIX>
__device__ __forceinline__ void attend_tile64(const ServeAttnParams &p, const TilePlan &plan, int block, char *lds) {
    using C = Tile64Cfg<T, HD>;
    constexpr int BM = C::BM, BN = C::BN;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, g4 = lane >> 4;
    const int group = p.n_head / p.n_head_kv, hd = p.head_dim;
    Item it;
    if (!find_item<PREFIX, true>(p, plan, block, group, it)) return;
    const Seq q = it.q;
    const int g = it.g, tile = it.tile;
    const int kend = tile_end<PREFIX>(p, q, tile, BM, group);
    const bool whole = plan.part0 < 0 || (plan.alone && it.size >= kend);
    const int part = plan.part0 + it.part, kb0 = min(it.part * it.size, kend), kb1 = min(kb0 + it.size, kend);
    if (it.part > 0 && kb0 >= kb1) return;
    // K: rows tid / PCS (and 256 / PCS on), dimensions 8 (tid % PCS); V: dimensions VD (tid % 64) of
    // the wave's eight keys 4 w + 0..3, 16 + 4 w + 0..3
    const int kpc = tid % C::PCS, krow = tid / C::PCS, vd = lane * C::VD;
    // (a padded dimension's thread reads zeros with a step of 0)
    const bool kin = kpc * 8 < hd, vin = vd < hd;
    const char *const Kg = kin ? (const char *)((const T *)p.k + (int64_t)g * hd + kpc * 8) : (const char *)zero_piece;
    const char *const Vg = vin ? (const char *)((const T *)p.v + (int64_t)g * hd + vd) : (const char *)zero_piece;
    const uint32_t ldk = kin ? (uint32_t)p.ldk * sizeof(T) : 0, ldv = vin ? (uint32_t)p.ldv * sizeof(T) : 0;
    const int32_t *const pages = PREFIX ? p.prefix_table : p.table + (int64_t)q.id * p.max_pages;
    const int page_mask = (1 << p.page_shift) - 1;
    vu4 kr[C::KU][C::KL];
    uint32_t vr[8][C::VW];
    int kid[C::KU], vid[2];
    auto load_ids = [&](int k0) {
        if (!p.table) return;
#pragma unroll
        for (int n = 0; n < C::KU; ++n) kid[n] = pages[min(k0 + krow + n * (256 / C::PCS), kb1 - 1) >> p.page_shift];
#pragma unroll
        for (int a = 0; a < 2; ++a) vid[a] = pages[min(k0 + 16 * a + 4 * wave, kb1 - 1) >> p.page_shift];
    };
    auto row_of = [&](const char *base, uint32_t ld, int id, int pos) {
        if (!p.table) return base + (int64_t)(q.row0 + pos) * ld;
        return base + (uint32_t)(pos & page_mask) * ld + (uint64_t)(uint32_t)id * (ld << p.page_shift);
    };
    auto take_v = [&](uint32_t (&to)[C::VW], gvu4 at) {
        if constexpr (C::VW == 4) {
            const vu4 x = *at;
#pragma unroll
            for (int e = 0; e < 4; ++e) to[e] = x[e];
        } else if constexpr (C::VW == 2) {
            const vu2 x = *(const __attribute__((address_space(1))) vu2 *)at;
            to[0] = x.x, to[1] = x.y;
        } else if constexpr (C::F32 || C::VD == 2) {
            to[0] = *(const __attribute__((address_space(1))) uint32_t *)at;
        } else {
            to[0] = *(const __attribute__((address_space(1))) uint16_t *)at;
        }
    };
    auto load_tile = [&](int k0) {
        const char *ka[C::KU], *va[2];
        bool held = true;
#pragma unroll
        for (int n = 0; n < C::KU; ++n) {
            ka[n] = row_of(Kg, ldk, kid[n], k0 + krow + n * (256 / C::PCS));
            held = held & (!p.table | ((uint32_t)kid[n] < (uint32_t)p.n_pages));
        }
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            va[a] = row_of(Vg, ldv, vid[a], k0 + 16 * a + 4 * wave);
            held = held & (!p.table | ((uint32_t)vid[a] < (uint32_t)p.n_pages));
        }
        if (k0 + BN <= kb1 && __all(held)) {
#pragma unroll
            for (int n = 0; n < C::KU; ++n)
#pragma unroll
                for (int x = 0; x < C::KL; ++x) kr[n][x] = *(gvu4)(uintptr_t)(ka[n] + 16 * x);
#pragma unroll
            for (int i = 0; i < 8; ++i) take_v(vr[i], (gvu4)(uintptr_t)(va[i >> 2] + (i & 3) * ldv));
            return;
        }
#pragma unroll
        for (int n = 0; n < C::KU; ++n) {
            const bool ok = (k0 + krow + n * (256 / C::PCS) < kb1) & (!p.table | ((uint32_t)kid[n] < (uint32_t)p.n_pages));
#pragma unroll
            for (int x = 0; x < C::KL; ++x) kr[n][x] = *piece(ka[n] + 16 * x, ok);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            take_v(vr[i], piece(va[i >> 2] + (i & 3) * ldv, (k0 + (i >> 2) * 16 + 4 * wave + (i & 3) < kb1) &
                                                                (!p.table | ((uint32_t)vid[i >> 2] < (uint32_t)p.n_pages))));
    };
    char *const Kw = lds + ((krow >> 4) * C::PCS + kpc) * C::KCH + (krow & 15) * 16;
    char *const Vw = lds + C::PL * C::KP + (lane >> 4) * C::VD * 1024 + (wave * 16 + l16) * 16;
    auto store_tile = [&]() {
#pragma unroll
        for (int n = 0; n < C::KU; ++n) {
            vu4 w[C::PL];
            if constexpr (C::F32) {
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    uint32_t u[3];
                    split3(__uint_as_float(kr[n][x >> 1][(x & 1) * 2]), __uint_as_float(kr[n][x >> 1][(x & 1) * 2 + 1]), u);
                    w[0][x] = u[0], w[1][x] = u[1], w[2][x] = u[2];
                }
            } else {
                w[0] = kr[n][0];
            }
            // (16 rows on where a block of keys has fewer threads)
            char *to = Kw + (256 / C::PCS >= 16 ? n * (256 / C::PCS / 16) * C::PCS * C::KCH : (n & 1) * (256 / C::PCS) * 16 + (n >> 1) * C::PCS * C::KCH);
#pragma unroll
            for (int y = 0; y < C::PL; ++y) *(vu4 *)(to + y * C::KP) = w[y];
        }
#pragma unroll
        for (int e = 0; e < C::VD; ++e) {
            vu4 w[C::PL];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                if constexpr (C::F32) {
                    uint32_t u[3];
                    split3(__uint_as_float(vr[2 * x][e]), __uint_as_float(vr[2 * x + 1][e]), u);
                    w[0][x] = u[0], w[1][x] = u[1], w[2][x] = u[2];
                } else {
                    w[0][x] = __builtin_amdgcn_perm(vr[2 * x + 1][e >> 1], vr[2 * x][e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
                }
            }
#pragma unroll
            for (int y = 0; y < C::PL; ++y) *(vu4 *)(Vw + e * 1024 + y * C::VP) = w[y];
        }
    };

    vu4 qf[C::PL][C::STEPS];
    if (kb0 < kb1) {
        load_ids(kb0);
        load_tile(kb0);
        load_ids(kb0 + BN);
    }
    const Row row = row_at<PREFIX>(p, q, tile * BM + wave * 16 + l16, group, g);
    if (!PREFIX && g4 == 0) tell_parts(p, plan, it, row, kend, whole);
    int lim_hi = row.lim, lim_lo = row.valid ? row.lim : INT32_MAX;
#pragma unroll
    for (int x = 8; x > 0; x >>= 1) {
        lim_hi = max(lim_hi, __shfl_xor(lim_hi, x, WAVE));
        lim_lo = min(lim_lo, __shfl_xor(lim_lo, x, WAVE));
    }
    lim_hi = __builtin_amdgcn_readfirstlane(lim_hi), lim_lo = __builtin_amdgcn_readfirstlane(lim_lo);
    {
        const T *Q = (const T *)p.q + row.t * p.ldq + (int64_t)row.head * hd;
#pragma unroll
        for (int j = 0; j < C::STEPS; ++j) {
            const int e = (4 * j + g4) * 8;
            const bool ok = row.valid && e < hd;
            const vu4 a = *piece(Q + e, ok);
            if constexpr (C::F32) {
                const vu4 b = *piece(Q + e + 4, ok);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    uint32_t u[3];
                    const vu4 &h = x < 2 ? a : b;
                    split3(__uint_as_float(h[(x & 1) * 2]), __uint_as_float(h[(x & 1) * 2 + 1]), u);
                    qf[0][j][x] = u[0], qf[1][j][x] = u[1], qf[2][j][x] = u[2];
                }
            } else {
                qf[0][j] = a;
            }
        }
    }
#pragma unroll
    for (int j = 0; j < C::STEPS; ++j) asm volatile("" : "+v"(qf[0][j]));  // (waited for here, as in the tiles of 128 rows)
    const float c = p.scale * LOG2E, slack = slack_of(c);  // (as in the tiles)
    float m = -INFINITY, l = 0.0f;
    vf4 o[C::VT];
#pragma unroll
    for (int t = 0; t < C::VT; ++t) o[t] = vf4{0.0f, 0.0f, 0.0f, 0.0f};
    const char *const Kr = lds + g4 * C::KCH + l16 * 16, *const Vr = lds + C::PL * C::KP + lane * 16;
    for (int k0 = kb0; k0 < kb1; k0 += BN) {
        store_tile();
        __syncthreads();
        if (k0 + BN < kb1) {
            load_tile(k0 + BN);
            load_ids(k0 + 2 * BN);
        }
        if (k0 <= lim_hi) {
            vf4 s[2] = {vf4{0.0f, 0.0f, 0.0f, 0.0f}, vf4{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
            for (int j = 0; j < C::STEPS; ++j) {
                vu4 k[2][C::PL];
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int y = 0; y < C::PL; ++y) k[b][y] = *(const vu4 *)(Kr + y * C::KP + (b * C::PCS + 4 * j) * C::KCH);
#pragma unroll
                for (int x = 6 - C::PRODUCTS; x < 6; ++x)
#pragma unroll
                    for (int b = 0; b < 2; ++b) s[b] = mfma16<typename C::Op>(k[b][SPLIT_A[x]], qf[SPLIT_B[x]][j], s[b]);
            }
            if (k0 + BN - 1 > lim_lo) {
                int lim = row.lim - k0 - 4 * g4;
                asm volatile("" : "+v"(lim));
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (b * 16 + i > lim) s[b][i] = -INFINITY;
            }
            float mt = s[0][0];
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) mt = fmaxf(mt, s[b][i]);
            mt = fmaxf(mt, __shfl_xor(mt, 16, WAVE));
            mt = fmaxf(mt, __shfl_xor(mt, 32, WAVE));
            if (__any(mt > m + slack)) {
                const float to = fmaxf(mt, m);
                const float shrink = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - to) * c);
                l *= shrink;
#pragma unroll
                for (int t = 0; t < C::VT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[t][i] *= shrink;
                m = to;
            }
            const float base = m == -INFINITY ? 0.0f : m * c;
            vu4 w[C::PL];
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const float e0 = __builtin_amdgcn_exp2f(fmaf(s[b][i], c, -base)), e1 = __builtin_amdgcn_exp2f(fmaf(s[b][i + 1], c, -base));
                    l += e0 + e1;
                    if constexpr (C::F32) {
                        uint32_t u[3];
                        split3(e0, e1, u);
                        w[0][b * 2 + i / 2] = u[0], w[1][b * 2 + i / 2] = u[1], w[2][b * 2 + i / 2] = u[2];
                    } else {
                        union { T e[2]; uint32_t u; } x;
                        x.e[0] = (T)e0, x.e[1] = (T)e1;
                        w[0][b * 2 + i / 2] = x.u;
                    }
                }
#pragma unroll
            for (int t = 0; t < C::VT; t += 2) {
                vu4 v[2][C::PL];
#pragma unroll
                for (int z = 0; z < 2; ++z)
#pragma unroll
                    for (int y = 0; y < C::PL; ++y) v[z][y] = *(const vu4 *)(Vr + y * C::VP + (t + z) * 1024);
#pragma unroll
                for (int x = 6 - C::PRODUCTS; x < 6; ++x)
#pragma unroll
                    for (int z = 0; z < 2; ++z) o[t + z] = mfma16<typename C::Op>(v[z][SPLIT_A[x]], w[SPLIT_B[x]], o[t + z]);
            }
        }
        __syncthreads();
    }
    l += __shfl_xor(l, 16, WAVE);
    l += __shfl_xor(l, 32, WAVE);

    // (as in the tiles: a row whose result is no number is computed again, key by key)
    float odd = l * 0.0f;
#pragma unroll
    for (int t = 0; t < C::VT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) odd = fmaf(o[t][i], 0.0f, odd);
    odd += __shfl_xor(odd, 16, WAVE);
    odd += __shfl_xor(odd, 32, WAVE);
    const bool again = row.valid && row.lim >= kb0 && odd != 0.0f;
    if (odd != 0.0f && !again) {
#pragma unroll
        for (int t = 0; t < C::VT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[t][i] = 0.0f;
    }
    uint32_t todo = (uint32_t)__ballot(again) & 0xffffu;
    if (row.valid && !again) {
        const bool seen = row.lim >= 0;
        const int64_t at = ((int64_t)part * p.T + row.t) * p.n_head + row.head;
        const float inv = whole ? (seen ? 1.0f / l : 0.0f) : 1.0f;
        T *out = (T *)p.out + row.t * p.ldo + (int64_t)row.head * hd;
        float *po = p.part_o + at * hd;
        // rows 4 g4 + i of blocks t0 .. t0 + VD - 1: 4 VD neighbouring dimensions
#pragma unroll
        for (int t0 = 0; t0 < C::VT; t0 += C::VD) {
            const int d = C::VD * ((t0 / C::VD) * 16 + 4 * g4);
            float e[4 * C::VD];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int x = 0; x < C::VD; ++x) e[i * C::VD + x] = o[t0 + x][i] * inv;
#pragma unroll
            for (int x = 0; x < C::VD; ++x) {
                if (d + 4 * x >= hd) continue;
                if (whole) {
                    T y[4] = {(T)e[4 * x], (T)e[4 * x + 1], (T)e[4 * x + 2], (T)e[4 * x + 3]};
                    __builtin_memcpy(__builtin_assume_aligned(out + d + 4 * x, sizeof y), y, sizeof y);
                } else {
                    *(vf4 *)(po + d + 4 * x) = vf4{e[4 * x], e[4 * x + 1], e[4 * x + 2], e[4 * x + 3]};
                }
            }
        }
        if (!whole && g4 == 0) p.part_ml[at] = make_float2(m, l);
    }
    while (todo) {
        const int n = __builtin_ctz(todo);
        todo &= todo - 1;
        const Row w = row_at<PREFIX>(p, q, tile * BM + wave * 16 + n, group, g);
        const Seq qs = PREFIX ? seq_at(p, (int)w.t) : q;
        float mr, lr, orow[4];
        attend_row<T>(p, qs, w.t, w.head, kb0, min(kb1, w.lim + 1), mr, lr, orow);
        store_row<T>(p, w.t, w.head, part, whole, true, mr, lr, orow);
    }
}

// ---- few rows ----
// A workgroup takes up to 16 query rows of one K/V head (a decoded token's query heads,
// a few drafted tokens), and its four waves take turns at the keys, KS each, every wave
// with a softmax of its own until they are joined at the end.  Nothing is shared while the
// keys stream by, so K and V go from memory to registers (two steps of them in flight)
// and straight into the products:
//   S^T = K Q^T   16 keys x 16 queries: lane l has query l % 16, keys 4 (l / 16) + i
//   O^T = V^T P^T with those keys in that order; lane l reads HD / 16 neighbouring
//                 dimensions of each key's row, of which the t-th belong to the t-th
//                 16 x 16 block, transposed (16-bit types) with v_perm.
// Bound by HBM: 2 hd elements per key against 4 hd operations per key and row.
template <typename T, int HD>
struct FewCfg {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int KB = F32 ? 1 : 2;              // blocks of 16 keys per step
    static constexpr int KS = 16 * KB;                  // keys per step
    static constexpr int EP = 16 / (int)sizeof(T);      // elements per piece
    static constexpr int STEPS = HD / (4 * EP);         // K pieces of a lane per block
    static constexpr int VW = HD / 16;                  // dimensions of a lane
    static constexpr int VK = 4 * KB;                   // keys of a lane
    static constexpr int VB = VW * (int)sizeof(T);      // bytes of a lane's row of V
    static constexpr int VP = (VB + 15) / 16;           // pieces of it
};

template <int HD>
struct FewLds {
    float joined[4][16][HD], ms[4][16], ls[4][16];
    int odd[16];
};

template <typename T, int HD, bool PREFIX>
__device__ __forceinline__ void attend_few(const ServeAttnParams &p, const TilePlan &plan, int block, char *lds) {
    using C = FewCfg<T, HD>;
    constexpr int BM = 16;
    FewLds<HD> &sh = *(FewLds<HD> *)lds;
    auto &joined = sh.joined;
    auto &ms = sh.ms;
    auto &ls = sh.ls;
    auto &odd = sh.odd;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, g4 = lane >> 4;
    const int group = p.n_head / p.n_head_kv, hd = p.head_dim;
    Item it;
    if (!find_item<PREFIX, false>(p, plan, block, group, it)) return;
    const Seq q = it.q;
    const int g = it.g, tile = it.tile;
    const int kend = tile_end<PREFIX>(p, q, tile, BM, group), key0 = min(plan.key0, kend), from = key0 & ~31;
    const bool whole = plan.part0 < 0 || (plan.alone && it.size >= kend - from);
    const int part = plan.part0 + it.part, kb0 = min(from + it.part * it.size, kend), kb1 = min(kb0 + it.size, kend);
    if (it.part > 0 && kb0 >= kb1) return;
    const char *const Kg = (const char *)((const T *)p.k + (int64_t)g * hd), *const Vg = (const char *)((const T *)p.v + (int64_t)g * hd);
    const uint32_t ldk = (uint32_t)p.ldk * sizeof(T), ldv = (uint32_t)p.ldv * sizeof(T);
    const int32_t *const pages = PREFIX ? p.prefix_table : p.table + (int64_t)q.id * p.max_pages;
    const int page_mask = (1 << p.page_shift) - 1;
    struct Step {
        vu4 k[C::KB][C::STEPS];
        vu4 v[C::VK][C::VP];
    };
    struct Ids {
        int k[C::KB], v[C::KB];
    };
    auto load_ids = [&](Ids &d, int k0) {
        if (!p.table) return;
#pragma unroll
        for (int b = 0; b < C::KB; ++b) {
            d.k[b] = pages[min(k0 + b * 16 + l16, kb1 - 1) >> p.page_shift];
            d.v[b] = pages[min(k0 + b * 16 + 4 * g4, kb1 - 1) >> p.page_shift];
        }
    };
    // the address of a position's row: one 64-bit product per group of rows of one page
    auto row_of = [&](const char *base, uint32_t ld, int id, int pos) {
        if (!p.table) return base + (int64_t)(q.row0 + pos) * ld;
        return base + (uint32_t)(pos & page_mask) * ld + (uint64_t)(uint32_t)id * (ld << p.page_shift);
    };
    auto load = [&](Step &x, const Ids &d, int k0) {
        bool held = true;
        if (p.table) {
#pragma unroll
            for (int b = 0; b < C::KB; ++b) held = held & ((uint32_t)d.k[b] < (uint32_t)p.n_pages) & ((uint32_t)d.v[b] < (uint32_t)p.n_pages);
        }
        if (hd == HD && k0 >= key0 && k0 + C::KS <= kb1 && __all(held)) {
#pragma unroll
            for (int b = 0; b < C::KB; ++b) {
                const char *kr = row_of(Kg, ldk, d.k[b], k0 + b * 16 + l16) + g4 * 16;
                const char *vr = row_of(Vg, ldv, d.v[b], k0 + b * 16 + 4 * g4) + l16 * C::VB;
#pragma unroll
                for (int j = 0; j < C::STEPS; ++j) x.k[b][j] = *(gvu4)(uintptr_t)(kr + j * 64);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < C::VP; ++j) {
                        const uintptr_t at = (uintptr_t)(vr + i * ldv + j * 16);
                        if constexpr (C::VB == 8) {
                            const vu2 h = *(const __attribute__((address_space(1))) vu2 *)at;
                            x.v[4 * b + i][j] = vu4{h.x, h.y, 0, 0};
                        } else {
                            x.v[4 * b + i][j] = *(gvu4)at;
                        }
                    }
            }
            return;
        }
#pragma unroll
        for (int b = 0; b < C::KB; ++b) {
            const int kp = k0 + b * 16 + l16, vp = k0 + b * 16 + 4 * g4;
            const bool kok = (kp >= key0) & (kp < kb1) & (!p.table | ((uint32_t)d.k[b] < (uint32_t)p.n_pages));
            const bool vok = !p.table | ((uint32_t)d.v[b] < (uint32_t)p.n_pages);
            const char *kr = row_of(Kg, ldk, d.k[b], kp) + g4 * 16, *vr = row_of(Vg, ldv, d.v[b], vp) + l16 * C::VB;
#pragma unroll
            for (int j = 0; j < C::STEPS; ++j) x.k[b][j] = *piece(kr + j * 64, kok & ((4 * j + g4) * C::EP < hd));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool ok = vok & (vp + i >= key0) & (vp + i < kb1);
#pragma unroll
                for (int j = 0; j < C::VP; ++j) {
                    const bool in = ok & (l16 * C::VW + j * C::EP < hd);
                    if constexpr (C::VB == 8) {
                        const vu2 h = *(const __attribute__((address_space(1))) vu2 *)piece(vr + i * ldv, in);
                        x.v[4 * b + i][j] = vu4{h.x, h.y, 0, 0};
                    } else {
                        x.v[4 * b + i][j] = *piece(vr + i * ldv + j * 16, in);
                    }
                }
            }
        }
    };

    constexpr int STRIDE = 4 * C::KS;
    const int first = kb0 + wave * C::KS;
    Step now, next;
    Ids ids;
    if (first < kb1) {
        load_ids(ids, first);
        const Ids held = ids;
        load_ids(ids, first + STRIDE);
        load(now, held, first);
    }
    int lim, lim_hi, lim_lo;
    vu4 qf[C::STEPS];
    {
        const Row row = row_at<PREFIX>(p, q, tile * BM + l16, group, g);
        if (!PREFIX && tid < 16) tell_parts(p, plan, it, row, kend - from, whole);
        lim = lim_hi = row.lim;
        lim_lo = row.valid ? lim : INT32_MAX;
        const T *Q = (const T *)p.q + row.t * p.ldq + (int64_t)row.head * hd;
#pragma unroll
        for (int j = 0; j < C::STEPS; ++j) {
            const int e = (4 * j + g4) * C::EP;
            qf[j] = *piece(Q + e, row.valid && e < hd);
        }
    }
#pragma unroll
    for (int x = 8; x > 0; x >>= 1) {
        lim_hi = max(lim_hi, __shfl_xor(lim_hi, x, WAVE));
        lim_lo = min(lim_lo, __shfl_xor(lim_lo, x, WAVE));
    }
    lim_hi = __builtin_amdgcn_readfirstlane(lim_hi), lim_lo = __builtin_amdgcn_readfirstlane(lim_lo);

    const float c = p.scale * LOG2E, slack = slack_of(c);  // (as in the tiles)
    float m = -INFINITY, l = 0.0f;
    vf4 o[C::VW];
#pragma unroll
    for (int t = 0; t < C::VW; ++t) o[t] = vf4{0.0f, 0.0f, 0.0f, 0.0f};
    auto compute = [&](const Step &x, int k0) {
        vf4 s[C::KB];
#pragma unroll
        for (int b = 0; b < C::KB; ++b) {
            s[b] = vf4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < C::STEPS; ++j) {
                if constexpr (C::F32) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        s[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(x.k[b][j][i]), __uint_as_float(qf[j][i]), s[b], 0, 0, 0);
                } else {
                    s[b] = mfma16<T>(x.k[b][j], qf[j], s[b]);
                }
            }
        }
        if (k0 < key0 || k0 + C::KS - 1 > lim_lo) {
#pragma unroll
            for (int b = 0; b < C::KB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int pos = k0 + b * 16 + 4 * g4 + i;
                    if (pos > lim || pos < key0) s[b][i] = -INFINITY;
                }
        }
        float mt = s[0][0];
#pragma unroll
        for (int b = 0; b < C::KB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) mt = fmaxf(mt, s[b][i]);
        mt = fmaxf(mt, __shfl_xor(mt, 16, WAVE));
        mt = fmaxf(mt, __shfl_xor(mt, 32, WAVE));
        if (__any(mt > m + slack)) {
            mt = fmaxf(mt, m);
            const float shrink = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mt) * c);
            l *= shrink;
#pragma unroll
            for (int t = 0; t < C::VW; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[t][i] *= shrink;
            m = mt;
        }
        const float base = m == -INFINITY ? 0.0f : m * c;
        union { T e[8]; vu4 u; } w;
#pragma unroll
        for (int b = 0; b < C::KB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[b][i] = __builtin_amdgcn_exp2f(fmaf(s[b][i], c, -base));
                l += s[b][i];
                if constexpr (!C::F32) w.e[4 * b + i] = (T)s[b][i];
            }
#pragma unroll
        for (int t = 0; t < C::VW; ++t) {
            if constexpr (C::F32) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    o[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(x.v[i][t >> 2][t & 3]), s[0][i], o[t], 0, 0, 0);
            } else {
                vu4 a;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    a[k] = __builtin_amdgcn_perm(x.v[2 * k + 1][t >> 3][(t & 7) >> 1], x.v[2 * k][t >> 3][(t & 7) >> 1], t & 1 ? 0x07060302u : 0x05040100u);
                o[t] = mfma16<T>(a, w.u, o[t]);
            }
        }
    };

    // The next step in flight during a step's products, the page ids of the one after it ahead
    // of that (loads return in order: a wait for an id must not be one for rows).
#pragma unroll
    for (int j = 0; j < C::STEPS; ++j) asm volatile("" : "+v"(qf[j]));  // (waited for here, as in the tiles)
    const int stop = min(kb1, lim_hi + 1);
    for (int k0 = first; k0 < stop; k0 += STRIDE) {
        if (k0 + STRIDE < stop) {
            const Ids held = ids;
            load_ids(ids, k0 + 2 * STRIDE);
            load(next, held, k0 + STRIDE);
        }
        compute(now, k0);
        now = next;
    }

    // the four waves' results: each to the common maximum, then summed
    l += __shfl_xor(l, 16, WAVE);
    l += __shfl_xor(l, 32, WAVE);
    if (g4 == 0) ms[wave][l16] = m, ls[wave][l16] = l;
    if (tid < BM) odd[tid] = 0;
    __syncthreads();
    {
        float mt = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) mt = fmaxf(mt, ms[w][l16]);
        const float base = mt == -INFINITY ? 0.0f : mt * c;
        const float shrink = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(fmaf(m, c, -base));
#pragma unroll
        for (int t = 0; t < C::VW; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) joined[wave][l16][(4 * g4 + i) * C::VW + t] = o[t][i] * shrink;
    }
    __syncthreads();
    // 256 / BM threads per row
    constexpr int TPR = 256 / BM, PER = HD / TPR;
    const int r = tid / TPR, d0 = (tid % TPR) * 4;
    const Row row = row_at<PREFIX>(p, q, tile * BM + r, group, g);
    float mt = -INFINITY, lt = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) mt = fmaxf(mt, ms[w][r]);
    const float base = mt == -INFINITY ? 0.0f : mt * c;
#pragma unroll
    for (int w = 0; w < 4; ++w)
        if (ms[w][r] != -INFINITY) lt = fmaf(ls[w][r], __builtin_amdgcn_exp2f(fmaf(ms[w][r], c, -base)), lt);
        else lt += ls[w][r];
    float4 v[PER / 4];
    float bad = lt * 0.0f;
#pragma unroll
    for (int x = 0; x < PER / 4; ++x) {
        const int d = d0 + x * TPR * 4;
        v[x] = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float4 a = *(const float4 *)&joined[w][r][d];
            v[x].x += a.x, v[x].y += a.y, v[x].z += a.z, v[x].w += a.w;
        }
        bad = fmaf(v[x].x, 0.0f, bad), bad = fmaf(v[x].y, 0.0f, bad), bad = fmaf(v[x].z, 0.0f, bad), bad = fmaf(v[x].w, 0.0f, bad);
    }
    // (as in the tiles: a row whose result is no number is computed again, key by key)
    if (bad != 0.0f) {
        if (row.valid && row.lim >= kb0) odd[r] = 1;
        else
            for (auto &x : v) x = make_float4(0, 0, 0, 0);
    }
    __syncthreads();
    if (row.valid && !odd[r]) {
        const bool seen = row.lim >= 0;
        const int64_t at = ((int64_t)part * p.T + row.t) * p.n_head + row.head;
        const float inv = whole ? (seen ? 1.0f / lt : 0.0f) : 1.0f;
#pragma unroll
        for (int x = 0; x < PER / 4; ++x) {
            const int d = d0 + x * TPR * 4;
            if (d >= hd) continue;
            if (whole) {
                T *out = (T *)p.out + row.t * p.ldo + (int64_t)row.head * hd + d;
                T e[4] = {(T)(v[x].x * inv), (T)(v[x].y * inv), (T)(v[x].z * inv), (T)(v[x].w * inv)};
                __builtin_memcpy(__builtin_assume_aligned(out, sizeof e), e, sizeof e);
            } else {
                *(float4 *)(p.part_o + at * hd + d) = v[x];
            }
        }
        if (!whole && tid % TPR == 0) p.part_ml[at] = make_float2(mt, lt);
    }
    for (int n = wave; n < BM; n += 4) {
        if (!odd[n]) continue;
        const Row w = row_at<PREFIX>(p, q, tile * BM + n, group, g);
        const Seq qs = PREFIX ? seq_at(p, (int)w.t) : q;
        float mr, lr, orow[4];
        attend_row<T>(p, qs, w.t, w.head, max(kb0, key0), min(kb1, w.lim + 1), mr, lr, orow);
        store_row<T>(p, w.t, w.head, part, whole, true, mr, lr, orow);
    }
}

// ---- launches ----
// A plan's rows: up to 16 per workgroup by the few-row form, tiles of 64, of 128 (16-bit types).
enum RowForm { ROWS_FEW, ROWS_64, ROWS_128 };
template <typename T, int HD, RowForm FORM, bool PREFIX>
__device__ __forceinline__ void attend(const ServeAttnParams &p, const TilePlan &plan, int block, char *lds) {
    if constexpr (FORM == ROWS_FEW) attend_few<T, HD, PREFIX>(p, plan, block, lds);
    else if constexpr (FORM == ROWS_64) attend_tile64<T, HD, PREFIX>(p, plan, block, lds);
    else attend_tile<T, HD, PREFIX>(p, plan, block, lds);
}
template <typename T, int HD, RowForm FORM>
constexpr size_t lds_of() {
    if constexpr (FORM == ROWS_FEW) return sizeof(FewLds<HD>);
    else if constexpr (FORM == ROWS_64) return Tile64Cfg<T, HD>::LDS;
    else return TileCfg<T, HD>::LDS;
}

template <typename T, int HD, RowForm FORM>
__global__ __launch_bounds__(256, HD == 256 ? 1 : 2) void attn_kernel(ServeAttnParams p, TilePlan keys) {
    extern __shared__ __align__(16) char lds[];
    attend<T, HD, FORM, false>(p, keys, blockIdx.x, lds);
}
// The shared prefix by the first workgroups, the sequences' own keys by the others.
template <typename T, int HD, RowForm FORM>
__global__ __launch_bounds__(256, HD == 256 ? 1 : 2) void attn_prefix_kernel(ServeAttnParams p, TilePlan prefix, TilePlan keys) {
    extern __shared__ __align__(16) char lds[];
    const int blocks = (int)prefix.items * p.n_head_kv;
    if ((int)blockIdx.x < blocks) attend<T, HD, FORM, true>(p, prefix, blockIdx.x, lds);
    else attend<T, HD, ROWS_FEW, false>(p, keys, blockIdx.x - blocks, lds);
}

// ---- joining parts ----
// One wave per (row, head): m = max_i m_i, o = sum_i 2^(c (m_i - m)) o_i over the same sum
// of l_i, for rows whose keys were cut into parts.  Four dimensions per lane and 64 / LPP
// parts side by side, LPP = the lanes of one row of parts; all loads of up to four such
// rounds in flight.
template <typename T, int LPP>
__global__ __launch_bounds__(256) void attn_join_kernel(ServeAttnParams p, TilePlan keys, TilePlan prefix) {
    constexpr int SIDE = WAVE / LPP;
    const int lane = threadIdx.x & 63, hd = p.head_dim, h = blockIdx.y;
    const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= p.T) return;
    const int told = p.parts[t * p.n_head + h];
    if (p.seq_off && (t < p.seq_off[0] || t >= p.seq_off[p.n_seq])) return;  // no row of a sequence
    if (told == 0) return;  // written whole
    const bool seen = told > 0;
    const int np = prefix.items ? prefix.splits : 0, parts = np + min(abs(told), keys.splits);
    const float c = p.scale * LOG2E;
    const int64_t step = p.T * p.n_head, at = t * p.n_head + h;
    auto place = [&](int i) { return (i < np ? prefix.part0 + i : keys.part0 + i - np) * step + at; };
    float m = -INFINITY;
    for (int i = lane; i < parts; i += WAVE) m = fmaxf(m, p.part_ml[place(i)].x);
    m = wave_max(m);
    const float base = m == -INFINITY ? 0.0f : m * c;
    float l = 0.0f;
    vf4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    const int d = lane % LPP * 4;
#pragma unroll 4
    for (int i = lane / LPP; i < parts; i += SIDE) {
        const float2 ml = p.part_ml[place(i)];
        const vf4 po = *(const vf4 *)(p.part_o + place(i) * hd + min(d, hd - 4));
        // (a part without a key that the row sees: -inf, and zeros; one whose scores are -inf or no
        // numbers: -inf, and sums whose NaN the weight 0 lets through)
        const float w = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(fmaf(ml.x, c, -base));
        l = fmaf(w, ml.y, l);
#pragma unroll
        for (int x = 0; x < 4; ++x) o[x] = fmaf(w, po[x], o[x]);
    }
#pragma unroll
    for (int x = LPP; x < WAVE; x <<= 1) {
        l += __shfl_xor(l, x, WAVE);
#pragma unroll
        for (int y = 0; y < 4; ++y) o[y] += __shfl_xor(o[y], x, WAVE);
    }
    if (lane < LPP && d < hd) {
        T e[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) e[x] = (T)(seen ? o[x] / l : 0.0f);
        __builtin_memcpy(__builtin_assume_aligned((T *)p.out + t * p.ldo + (int64_t)h * hd + d, sizeof e), e, sizeof e);
    }
}

// ---- plans ----
int hd_class(int head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }

struct AttnPlan {
    TilePlan keys, prefix;  // over the rows' own keys, and over the shared prefix
    int parts;              // partial results to join, 0: none
};

// seqs sequences of `rows` query rows per K/V head together, as the host knows them, whose
// rows see up to `most` keys from key0 on.  prefix: all rows, the same keys.
TilePlan plan_rows(const ServeAttnParams &p, int64_t seqs, int64_t rows, int64_t most, int64_t key0, bool prefix) {
    TilePlan t{};
    const int64_t avg = rows / std::max<int64_t>(seqs, 1);
    // Up to 16 rows of a sequence: the few-row form, which the tiles pass soon after (32
    // sequences of 500 to 2000 keys, 12 heads of 128: 30 rows bf16 22.4 against 20.2 us, f32
    // 38.7 against 37.3).  After a prefix it is always that: the tiles begin with key 0.
    // 16-bit prompts of up to about 450 tokens have tiles of 64 rows (8 of 400, 14 heads of 64: 16.3
    // against 20.7 us with 128; 32 of 200, 16 heads: 21.6 against 30.2; but 3 of 300 to 900, 12
    // heads of 128: 33.7 against 28.7, one of 4000: 139 against 95).
    const bool brief = !p.table && p.T <= 448 * seqs;
    t.bm = avg <= 16 || key0 > 0 ? 16 : p.dtype == GAJE_DTYPE_F32 || brief ? 64 : 128;
    t.key0 = (int32_t)key0;
    // Workgroups wanted: two for each of 256 CUs; over a prefix one, where every part costs
    // partial results of all rows (64 sequences over 16000 keys: 29.1 against 38.2 us), and beside
    // one of eight times the own keys or more half a CU's, which leaves fewer workgroups without an
    // item.
    t.blocks = prefix ? 8 : key0 >= 8 * most ? 7 : 9;
    // Parts of a prompt's own keys pay from 512 keys on (f32 prompts of up to 1500 tokens 67.6
    // against 75.1 us with 256, one f16 prompt of 1500 34.1 against 42.6), of a cache's from 256 (5
    // drafted tokens, f32, 37.3 against 49.4), a few rows' and a prefix's from 128.
    t.least = prefix || t.bm == 16 ? 128 : p.table ? 256 : 512;
    const int target = 1 << t.blocks;
    // ragged sequences end in a tile that is not full
    const int64_t tiles = prefix || p.prefix_table ? seqs * ((rows / seqs + t.bm - 1) / t.bm) : rows / t.bm + std::min(seqs, p.T);
    const int64_t blocks = tiles * p.n_head_kv;
    t.splits = 1;
    while (blocks < target && t.splits < 64 && t.splits * blocks < 16 * target && t.splits * t.least < most) t.splits *= 2;
    // a sequence has at most keys / size + 1 parts per tile, and half of its keys count at least
    // (and `splits` at most: a workgroup without an item still looks for one)
    t.items = std::min<int64_t>(tiles * t.splits, tiles + 2 * target / p.n_head_kv + 1);
    if (t.splits == 1) t.size = INT32_MAX / 2;
    if (prefix) {
        t.size = part_size(most * blocks / PART_UNIT, (int)most, t.splits, t.least, t.blocks);
        t.splits = (int)((most - 1) / t.size + 1);
        t.items = tiles * t.splits;
    }
    return t;
}

AttnPlan make_plan(const ServeAttnParams &p) {
    AttnPlan a{};
    const int64_t group = p.n_head / p.n_head_kv, most = p.table ? p.max_pages << p.page_shift : p.T;
    const int64_t first = p.prefix_table ? p.prefix_len : 0;  // (set for single tokens only)
    a.keys = plan_rows(p, p.n_seq, p.T * group, std::max<int64_t>(most - first, 1), first, false);
    a.keys.part0 = -1;
    if (first > 0) {
        a.prefix = plan_rows(p, 1, p.T * group, first, 0, true);
        a.prefix.part0 = 0;
        a.keys.part0 = a.prefix.splits;
        a.parts = a.prefix.splits + a.keys.splits;
    } else if (a.keys.splits > 1) {
        a.keys.part0 = 0;
        a.keys.alone = 1;
        a.parts = a.keys.splits;
    }
    return a;
}

int set_lds(const void *kernel, size_t lds, std::atomic<bool> *set) {
    int dev = 0;
    GAJE_HIP_CHECK(hipGetDevice(&dev));
    if (dev >= 0 && dev < 64 && set[dev].load()) return GAJE_OK;
    GAJE_HIP_CHECK(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    if (dev >= 0 && dev < 64) set[dev].store(true);
    return GAJE_OK;
}

template <typename T, int HD, RowForm FORM>
int launch_form(const ServeAttnParams &p, const AttnPlan &a, hipStream_t s) {
    static std::atomic<bool> set[2][64];
    const int64_t blocks = (a.prefix.items + a.keys.items) * p.n_head_kv;
    if (blocks > (int64_t)1 << 23)
        return set_error(GAJE_ERR_UNSUPPORTED, "attention over %lld tiles of rows (2^23 at most)", (long long)blocks);
    if (a.prefix.items) {
        constexpr size_t lds = std::max(lds_of<T, HD, FORM>(), lds_of<T, HD, ROWS_FEW>());
        GAJE_TRY(set_lds((const void *)attn_prefix_kernel<T, HD, FORM>, lds, set[1]));
        attn_prefix_kernel<T, HD, FORM><<<(unsigned)blocks, 256, lds, s>>>(p, a.prefix, a.keys);
    } else {
        constexpr size_t lds = lds_of<T, HD, FORM>();
        GAJE_TRY(set_lds((const void *)attn_kernel<T, HD, FORM>, lds, set[0]));
        attn_kernel<T, HD, FORM><<<(unsigned)blocks, 256, lds, s>>>(p, a.keys);
    }
    GAJE_HIP_CHECK(hipGetLastError());
    return GAJE_OK;
}

template <typename T, int HD>
int launch_head(const ServeAttnParams &p, const AttnPlan &a, hipStream_t s) {
    const int bm = a.prefix.items ? a.prefix.bm : a.keys.bm;
    if (bm == 16) return launch_form<T, HD, ROWS_FEW>(p, a, s);
    if (bm == 64) return launch_form<T, HD, ROWS_64>(p, a, s);
    if constexpr (sizeof(T) == 2) return launch_form<T, HD, ROWS_128>(p, a, s);
    return set_error(GAJE_ERR_HIP, "attention plan of %d rows", bm);
}

template <typename T>
int launch_typed(const ServeAttnParams &p, const AttnPlan &a, hipStream_t s) {
    const int hd = hd_class(p.head_dim);
    if (hd == 64) GAJE_TRY((launch_head<T, 64>(p, a, s)));
    else if (hd == 128) GAJE_TRY((launch_head<T, 128>(p, a, s)));
    else GAJE_TRY((launch_head<T, 256>(p, a, s)));
    if (a.parts) {
        const dim3 grid((unsigned)((p.T + 3) / 4), (unsigned)p.n_head);
        if (p.head_dim <= 64) attn_join_kernel<T, 16><<<grid, 256, 0, s>>>(p, a.keys, a.prefix);
        else if (p.head_dim <= 128) attn_join_kernel<T, 32><<<grid, 256, 0, s>>>(p, a.keys, a.prefix);
        else attn_join_kernel<T, 64><<<grid, 256, 0, s>>>(p, a.keys, a.prefix);
        GAJE_HIP_CHECK(hipGetLastError());
    }
    return GAJE_OK;
}

}  // namespace

int64_t serve_attn_workspace(const ServeAttnParams &p) {
    const int64_t parts = make_plan(p).parts, rows = (p.T * p.n_head + 3) & ~(int64_t)3;
    return parts ? rows * (parts * (8 + 4 * (int64_t)p.head_dim) + 4) : 0;
}

int launch_serve_attn(const ServeAttnParams &params, void *workspace, hipStream_t s) {
    ServeAttnParams p = params;
    const AttnPlan a = make_plan(p);
    if (!a.prefix.items) p.prefix_table = nullptr, p.prefix_len = 0;
    const int64_t rows = (p.T * p.n_head + 3) & ~(int64_t)3;
    p.part_o = (float *)workspace;
    p.part_ml = (float2 *)(p.part_o + a.parts * p.T * p.n_head * p.head_dim);
    p.parts = (int32_t *)(p.part_ml + a.parts * rows);
    if (p.dtype == GAJE_DTYPE_F32) return launch_typed<float>(p, a, s);
    if (p.dtype == GAJE_DTYPE_F16) return launch_typed<_Float16>(p, a, s);
    return launch_typed<__bf16>(p, a, s);
}

}  // namespace gaje
