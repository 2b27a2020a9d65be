// Softmax attention of many sequences: causal over packed prompts, over the pages of
// a KV cache, and over a prefix that all sequences share.
//
// Row t of sequence s with n rows sees keys 0 .. len - n + (t - first row) of its
// len keys.  Over those, with c = scale * log2(e):
//   m = max_j s_j,  o = sum_j 2^(c (s_j - m)) v_j / sum_j 2^(c (s_j - m)),
// s_j = q . k_j, all in f32.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "common.h"
#include "device_util.h"
#include "serve.h"

namespace gaje {
namespace {

constexpr float LOG2E = 1.44269504088896340736f;

template <typename T>
__device__ __forceinline__ float to_f32(T v) { return (float)v; }

// The rows of one sequence and its keys.
struct Seq {
    int64_t row0, rows;  // its rows of q and out
    int64_t len;         // its keys
    int64_t id;
};

__device__ __forceinline__ Seq seq_at(const ServeAttnParams &p, int64_t s) {
    Seq q;
    q.id = s;
    if (p.seq_off) {
        q.row0 = min(max((int64_t)p.seq_off[s], (int64_t)0), p.T);
        q.rows = max(min((int64_t)p.seq_off[s + 1], p.T) - q.row0, (int64_t)0);
    } else {
        q.row0 = s;
        q.rows = 1;
    }
    q.len = p.table ? min(max((int64_t)p.len[s], (int64_t)0), p.max_pages << p.page_shift) : q.rows;
    return q;
}

// The row of k and v that holds a sequence's position, -1 where its page is outside
// the pool.
__device__ __forceinline__ int64_t slot_at(const ServeAttnParams &p, const Seq &q, int64_t pos) {
    if (!p.table) return q.row0 + pos;
    const int32_t *row = pos < p.prefix_len && p.prefix_table ? p.prefix_table : p.table + q.id * p.max_pages;
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

// The sequence of row t, by the offsets (the last s with seq_off[s] <= t).
__device__ __forceinline__ int64_t seq_of_row(const ServeAttnParams &p, int64_t t) {
    if (!p.seq_off) return t;
    if (t < p.seq_off[0] || t >= p.seq_off[p.n_seq]) return -1;
    int64_t lo = 0, hi = p.n_seq;
    while (hi - lo > 1) {
        const int64_t mid = (lo + hi) >> 1;
        if (p.seq_off[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <typename T>
__global__ __launch_bounds__(256) void attn_row_kernel(ServeAttnParams p) {
    const int lane = threadIdx.x & 63, h = blockIdx.y;
    const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= p.T) return;
    const int64_t s = seq_of_row(p, t);
    if (s < 0) return;
    const Seq q = seq_at(p, s);
    const int64_t end = min(q.len - q.rows + (t - q.row0) + 1, q.len);
    float m, l, o[4];
    attend_row<T>(p, q, t, h, 0, end, m, l, o);
    T *out = (T *)p.out + t * p.ldo + (int64_t)h * p.head_dim;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < p.head_dim) out[lane + 64 * i] = (T)(end > 0 ? o[i] / l : 0.0f);
}

}  // namespace

int64_t serve_attn_workspace(const ServeAttnParams &) { return 0; }

int launch_serve_attn(const ServeAttnParams &p, void *, hipStream_t s) {
    const dim3 grid((unsigned)((p.T + 3) / 4), (unsigned)p.n_head);
    if (p.dtype == GAJE_DTYPE_F32) attn_row_kernel<float><<<grid, 256, 0, s>>>(p);
    else if (p.dtype == GAJE_DTYPE_F16) attn_row_kernel<_Float16><<<grid, 256, 0, s>>>(p);
    else attn_row_kernel<__bf16><<<grid, 256, 0, s>>>(p);
    GAJE_HIP_CHECK(hipGetLastError());
    return GAJE_OK;
}

}  // namespace gaje
