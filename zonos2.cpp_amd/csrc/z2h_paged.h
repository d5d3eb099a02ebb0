// z2h_paged.h — attention of a batch of sequences over a paged cache.
#pragma once
#include "z2h_common.h"
#include "z2h_ops_rules.h"

namespace z2d {

struct PlanArgs {
    const int32_t * row_start, * kv_len, * group_start, * prefix_len;
    int n_seq, n_rows, n_group, n_head, nkv, hd, cap;
    uint8_t * ws;
};
constexpr int PLAN_MAGIC = 0x50414745;

// the last index i of [0, n) with start[i] <= x (start ascending; -1: none)
__device__ __forceinline__ int last_at_or_before(const int32_t * start, int n, int x) {
    int lo = -1, hi = n;
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (start[m] <= x) lo = m; else hi = m;
    }
    return lo;
}

// per row: (cache rows it sees, its sequence, the sequence its prefix is read through, prefix rows)
__global__ void __launch_bounds__(256) k_paged_plan(PlanArgs a, int64_t rows_at) {
    int32_t * head = (int32_t *) a.ws;
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t == 0) { head[0] = PLAN_MAGIC; head[1] = a.n_rows; head[2] = a.n_head; head[3] = a.n_group; head[4] = a.n_seq; }
    if (t >= a.n_rows) return;
    int4 r = make_int4(0, 0, 0, 0);
    const int s = last_at_or_before(a.row_start, a.n_seq + 1, t);
    if (s >= 0 && s < a.n_seq) {
        const int r0 = a.row_start[s], m = a.row_start[s + 1] - r0, len = min(max(a.kv_len[s], 0), a.cap);
        r = make_int4(max(0, len - m + t - r0 + 1), s, s, 0);
        const int g = last_at_or_before(a.group_start, a.n_group + 1, s);
        if (g >= 0 && g < a.n_group) {
            r.z = min(max(a.group_start[g], 0), a.n_seq - 1);
            r.w = max(0, min(a.prefix_len[g], min(max(a.kv_len[r.z], 0), a.cap)));
        }
    }
    ((int4 *) (a.ws + rows_at))[t] = r;
}

struct PagedArgs {
    const void * k, * v;
    int64_t page_stride, qs, os, rows_at;
    const int32_t * table;
    int n_seq, table_len, n_pages, page_shift, nkv, n_head, n_rows, n_group;
    float scale;
    const void * q;
    void * out;
    uint8_t * ws;
};

// One (row, head) per block. 256 keys at a time: a key per thread for the scores, then a dim per thread for the values,
// with the running maximum and sum of the softmax.
template <int HD, typename T, typename TC>
__global__ void __launch_bounds__(256) k_paged_attn_row(PagedArgs a) {
    __shared__ float s_q[HD], s_p[256], s_red[8];
    const int32_t * head = (const int32_t *) a.ws;
    if (head[0] != PLAN_MAGIC || head[1] != a.n_rows || head[2] != a.n_head || head[3] != a.n_group || head[4] != a.n_seq) return;
    const int t = blockIdx.x, h = blockIdx.y, g = h / (a.n_head / a.nkv), tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int4 r = ((const int4 *) (a.ws + a.rows_at))[t];
    if (tid < HD) s_q[tid] = (float) ((const T *) a.q)[t * a.qs + (int64_t) h * HD + tid] * a.scale;
    float m = -__builtin_inff(), l = 0.0f, o = 0.0f;
    for (int k0 = 0; k0 < r.x; k0 += 256) {
        const int n = min(256, r.x - k0), key = k0 + tid;
        __syncthreads();
        float s = -__builtin_inff();
        if (tid < n) {
            const int page = max(0, z2o::page_of(a.table, a.n_seq, a.table_len, a.n_pages, a.page_shift, key < r.w ? r.z : r.y, key));
            const TC * kr = (const TC *) a.k + page * a.page_stride + (((int64_t) g << a.page_shift) + (key & ((1 << a.page_shift) - 1))) * HD;
            s = 0.0f;
            for (int d = 0; d < HD; ++d) s = __builtin_fmaf(s_q[d], (float) kr[d], s);
        }
        float mx = wave_max_f(s);
        if (lane == 0) s_red[wave] = mx;
        __syncthreads();
        mx = fmaxf(m, fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3])));
        const float p = tid < n ? z_expf(s - mx) : 0.0f, w = m == -__builtin_inff() ? 0.0f : z_expf(m - mx);
        const float ps = wave_tree_f(p);
        if (lane == 0) s_red[4 + wave] = ps;
        s_p[tid] = p;
        __syncthreads();
        l = l * w + ((s_red[4] + s_red[5]) + (s_red[6] + s_red[7]));
        m = mx;
        if (tid < HD) {
            o *= w;
            for (int i = 0; i < n; ++i) {
                const int ki = k0 + i;
                const int page = max(0, z2o::page_of(a.table, a.n_seq, a.table_len, a.n_pages, a.page_shift, ki < r.w ? r.z : r.y, ki));
                o = __builtin_fmaf(s_p[i], (float) ((const TC *) a.v)[page * a.page_stride + (((int64_t) g << a.page_shift) + (ki & ((1 << a.page_shift) - 1))) * HD + tid], o);
            }
        }
    }
    if (tid < HD) ((T *) a.out)[t * a.os + (int64_t) h * HD + tid] = (T) (l > 0.0f ? o / l : r.x > 0 ? o : 0.0f);
}

} // namespace z2d
