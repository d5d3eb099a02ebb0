// z2h_prompt.h — causal attention of packed prompts over their own rows.
//
//   o_r = sum_{i <= r} p_i v_i / sum p_i,  p_i = 2^(x_i - m),  x_i = scale log2(e) q_r.k_i
#pragma once
#include "z2h_common.h"
#include "z2h_ops_rules.h"
#include "z2h_tile.h"

namespace z2d {

struct PromptArgs {
    const int32_t * start;
    int n_seq, n_rows, n_head, nkv;
    const void * q, * k, * v;
    int64_t qs, ks, vs, os;
    void * out;
    float scale;
    int64_t block0;
};

__device__ __forceinline__ int prompt_start(const PromptArgs & a, int s) { return min(max(a.start[s], 0), a.n_rows); }

// The sequence that slot `slot` of tiles of `rows` rows belongs to, by one wave: a step narrows 64 times.
__device__ __forceinline__ int prompt_seq(const PromptArgs & a, int64_t slot, int rows, int lane) {
    int lo = 0, n = a.n_seq;                                     // among lo .. lo + n - 1; the last that begins at or before the slot
    while (n > 1) {
        const int step = (n + 63) / 64, s = lo + lane * step;
        const bool before = lane * step < n && z2o::prompt_slot(prompt_start(a, s), s, rows) <= slot;
        const unsigned long long b = __ballot(before);
        const int last = b ? 63 - __builtin_clzll(b) : 0;
        n = min(step, n - last * step);
        lo += last * step;
    }
    return lo;
}

// A (row, head) in plain fp32, by one wave: 64 keys at a time, a lane each for the scores, then the dims over the lanes. A value that is
// not finite reaches the row whatever its weight. s_q: HD floats of the wave's own.
template <int HD, typename T, int E>
__device__ __forceinline__ void prompt_walk(const PromptArgs & a, int first, int row, int head, float * s_q, float (&o)[E], float & l) {
    const int lane = threadIdx.x & 63, g = head / (a.n_head / a.nkv), d = E * lane;
    const T * src = (const T *) a.q + row * a.qs + (int64_t) head * HD;
    float mx = 0.0f;
    for (int i = lane; i < HD; i += 64) mx = fmaxf(mx, fabsf((float) src[i]));
    mx = wave_max_f(mx);
    int up = 0;                                                  // (a power of two keeps the scores of large queries finite)
    if (mx > 0.0f && mx < __builtin_inff()) (void) frexpf(mx, &up);
    up = max(up, -120);
    for (int i = lane; i < HD; i += 64) s_q[i] = a.scale == 0.0f ? 0.0f : ldexpf((float) src[i], -up);
    wait_lds();
    const float c = copysignf(fminf(ldexpf(fabsf(a.scale) * 1.44269504088896341f, up), 0x1p127f), a.scale);
    float m = -__builtin_inff();
    l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.0f;
    const T * kb = (const T *) a.k + (int64_t) g * HD, * vb = (const T *) a.v + (int64_t) g * HD;
    for (int key0 = first; key0 <= row; key0 += 64) {
        const T * k = kb + min(key0 + lane, row) * a.ks;
        float x[4] = {};
#pragma unroll 2
        for (int i = 0; i < HD / 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = __builtin_fmaf(s_q[4 * i + j], (float) k[4 * i + j], x[j]);
        float s = ((x[0] + x[1]) + (x[2] + x[3])) * c;
        if (key0 + lane > row) s = -__builtin_inff();
        if (__any(!(s < __builtin_inff()))) {                    // infinity or no number: nor is any weight a number
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = __builtin_nanf("");
            l = 1.0f;
            return;
        }
        const float mn = fmaxf(m, wave_max_f(s));
        const float w0 = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
        const float w = s == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(s - mn);
        m = mn;
        l = l * w0 + wave_tree_f(w);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = is_finite(o[e]) ? o[e] * w0 : o[e];
        const int n = min(64, row + 1 - key0);
        const bool weighs = s > -__builtin_inff();
        const unsigned long long live = __ballot(weighs);
        for (int i0 = 0; i0 < n; i0 += 4) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int i = min(i0 + u, n - 1);
                const float wi = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), i));
                if (i0 + u >= n || !(live >> i & 1)) continue;   // (a key without weight has none whatever its value)
                const T * v = vb + (key0 + i) * a.vs + d;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float y = d < HD ? (float) v[e] : 0.0f;
                    o[e] = is_finite(y) ? __builtin_fmaf(wi, y, o[e]) : o[e] + y;
                }
            }
        }
    }
}

template <int HD, typename T>
__global__ void __launch_bounds__(256) k_prompt_walk(PromptArgs a) {
    __shared__ float s_q[4][HD];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t id = (a.block0 + blockIdx.x) * 4 + wave;
    if (id >= (int64_t) a.n_rows * a.n_head) return;
    const int row = (int) (id / a.n_head), head = (int) (id % a.n_head);
    // (the sequence by a search over the table, one row at a time)
    int lo = -1, hi = a.n_seq;
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (prompt_start(a, m) <= row) lo = m; else hi = m;
    }
    if (lo < 0 || row >= prompt_start(a, lo + 1)) return;
    constexpr int E = HD >= 64 ? HD / 64 : 1;
    float o[E], l;
    prompt_walk<HD, T>(a, prompt_start(a, lo), row, head, s_q[wave], o, l);
    T * out = (T *) a.out + row * a.os + (int64_t) head * HD + E * lane;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (E * lane < HD)
#pragma unroll
        for (int e = 0; e < E; ++e) out[e] = (T) (o[e] * inv);
}

} // namespace z2d
