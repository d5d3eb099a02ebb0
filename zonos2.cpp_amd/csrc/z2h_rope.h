// z2h_rope.h — rotary positions of rows of heads, and appending rotated rows to a paged cache.
#pragma once
#include "z2h_common.h"
#include "z2h_ops_rules.h"

namespace z2d {

// cos and sin of `turn` turns (any double): reduced to the nearest quarter turn in 64 bits, then the Taylor polynomials
// of z_sincos on [-pi/4, pi/4].
__device__ __forceinline__ void turn_sincos(double turn, float & s, float & c) {
    const double f = turn - rint(turn);
    const double q = rint(4.0 * f);
    const float r = (float) ((f - 0.25 * q) * 6.28318530717958647692);
    const float r2 = r * r;
    float sp = 2.75573192e-6f;                                           // 1/9!
    sp = __builtin_fmaf(sp, r2, -1.98412698e-4f);
    sp = __builtin_fmaf(sp, r2, 8.33333333e-3f);
    sp = __builtin_fmaf(sp, r2, -1.66666667e-1f);
    const float sr = __builtin_fmaf(sp * r2, r, r);
    float cp = 2.48015873e-5f;                                           // 1/8!
    cp = __builtin_fmaf(cp, r2, -1.38888889e-3f);
    cp = __builtin_fmaf(cp, r2, 4.16666667e-2f);
    cp = __builtin_fmaf(cp, r2, -0.5f);
    const float cr = __builtin_fmaf(cp, r2, 1.0f);
    const int qi = ((int) q) & 3;
    s = qi == 0 ? sr : qi == 1 ? cr : qi == 2 ? -sr : -cr;
    c = qi == 0 ? cr : qi == 1 ? -sr : qi == 2 ? -cr : sr;
}

struct RopeArgs {
    double turn[z2o::MAX_ROPE_DIMS / 2];           // turns per position of each pair
    float mscale;
    int n_dims, hd, nh, nkv;
    const int32_t * seq, * pos;                    // seq NULL: rows of queries only
    const void * q, * k, * v;
    void * q_out, * kc, * vc;
    int64_t qs, qos, ks, vs, page_stride;
    const int32_t * table;
    int n_seq, table_len, n_pages, page_shift;
};

// One row per block: its pairs' cos and sin once, then every head. Pairs (and the dims behind them) over the threads.
template <typename T, typename TC, bool HALVES>
__global__ void __launch_bounds__(256) k_rope_append(RopeArgs a) {
    const int t = blockIdx.x, tid = threadIdx.x;
    const int seq = a.seq ? a.seq[t] : 0;
    if (a.seq && (seq < 0 || seq >= a.n_seq)) return;
    const int pos = a.pos[t], np = a.n_dims / 2, rest = a.hd - a.n_dims, U = np + rest, HL = 256 / U;
    const int u = tid % U, hl = tid / U;
    if (hl >= HL) return;
    int page = -1;
    if (a.k) page = z2o::page_of(a.table, a.n_seq, a.table_len, a.n_pages, a.page_shift, seq, pos);
    const int64_t cell = page < 0 ? 0 : page * a.page_stride + (int64_t) (pos & ((1 << a.page_shift) - 1)) * a.hd;
    const int64_t head_step = (int64_t) a.hd << a.page_shift;
    float c = 0.0f, s = 0.0f;
    const bool pair = u < np;
    if (pair) {
        turn_sincos((double) pos * a.turn[u], s, c);
        c *= a.mscale; s *= a.mscale;
    }
    const int i0 = pair ? (HALVES ? u : 2 * u) : a.n_dims + u - np, i1 = pair ? (HALVES ? u + np : 2 * u + 1) : i0;
    for (int h = hl; h < a.nh; h += HL) {
        const T * x = (const T *) a.q + t * a.qs + (int64_t) h * a.hd;
        T * y = (T *) a.q_out + t * a.qos + (int64_t) h * a.hd;
        const float x0 = (float) x[i0], x1 = (float) x[i1];
        if (!pair) y[i0] = (T) x0;
        else {
            y[i0] = (T) (x0 * c - x1 * s);
            y[i1] = (T) (x0 * s + x1 * c);
        }
    }
    if (page < 0) return;
    for (int g = hl; g < a.nkv; g += HL) {
        const T * x = (const T *) a.k + t * a.ks + (int64_t) g * a.hd, * v = (const T *) a.v + t * a.vs + (int64_t) g * a.hd;
        TC * y = (TC *) a.kc + cell + g * head_step, * w = (TC *) a.vc + cell + g * head_step;
        const float x0 = (float) x[i0], x1 = (float) x[i1];
        if (!pair) { y[i0] = (TC) x0; w[i0] = (TC) (float) v[i0]; }
        else {
            y[i0] = (TC) (x0 * c - x1 * s);
            y[i1] = (TC) (x0 * s + x1 * c);
            w[i0] = (TC) (float) v[i0];
            w[i1] = (TC) (float) v[i1];
        }
    }
}

} // namespace z2d
