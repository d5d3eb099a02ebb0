// z2h_moe.h — a mixture-of-experts layer for a few rows on the caller's tensors: routing, the experts' gated products, their weighted sum.
//
//   p = softmax(logits), the top_k of p + bias, w = p (or p / sum), out = sum_j w_j down (silu(gate x) * (up x))
//   k_moe_gate_up   every block routes all rows for itself (a wave per row); h = silu(gate x) * (up x) of all routes, fp32
//   k_moe_down      out = sum over the row's experts of w down h
#pragma once
#include "z2h_common.h"
#include "z2h_ops_rules.h"
#include "z2h_tile.h"

namespace z2d {

struct MoeArgs {
    const void * gate, * up, * down;
    int E, F, D, n, k, renorm;
    const float * logits, * bias;
    const void * x;
    int64_t xs, os;
    void * out;
    int32_t * sel;
    float * weights;
    int32_t * routes;                                            // [n][k] experts, -1: none
    float * w;                                                   // [n][k]
    float * h;                                                   // [n][k][F]
};

// score order as integers: larger is later, NaN does not come here
__device__ __forceinline__ long long score_key(double s) {
    const long long b = __builtin_bit_cast(long long, s + 0.0);  // (no -0)
    return b < 0 ? b ^ 0x7fffffffffffffffll : b;
}
template <int CTRL>
__device__ __forceinline__ long long dpp_ll(long long v) {
    return ((long long) dpp_i<CTRL>((int) (v >> 32)) << 32) | (unsigned) dpp_i<CTRL>((int) v);
}
// the wave's largest value, in all lanes
__device__ __forceinline__ long long wave_max_ll(long long v) {
    auto up = [](long long a, long long b) { return a > b ? a : b; };
    v = up(v, ((long long) up32_i((int) (v >> 32)) << 32) | (unsigned) up32_i((int) v));
    v = up(v, ((long long) up16_i((int) (v >> 32)) << 32) | (unsigned) up16_i((int) v));
    v = up(v, dpp_ll<DPP_ROW_SHL + 8>(v));
    v = up(v, dpp_ll<DPP_ROW_SHL + 4>(v));
    v = up(v, dpp_ll<DPP_ROW_SHL + 2>(v));
    v = up(v, dpp_ll<DPP_ROW_SHL + 1>(v));
    return ((long long) __builtin_amdgcn_readlane((int) (v >> 32), 0) << 32) | (unsigned) __builtin_amdgcn_readlane((int) v, 0);
}

// One row's experts and weights by one wave, into sel and w [k]. Experts are told apart by p + bias in 64 bits, without a bias by the logits
// themselves (the same order, and equal ones are equal).
__device__ __forceinline__ void route_row(const MoeArgs & a, int row, short * sel, float * w) {
    const int lane = threadIdx.x & 63;
    const float * z = a.logits + (int64_t) row * a.E;
    float mx = -__builtin_inff();
    bool bad = false;
    for (int e = lane; e < a.E; e += 64) {
        const float v = z[e];
        bad |= !(v < __builtin_inff());
        mx = fmaxf(mx, v);
    }
    mx = wave_max_f(mx);
    float sum = 0.0f;
    const float m0 = mx == -__builtin_inff() ? 0.0f : mx;
    for (int e = lane; e < a.E; e += 64) sum += z_expf(z[e] - m0);
    sum = wave_tree_f(sum);
    if (a.bias)
        for (int e = lane; e < a.E; e += 64) bad |= a.bias[e] != a.bias[e];
    if (__any(bad)) {
        if (lane < a.k) { sel[lane] = -1; w[lane] = __builtin_nanf(""); }
        return;
    }
    const float inv = 1.0f / sum;
    constexpr long long NONE = -0x7fffffffffffffffll - 1;
    long long last = 0x7fffffffffffffffll;                       // what was taken last: later ones come behind it
    int last_e = -1, found = 0;
    float total = 0.0f, mine = 0.0f;
    short mine_e = -1;
    for (; found < a.k; ++found) {
        long long best = NONE;
        int best_e = 0;
        for (int e = lane; e < a.E; e += 64) {
            const float v = z[e];
            if (v == -__builtin_inff()) continue;
            const long long key = score_key(a.bias ? (double) (z_expf(v - m0) * inv) + (double) a.bias[e] : (double) v);
            const bool behind = key < last || (key == last && e > last_e);
            if (behind && key > best) { best = key; best_e = e; }
        }
        const long long top = wave_max_ll(best);
        if (top == NONE) break;
        int e = best == top ? best_e : 0x7fffffff;               // of equal ones the lowest
#pragma unroll
        for (int o = 32; o; o >>= 1) e = min(e, __shfl_xor(e, o));
        last = top; last_e = e;
        const float p = z_expf(z[e] - m0) * inv;
        total += p;
        if (lane == found) { mine = p; mine_e = (short) e; }
    }
    if (lane < a.k) {
        sel[lane] = mine_e;
        w[lane] = a.renorm && found ? mine / total : mine;
    }
}

template <typename T, typename TW>
__global__ void __launch_bounds__(256) k_moe_gate_up(MoeArgs a) {
    __shared__ short s_sel[Z2H_MOE_ROWS_MAX * z2o::MOE_MAX_TOP];
    __shared__ float s_w[Z2H_MOE_ROWS_MAX * z2o::MOE_MAX_TOP];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int r = wave; r < a.n; r += 4) route_row(a, r, s_sel + r * a.k, s_w + r * a.k);
    __syncthreads();
    const int routes = a.n * a.k;
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < routes; i += 256) {
            a.routes[i] = s_sel[i];
            a.w[i] = s_w[i];
            if (a.sel) a.sel[i] = s_sel[i];
            if (a.weights) a.weights[i] = s_w[i];
        }
    for (int64_t o = (int64_t) blockIdx.x * 4 + wave; o < (int64_t) routes * a.F; o += (int64_t) gridDim.x * 4) {
        const int route = (int) (o / a.F), f = (int) (o % a.F), e = s_sel[route];
        if (e < 0) continue;
        const TW * g = (const TW *) a.gate + ((int64_t) e * a.F + f) * a.D, * u = (const TW *) a.up + ((int64_t) e * a.F + f) * a.D;
        const T * x = (const T *) a.x + (route / a.k) * a.xs;
        float sg = 0.0f, su = 0.0f;
        for (int d = lane; d < a.D; d += 64) {
            const float v = (float) x[d];
            sg = __builtin_fmaf((float) g[d], v, sg);
            su = __builtin_fmaf((float) u[d], v, su);
        }
        sg = wave_tree_f(sg);
        su = wave_tree_f(su);
        if (lane == 0) a.h[(int64_t) route * a.F + f] = z_silu(sg) * su;
    }
}

template <typename T, typename TW>
__global__ void __launch_bounds__(256) k_moe_down(MoeArgs a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int64_t o = (int64_t) blockIdx.x * 4 + wave; o < (int64_t) a.n * a.D; o += (int64_t) gridDim.x * 4) {
        const int row = (int) (o / a.D), d = (int) (o % a.D);
        float y = 0.0f;
        for (int j = 0; j < a.k; ++j) {
            const int e = a.routes[row * a.k + j];
            const float w = a.w[row * a.k + j];
            if (e < 0) {
                if (w != w) y = w;
                continue;
            }
            const TW * p = (const TW *) a.down + ((int64_t) e * a.D + d) * a.F;
            const float * h = a.h + (int64_t) (row * a.k + j) * a.F;
            float s = 0.0f;
            for (int f = lane; f < a.F; f += 64) s = __builtin_fmaf((float) p[f], h[f], s);
            y = __builtin_fmaf(w, wave_tree_f(s), y);
        }
        if (lane == 0) ((T *) a.out)[row * a.os + d] = (T) y;
    }
}

} // namespace z2d
