// z2h_verify.h — verification of drafted frames against the target's probabilities.
#pragma once
#include "z2h_common.h"
#include "z2h_ops_rules.h"

namespace z2d {

struct VerifyArgs {
    int n_seq, K, C, V;
    const int32_t * draft, * n_draft;
    const float * target, * temperature, * draft_probs;
    const double * u_accept, * u_draw;
    int32_t * n_accept, * codes;
    double * stats;                                // [row][2]: largest logit, mass over it
};

// the mass of a code whose logit is x in a row whose largest is mx (temperature > 0), or its probability
__device__ __forceinline__ double code_mass(float x, bool logits, double mx, double T) {
    return logits ? z_exp_d(((double) x - mx) / T) : (double) x;
}

// Of each logits row, one block: its largest logit and the sum of exp((x - largest) / temperature).
__global__ void __launch_bounds__(256) k_verify_stats(VerifyArgs a) {
    __shared__ double s_w[4];
    const int64_t row = blockIdx.x;
    const int s = (int) (row / ((int64_t) (a.K + 1) * a.C)), tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float * x = a.target + row * a.V;
    const double T = a.temperature[s];
    float mx = -__builtin_inff();
    for (int i = tid; i < a.V; i += 256) mx = fmaxf(mx, x[i]);
    mx = wave_max_f(mx);
    if (lane == 0) s_w[wave] = mx;
    __syncthreads();
    const double m = fmax(fmax(s_w[0], s_w[1]), fmax(s_w[2], s_w[3]));
    __syncthreads();
    double z = 0.0;
    if (T > 0.0) for (int i = tid; i < a.V; i += 256) z += z_exp_d(((double) x[i] - m) / T);
    z = wave_tree_d(z);
    if (lane == 0) s_w[wave] = z;
    __syncthreads();
    if (tid == 0) { a.stats[2 * row] = m; a.stats[2 * row + 1] = (s_w[0] + s_w[1]) + (s_w[2] + s_w[3]); }
}

// One block per (sequence, codebook): the first code that is not kept, then this codebook's code of the frame behind.
__global__ void __launch_bounds__(256) k_verify(VerifyArgs a) {
    extern __shared__ double s_piece[];            // mass of every 256 codes
    __shared__ int s_first, s_pick;
    __shared__ double s_tot;
    const int s = blockIdx.x / a.C, cb = blockIdx.x % a.C, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const bool logits = a.temperature != nullptr;
    const double T = logits ? a.temperature[s] : 1.0;
    const bool greedy = logits && !(T > 0.0);
    const int nd = a.n_draft ? min(max(a.n_draft[s], 0), a.K) : a.K, n_code = nd * a.C;
    const int64_t row0 = (int64_t) s * (a.K + 1) * a.C, d0 = (int64_t) s * a.K * a.C;
    if (tid == 0) s_first = n_code;
    __syncthreads();
    // the first of the row's largest logits, for greedy rows
    auto first_max = [&](int64_t row) {
        const float * x = a.target + row * a.V;
        for (int i = 0; i < a.V; ++i) if ((double) x[i] == a.stats[2 * row]) return i;
        return 0;
    };
    for (int j = tid; j < n_code; j += 256) {
        const int x = a.draft[d0 + j];
        const int64_t row = row0 + j;
        bool keep = x >= 0 && x < a.V;
        if (keep) {
            const double u = a.u_accept[d0 + j], q = a.draft_probs ? (double) a.draft_probs[(d0 + j) * a.V + x] : 1.0;
            if (greedy) keep = x == first_max(row) && u * q < 1.0;
            else if (logits) keep = u * q < code_mass(a.target[row * a.V + x], true, a.stats[2 * row], T) / a.stats[2 * row + 1];
            else keep = u * q < (double) a.target[row * a.V + x];
        }
        if (!keep) atomicMin(&s_first, j);
    }
    __syncthreads();
    const int first = s_first, k = first / a.C, c = first % a.C;
    const bool rejected = first < n_code;
    if (cb == 0 && tid == 0) a.n_accept[s] = k;
    if (rejected && cb < c) {
        if (tid == 0) a.codes[(int64_t) s * a.C + cb] = a.draft[d0 + (int64_t) k * a.C + cb];
        return;
    }
    const int64_t row = row0 + (int64_t) k * a.C + cb;
    const float * x = a.target + row * a.V;
    const double mx = logits ? a.stats[2 * row] : 0.0, Z = logits ? a.stats[2 * row + 1] : 1.0;
    const int best = greedy ? first_max(row) : 0;
    const int drafted = rejected ? a.draft[d0 + first] : -1;
    const float * qr = a.draft_probs && rejected ? a.draft_probs + (d0 + first) * a.V : nullptr;
    const int n_piece = (a.V + 255) / 256;
    for (int pass = rejected && cb == c ? 0 : 1; pass < 2; ++pass) {
        auto mass = [&](int i) {
            if (i >= a.V) return 0.0;
            double p = greedy ? (i == best ? 1.0 : 0.0) : code_mass(x[i], logits, mx, T) / Z;
            if (pass == 0) { p -= qr ? (double) qr[i] : i == drafted ? 1.0 : 0.0; p = p > 0.0 ? p : 0.0; }
            return p;
        };
        __syncthreads();
        for (int b = wave; b < n_piece; b += 4) {
            double w = 0.0;
            for (int e = 0; e < 4; ++e) w += mass(256 * b + 4 * lane + e);
            w = wave_tree_d(w);
            if (lane == 0) s_piece[b] = w;
        }
        __syncthreads();
        if (tid == 0) {
            double tot = 0.0, cum = 0.0;
            for (int b = 0; b < n_piece; ++b) tot += s_piece[b];
            const double want = a.u_draw[(int64_t) s * a.C + cb] * tot;
            int b = 0, last = 0;
            for (; b < n_piece; ++b) { if (s_piece[b] > 0.0) last = b; if (cum + s_piece[b] > want) break; cum += s_piece[b]; }
            const bool none = b == n_piece;          // rounding left no crossing: the last code with mass
            if (none) b = last;
            int pick = -1, lastc = 256 * b;
            for (int i = 256 * b; i < min(a.V, 256 * b + 256); ++i) {
                const double w = mass(i);
                if (w > 0.0) lastc = i;
                cum += w;
                if (!none && cum > want) { pick = i; break; }
            }
            s_pick = pick >= 0 ? pick : lastc;
            s_tot = tot;
        }
        __syncthreads();
        if (s_tot > 0.0 || pass == 1) break;
    }
    if (tid == 0) a.codes[(int64_t) s * a.C + cb] = s_pick;
}

} // namespace z2d
