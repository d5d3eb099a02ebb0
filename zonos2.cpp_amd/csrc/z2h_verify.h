// z2h_verify.h — verification of drafted frames against the target's probabilities.
//
// The codes of a sequence's drafts are tested independently (u q(x) < p(x)); the first that fails decides which row each
// codebook is drawn from, so every block finds it for itself from the handful of values it takes, and no launch waits for
// another's verdict. A draw needs the mass of a row twice, whole and up to the code: masses are summed in pieces of 256
// codes, the piece is found by a scan of the piece sums and the code by a scan of the piece. Everything is in 64 bits (an
// exponential there is about 25 instructions at the full rate), so that draws are those of the definition; sums are formed
// in a fixed order.
//   k_verify_stats   logits: a row's largest logit, its first place, and the mass over it
//   k_verify         rows of at most VERIFY_ONE codes: the verdict and the draw, one block per (sequence, codebook)
//   k_verify_sums / k_verify_pick   longer rows: piece sums by several blocks per row, then the draw
// Bound by reading the rows once and their exponentials where there are many codes, by the dependent loads of a verdict where
// there are few. Measured: 16 sequences x 4 frames x 9 codebooks of 1025 logits (3 MB) 5.5 + 8.8 us; 64 x 5 x 1 of 32000 probabilities
// 8.6 + 4.2 us (the row of each draw alone is read whole, 16 MB); 8 x 7 x 1 of 131072 logits (38 MB) 15.6 + 12.2 + 4.9 us: the
// first as long for its 8 million exponentials as for their loads.
#pragma once
#include "z2h_common.h"
#include "z2h_ops_rules.h"

namespace z2d {

struct VerifyStat { double max, mass; int64_t first; };          // of a chunk of a row
static_assert(sizeof(VerifyStat) == z2o::VERIFY_STAT_BYTES, "workspace layout");

struct VerifyDraw { int first, n_code; VerifyStat st; };         // a verdict and the numbers of the row that follows from it
static_assert(sizeof(VerifyDraw) == z2o::VERIFY_DRAW_BYTES, "workspace layout");

struct VerifyArgs {
    int n_seq, K, C, V, n_chunk, n_share;
    int64_t block0;                                              // of this launch of k_verify_stats
    const int32_t * draft, * n_draft;
    const float * target, * temperature, * draft_probs;
    const double * u_accept, * u_draw;
    int32_t * n_accept, * codes;
    VerifyStat * stats;                                          // [row][n_chunk]
    VerifyDraw * draws;                                          // [sequence][codebook]
    double * sums;                                               // [sequence][codebook][piece]
};

// exp(x) for x in [-708, 0]: z_exp_d's reduction and polynomial, with the whole part rounded in 32 bits and put into the
// exponent by an integer add (64-bit rounding and scaling instructions take four times as long as a 64-bit fma).
__device__ __forceinline__ double exp_core(double x) {
    const float nf = rintf((float) x * 1.44269504f);
    const double n = (double) nf;
    double r = __builtin_fma(-n, 0x1.62e42fee00000p-1, x);
    r = __builtin_fma(-n, 0x1.a39ef35793c76p-33, r);
    double p = 0x1.6124613a86d09p-33;                                    // 1/13!
    p = __builtin_fma(p, r, 0x1.1eed8eff8d898p-29);
    p = __builtin_fma(p, r, 0x1.ae64567f544e4p-26);
    p = __builtin_fma(p, r, 0x1.27e4fb7789f5cp-22);
    p = __builtin_fma(p, r, 0x1.71de3a556c734p-19);
    p = __builtin_fma(p, r, 0x1.a01a01a01a01ap-16);
    p = __builtin_fma(p, r, 0x1.a01a01a01a01ap-13);
    p = __builtin_fma(p, r, 0x1.6c16c16c16c17p-10);
    p = __builtin_fma(p, r, 0x1.1111111111111p-7);
    p = __builtin_fma(p, r, 0x1.5555555555555p-5);
    p = __builtin_fma(p, r, 0x1.5555555555555p-3);
    p = __builtin_fma(p, r, 0.5);
    p = __builtin_fma(p, r, 1.0);
    p = __builtin_fma(p, r, 1.0);
    const uint64_t b = __builtin_bit_cast(uint64_t, p) + ((uint64_t) (uint32_t) (int) nf << 52);
    return __builtin_bit_cast(double, b);
}
// exp(x) for x <= 0; 0 below -700 (z_exp_d is under 1e-304 there) and for what is no number
__device__ __forceinline__ double exp_mass(double x) {
    const double e = exp_core(fmax(x, -708.0));
    return x >= -700.0 ? e : 0.0;
}

// sum over the lanes up to this one
__device__ __forceinline__ double wave_scan_d(double v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double y = __shfl_up(v, o);
        if (lane >= o) v += y;
    }
    return v;
}

// One block of NT threads per (row, chunk): NT x 32 logits of a row, all requested before the first is used.
template <int NT>
__global__ void __launch_bounds__(NT) k_verify_stats(VerifyArgs a) {
    constexpr int NW = NT / 64, N = z2o::VERIFY_PER_THREAD;
    __shared__ double s_m[NW], s_z[NW];
    __shared__ int s_i[NW];
    const int id = (int) (a.block0 + blockIdx.x);
    const int64_t row = id / a.n_chunk;
    const int chunk = id % a.n_chunk;
    const int s = (int) (row / ((int64_t) (a.K + 1) * a.C)), k = (int) (row / a.C % (a.K + 1));
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c0 = chunk * NT * N;
    if (a.n_draft && k > min(max(a.n_draft[s], 0), a.K)) return;           // behind the last draft's successor
    const int n = min(NT * N, a.V - c0);
    const float * x = a.target + row * a.V + c0;
    const double T = a.temperature[s];
    float v[N], m = -__builtin_inff();
    // rows much shorter than a chunk take one round of it
    const int rounds = (n + 8 * NT - 1) / (8 * NT);
    // value e of round r is logit `place(r, e)`: long rows are read 16 bytes at a time
    auto place = [&](int r, int e) { return NT == 256 ? tid + NT * (8 * r + e) : 4 * (tid + NT * (2 * r + e / 4)) + e % 4; };
    const bool wide = NT > 256 && ((uintptr_t) x & 15) == 0 && n % 4 == 0;
#pragma unroll
    for (int r = 0; r < N / 8; ++r)
        if (r < rounds) {
            if (wide) {
#pragma unroll
                for (int e = 0; e < 8; e += 4) {
                    const int i = place(r, e);
                    const float4 y = i < n ? *(const float4 *) (x + i) : make_float4(m, m, m, m);
                    v[8 * r + e] = y.x; v[8 * r + e + 1] = y.y; v[8 * r + e + 2] = y.z; v[8 * r + e + 3] = y.w;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int i = place(r, e);
                    v[8 * r + e] = i < n ? x[i] : -__builtin_inff();
                }
            }
        }
    // Each thread on its own, eight logits at a time as they come in: its largest, and its mass over it.
    const double inv = 1.0 / T;
    double z = 0.0;
#pragma unroll
    for (int r = 0; r < N / 8; ++r)
        if (r < rounds) {
            float mr = m;
#pragma unroll
            for (int e = 0; e < 8; ++e) mr = fmaxf(mr, v[8 * r + e]);
            if (T > 0.0) {
                const double md = mr;
                z = r ? z * exp_mass(((double) m - md) * inv) : 0.0;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    // (hidden codes and the places behind the row's end add e^-708)
                    z += exp_core(fmax(((double) v[8 * r + e] - md) * inv, -708.0));
                }
            }
            m = mr;
        }
    const float wm = wave_max_f(m);
    int at = 0x7fffffff;
    if (!(T > 0.0)) {                                            // all mass on the first of the largest
#pragma unroll
        for (int r = 0; r < N / 8; ++r)
            if (r < rounds)
#pragma unroll
                for (int e = 0; e < 8; ++e) if (v[8 * r + e] == wm) at = min(at, place(r, e));
#pragma unroll
        for (int o = 32; o; o >>= 1) at = min(at, __shfl_xor(at, o));
    }
    if (lane == 0) { s_m[wave] = wm; s_i[wave] = at; }
    __syncthreads();
    double mx = s_m[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) mx = fmax(mx, s_m[w]);
    z = wave_tree_d(z * exp_mass(((double) m - mx) * inv));
    if (lane == 0) s_z[wave] = z;
    __syncthreads();
    if (tid == 0) {
        int first = 0x7fffffff;
        double mass = 0.0;
        for (int w = 0; w < NW; ++w) {
            if (s_m[w] == mx) first = min(first, s_i[w]);
            mass += s_z[w];
        }
        a.stats[row * a.n_chunk + chunk] = VerifyStat{mx, mass, c0 + (int64_t) (first < n ? first : 0)};
    }
}

// a whole row's numbers from its chunks' (eight at a time in flight)
__device__ __forceinline__ VerifyStat row_stat(const VerifyArgs & a, int64_t row, double T) {
    const VerifyStat * s = a.stats + row * a.n_chunk;
    if (a.n_chunk == 1) return s[0];
    VerifyStat r{-__builtin_inf(), 0.0, 0};
    constexpr int M = 8;
    const double inv = 1.0 / T;
    for (int c0 = 0; c0 < a.n_chunk; c0 += M) {
        VerifyStat t[M];
#pragma unroll
        for (int u = 0; u < M; ++u) t[u] = s[min(c0 + u, a.n_chunk - 1)];
        double m = r.max;
#pragma unroll
        for (int u = 0; u < M; ++u) if (t[u].max > m) { m = t[u].max; r.first = t[u].first; }
        if (T > 0.0) {
            double z = c0 ? r.mass * exp_mass((r.max - m) * inv) : 0.0;
#pragma unroll
            for (int u = 0; u < M; ++u) z += c0 + u < a.n_chunk ? t[u].mass * exp_mass((t[u].max - m) * inv) : 0.0;
            r.mass = z;
        }
        r.max = m;
    }
    return r;
}

// One (sequence, codebook): the verdict, and the masses of the row its code is drawn from.
struct VerifyRow {
    const float * x, * q;              // target row; draft row whose mass is taken off (or null)
    VerifyStat st;
    double inv_T, inv_mass;
    int V, drafted;                    // drafted: the code of all the draft's mass, where q is null (-1: none)
    bool logits, greedy, rest;

    // mass of code i, whose target value is x and whose draft probability is qi
    __device__ __forceinline__ double mass(int i, float xi, float qi, bool off) const {
        double p = greedy ? (i == st.first ? 1.0 : 0.0) : logits ? exp_mass(((double) xi - st.max) * inv_T) * inv_mass : (double) xi;
        if (off) { p -= q ? (double) qi : i == drafted ? 1.0 : 0.0; p = p > 0.0 ? p : 0.0; }
        return p;
    }
    __device__ __forceinline__ double mass_at(int i, bool off) const { return i < V ? mass(i, x[i], q && off ? q[i] : 0.0f, off) : 0.0; }
    // sum over piece b's 256 codes, by a wave
    // (pieces n >= live are left out)
    template <int NB>
    __device__ __forceinline__ void pieces(const int (&b)[NB], int live, bool off, double (&sum)[NB]) const {
        const int lane = threadIdx.x & 63;
        float xv[NB][4], qv[NB][4];
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = 256 * b[n] + 64 * e + lane, j = i < V ? i : V - 1;
                xv[n][e] = x[j];
                qv[n][e] = q && off ? q[j] : 0.0f;
            }
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            if (n >= live) break;
            double w = 0.0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = 256 * b[n] + 64 * e + lane;
                const double p = mass(i, xv[n][e], qv[n][e], off);
                w += i < V ? p : 0.0;
            }
            sum[n] = wave_tree_d(w);
        }
    }
};

__device__ __forceinline__ int verify_codes(const VerifyArgs & a, int s) { return (a.n_draft ? min(max(a.n_draft[s], 0), a.K) : a.K) * a.C; }

// The block's verdict on a sequence: the index of the first code that is not kept (or of the code behind the last).
// A thread's values are requested before the number of drafts is known: the buffers hold all K.
constexpr int KEPT_STATS = 256;
struct Verdict { int first; VerifyStat stat[KEPT_STATS]; };        // of code j's row, those of the frame behind the drafts too
__device__ __forceinline__ int verify_first(const VerifyArgs & a, int s, int & n_code, Verdict & o) {
    const bool logits = a.temperature != nullptr;
    const double T = logits ? (double) a.temperature[s] : 1.0;
    const bool greedy = logits && !(T > 0.0);
    const int64_t row0 = (int64_t) s * (a.K + 1) * a.C, d0 = (int64_t) s * a.K * a.C;
    if (threadIdx.x == 0) o.first = 0x7fffffff;
    n_code = verify_codes(a, s);
    __syncthreads();
    const int all = a.K * a.C;
    for (int j = threadIdx.x; j < all + a.C; j += blockDim.x) {
        const int jd = min(j, all - 1), x = all ? a.draft[d0 + jd] : 0, xc = min(max(x, 0), a.V - 1);
        const double u = all ? a.u_accept[d0 + jd] : 0.0;
        if (j >= n_code) {
            if (logits && j < n_code + a.C && j < KEPT_STATS) o.stat[j] = row_stat(a, row0 + j, T);
            break;
        }
        const double q = a.draft_probs ? (double) a.draft_probs[(d0 + j) * a.V + xc] : 1.0;
        const float t = a.target[(row0 + j) * a.V + xc];
        double p = t;
        if (logits) {
            const VerifyStat st = row_stat(a, row0 + j, T);
            if (j < KEPT_STATS) o.stat[j] = st;
            p = greedy ? (x == st.first ? 1.0 : 0.0) : exp_mass(((double) t - st.max) * (1.0 / T)) / st.mass;
        }
        if (!(x == xc && u * q < p)) atomicMin(&o.first, j);
    }
    __syncthreads();
    return min(o.first, n_code);
}

__device__ __forceinline__ const VerifyStat * kept_stat(const VerifyArgs & a, const Verdict & v, int first, int cb) {
    const int j = first / a.C * a.C + cb;
    return j < KEPT_STATS ? &v.stat[j] : nullptr;
}

// false: the code is the draft's own (taken over here)
__device__ __forceinline__ bool verify_row(const VerifyArgs & a, int s, int cb, int first, int n_code, const VerifyStat * st, bool write, VerifyRow & r) {
    const int k = first / a.C, c = first % a.C;
    const bool rejected = first < n_code;
    const int64_t d0 = (int64_t) s * a.K * a.C;
    if (write && cb == 0 && threadIdx.x == 0) a.n_accept[s] = k;
    if (rejected && cb < c) {
        if (write && threadIdx.x == 0) a.codes[(int64_t) s * a.C + cb] = a.draft[d0 + (int64_t) k * a.C + cb];
        return false;
    }
    const int64_t row = ((int64_t) s * (a.K + 1) + k) * a.C + cb;
    r.logits = a.temperature != nullptr;
    const double T = r.logits ? (double) a.temperature[s] : 1.0;
    r.greedy = r.logits && !(T > 0.0);
    r.inv_T = 1.0 / T;
    r.x = a.target + row * a.V;
    r.V = a.V;
    r.rest = rejected && cb == c;
    r.q = r.rest && a.draft_probs ? a.draft_probs + (d0 + first) * a.V : nullptr;
    r.drafted = r.rest ? a.draft[d0 + first] : -1;
    if (r.logits) { r.st = st ? *st : row_stat(a, row, T); r.inv_mass = 1.0 / r.st.mass; }
    return true;
}

// piece sums of a row over the waves of the block: pieces [b0, b1) to out[b]
__device__ __forceinline__ void row_pieces(const VerifyRow & r, bool off, int b0, int b1, double * out) {
    constexpr int NB = 4, NW = 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int b = __builtin_amdgcn_readfirstlane(b0 + wave); b < b1; b += NB * NW) {
        int at[NB];
        double sum[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) at[n] = min(b + n * NW, b1 - 1);
        r.template pieces<NB>(at, (b1 - b + NW - 1) / NW, off, sum);
#pragma unroll
        for (int n = 0; n < NB; ++n)
            if (lane == 0 && b + n * NW < b1) out[b + n * NW] = sum[n];
    }
}

// by one wave: the code that u draws from a row's masses, given its piece sums; -1 where the row has no mass
__device__ __forceinline__ int pick_code(const VerifyRow & r, bool off, const double * sum, int n_piece, double u) {
    const int lane = threadIdx.x & 63;
    // a run of pieces per lane; the run, then the piece in it
    const int per = (n_piece + 63) / 64, p0 = per * lane, p1 = min(n_piece, p0 + per);
    double own_run = 0.0;
    for (int b = p0; b < p1; b += 8) {
        double t[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = b + e < p1 ? sum[b + e] : 0.0;
#pragma unroll
        for (int e = 0; e < 8; ++e) own_run += t[e];
    }
    const double runs = wave_scan_d(own_run), total = __shfl(runs, 63);
    if (!(total > 0.0)) return -1;
    const double want = u * total;
    const uint64_t over = __ballot(own_run > 0.0 && runs > want), some = __ballot(own_run > 0.0);
    const bool none = over == 0;                                 // rounding left no crossing: the last code with mass
    const int l = none ? 63 - __builtin_clzll(some) : __ffsll((unsigned long long) over) - 1;
    double base = l > 0 ? __shfl(runs, max(l - 1, 0)) : 0.0;
    const int q0 = per * l, nq = min(n_piece, q0 + per) - q0;    // at most 64 pieces
    const double ws = lane < nq ? sum[q0 + lane] : 0.0, cum_p = wave_scan_d(ws);
    const uint64_t over_p = __ballot(ws > 0.0 && base + cum_p > want), some_p = __ballot(ws > 0.0);
    const bool none_p = none || over_p == 0;
    const int lp = none_p ? 63 - __builtin_clzll(some_p | 1) : __ffsll((unsigned long long) over_p) - 1;
    base += lp > 0 ? __shfl(cum_p, max(lp - 1, 0)) : 0.0;
    const int piece = q0 + lp;
    double w[4], own = 0.0;
#pragma unroll
    for (int e = 0; e < 4; ++e) { w[e] = r.mass_at(256 * piece + 4 * lane + e, off); own += w[e]; }
    const double cum = wave_scan_d(own);
    double run = base + (cum - own);
    int hit = 0x7fffffff, end = -1;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        run += w[e];
        if (w[e] > 0.0) {
            end = 256 * piece + 4 * lane + e;
            if (!none_p && run > want) hit = min(hit, end);
        }
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) { hit = min(hit, __shfl_xor(hit, o)); end = max(end, __shfl_xor(end, o)); }
    return hit != 0x7fffffff ? hit : end;
}

__global__ void __launch_bounds__(256) k_verify(VerifyArgs a) {
    __shared__ double s_sum[z2o::VERIFY_ONE / 256];
    __shared__ Verdict s_v;
    __shared__ int s_none;
    const int s = blockIdx.x / a.C, cb = blockIdx.x % a.C, n_piece = (a.V + 255) / 256;
    int n_code;
    const int first = verify_first(a, s, n_code, s_v);
    VerifyRow r{};
    if (!verify_row(a, s, cb, first, n_code, kept_stat(a, s_v, first, cb), true, r)) return;
    const int64_t at = (int64_t) s * a.C + cb;
    for (bool off = r.rest;; off = false) {
        row_pieces(r, off, 0, n_piece, s_sum);
        __syncthreads();
        if (threadIdx.x < 64) {
            const int code = pick_code(r, off, s_sum, n_piece, a.u_draw[at]);
            if (threadIdx.x == 0) {
                s_none = code < 0;
                a.codes[at] = max(code, 0);
            }
        }
        __syncthreads();
        if (!off || !s_none) break;                              // no mass in the rest: from p itself
    }
}

// One block per (sequence, codebook, share of the row's pieces).
__global__ void __launch_bounds__(256) k_verify_sums(VerifyArgs a) {
    __shared__ Verdict s_v;
    const int draw = blockIdx.x / a.n_share, share = blockIdx.x % a.n_share, s = draw / a.C, cb = draw % a.C, n_piece = (a.V + 255) / 256;
    int n_code;
    const int first = verify_first(a, s, n_code, s_v);
    VerifyRow r{};
    if (!verify_row(a, s, cb, first, n_code, kept_stat(a, s_v, first, cb), false, r)) {
        if (share == 0 && threadIdx.x == 0) a.draws[draw] = VerifyDraw{first, n_code, VerifyStat{}};
        return;
    }
    if (share == 0 && threadIdx.x == 0) a.draws[draw] = VerifyDraw{first, n_code, r.st};
    const int per = (n_piece + a.n_share - 1) / a.n_share, b0 = share * per;
    row_pieces(r, r.rest, b0, min(n_piece, b0 + per), a.sums + (int64_t) draw * n_piece);
}

__global__ void __launch_bounds__(256) k_verify_pick(VerifyArgs a) {
    __shared__ int s_none;
    const int s = blockIdx.x / a.C, cb = blockIdx.x % a.C, n_piece = (a.V + 255) / 256;
    const VerifyDraw v = a.draws[blockIdx.x];
    VerifyRow r{};
    if (!verify_row(a, s, cb, v.first, v.n_code, &v.st, true, r)) return;
    const int64_t at = (int64_t) s * a.C + cb;
    double * sum = a.sums + at * n_piece;
    for (bool off = r.rest;; off = false) {
        if (threadIdx.x < 64) {
            const int code = pick_code(r, off, sum, n_piece, a.u_draw[at]);
            if (threadIdx.x == 0) {
                s_none = code < 0;
                a.codes[at] = max(code, 0);
            }
        }
        __syncthreads();
        if (!off || !s_none) break;
        row_pieces(r, false, 0, n_piece, sum);              // no mass in the rest: from p itself
        __syncthreads();
    }
}

} // namespace z2d
