// z2h_moe.h — a mixture-of-experts layer for a few rows on the caller's tensors: routing, the experts' gated products, their weighted sum.
//
//   p = softmax(logits), the top_k of p + bias, w = p (or p / sum), out = sum_j w_j down (silu(gate x) * (up x))
//   k_moe_gate_up   every block routes all rows for itself (a wave per row), then takes an equal share of the tiles of 8 gate and 8 up rows of
//                   the experts that a row takes; h = silu(gate x) * (up x) in fp32
//   k_moe_down      16 dims of out per block (and a share of the experts' hidden dims), all rows; shares are joined by the last block of them
// Both read every weight that they need once and are bound by that: weights go from memory to the left operand of v_mfma_f32_16x16x32, 16 rows of
// the matrix by 32 of its columns per instruction, and up to 16 rows of x or h are the right operand, so that the products cost the
// same for 1 to 16 of them.
#pragma once
#include "z2h_common.h"
#include "z2h_ops_rules.h"
#include "z2h_tile.h"

namespace z2d {

constexpr int MOE_WAVES = 8, MOE_T = 64 * MOE_WAVES;
constexpr int MOE_ROWS = Z2H_MOE_ROWS_MAX, MOE_MASKS = MOE_ROWS / 32;

// an expert that some rows take: their bits, and the place of the first of their routes (in the order of the rows)
struct MoeTouched { int e, pos0; unsigned rows[MOE_MASKS]; };
struct MoeTable { int n, spare[3]; unsigned no_number[MOE_MASKS]; };     // touched experts; rows without a number
static_assert(sizeof(MoeTouched) == 24 && sizeof(MoeTable) == 32, "workspace layout");

struct MoeArgs {
    const void * gate, * up, * down;
    int E, F, D, n, k, renorm, shares, tiles;
    const float * logits, * bias;
    const void * x;
    int64_t xs, os;
    void * out;
    int32_t * sel;
    float * weights;
    MoeTable * table;
    MoeTouched * touched;
    float * w;                                                   // [n k] weights of the routes, by place
    int32_t * tickets;                                           // [tiles of out]
    float * h;                                                   // [n k][F], by place
    float * parts;                                               // [shares][n][D]
};

typedef float v4f_t __attribute__((ext_vector_type(4)));
template <typename TW>
__device__ __forceinline__ v4f_t mfma16(typename Vec8<TW>::type a, typename Vec8<TW>::type b, v4f_t c) {
    if constexpr (__is_same(TW, _Float16)) return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// ---- routing
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

// One row's experts and weights by one wave, into sel and w [k]; false: the row has no number. Experts are told apart by p + bias in 64 bits,
// without a bias by the logits themselves (the same order, and equal ones are equal). Expert 64 i + lane is entry i of the lane's.
template <int EPL>
__device__ __forceinline__ bool route_row(const MoeArgs & a, int row, short * sel, float * w) {
    const int lane = threadIdx.x & 63;
    const float * src = a.logits + (int64_t) row * a.E;
    constexpr long long NONE = -0x7fffffffffffffffll - 1;
    float z[EPL], p[EPL], b[EPL];
    float mx = -__builtin_inff(), sum = 0.0f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
        const int e = 64 * i + lane;
        z[i] = e < a.E ? src[e] : -__builtin_inff();
        b[i] = a.bias && e < a.E ? a.bias[e] : 0.0f;
        bad |= !(z[i] < __builtin_inff()) || b[i] != b[i];
        mx = fmaxf(mx, z[i]);
    }
    mx = wave_max_f(mx);
    const float m0 = mx == -__builtin_inff() ? 0.0f : mx;
#pragma unroll
    for (int i = 0; i < EPL; ++i) sum += p[i] = z_expf(z[i] - m0);
    const float inv = 1.0f / wave_tree_f(sum);
    if (__any(bad)) {
        if (lane < a.k) { sel[lane] = -1; w[lane] = __builtin_nanf(""); }
        return false;
    }
    long long key[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
        p[i] *= inv;
        key[i] = z[i] == -__builtin_inff() ? NONE : score_key(a.bias ? (double) p[i] + (double) b[i] : (double) z[i]);
    }
    float total = 0.0f, mine = 0.0f;
    short mine_e = -1;
    for (int found = 0; found < a.k; ++found) {
        long long best = key[0];
#pragma unroll
        for (int i = 1; i < EPL; ++i) best = key[i] > best ? key[i] : best;
        const long long top = wave_max_ll(best);
        if (top == NONE) break;
        bool open = true;                                        // of equal ones the lowest
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
            const unsigned long long same = __ballot(key[i] == top);
            if (open && same) {
                const int at = __builtin_ctzll(same);
                const float pe = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, p[i]), at));
                total += pe;
                if (lane == found) { mine = pe; mine_e = (short) (64 * i + at); }
                if (lane == at) key[i] = NONE;
                open = false;
            }
        }
    }
    if (lane < a.k) {
        sel[lane] = mine_e;
        w[lane] = a.renorm && total > 0.0f ? mine / total : mine;
    }
    return true;
}

struct MoeRouting {
    short sel[MOE_ROWS * z2o::MOE_MAX_TOP];
    float w[MOE_ROWS * z2o::MOE_MAX_TOP];
    unsigned rows[z2o::MOE_MAX_EXPERTS][MOE_MASKS], no_number[MOE_MASKS];
    short list[z2o::MOE_MAX_EXPERTS], pos0[z2o::MOE_MAX_EXPERTS];        // touched experts in order, and their first routes' places
    int wave[MOE_WAVES], n;
};

// All rows' routes, and of every expert the rows that take it; by the whole block.
__device__ __forceinline__ void route(const MoeArgs & a, MoeRouting & s) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int i = tid; i < a.E * MOE_MASKS; i += MOE_T) (&s.rows[0][0])[i] = 0;
    if (tid < MOE_MASKS) s.no_number[tid] = 0;
    __syncthreads();
    for (int r = wave; r < a.n; r += MOE_WAVES) {
        short * sel = s.sel + r * a.k;
        float * w = s.w + r * a.k;
        const bool ok = a.E <= 64 ? route_row<1>(a, r, sel, w) : a.E <= 256 ? route_row<4>(a, r, sel, w) : route_row<16>(a, r, sel, w);
        if (!ok && lane == 0) atomicOr(&s.no_number[r >> 5], 1u << (r & 31));
        if (ok && lane < a.k && sel[lane] >= 0) atomicOr(&s.rows[sel[lane]][r >> 5], 1u << (r & 31));
    }
    __syncthreads();
    int total = 0;                                               // touched experts << 16 | routes
    for (int e0 = 0; e0 < a.E; e0 += MOE_T) {
        const int e = e0 + tid;
        int routes = 0;
        if (e < a.E)
            for (int i = 0; i < MOE_MASKS; ++i) routes += __popc(s.rows[e][i]);
        const int mine = routes ? 0x10000 | routes : 0;
        int x = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(x, o);
            if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 63) s.wave[wave] = x;
        __syncthreads();
        int below = total;
        for (int w = 0; w < MOE_WAVES; ++w) {
            if (w < wave) below += s.wave[w];
            total += s.wave[w];
        }
        below += x - mine;
        if (routes) { s.list[below >> 16] = (short) e; s.pos0[below >> 16] = (short) (below & 0xffff); }
    }
    if (tid == 0) s.n = total >> 16;
    __syncthreads();
}
// the i-th row that takes an expert (it has more)
__device__ __forceinline__ int nth_row(const unsigned * rows, int i) {
    int word = 0;
#pragma unroll
    for (int m = 0; m < MOE_MASKS - 1; ++m) {
        const int c = __popc(rows[word]);
        if (i >= c) { i -= c; ++word; }
    }
    unsigned w = rows[word];
    for (; i > 0; --i) w &= w - 1;
    return 32 * word + __builtin_ctz(w);
}
// rows below `row` that take an expert
__device__ __forceinline__ int rows_before(const unsigned * rows, int row) {
    int n = 0;
#pragma unroll
    for (int m = 0; m < MOE_MASKS; ++m) n += __popc(32 * m + 32 <= row ? rows[m] : 32 * m <= row ? rows[m] & ((1u << (row & 31)) - 1) : 0u);
    return n;
}

// ---- right operands
// 8 values of a row from memory (its address may be any)
template <typename T>
__device__ __forceinline__ void load8(const T * p, float (&x)[8]) {
    if (((uintptr_t) p & 15) == 0) {
        constexpr int N = 16 / (int) sizeof(T);
        typedef T tv __attribute__((ext_vector_type(N)));
#pragma unroll
        for (int i = 0; i < 8; i += N) {
            const tv y = *(const tv *) (p + i);
#pragma unroll
            for (int j = 0; j < N; ++j) x[i + j] = (float) y[j];
        }
    } else
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float) p[i];
}
// the largest of a column's values, whose four lanes are 16 apart
__device__ __forceinline__ float column_max(float v) {
    v = fmaxf(v, other_half(v));
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    const unsigned r0 = r[0], r1 = r[1];
    return fmaxf(__builtin_bit_cast(float, r0), __builtin_bit_cast(float, r1));
}
// fp32 columns as two numbers of the weights' type each. f16: brought to [2^7, 2^8) by a power of two first, so that both parts together keep
// every value to 2^-22 of the column's largest; `back` undoes it.
template <int FR, typename TW>
struct SplitColumn {
    typedef typename Vec8<TW>::type v8;
    v8 hi[FR], lo[FR];
    float back;
    __device__ __forceinline__ void set(const float (&x)[FR][8]) {
        float up = 1.0f;
        back = 1.0f;
        if constexpr (__is_same(TW, _Float16)) {
            float mx = 0.0f;
#pragma unroll
            for (int i = 0; i < FR; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) mx = fmaxf(mx, fabsf(x[i][j]));
            mx = column_max(mx);
            int e = 8;
            if (mx > 0.0f && mx < __builtin_inff()) (void) frexpf(mx, &e);
            e = max(e, -110);
            up = ldexpf(1.0f, 8 - e);
            back = ldexpf(1.0f, e - 8);
        }
#pragma unroll
        for (int i = 0; i < FR; ++i)
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                typedef typename Pair<float>::type f2;
                typedef typename Pair<TW>::type c2;
                const f2 y = {x[i][j] * up, x[i][j + 1] * up};
                const c2 h = __builtin_convertvector(y, c2), l = __builtin_convertvector(two_rest(y, h), c2);
                hi[i][j] = h[0]; hi[i][j + 1] = h[1];
                lo[i][j] = l[0]; lo[i][j + 1] = l[1];
            }
    }
};

// ---- gate and up
constexpr int MOE_FR = 8;                                        // operands of a wave in a pass: 256 columns of the matrix
// NT tiles of 16 rows of x. The wave's columns are one of eight slices of up to 2048; tiles of 16 matrix rows (8 of gate, 8 of up) follow each
// other, the next one's weights on their way while this one is multiplied, and the slices' sums meet in LDS.
template <typename T, typename TW, int NT>
__global__ void __launch_bounds__(MOE_T, NT == 1 ? 4 : 2) k_moe_gate_up(MoeArgs a) {
    constexpr bool SPLIT = sizeof(T) == 4;
    typedef typename Vec8<TW>::type v8;
    __shared__ MoeRouting s;
    __shared__ float s_sum[2][MOE_WAVES][NT][256];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    route(a, s);
    if (blockIdx.x == 0) {
        for (int i = tid; i < a.n * a.k; i += MOE_T) {
            if (a.sel) a.sel[i] = s.sel[i];
            if (a.weights) a.weights[i] = s.w[i];
        }
        for (int i = tid; i < a.tiles; i += MOE_T) a.tickets[i] = 0;
        if (tid == 0) a.table->n = s.n;
        if (tid < MOE_MASKS) a.table->no_number[tid] = s.no_number[tid];
        for (int t = tid; t < s.n; t += MOE_T) {
            MoeTouched x{s.list[t], s.pos0[t], {}};
            for (int i = 0; i < MOE_MASKS; ++i) x.rows[i] = s.rows[x.e][i];
            a.touched[t] = x;
        }
        for (int r = tid; r < a.n; r += MOE_T)
            for (int j = 0; j < a.k; ++j) {
                const int e = s.sel[r * a.k + j];
                if (e < 0) continue;
                int t = 0;
                for (int hi = s.n; hi - t > 1;) { const int m = (t + hi) >> 1; if (s.list[m] <= e) t = m; else hi = m; }
                a.w[s.pos0[t] + rows_before(s.rows[e], r)] = s.w[r * a.k + j];
            }
    }
    const int per = a.F / 8, n_tiles = s.n * per, frags = (a.D + 31) / 32;
    const int t0 = (int) ((int64_t) n_tiles * blockIdx.x / gridDim.x), t1 = (int) ((int64_t) n_tiles * (blockIdx.x + 1) / gridDim.x);
    const int passes = (frags + MOE_FR * MOE_WAVES - 1) / (MOE_FR * MOE_WAVES), mine = (frags + passes * MOE_WAVES - 1) / (passes * MOE_WAVES);
    const int k8 = 8 * (lane >> 4), col = lane & 15, r16 = lane & 15;
    // the lane's matrix row of tile i of an expert: gate for lanes' rows 0 .. 7, up behind them
    const TW * mat = (const TW *) (r16 < 8 ? a.gate : a.up) + (int64_t) (r16 & 7) * a.D + k8;
    int buf = 0;
    for (int from = t0; from < t1;) {
        const int t = from / per, e = s.list[t], to = min(t1, (t + 1) * per);
        int count = 0;
#pragma unroll
        for (int i = 0; i < MOE_MASKS; ++i) count += __popc(s.rows[e][i]);
        const TW * base = mat + ((int64_t) e * a.F - (int64_t) t * per * 8) * a.D;      // + tile * 8 rows
        for (int c0 = 0; c0 < count; c0 += 16 * NT) {
            for (int tile = from; tile < to; ++tile) {
                v4f_t sum[NT];
#pragma unroll
                for (int c = 0; c < NT; ++c) sum[c] = v4f_t{};
                for (int pass = 0; pass < passes; ++pass) {
                    const int f0 = (pass * MOE_WAVES + wave) * mine;
                    v8 w[MOE_FR];
                    const TW * p = base + (int64_t) tile * 8 * a.D + 32 * f0;
#pragma unroll
                    for (int i = 0; i < MOE_FR; ++i) w[i] = i < mine && 32 * (f0 + i) + k8 < a.D ? *(const v8 *) (p + 32 * i) : v8{};
#pragma unroll
                    for (int c = 0; c < NT; ++c) {
                        const int at = c0 + 16 * c + col;
                        const bool live = at < count;
                        const T * x = (const T *) a.x + (live ? nth_row(s.rows[e], at) : 0) * a.xs + 32 * f0 + k8;
                        float y[MOE_FR][8];
#pragma unroll
                        for (int i = 0; i < MOE_FR; ++i) {
                            if (live && i < mine && 32 * (f0 + i) + k8 < a.D) load8(x + 32 * i, y[i]);
                            else
#pragma unroll
                                for (int j = 0; j < 8; ++j) y[i][j] = 0.0f;
                        }
                        if constexpr (SPLIT) {
                            SplitColumn<MOE_FR, TW> b;
                            b.set(y);
                            v4f_t part{};
#pragma unroll
                            for (int i = 0; i < MOE_FR; ++i) {
                                part = mfma16<TW>(w[i], b.hi[i], part);
                                part = mfma16<TW>(w[i], b.lo[i], part);
                            }
#pragma unroll
                            for (int i = 0; i < 4; ++i) sum[c][i] = __builtin_fmaf(part[i], b.back, sum[c][i]);
                        } else {
#pragma unroll
                            for (int i = 0; i < MOE_FR; ++i) {
                                v8 b;
#pragma unroll
                                for (int j = 0; j < 8; ++j) b[j] = (TW) y[i][j];
                                sum[c] = mfma16<TW>(w[i], b, sum[c]);
                            }
                        }
                    }
                }
#pragma unroll
                for (int c = 0; c < NT; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s_sum[buf][wave][c][(4 * (lane >> 4) + i) * 16 + col] = sum[c][i];
                lds_sync();
                for (int i = tid; i < NT * 128; i += MOE_T) {
                    const int c = i >> 7, row = (i >> 3) & 15, f = i & 7;
                    if (c0 + 16 * c + row < count) {
                        float g = 0.0f, u = 0.0f;
#pragma unroll
                        for (int v = 0; v < MOE_WAVES; ++v) {
                            g += s_sum[buf][v][c][f * 16 + row];
                            u += s_sum[buf][v][c][(f + 8) * 16 + row];
                        }
                        a.h[(int64_t) (s.pos0[t] + c0 + 16 * c + row) * a.F + (tile - t * per) * 8 + f] = z_silu(g) * u;
                    }
                }
                buf ^= 1;
            }
        }
        from = to;
    }
}

// ---- down
constexpr int MOE_DF = 4;                                        // operands of a unit: 128 hidden dims of an expert
// 16 dims of out and all rows (CT tiles of 16) per block, over its share of the units (an expert's 128 hidden dims), dealt to the waves in runs.
// The right operand is w h of the rows that take the expert, 0 for the others, whose sums it does not reach whatever the weights hold.
template <typename T, typename TW, int CT>
__global__ void __launch_bounds__(MOE_T, CT <= 2 ? 4 : 2) k_moe_down(MoeArgs a) {
    typedef typename Vec8<TW>::type v8;
    __shared__ float s_sum[MOE_WAVES][CT][256];
    __shared__ int s_last;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = uniform(&a.table->n)[0], chunks = (a.F + 32 * MOE_DF - 1) / (32 * MOE_DF), units = n * chunks;
    const int share = (int) blockIdx.y * MOE_WAVES + wave, shares = a.shares * MOE_WAVES;
    const int u0 = (int) ((int64_t) units * share / shares), u1 = (int) ((int64_t) units * (share + 1) / shares);
    const int k8 = 8 * (lane >> 4), col = lane & 15, d = 16 * (int) blockIdx.x + col;
    const TW * mat = (const TW *) a.down + (int64_t) min(d, a.D - 1) * a.F + k8;
    v4f_t sum[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) sum[c] = v4f_t{};
    for (int u = u0; u < u1; ++u) {
        const MoeTouched t = uniform_copy(a.touched + u / chunks);
        const int f0 = u % chunks * 32 * MOE_DF;
        v8 w[MOE_DF];
        const TW * p = mat + (int64_t) t.e * a.D * a.F + f0;
#pragma unroll
        for (int i = 0; i < MOE_DF; ++i) w[i] = d < a.D && f0 + 32 * i + k8 < a.F ? *(const v8 *) (p + 32 * i) : v8{};
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            if (!((t.rows[c >> 1] >> (16 * (c & 1))) & 0xffffu)) continue;
            const int row = 16 * c + col;
            const bool live = t.rows[c >> 1] >> (row & 31) & 1;
            const int pos = live ? t.pos0 + rows_before(t.rows, row) : 0;
            const float wt = live ? a.w[pos] : 0.0f;
            const float * h = a.h + (int64_t) pos * a.F + f0 + k8;
            float y[MOE_DF][8];
#pragma unroll
            for (int i = 0; i < MOE_DF; ++i) {
                if (live && f0 + 32 * i + k8 < a.F) load8(h + 32 * i, y[i]);
                else
#pragma unroll
                    for (int j = 0; j < 8; ++j) y[i][j] = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) y[i][j] *= wt;
            }
            SplitColumn<MOE_DF, TW> b;
            b.set(y);
            v4f_t part{};
#pragma unroll
            for (int i = 0; i < MOE_DF; ++i) {
                part = mfma16<TW>(w[i], b.hi[i], part);
                part = mfma16<TW>(w[i], b.lo[i], part);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[c][i] = live ? __builtin_fmaf(part[i], b.back, sum[c][i]) : sum[c][i];
        }
    }
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) s_sum[wave][c][(4 * (lane >> 4) + i) * 16 + col] = sum[c][i];
    __syncthreads();
    auto store = [&](int row, int d, float v) {
        if (a.table->no_number[row >> 5] >> (row & 31) & 1) v = __builtin_nanf("");
        ((T *) a.out)[row * a.os + d] = (T) v;
    };
    for (int i = tid; i < CT * 256; i += MOE_T) {
        const int row = i >> 4, dd = i & 15, at = 16 * (int) blockIdx.x + dd;
        if (row >= a.n || at >= a.D) continue;
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < MOE_WAVES; ++w) v += s_sum[w][row >> 4][dd * 16 + (row & 15)];
        if (a.shares == 1) store(row, at, v);
        else a.parts[((int64_t) blockIdx.y * a.n + row) * a.D + at] = v;
    }
    if (a.shares == 1) return;
    // the last block of a tile's joins what all have left, in their order
    __threadfence();
    __syncthreads();
    if (tid == 0) s_last = __hip_atomic_fetch_add(a.tickets + blockIdx.x, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == a.shares - 1;
    __syncthreads();
    if (!s_last) return;
    for (int i = tid; i < CT * 256; i += MOE_T) {
        const int row = i >> 4, at = 16 * (int) blockIdx.x + (i & 15);
        if (row >= a.n || at >= a.D) continue;
        float v = 0.0f;
        for (int p = 0; p < a.shares; ++p) v += a.parts[((int64_t) p * a.n + row) * a.D + at];
        store(row, at, v);
    }
}

} // namespace z2d
