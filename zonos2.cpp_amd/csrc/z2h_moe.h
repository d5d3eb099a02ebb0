// z2h_moe.h — a mixture-of-experts layer for a few rows on the caller's tensors: routing, the experts' gated products, their weighted sum.
//
//   p = softmax(logits), the top_k of p + bias, w = p (or p / sum), out = sum_j w_j down (silu(gate x) * (up x))
//   k_moe_route     more than eight rows or 256 experts: each row's experts and weights, a wave per row
//   k_moe_gate_up   every block lists the experts that a row takes (without k_moe_route: after routing all rows for itself), then takes an equal
//                   share of the tiles of 8 gate and 8 up rows of those experts; h = silu(gate x) * (up x) in fp32
//   k_moe_down      16 dims of out per block (and a share of the experts' hidden dims), all rows; shares are joined by the last block of them
// Both products read every weight that they need once and are bound by that: weights go from memory to the left operand of
// v_mfma_f32_16x16x32, 16 rows of the matrix by 32 of its columns per instruction, and up to 16 rows of x or h are the right operand, so that
// the products cost the same for 1 to 16 of them. A row of x goes there as it is (fp32: as two fp16 numbers), h as two fp16 or three bf16 numbers.
// Measured, bf16 weights: 64 rows, 6 of 64 experts of 1032 x 2048: 210 us, 3.9 TB/s of weights (k_moe_route 5, k_moe_gate_up 126 for
// 541 MB, k_moe_down 76 for 270 MB); fp16, 16 rows, 4 of 32 experts of 1536 x 2048: 114 to 118 us, 4.6 TB/s; fp32 rows, one row: 26 us, 2.9 TB/s,
// of which 12 are two launches, routing and the join (a layer of 8 x 32 takes 13 to 14). A copy reaches 5.15 TB/s: both products let memory
// stand still between their tiles, since they wait for the weights that they have requested ahead (see there).
#pragma once
#include "z2h_common.h"
#include "z2h_ops_rules.h"
#include "z2h_tile.h"

namespace z2d {

constexpr int MOE_WAVES = 8, MOE_T = 64 * MOE_WAVES;
constexpr int MOE_ROWS = Z2H_MOE_ROWS_MAX, MOE_MASKS = MOE_ROWS / 32;

// an expert that some rows take: their bits, the place of the first of their routes (in the order of the rows), and the turns of 16 rows that the
// experts before it take
struct MoeTouched { short e, pos0; int turn0; unsigned rows[MOE_MASKS]; };
struct MoeTable { int n, turns, spare[2]; unsigned no_number[MOE_MASKS]; };      // touched experts and their turns; rows without a number
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
    int32_t * row_sel;                                           // [n k] of k_moe_route; null: every block routes for itself
    float * row_w;
    float * w;                                                   // [n k] weights of the routes, by place
    int32_t * tickets;                                           // [tiles of out]
    int hs;
    float * h;                                                   // [n k][hs], by place; see k_moe_down for the columns' order
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

// One row's experts and weights by one wave, into sel and w [k]; a row without a number: -1 and NaN. Probabilities and p + bias are formed in 64 bits
// (without a bias the logits themselves tell experts apart), and weights are rounded once. Weights that are to sum to one are formed relative
// to the largest chosen logit: a bias may keep the others out by any distance. Expert 64 i + lane is entry i of the lane's.
template <int EPL, typename S>
__device__ __forceinline__ void route_row(const MoeArgs & a, int row, S * sel, float * w) {
    const int lane = threadIdx.x & 63;
    const float * src = a.logits + (int64_t) row * a.E;
    constexpr long long NONE = -0x7fffffffffffffffll - 1;
    float z[EPL], b[EPL];
    float mx = -__builtin_inff();
    bool bad = false;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
        const int e = 64 * i + lane;
        z[i] = e < a.E ? src[e] : -__builtin_inff();
        b[i] = a.bias && e < a.E ? a.bias[e] : 0.0f;
        bad |= !(z[i] < __builtin_inff()) || b[i] != b[i];
        mx = fmaxf(mx, z[i]);
    }
    if (__any(bad)) {
        if (lane < a.k) { sel[lane] = -1; w[lane] = __builtin_nanf(""); }
        return;
    }
    mx = wave_max_f(mx);
    const double m0 = mx == -__builtin_inff() ? 0.0 : (double) mx;
    double p[EPL], sum = 0.0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) sum += p[i] = z_exp_d((double) z[i] - m0);
    sum = wave_tree_d(sum);
    const double inv = 1.0 / sum;
    long long key[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i)
        key[i] = z[i] == -__builtin_inff() ? NONE : score_key(a.bias ? p[i] * inv + (double) b[i] : (double) z[i]);
    float mine = -__builtin_inff();
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
                const float ze = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, z[i]), at));
                if (lane == found) { mine = ze; mine_e = (short) (64 * i + at); }
                if (lane == at) key[i] = NONE;
                open = false;
            }
        }
    }
    const double from = a.renorm ? (double) wave_max_f(mine) : m0;
    const double we = mine_e < 0 ? 0.0 : z_exp_d((double) mine - from);
    if (a.renorm) sum = wave_tree_d(we);
    if (lane < a.k) {
        sel[lane] = mine_e;
        w[lane] = mine_e < 0 ? 0.0f : (float) (we / sum);
    }
}
// Up to this many experts a block of k_moe_gate_up may route for itself; 16 to a lane do not fit its registers (bf16, 300 experts: 8 rows 22.7 us with
// the launch, 24.0 without and 11 registers spilled; 1 row 21.9 and 21.0).
constexpr int MOE_OWN_EXPERTS = 256;
template <int MAX, typename S>
__device__ __forceinline__ void route_any(const MoeArgs & a, int row, S * sel, float * w) {
    if (a.E <= 64) route_row<1>(a, row, sel, w);
    else if (MAX <= 256 || a.E <= 256) route_row<4>(a, row, sel, w);
    else route_row<16>(a, row, sel, w);
}
// Each row once, in a launch of its own: 4 us for 64 rows of 64 experts, 13 when every block of k_moe_gate_up does all.
__global__ void __launch_bounds__(64) k_moe_route(MoeArgs a) {
    route_any<z2o::MOE_MAX_EXPERTS>(a, blockIdx.x, a.row_sel + blockIdx.x * a.k, a.row_w + blockIdx.x * a.k);
}

struct MoeRouting {
    short sel[MOE_ROWS * z2o::MOE_MAX_TOP];
    float w[MOE_ROWS * z2o::MOE_MAX_TOP];
    unsigned rows[z2o::MOE_MAX_EXPERTS][MOE_MASKS], no_number[MOE_MASKS];
    short list[z2o::MOE_MAX_EXPERTS], pos0[z2o::MOE_MAX_EXPERTS];        // touched experts in order, and their first routes' places
    short turn0[2][z2o::MOE_MAX_EXPERTS];                                // turns of 16 rows and of the kernel's own of the experts before
    unsigned long long wave[MOE_WAVES];
    int n, turns[2];
};

// All rows' routes, and of every expert the rows that take it; by the whole block. An expert takes a turn per ROWS rows.
template <int ROWS>
__device__ __forceinline__ void route(const MoeArgs & a, MoeRouting & s) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int i = tid; i < a.E * MOE_MASKS; i += MOE_T) (&s.rows[0][0])[i] = 0;
    if (tid < MOE_MASKS) s.no_number[tid] = 0;
    __syncthreads();
    if (a.row_sel)
        for (int i = tid; i < a.n * a.k; i += MOE_T) {
            s.sel[i] = (short) a.row_sel[i];
            s.w[i] = a.row_w[i];
        }
    else
        for (int r = wave; r < a.n; r += MOE_WAVES) route_any<MOE_OWN_EXPERTS>(a, r, s.sel + r * a.k, s.w + r * a.k);
    __syncthreads();
    for (int i = tid; i < a.n * a.k; i += MOE_T) {
        const int r = i / a.k, e = s.sel[i];
        if (e >= 0) atomicOr(&s.rows[e][r >> 5], 1u << (r & 31));
        else if (s.w[i] != s.w[i]) atomicOr(&s.no_number[r >> 5], 1u << (r & 31));
    }
    __syncthreads();
    unsigned long long total = 0;                                // 16 bits each: touched experts, turns of ROWS rows, of 16 rows, routes
    for (int e0 = 0; e0 < a.E; e0 += MOE_T) {
        const int e = e0 + tid;
        int routes = 0;
        if (e < a.E)
            for (int i = 0; i < MOE_MASKS; ++i) routes += __popc(s.rows[e][i]);
        const unsigned long long mine = ((unsigned long long) ((routes ? 0x10000 : 0) | (routes + ROWS - 1) / ROWS) << 32) |
                                        (unsigned) ((routes + 15) / 16 << 16 | routes);
        unsigned long long x = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const unsigned long long y = __shfl_up(x, o);
            if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 63) s.wave[wave] = x;
        __syncthreads();
        unsigned long long below = total;
        for (int w = 0; w < MOE_WAVES; ++w) {
            if (w < wave) below += s.wave[w];
            total += s.wave[w];
        }
        below += x - mine;
        if (routes) {
            const int t = (int) (below >> 48);
            s.list[t] = (short) e;
            s.pos0[t] = (short) below;
            s.turn0[0][t] = (short) (below >> 16);
            s.turn0[1][t] = (short) (below >> 32);
        }
    }
    if (tid == 0) { s.n = (int) (total >> 48); s.turns[0] = (int) (total >> 16 & 0xffff); s.turns[1] = (int) (total >> 32 & 0xffff); }
    __syncthreads();
}
// the i-th row that takes an expert (it has more)
__device__ __forceinline__ int nth_row(const unsigned * rows, int i) {
    int word = 0;
    unsigned w = rows[0];
#pragma unroll
    for (int m = 1; m < MOE_MASKS; ++m) {
        const int c = __popc(w);
        if (word == m - 1 && i >= c) { i -= c; word = m; w = rows[m]; }
    }
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
// fp32 columns as numbers of the weights' type. f16: two each, brought to [2^7, 2^8) by a power of two first, so that both parts together keep
// every value to 2^-22 of the column's largest; `back` undoes it. bf16: three each, which keep every value to 2^-24 of itself (two keep
// 2^-16: outputs that are differences of nearly equal terms lose as many of their bits; 64 rows 210 us in place of 209, 5 rows 54 in place of 53).
template <int FR, typename TW>
struct SplitColumn {
    static constexpr int PARTS = __is_same(TW, _Float16) ? 2 : 3;
    typedef typename Vec8<TW>::type v8;
    v8 part[PARTS][FR];
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
                f2 y = {x[i][j] * up, x[i][j + 1] * up};
#pragma unroll
                for (int q = 0; q < PARTS; ++q) {
                    const c2 h = __builtin_convertvector(y, c2);
                    part[q][i][j] = h[0]; part[q][i][j + 1] = h[1];
                    if (q + 1 < PARTS) y = two_rest(y, h);
                }
            }
    }
};

// ---- gate and up
// Blocks of one compute unit at a time: two where the registers allow it.
template <typename T, int NT>
constexpr int moe_per_cu() { return sizeof(T) == 2 && NT == 1 ? 2 : 1; }
constexpr int MOE_FR = 8;                                        // operands of a wave in a pass: 256 columns of the matrix

// A block's or wave's part u0 .. u1 of the units, which are every touched expert's pieces (tiles, chunks) times its turns, so that parts take
// the same time (without the turns: k_moe_gate_up 205 us in place of 126 for 64 rows most of which take the same few of 64 experts). A piece
// belongs to the part with its first unit.
struct MoePieces {
    int from, to;
    __device__ __forceinline__ MoePieces(int u0, int u1, int base, int pieces, int turns) {
        from = max(u0 - base, 0);
        to = u1 - base;
        if (turns > 1) { from = (from + turns - 1) / turns; to = (to + turns - 1) / turns; }
        to = min(to, pieces);
    }
};
// The tiles of 16 matrix rows (8 of gate, 8 of up) that a block has, in the order in which it takes them: for every ROWS rows of x that take the
// expert, all its tiles. Columns go in passes of up to 2048; with more than one, MOE_GROUP tiles take a pass before their next one, so that
// the right operands are formed once for all of them (64 rows, 4 of 32 experts of 1536 x 4096: 294 us in place of 534 in fp32,
// 295 in place of 373 in f16).
constexpr int MOE_GROUP = 16;
template <int ROWS>
struct MoeCursor {
    int t, tile, pass, c0, e, count, from, to, g0;
    // from expert t_ on; false: the block has nothing there
    __device__ __forceinline__ bool enter(const MoeRouting & s, int t_, int per, int u0, int u1) {
        pass = c0 = 0;
        for (t = t_; t < s.n; ++t) {
            const int base = __builtin_amdgcn_readfirstlane((int) s.turn0[1][t]) * per;
            if (base >= u1) return false;
            e = __builtin_amdgcn_readfirstlane((int) s.list[t]);
            count = 0;
#pragma unroll
            for (int i = 0; i < MOE_MASKS; ++i) count += __popc(s.rows[e][i]);
            count = __builtin_amdgcn_readfirstlane(count);
            const MoePieces x(u0, u1, base, per, (count + ROWS - 1) / ROWS);
            tile = g0 = from = x.from;
            to = x.to;
            if (from < to) return true;
        }
        return false;
    }
    // false: that was the last
    __device__ __forceinline__ bool next(const MoeRouting & s, int per, int u0, int u1, int passes) {
        if (++tile < (passes > 1 ? min(g0 + MOE_GROUP, to) : to)) return true;
        if (++pass < passes) { tile = g0; return true; }
        pass = 0;
        g0 = tile;
        if (tile < to) return true;
        if (c0 + ROWS < count) { tile = g0 = from; c0 += ROWS; return true; }
        return enter(s, t + 1, per, u0, u1);
    }
};

// NT tiles of 16 rows of x stay in registers while the expert's tiles pass by. The next tile's weights are requested before the present one's
// products, but arrive before them too: all of these loads are made under conditions, so that the compiler cannot count which may be left
// on their way, and it waits for every one before it multiplies. A wave has one of eight slices of the columns; the slices' sums meet in LDS.
template <typename T, typename TW, int NT>
__global__ void __launch_bounds__(MOE_T, (2 * moe_per_cu<T, NT>())) k_moe_gate_up(MoeArgs a) {
    constexpr bool SPLIT = sizeof(T) == 4;
    typedef typename Vec8<TW>::type v8;
    __shared__ MoeRouting s;
    __shared__ float s_sum[2][MOE_WAVES][NT][256], s_acc[MOE_GROUP][2][128 * NT];       // of a tile's earlier passes
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    route<16 * NT>(a, s);
    if (blockIdx.x == gridDim.x - 1) {
        for (int i = tid; i < a.n * a.k; i += MOE_T) {
            if (a.sel) a.sel[i] = s.sel[i];
            if (a.weights) a.weights[i] = s.w[i];
        }
        for (int i = tid; i < a.tiles; i += MOE_T) a.tickets[i] = 0;
        if (tid == 0) { a.table->n = s.n; a.table->turns = s.turns[0]; }
        if (tid < MOE_MASKS) a.table->no_number[tid] = s.no_number[tid];
        for (int t = tid; t < s.n; t += MOE_T) {
            MoeTouched x{s.list[t], s.pos0[t], s.turn0[0][t], {}};
            for (int i = 0; i < MOE_MASKS; ++i) x.rows[i] = s.rows[x.e][i];
            a.touched[t] = x;
        }
        for (int i = tid; i < a.n * a.k; i += MOE_T) {
            const int e = s.sel[i];
            if (e < 0) continue;
            int t = 0;
            for (int hi = s.n; hi - t > 1;) { const int m = (t + hi) >> 1; if (s.list[m] <= e) t = m; else hi = m; }
            a.w[s.pos0[t] + rows_before(s.rows[e], i / a.k)] = s.w[i];
        }
    }
    const int per = a.F / 8, units = __builtin_amdgcn_readfirstlane(s.turns[1]) * per, frags = (a.D + 31) / 32;
    const int u0 = (int) ((int64_t) units * blockIdx.x / gridDim.x), u1 = (int) ((int64_t) units * (blockIdx.x + 1) / gridDim.x);
    if (u0 >= u1) return;
    int t0 = 0;                                                  // the expert of unit u0
    for (int hi = __builtin_amdgcn_readfirstlane(s.n); hi - t0 > 1;) {
        const int m = (t0 + hi) >> 1;
        if (__builtin_amdgcn_readfirstlane((int) s.turn0[1][m]) * per <= u0) t0 = m;
        else hi = m;
    }
    MoeCursor<16 * NT> cur, nxt;
    if (!cur.enter(s, t0, per, u0, u1)) return;
    const int passes = (frags + MOE_FR * MOE_WAVES - 1) / (MOE_FR * MOE_WAVES), mine = (frags + passes * MOE_WAVES - 1) / (passes * MOE_WAVES);
    const int k8 = 8 * (lane >> 4), col = lane & 15;
    // the lane's matrix row of an expert's first tile: gate for rows 0 .. 7 of the operand, up behind them
    const TW * mat = (const TW *) (col < 8 ? a.gate : a.up) + (int64_t) (col & 7) * a.D + k8;
    auto inside = [&](int f0, int i) __attribute__((always_inline)) { return i < mine && 32 * (f0 + i) + k8 < a.D; };
    auto request = [&](const MoeCursor<16 * NT> & c, v8 (&w)[MOE_FR]) __attribute__((always_inline)) {
        const int f0 = (c.pass * MOE_WAVES + wave) * mine;
        const TW * p = mat + ((int64_t) c.e * a.F + c.tile * 8) * a.D + 32 * f0;
#pragma unroll
        for (int i = 0; i < MOE_FR; ++i) w[i] = inside(f0, i) ? *(const v8 *) (p + 32 * i) : v8{};
    };
    SplitColumn<MOE_FR, TW> b[NT];                               // 16-bit rows: the first part alone
    auto columns = [&](const MoeCursor<16 * NT> & c) __attribute__((always_inline)) {
        const int f0 = (c.pass * MOE_WAVES + wave) * mine;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int at = c.c0 + 16 * n + col;
            const bool live = at < c.count;
            const T * x = (const T *) a.x + (live ? nth_row(s.rows[c.e], at) : 0) * a.xs + 32 * f0 + k8;
            if constexpr (SPLIT) {
                float y[MOE_FR][8];
#pragma unroll
                for (int i = 0; i < MOE_FR; ++i) {
                    if (live && inside(f0, i)) load8(x + 32 * i, y[i]);
                    else
#pragma unroll
                        for (int j = 0; j < 8; ++j) y[i][j] = 0.0f;
                }
                b[n].set(y);
            } else {
                const bool wide = ((uintptr_t) x & 15) == 0;
#pragma unroll
                for (int i = 0; i < MOE_FR; ++i) {
                    b[n].part[0][i] = v8{};
                    if (live && inside(f0, i)) {
                        if (wide) b[n].part[0][i] = *(const v8 *) (x + 32 * i);
                        else
#pragma unroll
                            for (int j = 0; j < 8; ++j) b[n].part[0][i][j] = x[32 * i + j];
                    }
                }
            }
        }
    };
    v4f_t sum[NT];
    int buf = 0;
    bool fresh = true, more;                                     // the right operands have to be formed anew
    auto step = [&](const v8 (&w)[MOE_FR], v8 (&ahead)[MOE_FR]) __attribute__((always_inline)) {
        nxt = cur;
        more = nxt.next(s, per, u0, u1, passes);
        if (more) request(nxt, ahead);
        if (fresh) columns(cur);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            v4f_t part{};
#pragma unroll
            for (int i = 0; i < MOE_FR; ++i) {
                part = mfma16<TW>(w[i], b[n].part[0][i], part);
                if constexpr (SPLIT) part = mfma16<TW>(w[i], b[n].part[1][i], part);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[n][i] = SPLIT ? part[i] * b[n].back : part[i];
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) s_sum[buf][wave][n][(4 * (lane >> 4) + i) * 16 + col] = sum[n][i];
        lds_sync();
        if (tid < NT * 128) {
            int id = tid;
            asm volatile("" : "+v"(id));                         // (formed here anew: kept over the loop, these would not fit its registers)
            const int n = id >> 7, row = (id >> 3) & 15, f = id & 7, at = cur.c0 + 16 * n + row;
            if (at < cur.count) {
                float g = 0.0f, u = 0.0f;
#pragma unroll
                for (int v = 0; v < MOE_WAVES; ++v) {
                    g += s_sum[buf][v][n][f * 16 + row];
                    u += s_sum[buf][v][n][(f + 8) * 16 + row];
                }
                float (& acc)[2][128 * NT] = s_acc[cur.tile - cur.g0 & (MOE_GROUP - 1)];         // (0 with one pass)
                if (cur.pass) { g += acc[0][id]; u += acc[1][id]; }
                if (cur.pass < passes - 1) { acc[0][id] = g; acc[1][id] = u; }
                else a.h[(int64_t) (s.pos0[cur.t] + at) * a.hs + ((cur.tile >> 2) * 32 + (cur.tile & 3) * 4) + ((f & 4) * 4 + (f & 3))] = z_silu(g) * u;
            }
        }
        buf ^= 1;                                                // (the next tile's sums go elsewhere: one barrier per tile)
        fresh = more && (nxt.pass != cur.pass || nxt.t != cur.t || nxt.c0 != cur.c0);
        cur = nxt;
    };
    v8 w0[MOE_FR], w1[MOE_FR];
    request(cur, w0);
    for (;;) {
        step(w0, w1);
        if (!more) break;
        step(w1, w0);
        if (!more) break;
    }
}

// ---- down
constexpr int MOE_DF = 4, MOE_DW = 4, MOE_DT = 64 * MOE_DW;      // operands of a unit: 128 hidden dims of an expert; waves of a block
// 16 dims of out and all rows per block, over its share of the units (128 hidden dims of an expert), dealt to the waves in turn, so that they read
// the matrix row by row together (in runs of their own: 81 us in place of 78 for 64 rows and 64 experts of 1032 x 2048). The right operand is w h
// of 16 rows that take the expert; its sums go to the rows' places in LDS when the wave turns to other rows. The next unit's weights and h are
// requested before this one is multiplied; as in k_moe_gate_up they are conditional loads, and all but one or two are waited for first. h comes
// from the caches as often as there are tiles of out: of 32 of its columns, the first four of every eight lie before the others, so that the four
// lanes of a row, who have eight columns each, read 64 bytes in a row at a time (64 rows, 64 experts of 1032 x 2048: the layer 211 us in place of
// 217). Without any reads of h it would take 20 us less. (32 dims per block, which halves them, leave registers for two blocks per compute unit in
// place of three: 206 us there, 31 in place of 27 for a layer of 8 x 32; 12 waves over 64 dims, for the near cache's sake: 82 us in place of 78 in
// this kernel.)
template <typename T, typename TW>
__global__ void __launch_bounds__(MOE_DT, 3) k_moe_down(MoeArgs a) {
    typedef typename Vec8<TW>::type v8;
    extern __shared__ __attribute__((aligned(16))) float s_out[];        // [waves][n][16]
    __shared__ int s_last;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    float * out = s_out + wave * a.n * 16;
    for (int i = lane; i < a.n * 4; i += 64) ((v4f_t *) out)[i] = v4f_t{};
    const int n_max = min(a.E, a.n * a.k), turn0 = lane < n_max ? a.touched[lane].turn0 : 0;
    const int n = uniform(&a.table->n)[0], chunks = (a.F + 32 * MOE_DF - 1) / (32 * MOE_DF), units = uniform(&a.table->turns)[0] * chunks;
    const int u0 = (int) ((int64_t) units * blockIdx.y / a.shares), u1 = (int) ((int64_t) units * (blockIdx.y + 1) / a.shares);
    int t0 = __popcll(__ballot(lane < n && turn0 * chunks <= u0)) - 1;   // the expert of unit u0
    for (int i = 64 + lane; i - lane < n; i += 64) t0 += __popcll(__ballot(i < n && a.touched[i].turn0 * chunks <= u0));
    const int k8 = 8 * (lane >> 4), col = lane & 15, d = 16 * (int) blockIdx.x + col;
    const TW * mat = (const TW *) a.down + (int64_t) min(d, a.D - 1) * a.F + k8;
    struct Unit { int u, t, from, to, c0, count; MoeTouched x; };
    auto enter = [&](Unit & c, int t) __attribute__((always_inline)) {
        c.c0 = 0;
        for (c.t = t; c.t < n; ++c.t) {
            c.x = uniform_copy(a.touched + c.t);
            if (c.x.turn0 * chunks >= u1) return false;
            c.count = 0;
#pragma unroll
            for (int i = 0; i < MOE_MASKS; ++i) c.count += __popc(c.x.rows[i]);
            const MoePieces x(u0, u1, c.x.turn0 * chunks, chunks, (c.count + 15) / 16);
            c.u = c.from = x.from + ((wave - c.t * chunks - x.from) & (MOE_DW - 1));
            c.to = x.to;
            if (c.from < c.to) return true;
        }
        return false;
    };
    auto next = [&](Unit & c) __attribute__((always_inline)) {
        if ((c.u += MOE_DW) < c.to) return true;
        if (c.c0 + 16 < c.count) { c.u = c.from; c.c0 += 16; return true; }
        return enter(c, c.t + 1);
    };
    struct Data { v8 w[MOE_DF]; float h[MOE_DF][8], weight; };
    auto request = [&](const Unit & c, Data & x) __attribute__((always_inline)) {
        const int f0 = c.u * 32 * MOE_DF, at = c.c0 + col;
        const TW * p = mat + (int64_t) c.x.e * a.D * a.F + f0;
        const int pos = c.x.pos0 + min(at, c.count - 1);
        const float * h = a.h + (int64_t) pos * a.hs + f0 + 4 * (lane >> 4);
#pragma unroll
        for (int i = 0; i < MOE_DF; ++i) {
            const bool in = f0 + 32 * i + k8 < a.F;
            x.w[i] = d < a.D && in ? *(const v8 *) (p + 32 * i) : v8{};
            v4f_t y0{}, y1{};
            if (at < c.count && in) { y0 = *(const v4f_t *) (h + 32 * i); y1 = *(const v4f_t *) (h + 32 * i + 16); }
#pragma unroll
            for (int j = 0; j < 4; ++j) { x.h[i][j] = y0[j]; x.h[i][4 + j] = y1[j]; }
        }
        x.weight = a.w[pos];
    };
    v4f_t sum{};
    Unit cur, nxt;
    bool more = u0 < u1 && enter(cur, t0);
    auto step = [&](const Data & x, Data & ahead) __attribute__((always_inline)) {
        nxt = cur;
        more = next(nxt);
        if (more) request(nxt, ahead);
        SplitColumn<MOE_DF, TW> b;
        b.set(x.h);
        v4f_t part{};
#pragma unroll
        for (int i = 0; i < MOE_DF; ++i)
#pragma unroll
            for (int q = 0; q < b.PARTS; ++q) part = mfma16<TW>(x.w[i], b.part[q][i], part);
        const float back = b.back * x.weight;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = __builtin_fmaf(part[i], back, sum[i]);
        if (!more || nxt.t != cur.t || nxt.c0 != cur.c0) {
            if (cur.c0 + col < cur.count) {
                v4f_t * to = (v4f_t *) (out + nth_row(cur.x.rows, cur.c0 + col) * 16 + 4 * (lane >> 4));
                *to += sum;
            }
            sum = v4f_t{};
        }
        cur = nxt;
    };
    if (more) {
        Data x0, x1;
        request(cur, x0);
        for (;;) {
            step(x0, x1);
            if (!more) break;
            step(x1, x0);
            if (!more) break;
        }
    }
    __syncthreads();
    auto store = [&](int row, int at, float v) {
        if (a.table->no_number[row >> 5] >> (row & 31) & 1) v = __builtin_nanf("");
        ((T *) a.out)[row * a.os + at] = (T) v;
    };
    for (int i = tid; i < a.n * 16; i += MOE_DT) {
        const int row = i >> 4, at = 16 * (int) blockIdx.x + (i & 15);
        if (at >= a.D) continue;
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < MOE_DW; ++w) v += s_out[w * a.n * 16 + i];
        if (a.shares == 1) store(row, at, v);
        else __hip_atomic_store(a.parts + ((int64_t) blockIdx.y * a.n + row) * a.D + at, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (a.shares == 1) return;
    // the last block of a tile's joins what all have left, in their order. What it joins is stored and read past the caches of one part of the
    // chip, and every wave's stores have arrived before its block takes a ticket (a fence of the whole chip here writes its caches back:
    // 75 us in place of 10 for one row).
    wait_loads_but<0>();
    __syncthreads();
    if (tid == 0) s_last = __hip_atomic_fetch_add(a.tickets + blockIdx.x, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.shares - 1;
    __syncthreads();
    if (!s_last) return;
    for (int i = tid; i < a.n * 16; i += MOE_DT) {
        const int row = i >> 4, at = 16 * (int) blockIdx.x + (i & 15);
        if (at >= a.D) continue;
        float v = 0.0f, x[z2o::MOE_SHARES];                      // (all requested before the first is added)
#pragma unroll
        for (int p = 0; p < z2o::MOE_SHARES; ++p)
            x[p] = p < a.shares ? __hip_atomic_load(a.parts + ((int64_t) p * a.n + row) * a.D + at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0f;
#pragma unroll
        for (int p = 0; p < z2o::MOE_SHARES; ++p) v += x[p];
        store(row, at, v);
    }
}

} // namespace z2d
