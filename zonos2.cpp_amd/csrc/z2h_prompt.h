// z2h_prompt.h — causal attention of packed prompts over their own rows.
//
//   o_r = sum_{i <= r} p_i v_i / sum p_i,  p_i = 2^(x_i - m),  x_i = scale log2(e) q_r.k_i
//
// The running maximum m moves only where a score exceeds it by 2^8, so that sums are seldom scaled. 4 hd flops per row-head and key and 2 hd more for
// the weights' second parts: long prompts are bound by the products (one of 8191 rows, 32 heads of 128, bf16: 730 us, 1.1 PFLOP/s with the
// second parts, which is what a matrix product of 8192 reaches; 24 of 16 to 2000 rows, 32 heads of 64: 97 us, 0.86), short ones by a
// chain of loads and by code that runs once (8 of 256 rows, 16 heads of 128, f16: 14.7 to 16.3 us; one of 37, fp32: 7.8, of which 2.7 are the launch).
// fp32 products reach 151 TFLOP/s: 8191 rows, 32 heads of 128 take 4.1 ms of which they need 3.6; 2000 rows, 16 heads 265 us (109), 16 of 256 rows
// 75 (29), by the cut and by what PromptLoad says.
#pragma once
#include "z2h_common.h"
#include "z2h_ops_rules.h"
#include "z2h_tile.h"

namespace z2d {

typedef float v4f_t __attribute__((ext_vector_type(4)));

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

// A (row, head) in plain fp32, by one wave: 64 keys at a time, a lane each for the scores, then the dims over the lanes. o is the mean by weight of
// the values so far, so that it is finite where they are. A value that is not finite reaches the row whatever its weight. s_q: HD floats of
// the wave's own.
template <int HD, typename T, int E>
__device__ __forceinline__ void prompt_walk(const PromptArgs & a, int first, int row, int head, float * s_q, float (&o)[E]) {
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
    float m = -__builtin_inff(), l = 0.0f;
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
            return;
        }
        const float mn = fmaxf(m, wave_max_f(s));
        const float w0 = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
        float w = s == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(s - mn);
        m = mn;
        const float old = l * w0, sum = old + wave_tree_f(w), inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        l = sum;
        w *= inv;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = is_finite(o[e]) ? o[e] * (old * inv) : o[e];
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

// The lane's part of a row-head's query, whose sign and (fp32) a power of two of whose size are taken out: scores are `c` times the products, in
// units of log2. whole: the largest of all lanes that have a part of the row-head; beside: requests that go out behind the query's.
template <typename T, int QN, typename D, typename W, typename B>
__device__ __forceinline__ float prompt_query(const PromptArgs & a, const T * src, bool live, D dim, float (&x)[QN], W whole, B beside) {
    const bool zero = !live || a.scale == 0.0f;
    const float sign = a.scale < 0.0f ? -1.0f : 1.0f;
    float c = zero ? 1.0f : fabsf(a.scale) * 1.44269504088896341f;
    constexpr int N = 16 / (int) sizeof(T);
    typedef T tv __attribute__((ext_vector_type(N)));
    tv y[QN / N];
    if (((uintptr_t) src & 15) == 0) {
#pragma unroll
        for (int i = 0; i < QN / N; ++i) y[i] = *(const tv *) (src + dim(N * i));
    } else
#pragma unroll
        for (int i = 0; i < QN; ++i) y[i / N][i % N] = src[dim(i)];
    beside();
#pragma unroll
    for (int i = 0; i < QN; ++i) x[i] = (float) y[i / N][i % N];
    float up = sign;
    if constexpr (sizeof(T) == 4) {
        // a power of two keeps the scores of large queries finite, and those of tiny ones from vanishing
        float mx = 0.0f;
#pragma unroll
        for (int i = 0; i < QN; ++i) mx = fmaxf(mx, fabsf(x[i]));
        mx = whole(mx);
        int e = 0;
        if (mx > 0.0f && mx < __builtin_inff()) (void) frexpf(mx, &e);
        e = min(-e, 120);
        up = ldexpf(sign, e);
        c = zero ? 1.0f : ldexpf(c, -e);
    }
#pragma unroll
    for (int i = 0; i < QN; ++i) x[i] = zero ? 0.0f : x[i] * up;
    return fminf(fmaxf(c, 0x1p-126f), 0x1p127f);                  // hidden scores stay -inf whatever the scale
}

// A row-head formed once more in plain fp32, and stored; by one wave
template <int HD, typename T>
__device__ __forceinline__ void prompt_again(const PromptArgs & a, int first, int row, int head, float * s_q, int lane) {
    constexpr int E = HD >= 64 ? HD / 64 : 1;
    float x[E];
    prompt_walk<HD, T>(a, first, row, head, s_q, x);
    T * out = (T *) a.out + row * a.os + (int64_t) head * HD + E * lane;
    if (E * lane < HD)
#pragma unroll
        for (int e = 0; e < E; ++e) out[e] = (T) x[e];
}

// Rows of T in LDS, stored as they are with their 16-byte pieces permuted by row: keys so that 32 rows' pieces of the same dims take all
// banks, values so that transposing reads (16 bits) or two rows 4 apart (fp32) do.
template <int HD, typename T>
struct Rows {
    static constexpr int N = 16 / (int) sizeof(T), NC = HD / N, RP = NC >= 16 ? 1 : 16 / NC;   // elements and pieces, rows per 256 bytes
    static __device__ __forceinline__ int k_perm(int row) { return (row / RP) & (NC < 16 ? NC - 1 : 15); }
    static __device__ __forceinline__ int v_perm(int row) {
        if constexpr (sizeof(T) == 2) return 4 * ((row / RP) & (NC / 4 - 1));
        else return NC >= 16 ? 8 * ((row >> 2) & 1) : 0;
    }
    static __device__ __forceinline__ int k_at(int row, int piece) { return row * HD + (piece ^ k_perm(row)) * N; }
    static __device__ __forceinline__ int v_at(int row, int piece) { return row * HD + (piece ^ v_perm(row)) * N; }
};

// One wave's 32 row-heads against 32 NT keys. S^T = K Q^T leaves a lane one row-head's scores (16 of 32 keys, the lane 32 away the others) in
// the order in which they are the right operand of O^T = V^T P^T: weights never move between lanes.
template <int HD, typename T> struct PromptMath;

// 16 bits: v_mfma_f32_32x32x16; the weights meet the values as two numbers of the type, the second carrying what the first's rounding leaves.
// One alone (2^-12, 2^-9 on average) would err as much as the output's own rounding over any number of keys.
template <int HD, typename T>
struct PromptMath {
    static constexpr int NT = 2, KS = HD / 16, DT = HD / 32, BIAS = __is_same(T, _Float16) ? 6 : 0;
    typedef typename Vec8<T>::type v8;
    typedef Rows<HD, T> R;
    v8 q[KS], p[2 * NT], pl[2 * NT];
    int k_place[KS], v_place[DT];

    __device__ __forceinline__ void init(const float (&x)[KS * 8], int lane) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int j = 0; j < 8; ++j) q[ks][j] = (T) x[8 * ks + j];
        const int i16 = lane & 15, r = 4 * (lane >> 5) + (i16 >> 2);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) k_place[ks] = R::k_at(lane & 31, 2 * ks + (lane >> 5));
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const int d = 32 * dt + 16 * ((lane >> 4) & 1) + 4 * (i16 & 3);
            v_place[dt] = R::v_at(r, d >> 3) + (d & 7);
        }
    }
    // dims that the lane holds of its query, in the order of init's x
    static __device__ __forceinline__ int dim(int i, int lane) { return 16 * (i >> 3) + 8 * (lane >> 5) + (i & 7); }
    static constexpr int QN = KS * 8;

    // (keys are requested four products ahead: the compiler by itself reads, waits and multiplies in turn)
    template <typename B>
    __device__ __forceinline__ void scores(v16f_t (&s)[NT], const T * sk, B beside) const {
        constexpr int AHEAD = 4 < NT * KS ? 4 : NT * KS;
        v8 f[AHEAD];
        auto read = [&](int i) __attribute__((always_inline)) { return *(const v8 *) (sk + k_place[i / NT] + 32 * (i % NT) * HD); };
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n] = v16f_t{};
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) f[i] = read(i);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < NT * KS; ++i) {
            s[i % NT] = mfma32<T>(f[i % AHEAD], q[i / NT], s[i % NT]);
            if (i + AHEAD < NT * KS) f[i % AHEAD] = read(i + AHEAD);
            beside(i, NT * KS);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    __device__ __forceinline__ float weigh(v16f_t (&s)[NT], float c, float mu) {
        float sum = 0.0f;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                typedef typename Pair<float>::type f2;
                typedef typename Pair<T>::type c2;
                const f2 w = {__builtin_amdgcn_exp2f(__builtin_fmaf(s[n][i], c, -mu)), __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][i + 1], c, -mu))};
                const c2 hi = __builtin_convertvector(w, c2);
                const c2 lo = __builtin_convertvector(two_rest(w, hi), c2);
                p[2 * n + (i >> 3)][i & 7] = hi[0];
                p[2 * n + (i >> 3)][(i & 7) + 1] = hi[1];
                pl[2 * n + (i >> 3)][i & 7] = lo[0];
                pl[2 * n + (i >> 3)][(i & 7) + 1] = lo[1];
                sum += w[0];
                sum += w[1];
            }
        return sum;
    }
    // V^T operand of 16 keys from LDS row r0 on, dims 32 dt ..: lanes 16 g + i read keys 4 (g / 2) + i / 4, dims 16 (g & 1) + 4 (i & 3)
    __device__ __forceinline__ v8 values(const T * sv, int r0, int dt) const {
        const T * at = sv + v_place[dt] + r0 * HD;
        typedef __attribute__((address_space(3))) s4_t lds4;
        const s4_t x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *) at);
        const s4_t x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *) (at + 8 * HD));
        return __builtin_bit_cast(v8, __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    __device__ __forceinline__ void add(v16f_t (&o)[DT], const T * sv) const {
#pragma unroll
        for (int t = 0; t < 2 * NT; ++t)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const v8 v = values(sv, 16 * t, dt);
                o[dt] = mfma32<T>(v, p[t], o[dt]);
                o[dt] = mfma32<T>(v, pl[t], o[dt]);
            }
    }
};

// fp32: v_mfma_f32_32x32x2, products and weights in fp32 (1/16 of the 16-bit rate).
template <int HD>
struct PromptMath<HD, float> {
    static constexpr int NT = 1, DT = HD / 32, BIAS = 0, QN = HD / 2;
    typedef Rows<HD, float> R;
    float q[QN];
    float p[16];
    int k_row, k_xor, v_at[DT];
    typedef float v4 __attribute__((ext_vector_type(4)));

    __device__ __forceinline__ void init(const float (&x)[QN], int lane) {
#pragma unroll
        for (int i = 0; i < QN; ++i) q[i] = x[i];
        k_row = (lane & 31) * HD;
        k_xor = (lane >> 5) ^ R::k_perm(lane & 31);              // (of the pieces 2 j + half, the row's permutation)
        const int row = 4 * (lane >> 5);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) v_at[dt] = R::v_at(row, 8 * dt + ((lane & 31) >> 2)) + (lane & 3);
    }
    static __device__ __forceinline__ int dim(int i, int lane) { return 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3); }
    template <typename B>
    __device__ __forceinline__ void scores(v16f_t (&s)[NT], const float * sk, B beside) const {
        s[0] = v16f_t{};
#pragma unroll
        for (int j = 0; j < HD / 8; ++j) {
            beside(j, HD / 8);
            const v4 k = *(const v4 *) (sk + k_row + ((2 * j) ^ k_xor) * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(k[e], q[4 * j + e], s[0], 0, 0, 0);
        }
    }
    __device__ __forceinline__ float weigh(v16f_t (&s)[NT], float c, float mu) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][i], c, -mu));
            sum += p[i];
        }
        return sum;
    }
    // register i of a lane's half h is key 8 (i / 4) + 4 h + i % 4
    __device__ __forceinline__ void add(v16f_t (&o)[DT], const float * sv) const {
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
                o[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(sv[v_at[dt] + (8 * (i >> 2) + (i & 3)) * HD], p[i], o[dt], 0, 0, 0);
    }
};

// A wave's rows and running sums.
template <int HD, typename T>
struct PromptWave {
    typedef PromptMath<HD, T> M;
    M math;
    v16f_t o[M::DT];
    float m, l, c;                                               // m includes -BIAS: f16 weights up to 2^14, kept to 2^-24
    int vis;                                                     // keys that the lane's row sees

    // row-heads first_rh .. + 31 of rows row0 .. row0 + rows - 1, whose first sees `before` + 1 keys
    template <typename B>
    __device__ __forceinline__ void init(const PromptArgs & a, int row0, int rows, int before, int g, int first_rh, int lane, B beside) {
        const int group = a.n_head / a.nkv, rh = first_rh + (lane & 31);
        const bool live = rh < rows * group;
        const int r = live ? rh / group : 0, head = g * group + (live ? rh % group : 0);
        const T * src = (const T *) a.q + (row0 + r) * a.qs + (int64_t) head * HD;
        vis = live ? before + r + 1 : 0x7fffffff;
        float x[M::QN];
        c = prompt_query<T, M::QN>(a, src, live, [&](int i) { return M::dim(i, lane); }, x, [](float mx) { return fmaxf(mx, other_half(mx)); }, beside);
        math.init(x, lane);
        m = -__builtin_inff();
        l = 0.0f;
#pragma unroll
        for (int dt = 0; dt < M::DT; ++dt) o[dt] = v16f_t{};
    }

    // keys key0 .. key0 + 32 NT (counted from the sequence's first) in LDS; those at or behind `vis` are hidden
    template <typename B>
    __device__ __forceinline__ void step(const T * sk, const T * sv, int key0, int lane, B beside) {
        constexpr int NT = M::NT;
        v16f_t s[NT];
        math.scores(s, sk, beside);
        if (__any(key0 + 32 * NT > vis)) {
            const int h4 = 4 * (lane >> 5);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (key0 + 32 * n + 8 * (i >> 2) + h4 + (i & 3) >= vis) s[n][i] = -__builtin_inff();
        }
        float mx = s[0][0];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[n][i]);
        mx = fmaxf(mx, other_half(mx)) * c;
        // the maximum moves only where a score exceeds it by 2^8: rarely behind the first keys
        const bool up = mx > m + (8.0f + M::BIAS);
        if (__any(up)) {
            const float mn = up ? mx - M::BIAS : m;
            const float w = mn == m || m == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(m - mn);   // (nothing to scale yet)
            m = mn;
            l *= w;
#pragma unroll
            for (int dt = 0; dt < M::DT; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[dt][i] *= w;
        }
        l += math.weigh(s, c, m == -__builtin_inff() ? 0.0f : m);
        math.add(o, sv);
    }

    // The sums over other keys of the same row-heads, four at a time. (A part without weights may hold anything: NaN, which is formed once more.)
    template <typename F>
    __device__ __forceinline__ void join(float m2, float l2, F o2) {
        const float mn = fmaxf(m, m2);
        const float w = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - mn), w2 = m2 == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m2 - mn);
        // (both of a row-head's lanes have the same maxima)
        m = mn;
        l = l * w + l2 * w2;
#pragma unroll
        for (int dt = 0; dt < M::DT; ++dt)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const v4f_t x = o2(dt, i);
#pragma unroll
                for (int j = 0; j < 4; ++j) o[dt][i + j] = __builtin_fmaf(o[dt][i + j], w, x[j] * w2);
            }
    }

    // What is not finite meets both parts of a weight, and hidden rows' weights of 0: the product is then NaN where the definition has infinity or
    // leaves it out, and sums of weights up to 2^8 (f16: 2^14) times the largest values may be infinite where their mean is not. So a row-head
    // that holds either is formed once more, in plain fp32: a wave's up to 32 one after the other, so that a value that is no number in the
    // first of 2000 rows (16 heads of 128) costs 14 ms in place of 0.05, in the first of 8191 (32 heads) 148 in place of 0.76.
    // The others' rows go through LDS, so that 16 bytes per lane make whole rows of the output. s_own: 32 HD T of LDS of the wave's own.
    // (What runs once per block is as little code as can be: a new instruction line of 64 bytes takes 70 ns.)
    __device__ __forceinline__ void store(const PromptArgs & a, int first, int row0, int rows, int g, int first_rh, int lane, T * s_own) {
        typedef Rows<HD, T> R;
        const int group = a.n_head / a.nkv, heads = rows * group, rh = first_rh + (lane & 31);
        l += other_half(l);
        float odd[2] = {l * 0.0f, 0.0f};                         // 0, or NaN where any is not finite
#pragma unroll
        for (int dt = 0; dt < M::DT; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) odd[i & 1] = __builtin_fmaf(o[dt][i], 0.0f, odd[i & 1]);
        odd[0] += odd[1];
        odd[0] += other_half(odd[0]);
        unsigned again = (unsigned) __ballot(rh < heads && odd[0] != 0.0f);
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int dt = 0; dt < M::DT; ++dt)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int d = 32 * dt + 2 * i + 4 * (lane >> 5);
                typedef T t4 __attribute__((ext_vector_type(4)));
                *(t4 *) (s_own + R::k_at(lane & 31, d / R::N) + d % R::N) = __builtin_convertvector(
                    (v4f_t{o[dt][i] * inv, o[dt][i + 1] * inv, o[dt][i + 2] * inv, o[dt][i + 3] * inv}), t4);
            }
        wait_lds();
        const bool wide = (uintptr_t) a.out % 16 == 0 && a.os * (int64_t) sizeof(T) % 16 == 0;
        const float part = 1.0f / group;
#pragma unroll 2
        for (int j = 0; j < R::NC / 2; ++j) {
            const int row = (64 * j + lane) / R::NC, piece = lane % R::NC, at = first_rh + row;
            const int r = (int) ((at + 0.5f) * part);            // (at / group: both are below 2^8)
            typedef T tv __attribute__((ext_vector_type(R::N)));
            const tv x = *(const tv *) (s_own + R::k_at(row, piece));
            if (at >= heads || again >> row & 1) continue;
            T * out = (T *) a.out + (row0 + r) * a.os + (int64_t) (g * group + at - r * group) * HD + piece * R::N;
            if (wide) *(tv *) out = x;
            else
#pragma unroll
                for (int e = 0; e < R::N; ++e) out[e] = x[e];
        }
        for (; again; again &= again - 1) {
            const int at = first_rh + __builtin_ctz(again);
            prompt_again<HD, T>(a, first, row0 + at / group, g * group + at % group, (float *) s_own, lane);
        }
    }
};

// Brings 16 rows of K or V to LDS at a time. ALIGNED: every piece is 16 bytes that may be loaded at once, straight to LDS; else by elements.
// (fp32: whether a wave brings keys or values in a part is not known before it runs, and the compiler keeps the pieces' places in scratch memory, 12
// bytes per lane, up to 72 where they are not aligned; reading them waits for the loads to LDS before.)
template <int HD, typename T, bool ALIGNED>
struct PromptLoad {
    typedef Rows<HD, T> R;
    static constexpr int ROWS = 64 / R::NC, N = 16 / ROWS;       // rows per instruction, instructions for 16 rows
    const T * k, * v;                                            // the key head's first row of the sequence
    int64_t ks, vs;
    int last, row, piece_k[N], piece_v[N];                       // of the lane: its row, its pieces' first elements
    __device__ __forceinline__ PromptLoad(const PromptArgs & a, int first, int n_keys, int g, int lane)
        : k((const T *) a.k + first * a.ks + (int64_t) g * HD), v((const T *) a.v + first * a.vs + (int64_t) g * HD), ks(a.ks), vs(a.vs),
          last(n_keys - 1), row(lane / R::NC) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            piece_k[i] = ((lane % R::NC) ^ R::k_perm(i * ROWS + row)) * R::N;
            piece_v[i] = ((lane % R::NC) ^ R::v_perm(i * ROWS + row)) * R::N;
        }
    }
    static __device__ __forceinline__ void move(const T * from, T * to, int lane) {
        if constexpr (ALIGNED) to_lds(from, to);
        else {
            T x[R::N];
#pragma unroll
            for (int j = 0; j < R::N; ++j) x[j] = from[j];
#pragma unroll
            for (int j = 0; j < R::N; ++j) to[lane * R::N + j] = x[j];
        }
    }
    // rows key .. key + 15 (a multiple of 16) to the rows of LDS at `to`; rows behind the sequence's end are its last one again
    __device__ __forceinline__ void keys16(int key, T * to, int lane) const {
#pragma unroll
        for (int i = 0; i < N; ++i) move(k + min(key + i * ROWS + row, last) * ks + piece_k[i], to + i * ROWS * HD, lane);
    }
    __device__ __forceinline__ void values16(int key, T * to, int lane) const {
#pragma unroll
        for (int i = 0; i < N; ++i) move(v + min(key + i * ROWS + row, last) * vs + piece_v[i], to + i * ROWS * HD, lane);
    }
};

// What a block has to do: rows row0 .. row0 + rows - 1 of a sequence that begins at row `first`, with key head g. Long tiles come first.
struct PromptTile { int first, row0, rows, g; };
__device__ __forceinline__ PromptTile prompt_tile(const PromptArgs & a, int tile_rows, int lane) {
    const int64_t id = a.block0 + blockIdx.x;
    const int64_t slot = z2o::prompt_slots(a.n_rows, a.n_seq, tile_rows) - 1 - id / a.nkv;
    PromptTile t;
    t.g = (int) (id % a.nkv);
    const int s = prompt_seq(a, slot, tile_rows, lane), start = prompt_start(a, s), end = prompt_start(a, s + 1);
    const int64_t at = start + (slot - z2o::prompt_slot(start, s, tile_rows)) * tile_rows;
    t.first = start;
    t.row0 = (int) min(max(at, (int64_t) 0), (int64_t) a.n_rows);
    t.rows = max(0, min(tile_rows, end - t.row0));
    if (at < start) t.rows = 0;
    return t;
}

// ---- few tiles: 16 row-heads per block, the keys dealt to its four waves
// the largest (or the sum) of a column's values, whose four lanes are 16 apart
template <bool SUM>
__device__ __forceinline__ float column(float v) {
    auto both = [](float a, float b) { return SUM ? a + b : fmaxf(a, b); };
    v = both(v, other_half(v));
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    const unsigned r0 = r[0], r1 = r[1];
    return both(__builtin_bit_cast(float, r0), __builtin_bit_cast(float, r1));
}
template <typename T, int N, bool ALIGNED>
__device__ __forceinline__ void load_piece(const T * p, T (&x)[N]) {
    if constexpr (ALIGNED) {
        typedef T tv __attribute__((ext_vector_type(N)));
        const tv y = *(const tv *) p;
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = y[i];
    } else
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = p[i];
}

// One wave's 16 row-heads (a lane: row-head lane % 16, group g = lane / 16 of four) against KEYS keys at a time: keys from memory to registers, 16-bit
// values through LDS (transposed as they are read), fp32 values to registers too.
template <int HD, typename T, bool ALIGNED>
struct SmallMath {
    static constexpr int KEYS = 32, KS = HD / 32, DT = HD / 16, BIAS = __is_same(T, _Float16) ? 6 : 0, QN = HD / 4;
    static constexpr int NC = HD / 8, RP = NC >= 16 ? 1 : 16 / NC, ROWS = 64 / NC, LDS = 2 * KEYS * HD;
    typedef typename Vec8<T>::type v8;
    v8 q[KS];
    struct Data { v8 k[2][KS]; };
    static __device__ __forceinline__ int perm(int row) { return 2 * ((row / RP) & (NC / 2 - 1)); }
    static __device__ __forceinline__ int dim(int i, int g) { return 32 * (i >> 3) + 8 * g + (i & 7); }
    // dim of register i of o's tile t
    static __device__ __forceinline__ int out_dim(int t, int i, int g) { return 16 * t + 4 * g + i; }
    __device__ __forceinline__ void init(const float (&x)[QN]) {
#pragma unroll
        for (int i = 0; i < QN; ++i) q[i >> 3][i & 7] = (T) x[i];
    }
    __device__ __forceinline__ void request(Data & d, const T * k, int64_t ks, const T * v, int64_t vs, int key, int last, T * lds, int lane) const {
        const int l = lane & 15, g = lane >> 4;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                T x[8];
                load_piece<T, 8, ALIGNED>(k + min(key + 16 * t + l, last) * ks + 32 * i + 8 * g, x);
#pragma unroll
                for (int j = 0; j < 8; ++j) d.k[t][i][j] = x[j];
            }
        const int row = lane / NC, piece = lane % NC;
#pragma unroll
        for (int r = 0; r < KEYS; r += ROWS) {
            const T * from = v + min(key + r + row, last) * vs + (piece ^ perm(r + row)) * 8;
            if constexpr (ALIGNED) to_lds(from, lds + r * HD);
            else {
                T x[8];
                load_piece<T, 8, false>(from, x);
#pragma unroll
                for (int j = 0; j < 8; ++j) lds[r * HD + lane * 8 + j] = x[j];
            }
        }
    }
    // register i of s: key key0 + key_of(i, g)
    static constexpr int SN = 8;
    static __device__ __forceinline__ int key_of(int i, int g) { return 16 * (i >> 2) + 4 * g + (i & 3); }
    __device__ __forceinline__ void scores(const Data & d, float (&s)[SN]) const {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            v4f_t x{};
#pragma unroll
            for (int i = 0; i < KS; ++i) x = mfma16(d.k[t][i], q[i], x);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[4 * t + i] = x[i];
        }
    }
    static __device__ __forceinline__ v4f_t mfma16(v8 a, v8 b, v4f_t c) {
        if constexpr (__is_same(T, _Float16)) return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    __device__ __forceinline__ void add(const Data &, const float (&w)[SN], v4f_t (&o)[DT], const T * lds, int lane) const {
        v8 hi, lo;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            typedef typename Pair<float>::type f2;
            typedef typename Pair<T>::type c2;
            const f2 y = {w[i], w[i + 1]};
            const c2 h = __builtin_convertvector(y, c2), r = __builtin_convertvector(two_rest(y, h), c2);
            hi[i] = h[0]; hi[i + 1] = h[1];
            lo[i] = r[0]; lo[i + 1] = r[1];
        }
        const int l = lane & 15, row = 4 * (lane >> 4) + (l >> 2);
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            const int d = 16 * t + 4 * (l & 3);
            typedef __attribute__((address_space(3))) s4_t lds4;
            // (rows 16 apart are permuted alike)
            const T * at = lds + row * HD + ((d >> 3) ^ perm(row)) * 8 + (d & 7);
            const s4_t x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *) at);
            const s4_t x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *) (at + 16 * HD));
            const v8 v = __builtin_bit_cast(v8, __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7));
            o[t] = mfma16(v, hi, o[t]);
            o[t] = mfma16(v, lo, o[t]);
        }
    }
};
template <int HD, bool ALIGNED>
struct SmallMath<HD, float, ALIGNED> {
    static constexpr int KEYS = 16, DT = HD / 16, BIAS = 0, QN = HD / 4, SN = 4, LDS = HD * 16;
    static constexpr int VE = HD >= 64 ? 4 : 2, VQ = DT / VE;     // values: VQ pieces of VE dims of a row per lane
    float q[QN];
    struct Data { float k[QN], v[4][VQ][VE]; };
    static __device__ __forceinline__ int dim(int i, int g) { return 16 * (i >> 2) + 4 * g + (i & 3); }
    static __device__ __forceinline__ int out_dim(int t, int i, int g) { return t / VE * 16 * VE + (4 * g + i) * VE + t % VE; }
    static __device__ __forceinline__ int key_of(int i, int g) { return 4 * g + i; }
    __device__ __forceinline__ void init(const float (&x)[QN]) {
#pragma unroll
        for (int i = 0; i < QN; ++i) q[i] = x[i];
    }
    __device__ __forceinline__ void request(Data & d, const float * k, int64_t ks, const float * v, int64_t vs, int key, int last, float *, int lane) const {
        const int l = lane & 15, g = lane >> 4;
        const float * row = k + min(key + l, last) * ks + 4 * g;
#pragma unroll
        for (int j = 0; j < QN / 4; ++j) {
            float x[4];
            load_piece<float, 4, ALIGNED>(row + 16 * j, x);
#pragma unroll
            for (int e = 0; e < 4; ++e) d.k[4 * j + e] = x[e];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < VQ; ++j) load_piece<float, VE, ALIGNED>(v + min(key + 4 * g + i, last) * vs + 16 * VE * j + VE * l, d.v[i][j]);
    }
    __device__ __forceinline__ void scores(const Data & d, float (&s)[SN]) const {
        v4f_t x[4] = {};                                         // (four chains: a product waits for the one before it in its own)
#pragma unroll
        for (int i = 0; i < QN; ++i) x[i & 3] = __builtin_amdgcn_mfma_f32_16x16x4f32(d.k[i], q[i], x[i & 3], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = (x[0][i] + x[1][i]) + (x[2][i] + x[3][i]);
    }
    __device__ __forceinline__ void add(const Data & d, const float (&w)[SN], v4f_t (&o)[DT], const float *, int) const {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int t = 0; t < DT; ++t) o[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(d.v[i][t / VE][t % VE], w[i], o[t], 0, 0, 0);
    }
};

// The next keys and values are requested before the present step's products. Those with the keys go on beside them; before those with 16-bit values the
// compiler waits for the requested ones too, since it takes both buffers, halves of one array, for the same memory. fp32 heads of 128 take all
// 256 registers and keep 8 more values in scratch memory (36 bytes per lane), read again in each step.
template <int HD, typename T, bool ALIGNED>
__global__ void __launch_bounds__(256, 2) k_prompt_small(PromptArgs a) {
    typedef SmallMath<HD, T, ALIGNED> M;
    constexpr int DT = M::DT, SN = M::SN;
    // of every wave: two buffers of values, then its sums [16][HD]
    constexpr int BYTES = M::LDS * (int) sizeof(T) > 16 * HD * 4 ? M::LDS * (int) sizeof(T) : 16 * HD * 4;
    __shared__ __attribute__((aligned(1024))) uint8_t s_lds[4][BYTES];
    __shared__ float s_m[4][16], s_l[4][16];
    __shared__ int s_again[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), group = a.n_head / a.nkv, col = lane & 15, g = lane >> 4;
    const PromptTile t = prompt_tile(a, z2o::small_rows(group), lane);
    if (t.rows <= 0) return;
    const int before = t.row0 - t.first, n_keys = before + t.rows, heads = t.rows * group;
    const T * k = (const T *) a.k + t.first * a.ks + (int64_t) t.g * HD, * v = (const T *) a.v + t.first * a.vs + (int64_t) t.g * HD;
    T * lds = (T *) s_lds[wave];
    typename M::Data d0, d1;
    M math;
    int key = M::KEYS * wave;
    // the queries
    const bool live = col < heads;
    const int r = live ? col / group : 0, head = t.g * group + (live ? col % group : 0), vis = before + r + 1;
    float c, m = -__builtin_inff(), l = 0.0f;
    {
        float x[M::QN];
        c = prompt_query<T, M::QN>(a, (const T *) a.q + (t.row0 + r) * a.qs + (int64_t) head * HD, live, [&](int i) { return M::dim(i, g); }, x,
                                   [](float mx) { return column<false>(mx); },
                                   [&]() __attribute__((always_inline)) { if (key < n_keys) math.request(d0, k, a.ks, v, a.vs, key, n_keys - 1, lds, lane); });
        math.init(x);
    }
    v4f_t o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) o[i] = v4f_t{};
    auto step = [&](typename M::Data & d, typename M::Data & ahead, T * here, T * there) __attribute__((always_inline)) {
        wait_loads_but<0>();                                     // (the values in LDS)
        const bool more = key + 4 * M::KEYS < n_keys;
        if (more) math.request(ahead, k, a.ks, v, a.vs, key + 4 * M::KEYS, n_keys - 1, there, lane);
        float s[SN];
        math.scores(d, s);
        float mx = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < SN; ++i) {
            if (key + M::key_of(i, g) >= vis) s[i] = -__builtin_inff();
            mx = fmaxf(mx, s[i]);
        }
        mx = column<false>(mx) * c;
        const bool up = mx > m + (8.0f + M::BIAS);
        if (__any(up)) {
            const float mn = up ? mx - M::BIAS : m;
            const float w = mn == m || m == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= w;
#pragma unroll
            for (int i = 0; i < DT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[i][j] *= w;
        }
        const float mu = m == -__builtin_inff() ? 0.0f : m;
        float w[SN];
#pragma unroll
        for (int i = 0; i < SN; ++i) {
            w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -mu));
            l += w[i];
        }
        math.add(d, w, o, here, lane);
        key += 4 * M::KEYS;
    };
    T * other = lds + M::LDS / 2;
    while (key < n_keys) {
        step(d0, d1, lds, other);
        if (key >= n_keys) break;
        step(d1, d0, other, lds);
    }
    // ---- the waves' sums together, 16 threads per row-head
    l = column<true>(l);
    wait_lds();
    float * mine = (float *) s_lds[wave];
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) mine[col * HD + ((M::out_dim(i, j, g) + 4 * col) & (HD - 1))] = o[i][j];
    if (g == 0) { s_m[wave][col] = m; s_l[wave][col] = l; }
    if (tid < 16) s_again[tid] = 0;
    __syncthreads();
    const int rh = tid >> 4;
    const float mm = fmaxf(fmaxf(s_m[0][rh], s_m[1][rh]), fmaxf(s_m[2][rh], s_m[3][rh]));
    float f[4], sum = 0.0f, y[HD / 16];
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) y[i] = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        f[w] = s_m[w][rh] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(s_m[w][rh] - mm);
        sum = __builtin_fmaf(f[w], s_l[w][rh], sum);
        if (s_m[w][rh] != -__builtin_inff() || s_l[w][rh] != 0.0f)
#pragma unroll
            for (int i = 0; i < HD / 16; ++i) y[i] = __builtin_fmaf(f[w], ((const float *) s_lds[w])[rh * HD + (((tid & 15) * (HD / 16) + i + 4 * rh) & (HD - 1))], y[i]);
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    bool odd = !is_finite(sum);
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) odd |= !is_finite(y[i]);
    if (odd) s_again[rh] = 1;
    __syncthreads();
    if (rh < heads && !s_again[rh]) {
        T * out = (T *) a.out + (t.row0 + rh / group) * a.os + (int64_t) (t.g * group + rh % group) * HD + (tid & 15) * (HD / 16);
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) out[i] = (T) (y[i] * inv);
    }
    for (int i = wave; i < heads; i += 4)
        if (s_again[i]) prompt_again<HD, T>(a, t.first, t.row0 + i / group, t.g * group + i % group, (float *) s_lds[wave], lane);
}

// ---- many tiles: 128 row-heads per block
// Four waves of 32 row-heads each over the same keys, 32 NT at a time in LDS, the next ones on their way into the other buffer. HALVES 2: eight
// waves, the second four over every other 32 NT keys; their sums are joined in LDS.
template <int HD, typename T, bool ALIGNED, int HALVES>
__global__ void __launch_bounds__(256 * HALVES, 2) k_prompt(PromptArgs a) {
    constexpr int KEYS = 32 * PromptMath<HD, T>::NT, DT = PromptMath<HD, T>::DT;
    __shared__ __attribute__((aligned(1024))) T s_k0[HALVES][KEYS * HD], s_k1[HALVES][KEYS * HD], s_v0[HALVES][KEYS * HD], s_v1[HALVES][KEYS * HD];
    __shared__ float s_ml[HALVES == 2 ? 4 : 1][2][64];
    const int lane = threadIdx.x & 63, group = a.n_head / a.nkv;
    const int wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6) & 3, half = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 8);
    const PromptTile t = prompt_tile(a, z2o::tile_rows(group), lane);
    if (t.rows <= 0) return;
    const int before = t.row0 - t.first, n_keys = before + t.rows;
    const PromptLoad<HD, T, ALIGNED> load(a, t.first, n_keys, t.g, lane);
    // this wave's part i of 2 KEYS / 64 of the rows to bring: 16 of K or of V
    constexpr int PARTS = KEYS / 32;
    auto bring_part = [&](int i, int key, T * sk, T * sv) __attribute__((always_inline)) {
        const int part = 4 * i + wave;
        if (part < KEYS / 16) load.keys16(key + 16 * part, sk + 16 * part * HD, lane);
        else load.values16(key + 16 * (part - KEYS / 16), sv + 16 * (part - KEYS / 16) * HD, lane);
    };
    auto bring = [&](int key, T * sk, T * sv) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PARTS; ++i) bring_part(i, key, sk, sv);
    };
    int key = half * KEYS;
    PromptWave<HD, T> w;
    w.init(a, t.row0, t.rows, before, t.g, 32 * wave, lane, [&]() __attribute__((always_inline)) {
        if (key < n_keys) bring(key, s_k0[half], s_v0[half]);
    });
    // the wave's rows see keys up to `mine`
    const int mine = 32 * wave < t.rows * group ? before + min(t.rows, (32 * wave + 31) / group + 1) : 0;
    auto stage = [&](const T * sk, const T * sv, T * ok, T * ov) __attribute__((always_inline)) {
        wait_loads_but<0>();
        __syncthreads();
        const int next = key + HALVES * KEYS;
        if (key < mine)
            w.step(sk, sv, key, lane, [&](int i, int n) __attribute__((always_inline)) {
                if (i % (n / PARTS) == 0 && next < n_keys) bring_part(i / (n / PARTS), next, ok, ov);
            });
        else if (next < n_keys) bring(next, ok, ov);
        key += HALVES * KEYS;
    };
    // (both halves take the first one's number of steps: they share the barriers)
    for (int at = 0; at < n_keys;) {
        stage(s_k0[half], s_v0[half], s_k1[half], s_v1[half]);
        if ((at += HALVES * KEYS) >= n_keys) break;
        stage(s_k1[half], s_v1[half], s_k0[half], s_v0[half]);
        at += HALVES * KEYS;
    }
    __syncthreads();
    if constexpr (HALVES == 2) {
        float * to = (float *) (wave < 2 ? wave ? s_k1[0] : s_k0[0] : wave == 2 ? s_v0[0] : s_v1[0]);    // 32 HD floats each at least
        if (half) {
            s_ml[wave][0][lane] = w.m;
            s_ml[wave][1][lane] = w.l;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int i = 0; i < 16; i += 4) *(v4f_t *) (to + ((16 * dt + i) * 16 + lane) * 4) = v4f_t{w.o[dt][i], w.o[dt][i + 1], w.o[dt][i + 2], w.o[dt][i + 3]};
        }
        __syncthreads();
        if (half) return;
        w.join(s_ml[wave][0][lane], s_ml[wave][1][lane], [&](int dt, int i) { return *(const v4f_t *) (to + ((16 * dt + i) * 16 + lane) * 4); });
        wait_lds();
        w.store(a, t.first, t.row0, t.rows, t.g, 32 * wave, lane, (T *) to);
    } else {
        constexpr int PER = KEYS / 32;                           // waves' rows that a buffer holds
        T * to = wave / PER == 0 ? s_k0[0] : wave / PER == 1 ? s_k1[0] : wave / PER == 2 ? s_v0[0] : s_v1[0];
        w.store(a, t.first, t.row0, t.rows, t.g, 32 * wave, lane, to + wave % PER * 32 * HD);
    }
}

} // namespace z2d
