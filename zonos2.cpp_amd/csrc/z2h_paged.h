// z2h_paged.h — attention of a batch of sequences over a paged cache, groups of which share a prefix.
//
//   o = sum_i p_i v_i / sum_i p_i,  p_i = 2^(x_i - m),  x_i = scale log2(e) q.k_i
// in one pass over the keys with a running m; partial (m, sum p, sum p v) of disjoint keys join by scaling to the larger m. So a
// row's keys may be cut anywhere: its group's shared prefix is walked once for all rows of the group (their queries side
// by side in one product), the rest of its keys with its own sequence, and both in chunks of alike work.
//   k_paged_plan     one block: tiles, chunks and the places of their partial results, from the lengths (z2h_ops_rules.h)
//   k_paged_attn     one item = (tile of query rows, key head, chunk of keys) per block
//   k_paged_join     one wave per (row, head): its chunks' partial results
// Single tokens are bound by reading the cache once; groups of many rows and prompt chunks by the products and the exponentials.
#pragma once
#include "z2h_common.h"
#include "z2h_ops_rules.h"

namespace z2d {

constexpr int PLAN_MAGIC = 0x50414745;
enum { PH_MAGIC = 0, PH_ROWS, PH_HEADS, PH_GROUPS, PH_SEQS, PH_KV_HEADS, PH_ITEMS, PH_CHUNK };

// per row: what it sees, and where its partial results are: chunk c, key head g, head h of the group at
// base + c * step + g * (step / key heads) + h, in its group's prefix and in its own keys
struct PlanRow { int vis, pre_base, pre_n, pre_step, own_base, own_n, own_step, spare; };
struct PlanTile { int row0, rows, key0, key1, seq, chunks, item0, part0; };
struct PlanItem { int row0, rows, key0, key1, seq, head, part0, direct; };
static_assert(sizeof(PlanRow) == 32 && sizeof(PlanTile) == 32 && sizeof(PlanItem) == 32, "workspace layout");

struct PlanArgs {
    const int32_t * row_start, * kv_len, * group_start, * prefix_len;
    int n_seq, n_rows, n_group, n_head, nkv, cap, target;
    int32_t * head;
    PlanRow * rows;
    PlanTile * tiles;
    PlanItem * items;
    int max_tiles, max_items, max_parts;
};

// the last index i of [0, n) with start[i] <= x (start ascending; -1: none)
__device__ __forceinline__ int last_at_or_before(const int32_t * start, int n, int x) {
    int lo = -1, hi = n;
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (start[m] <= x) lo = m; else hi = m;
    }
    return lo;
}

constexpr int PLAN_T = 1024;
// sum of v over the lower threads of the block, and the block's total
__device__ __forceinline__ int block_scan(int v, int * s_wave, int & total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 63) s_wave[wave] = x;
    __syncthreads();
    int below = 0, all = 0;
#pragma unroll
    for (int w = 0; w < PLAN_T / 64; ++w) {
        if (w < wave) below += s_wave[w];
        all += s_wave[w];
    }
    total = all;
    return below + x - v;
}

// One block. Everything is clamped to the tables' sizes, so that whatever the lengths say no entry leads outside the buffers.
__global__ void __launch_bounds__(PLAN_T) k_paged_plan(PlanArgs a) {
    __shared__ int s_wave[PLAN_T / 64];
    __shared__ unsigned long long s_total;
    constexpr int LDS_TILES = 4096;
    __shared__ int s_item0[LDS_TILES];
    const int tid = threadIdx.x, group = a.n_head / a.nkv, tr = z2o::tile_rows(group);
    for (int t = tid; t < a.n_rows; t += PLAN_T) a.rows[t] = PlanRow{0, 0, 0, 0, 0, 0, 0, 0};
    if (tid == 0) {
        s_total = 0;
        a.head[PH_MAGIC] = PLAN_MAGIC; a.head[PH_ROWS] = a.n_rows; a.head[PH_HEADS] = a.n_head; a.head[PH_GROUPS] = a.n_group;
        a.head[PH_SEQS] = a.n_seq; a.head[PH_KV_HEADS] = a.nkv;
    }
    auto start_of = [&](int s) { return min(max(a.row_start[s], 0), a.n_rows); };
    auto len_of = [&](int s) { return min(max(a.kv_len[s], 0), a.cap); };
    auto group_of = [&](int g) { return min(max(a.group_start[g], 0), a.n_seq); };
    // ---- tiles of every span: the groups' prefixes, then the sequences' own keys
    int n_tiles = 0;
    unsigned long long work = 0;
    for (int base = 0; base < a.n_group + a.n_seq; base += PLAN_T) {
        const int x = base + tid;
        int r0 = 0, r1 = 0, key0 = 0, key1 = 0, seq = 0, len = 0;
        const bool own = x >= a.n_group;
        if (x < a.n_group) {
            const int s0 = group_of(x), s1 = group_of(x + 1);
            if (s0 < s1) {
                r0 = start_of(s0); r1 = start_of(s1); seq = s0;
                key1 = max(0, min(a.prefix_len[x], len_of(s0)));
            }
        } else if (x < a.n_group + a.n_seq) {
            seq = x - a.n_group;
            r0 = start_of(seq); r1 = start_of(seq + 1); len = key1 = len_of(seq);
            const int g = last_at_or_before(a.group_start, a.n_group + 1, seq);
            if (g >= 0 && g < a.n_group) key0 = max(0, min(a.prefix_len[g], len_of(group_of(g))));
        }
        const bool some = r1 > r0 && (own || key1 > 0);
        int all;
        const int at = n_tiles + block_scan(some ? (r1 - r0 + tr - 1) / tr : 0, s_wave, all);
        n_tiles = min(n_tiles + all, a.max_tiles);
        if (some)
            for (int i = 0, r = r0; r < r1; ++i, r += tr) {
                if (at + i >= a.max_tiles) break;
                const int rows = min(tr, r1 - r);
                // own keys: up to what the tile's last row sees
                const int end = own ? max(key0, min(key1, len - (r1 - r0) + (r + rows - r0))) : key1;
                a.tiles[at + i] = PlanTile{r, rows, key0, end, seq, own ? (len - (r1 - r0) + (r - r0)) : -1, 0, own};
                work += (unsigned long long) z2o::tile_keys(key0, end) * a.nkv;
            }
    }
    atomicAdd(&s_total, work);                         // integers: the order does not matter
    __syncthreads();
    const int chunk = z2o::chunk_keys((int64_t) s_total, a.target);
    // ---- chunks of every tile, the places of its items and partial results, and its rows' entries
    int n_items = 0, n_parts = 0;
    for (int base = 0; base < n_tiles; base += PLAN_T) {
        const int i = base + tid;
        PlanTile t{};
        if (i < n_tiles) t = a.tiles[i];
        const int see0 = t.chunks;                     // (own tiles: cache rows before the first row's own)
        const bool own = t.part0;
        const int chunks = i < n_tiles ? z2o::chunk_count(z2o::tile_keys(t.key0, t.key1), chunk) : 0, heads = t.rows * group;
        int items, parts;
        t.chunks = chunks;
        t.item0 = n_items + block_scan(chunks * a.nkv, s_wave, items);
        t.part0 = n_parts + block_scan(chunks * a.nkv * heads, s_wave, parts);
        n_items = min(n_items + items, a.max_items);
        n_parts = min(n_parts + parts, a.max_parts);
        if (i < n_tiles) {
            if (t.part0 + chunks * a.nkv * heads > a.max_parts) t.chunks = 0;   // (cannot be, by the sizes' rule)
            a.tiles[i] = t;
            if (i < LDS_TILES) s_item0[i] = t.item0;
            for (int r = 0; r < t.rows; ++r) {
                PlanRow & p = a.rows[t.row0 + r];
                const int part = t.part0 + r * group, step = a.nkv * heads;
                if (own) { p.vis = max(0, see0 + r + 1); p.own_base = part; p.own_n = t.chunks; p.own_step = step; }
                else { p.pre_base = part; p.pre_n = t.chunks; p.pre_step = step; }
            }
        }
    }
    __syncthreads();
    if (tid == 0) { a.head[PH_ITEMS] = n_items; a.head[PH_CHUNK] = chunk; }
    // ---- items: chunk by chunk of a tile, its key heads side by side
    for (int i = tid; i < n_items; i += PLAN_T) {
        int lo = 0, hi = n_tiles;
        while (hi - lo > 1) {
            const int m = (lo + hi) >> 1;
            if ((m < LDS_TILES ? s_item0[m] : a.tiles[m].item0) <= i) lo = m; else hi = m;
        }
        const PlanTile t = a.tiles[lo];
        const int c = (i - t.item0) / a.nkv, g = (i - t.item0) % a.nkv, from = (t.key0 & ~63) + c * chunk;
        if (c >= t.chunks) { a.items[i] = PlanItem{0, 0, 0, 0, 0, 0, 0, 0}; continue; }
        const bool direct = t.chunks == 1 && a.rows[t.row0].pre_n == 0 && a.rows[t.row0].own_n == 1;
        a.items[i] = PlanItem{t.row0, t.rows, max(t.key0, from), min(t.key1, from + chunk), t.seq, g,
                              t.part0 + (c * a.nkv + g) * t.rows * group, direct};
    }
}

struct PagedArgs {
    const void * k, * v;
    int64_t page_stride, qs, os;
    const int32_t * table;
    int n_seq, table_len, n_pages, page_shift, nkv, n_head, n_rows, n_group;
    float scale;
    const void * q;
    void * out;
    const int32_t * head;
    const PlanRow * rows;
    const PlanItem * items;
    float2 * part_ml;
    float * part_o;
};

__device__ __forceinline__ bool plan_fits(const PagedArgs & a) {
    return a.head[PH_MAGIC] == PLAN_MAGIC && a.head[PH_ROWS] == a.n_rows && a.head[PH_HEADS] == a.n_head && a.head[PH_GROUPS] == a.n_group &&
           a.head[PH_SEQS] == a.n_seq && a.head[PH_KV_HEADS] == a.nkv;
}

typedef float v16f_t __attribute__((ext_vector_type(16)));
typedef unsigned u4_t __attribute__((ext_vector_type(4)));
typedef short s4_t __attribute__((ext_vector_type(4)));
typedef short s8_t __attribute__((ext_vector_type(8)));
template <typename TC> struct Vec8 { typedef TC type __attribute__((ext_vector_type(8))); };

template <typename TC>
__device__ __forceinline__ v16f_t mfma32(typename Vec8<TC>::type a, typename Vec8<TC>::type b, v16f_t c) {
    if constexpr (__is_same(TC, _Float16)) return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
// the value of the lane 32 away
__device__ __forceinline__ float other_half(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    const unsigned r0 = r[0], r1 = r[1];
    return __builtin_bit_cast(float, (threadIdx.x & 32) ? r0 : r1);
}

// k_paged_attn: 4 waves. A wave holds the queries of 32 row-heads as the right operand of S^T = K Q^T and their O^T = V^T P^T:
// with v_mfma_f32_32x32x16 a lane then has one row-head's scores (16 of 32 keys, the lane 32 away the others), and a
// product's output registers 8 t .. 8 t + 7 are, in their order, the right operand of the next product's step t over the keys
// {16 t + 4 h + j, 16 t + 8 + 4 h + j} (h the lane's half, j < 4): P never moves between lanes. V^T's operand for these keys is two
// transposing LDS reads of 4 keys x 16 dims each from V rows stored as they are. K and V rows lie in LDS with their 16-byte
// pieces permuted by row, so that both reads take all banks.
template <int HD>
struct Tile {
    static constexpr int NC = HD / 8, RP = 128 / HD;             // 16-byte pieces of a row, rows per 256 bytes
    // (rows of the same place in 32 are permuted alike)
    static __device__ __forceinline__ int k_at(int row, int piece) { return row * HD + ((piece ^ ((row / RP) & (NC - 1))) * 8); }
    static __device__ __forceinline__ int v_at(int row, int piece) { return row * HD + ((piece ^ (4 * ((row / RP) & (NC / 4 - 1)))) * 8); }
};

template <int HD, typename T, typename TC>
struct AttnWave {
    typedef typename Vec8<TC>::type v8;
    static constexpr int KS = HD / 16, DT = HD / 32, BIAS = __is_same(TC, _Float16) ? 6 : 0;
    static constexpr bool SPLIT = __is_same(T, float);           // fp32 queries and weights as two f16 each
    v8 q[KS], ql[SPLIT ? KS : 1];
    v16f_t o[DT];
    float m, l, c;                                               // m includes -BIAS: f16 weights up to 2^14, kept to 2^-24
    int vis;

    __device__ __forceinline__ void init(const PagedArgs & a, const PlanItem & it, int first_rh, int lane) {
        const int group = a.n_head / a.nkv, rh = first_rh + (lane & 31), h8 = 8 * (lane >> 5);
        const bool live = rh < it.rows * group;
        const int row = it.row0 + (live ? rh / group : 0), head = it.head * group + (live ? rh % group : 0);
        const T * src = (const T *) a.q + row * a.qs + (int64_t) head * HD;
        vis = live ? a.rows[row].vis : 0x7fffffff;
        const bool zero = !live || a.scale == 0.0f;
        const float sign = a.scale < 0.0f ? -1.0f : 1.0f;
        c = zero ? 1.0f : fabsf(a.scale) * 1.44269504088896341f;
        const bool wide = ((uintptr_t) src & 15) == 0;
        float x[KS][8];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            if (wide) {
                typedef T tv __attribute__((ext_vector_type(16 / sizeof(T))));
                const tv * p = (const tv *) (src + 16 * ks + h8);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[ks][j] = (float) p[j / (16 / (int) sizeof(T))][j % (16 / sizeof(T))];
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[ks][j] = (float) src[16 * ks + h8 + j];
            }
        }
        float up = sign;
        if constexpr (SPLIT) {
            // a power of two brings the row-head's largest value to [2^7, 2^8): hi + lo then keep every value to 2^-22 of it
            float mx = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int j = 0; j < 8; ++j) mx = fmaxf(mx, fabsf(x[ks][j]));
            mx = fmaxf(mx, other_half(mx));
            int e = 0;
            if (mx > 0.0f && mx < __builtin_inff()) (void) frexpf(mx, &e);
            e = mx > 0.0f && mx < __builtin_inff() ? 8 - e : 0;
            e = min(e, 120);
            up = ldexpf(sign, e);
            c = zero ? 1.0f : ldexpf(c, -e);
        }
        c = fminf(fmaxf(c, 0x1p-126f), 0x1p127f);                 // hidden scores stay -inf whatever the scale
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float y = zero ? 0.0f : x[ks][j] * up;
                q[ks][j] = (TC) y;
                if constexpr (SPLIT) ql[ks][j] = (TC) (y - (float) q[ks][j]);
            }
        m = -__builtin_inff();
        l = 0.0f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[dt][i] = 0.0f;
    }

    // scores of NT tiles of 32 keys whose rows lie at LDS rows r0, r0 + 32, ...
    template <int NT>
    __device__ __forceinline__ void scores(v16f_t (&s)[NT], const TC * sk, int r0, int lane) const {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            v16f_t acc = {};
            const TC * rows = sk + (r0 + 32 * n) * HD;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const v8 kf = *(const v8 *) (rows + Tile<HD>::k_at(lane & 31, 2 * ks + (lane >> 5)));
                acc = mfma32<TC>(kf, q[ks], acc);
                if constexpr (SPLIT) acc = mfma32<TC>(kf, ql[ks], acc);
            }
            s[n] = acc;
        }
    }

    // keys key0 .. key0 + 32 NT of the tiles; keys outside [from, min(to, vis)) are hidden
    template <int NT>
    __device__ __forceinline__ void step(const TC * sk, const TC * sv, int r0, int key0, int from, int to, int lane) {
        v16f_t s[NT];
        scores<NT>(s, sk, r0, lane);
        const int end = min(to, vis), h4 = 4 * (lane >> 5);
        const bool edge = __any(key0 < from || key0 + 32 * NT > end);
        if (edge) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int key = key0 + 32 * n + 8 * (i >> 2) + h4 + (i & 3);
                    if (key < from || key >= end) s[n][i] = -__builtin_inff();
                }
        }
        float mx = s[0][0];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[n][i]);
        mx = fmaxf(mx, other_half(mx)) * c;
        // the maximum moves only where a score exceeds it by 2^8: rarely behind the first keys
        if (__any(mx > m + (8.0f + BIAS))) {
            const float mn = mx > m + (8.0f + BIAS) ? mx - BIAS : m;
            const float w = mn == m ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= w;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[dt][i] *= w;
        }
        if (edge) infinite_values<NT>(s, sv, r0, lane);
        const float mu = m == -__builtin_inff() ? 0.0f : m;
        v8 p[2 * NT], pl[SPLIT ? 2 * NT : 1];
        float sum = 0.0f;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][i], c, -mu));
                const TC hi = (TC) w;
                p[2 * n + (i >> 3)][i & 7] = hi;
                if constexpr (SPLIT) pl[2 * n + (i >> 3)][i & 7] = (TC) (w - (float) hi);
                // the sum is over the weights as the products take them, so that their rounding has no mean effect
                sum += SPLIT ? w : (float) hi;
            }
        l += sum;
#pragma unroll
        for (int t = 0; t < 2 * NT; ++t)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                s8_t v = values(sv, r0 + 16 * t, dt, lane);
                if (edge) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = not_finite(v[j]) ? (short) 0 : v[j];
                }
                const v8 vf = __builtin_bit_cast(v8, v);
                o[dt] = mfma32<TC>(vf, p[t], o[dt]);
                if constexpr (SPLIT) o[dt] = mfma32<TC>(vf, pl[t], o[dt]);
            }
    }

    // V^T operand of 16 keys from LDS row r0 on, dims 32 dt ..: lanes 16 g + i read keys 4 (g / 2) + i / 4, dims 16 (g & 1) + 4 (i & 3)
    static __device__ __forceinline__ s8_t values(const TC * sv, int r0, int dt, int lane) {
        const int i16 = lane & 15, r = 4 * (lane >> 5) + (i16 >> 2), d = 32 * dt + 16 * ((lane >> 4) & 1) + 4 * (i16 & 3);
        const TC * at = sv + r0 * HD + Tile<HD>::v_at(r, d >> 3) + (d & 7);
        typedef __attribute__((address_space(3))) s4_t lds4;
        const s4_t x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *) at);
        const s4_t x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *) (at + 8 * HD));
        return __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    static constexpr unsigned EXP = __is_same(TC, _Float16) ? 0x7c00u : 0x7f80u;
    static __device__ __forceinline__ bool not_finite(short x) { return ((unsigned) (unsigned short) x & EXP) == EXP; }

    // Where some rows hide keys that others see, a hidden value that is not finite must not reach them as 0 x inf: `step` leaves such
    // values out of its operand, and here rows that see one get infinity (or both infinities: NaN) by a product of indicators.
    template <int NT>
    __device__ __forceinline__ void infinite_values(const v16f_t (&s)[NT], const TC * sv, int r0, int lane) {
#pragma unroll
        for (int t = 0; t < 2 * NT; ++t)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const s8_t v = values(sv, r0 + 16 * t, dt, lane);
                bool any = false;
#pragma unroll
                for (int j = 0; j < 8; ++j) any |= not_finite(v[j]);
                if (!__any(any)) continue;
                v8 seen;
#pragma unroll
                for (int j = 0; j < 8; ++j) seen[j] = (TC) (s[t >> 1][8 * (t & 1) + j] == -__builtin_inff() ? 0.0f : 1.0f);
#pragma unroll
                for (int sign = 0; sign < 2; ++sign) {
                    v8 is;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const unsigned x = (unsigned short) v[j];
                        const bool nan = (x & 0x7fffu) != EXP, neg = x & 0x8000u;
                        is[j] = (TC) (not_finite(v[j]) && (nan || neg == (sign == 1)) ? 1.0f : 0.0f);
                    }
                    const v16f_t z = {};
                    const v16f_t hit = mfma32<TC>(is, seen, z);
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (hit[i] > 0.0f) o[dt][i] += sign ? -__builtin_inff() : __builtin_inff();
                }
            }
    }
};

template <typename T>
__device__ __forceinline__ void store4(T * p, float x0, float x1, float x2, float x3) {
    typedef T tv __attribute__((ext_vector_type(4)));
    if (((uintptr_t) p & (4 * sizeof(T) - 1)) == 0) {
        tv v = {(T) x0, (T) x1, (T) x2, (T) x3};
        *(tv *) p = v;
    } else {
        p[0] = (T) x0; p[1] = (T) x1; p[2] = (T) x2; p[3] = (T) x3;
    }
}

template <int HD, typename T, typename TC>
__global__ void __launch_bounds__(256, 2) k_paged_attn(PagedArgs a) {
    constexpr int NC = HD / 8, ROWS = 128;
    __shared__ __attribute__((aligned(16))) TC s_kv[2 * ROWS * HD];
    __shared__ float2 s_ml[4][32];
    TC * s_k = s_kv, * s_v = s_kv + ROWS * HD;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, group = a.n_head / a.nkv;
    if (!plan_fits(a)) return;
    const int n_items = a.head[PH_ITEMS], mask = (1 << a.page_shift) - 1;
    for (int item = blockIdx.x; item < n_items; item += gridDim.x) {
        const PlanItem it = a.items[item];
        const int heads = it.rows * group;
        if (heads == 0) continue;
        const int64_t head_at = (int64_t) it.head << a.page_shift;
        // elements from the start of k and v to the 16 rows that begin with `key` (one page holds them; the wave is of one mind)
        auto rows_at = [&](int key) __attribute__((always_inline)) {
            key = __builtin_amdgcn_readfirstlane(key);
            const int page = max(0, z2o::page_of(a.table, a.n_seq, a.table_len, a.n_pages, a.page_shift, it.seq, key));
            return (int64_t) __builtin_amdgcn_readfirstlane(page) * a.page_stride + (head_at + (key & mask)) * HD;
        };
        AttnWave<HD, T, TC> w;
        if (heads <= z2o::NARROW_RH) {
            // ---- every wave takes 32 keys of each 128 and has its own part of LDS: nothing to wait for but its loads
            constexpr int N = 32 * NC / 64;                      // loads of 16 bytes per lane: 32 rows
            u4_t kr[N], vr[N];
            TC * wk = s_k + 32 * wave * HD, * wv = s_v + 32 * wave * HD;
            const int lrow = lane / NC, piece = lane % NC;
            auto load = [&](int64_t at0, int64_t at1) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int row = i * (64 / NC) + lrow;
                    const int64_t at = (i < N / 2 ? at0 : at1) + (row & 15) * HD + 8 * piece;
                    kr[i] = *(const u4_t *) ((const TC *) a.k + at);
                    vr[i] = *(const u4_t *) ((const TC *) a.v + at);
                }
            };
            int key = (it.key0 & ~31) + 32 * wave;
            load(rows_at(key), rows_at(key + 16));
            int64_t n0 = rows_at(key + 128), n1 = rows_at(key + 144);
            w.init(a, it, 0, lane);
            for (; key < it.key1; key += 128) {
                const bool cut = key < it.key0 || key + 32 > it.key1;     // rows of no key: not read into the products
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int row = i * (64 / NC) + lrow;
                    if (cut && (key + row < it.key0 || key + row >= it.key1)) vr[i] = u4_t{0, 0, 0, 0};
                    *(u4_t *) (wk + Tile<HD>::k_at(row, piece)) = kr[i];
                    *(u4_t *) (wv + Tile<HD>::v_at(row, piece)) = vr[i];
                }
                if (key + 128 < it.key1) {
                    load(n0, n1);
                    n0 = rows_at(key + 256); n1 = rows_at(key + 272);
                }
                asm volatile("" ::: "memory");
                w.template step<1>(wk, wv, 0, key, it.key0, it.key1, lane);
                asm volatile("" ::: "memory");
            }
            // ---- the four waves' results, scaled to one maximum, meet in LDS
            w.l += other_half(w.l);
            if (lane < 32) s_ml[wave][lane] = make_float2(w.m, w.l);
            __syncthreads();
            const int rh = lane & 31;
            const float m = fmaxf(fmaxf(s_ml[0][rh].x, s_ml[1][rh].x), fmaxf(s_ml[2][rh].x, s_ml[3][rh].x));
            const float f = w.m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(w.m - m);
            float * s_o = (float *) s_kv;                        // [4][32][HD]: the block's LDS exactly
            static_assert(4 * 32 * HD * 4 <= sizeof(TC) * 2 * ROWS * HD, "merge area");
            if (rh < heads) {
#pragma unroll
                for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
                    for (int i = 0; i < 16; i += 4)
                        *(float4 *) (s_o + (wave * 32 + rh) * HD + 32 * dt + 2 * i + 4 * (lane >> 5)) =
                            make_float4(w.o[dt][i] * f, w.o[dt][i + 1] * f, w.o[dt][i + 2] * f, w.o[dt][i + 3] * f);
            }
            __syncthreads();
            for (int e = tid; e < heads * (HD / 4); e += 256) {
                const int r = e / (HD / 4), d = 4 * (e % (HD / 4));
                float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                float mm = s_ml[0][r].x, ll = 0.0f;
#pragma unroll
                for (int i = 1; i < 4; ++i) mm = fmaxf(mm, s_ml[i][r].x);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 ml = s_ml[i][r];
                    const float4 y = *(const float4 *) (s_o + (i * 32 + r) * HD + d);
                    ll += ml.x == -__builtin_inff() ? 0.0f : ml.y * __builtin_amdgcn_exp2f(ml.x - mm);
                    x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
                }
                if (it.direct) {
                    const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
                    store4((T *) a.out + (it.row0 + r / group) * a.os + (int64_t) (it.head * group + r % group) * HD + d,
                           x.x * inv, x.y * inv, x.z * inv, x.w * inv);
                } else {
                    *(float4 *) (a.part_o + (int64_t) (it.part0 + r) * HD + d) = x;
                    if (d == 0) a.part_ml[it.part0 + r] = make_float2(mm, ll);
                }
            }
            __syncthreads();
        } else {
            // ---- every wave takes 32 row-heads; 64 keys at a time in LDS for all, the next 64 on their way in registers
            constexpr int N = 16 * NC / 64;                      // loads per lane: the wave's 16 of the 64 rows
            u4_t kr[N], vr[N];
            const int lrow = 16 * wave + lane / NC, piece = lane % NC;
            auto load = [&](int64_t at0) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int64_t at = at0 + (i * (64 / NC) + lane / NC) * HD + 8 * piece;
                    kr[i] = *(const u4_t *) ((const TC *) a.k + at);
                    vr[i] = *(const u4_t *) ((const TC *) a.v + at);
                }
            };
            auto put = [&](int key, int buf) __attribute__((always_inline)) {
                const bool cut = key < it.key0 || key + 64 > it.key1;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int row = lrow + i * (64 / NC);
                    if (cut && (key + row < it.key0 || key + row >= it.key1)) vr[i] = u4_t{0, 0, 0, 0};
                    *(u4_t *) (s_k + 64 * buf * HD + Tile<HD>::k_at(row, piece)) = kr[i];
                    *(u4_t *) (s_v + 64 * buf * HD + Tile<HD>::v_at(row, piece)) = vr[i];
                }
            };
            int key = it.key0 & ~63, buf = 0;
            const int mine = 16 * wave;
            load(rows_at(key + mine));
            int64_t next = rows_at(key + 64 + mine);
            w.init(a, it, 32 * wave, lane);
            put(key, 0);
            lds_sync();
            const bool live = 32 * wave < heads;
            for (; key < it.key1; key += 64, buf ^= 1) {
                const bool more = key + 64 < it.key1;
                if (more) {
                    load(next);
                    next = rows_at(key + 128 + mine);
                }
                if (live) w.template step<2>(s_k, s_v, 64 * buf, key, it.key0, it.key1, lane);
                if (more) put(key + 64, buf ^ 1);
                lds_sync();
            }
            w.l += other_half(w.l);
            const int rh = 32 * wave + (lane & 31);
            if (rh < heads) {
                const float inv = !it.direct ? 1.0f : w.l == 0.0f ? 0.0f : 1.0f / w.l;
                T * out = (T *) a.out + (it.row0 + rh / group) * a.os + (int64_t) (it.head * group + rh % group) * HD;
                float * part = a.part_o + (int64_t) (it.part0 + rh) * HD;
#pragma unroll
                for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const int d = 32 * dt + 2 * i + 4 * (lane >> 5);
                        const float4 x = make_float4(w.o[dt][i] * inv, w.o[dt][i + 1] * inv, w.o[dt][i + 2] * inv, w.o[dt][i + 3] * inv);
                        if (it.direct) store4(out + d, x.x, x.y, x.z, x.w);
                        else *(float4 *) (part + d) = x;
                    }
                if (!it.direct && lane < 32) a.part_ml[it.part0 + rh] = make_float2(w.m, w.l);
            }
        }
    }
}

// One wave per (row, head): weights of its partial results from their maxima (a lane each, 64 at a time), then the dims over the lanes.
template <int HD, typename T>
__global__ void __launch_bounds__(256) k_paged_join(PagedArgs a) {
    if (!plan_fits(a)) return;
    const int lane = threadIdx.x & 63, id = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= a.n_rows * a.n_head) return;
    const int row = id / a.n_head, head = id % a.n_head, group = a.n_head / a.nkv, g = head / group;
    const PlanRow r = a.rows[row];
    if (r.pre_n == 0 && r.own_n == 1) return;                    // stored by its only chunk
    const int n = r.pre_n + r.own_n;
    auto part = [&](int i) {
        const bool pre = i < r.pre_n;
        const int step = pre ? r.pre_step : r.own_step;
        return (pre ? r.pre_base + i * step : r.own_base + (i - r.pre_n) * step) + g * (step / a.nkv) + head % group;
    };
    constexpr int E = HD >= 64 ? HD / 64 : 1;
    const int d = E * lane;
    float m = -__builtin_inff(), l = 0.0f, o[E] = {};
    for (int i0 = 0; i0 < n; i0 += 64) {
        const float2 ml = i0 + lane < n ? a.part_ml[part(i0 + lane)] : make_float2(-__builtin_inff(), 0.0f);
        const float mn = fmaxf(m, wave_max_f(ml.x));
        const float w = ml.x == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(ml.x - mn);
        const float w0 = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l = l * w0 + wave_tree_f(w * ml.y);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] *= w0;
        const int k = min(64, n - i0);
        constexpr int MB = 4;                                    // loads in flight
        for (int i = 0; i < k; i += MB) {
            float x[MB][E];
#pragma unroll
            for (int u = 0; u < MB; ++u) {
                const float * p = a.part_o + (int64_t) part(i0 + min(i + u, k - 1)) * HD + d;
#pragma unroll
                for (int e = 0; e < E; ++e) x[u][e] = d < HD ? p[e] : 0.0f;
            }
#pragma unroll
            for (int u = 0; u < MB; ++u) {
                const float wi = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), min(i + u, 63)));
                if (i + u < k)
#pragma unroll
                    for (int e = 0; e < E; ++e) o[e] = __builtin_fmaf(wi, x[u][e], o[e]);
            }
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T * out = (T *) a.out + row * a.os + (int64_t) head * HD + d;
    if (d < HD)
#pragma unroll
        for (int e = 0; e < E; ++e) out[e] = (T) (o[e] * inv);
}

} // namespace z2d
