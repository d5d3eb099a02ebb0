// z2h_paged.h — attention of a batch of sequences over a paged cache, groups of which share a prefix.
//
//   o = sum_i p_i v_i / sum_i p_i,  p_i = 2^(x_i - m),  x_i = scale log2(e) q.k_i
// in one pass over the keys with a running m; partial (m, sum p, sum p v) of disjoint keys join by scaling to the larger m. So a
// row's keys may be cut anywhere: its group's shared prefix is walked once for all rows of the group (their queries side
// by side in one product), the rest of its keys with its own sequence, and both where shares of equal work end.
//   k_paged_plan     one block: tiles of query rows, the shares and the places of partial results, from the lengths (z2h_ops_rules.h)
//   k_paged_attn     a share of the wide strips per block and of the narrow ones per wave
//   k_paged_join     a wave per (row, head), or a block of four while the device holds them all: its pieces' partial results, and rows
//                    that hold NaN once more
// Single tokens are bound by reading the cache once; groups of many rows and prompt chunks by the products and the exponentials.
// Measured (attention + join): 64 single rows over 2048 shared and 16 to 2048 own keys, 4 key heads of 128: 22.1 + 5.4 us for
// 60 MB; 256 rows over 16384 shared keys, 8 key heads of 128, 32 query heads: 129 + 10 us for 253 MB and 69 GFLOP (103 with the
// products of the weights' second parts, at 800 TFLOP/s); 4 prompt chunks of 333 rows behind 1500 shared ones: 48.7 + 11.6 us; one row over
// 700 keys: 10.1 + 3.7 us, of dependent loads. The plan: 20 us for one sequence, 30 for 64, 44 for 256.
#pragma once
#include "z2h_common.h"
#include "z2h_ops_rules.h"
#include "z2h_tile.h"

namespace z2d {

constexpr int PLAN_MAGIC = 0x50414745;
enum { PH_MAGIC = 0, PH_ROWS, PH_HEADS, PH_GROUPS, PH_SEQS, PH_KV_HEADS, PH_SHIFT, PH_KIND, PH_COUNT = PH_KIND + 6 };
enum { PK_TILES = 0, PK_SHARE, PK_HEAD };                        // of each kind, narrow then wide, from PH_KIND on

// per row: what it sees, and its tiles in its group's prefix and in its own keys (-1: none), and its place in their row-heads
struct PlanRow { int vis, pre_tile, pre_at, own_tile, own_at, spare[3]; };
// A tile's strips begin at `begin` + key head x pitch in the row of all strips of its kind; partial result `at` of its strip g is at part0 +
// (g x pieces + at) x row-heads, `pieces` the most that any of its strips has; alone: its rows have no other tile. Wide tiles are
// kept from the table's first place on, narrow ones from its last backwards.
struct PlanTile { int row0, rows, key0, key1, seq, alone, begin, part0; };
// a piece of a strip: query rows, keys, and where its results go
struct PlanItem { int row0, rows, key0, key1, seq, head, part0, direct; };
// what a block (wide) or a wave (narrow) begins with: its share's first piece (rows 0: none), and the strip that may have the next (tile
// of its kind -1: none)
struct PlanShare { PlanItem it; int share, tile, head, spare[5]; };
// of a tile's strip: its first partial result, its pieces, the tile's row-heads, and whether its only piece stores the rows itself
struct PlanStrip { int part0; unsigned short pieces; unsigned char heads, stored; };
static_assert(sizeof(PlanRow) == 32 && sizeof(PlanTile) == 32 && sizeof(PlanShare) == 64 && sizeof(PlanStrip) == 8, "workspace layout");

struct PlanArgs {
    const int32_t * row_start, * kv_len, * group_start, * prefix_len;
    int n_seq, n_rows, n_group, n_head, nkv, cap, blocks;
    int32_t * head;
    PlanRow * rows;
    PlanTile * tiles;
    PlanStrip * strips;                                          // [tile's place][key head]
    PlanShare * shares;                                          // [blocks] wide, [blocks][4] narrow
    int max_tiles, max_parts;
};

__device__ __forceinline__ int tile_place(int i, bool wide, int max_tiles) { return wide ? i : max_tiles - 1 - i; }

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

struct PlanKind {
    z2o::Cut cut;
    int tiles, shift, max_tiles, nkv, group;
    bool wide;
    // the next piece that share b has, from the tile's strip `head` on: (tile, head) is then the strip behind it
    // (KERNEL: not in the kernel that writes the tiles)
    template <bool KERNEL>
    __device__ __forceinline__ bool next(const PlanTile * all, int b, int & tile, int & head, PlanItem & it) const {
        while (tile < tiles) {
            PlanTile t;
            if constexpr (KERNEL) t = uniform_copy(all + tile_place(tile, wide, max_tiles));
            else t = all[tile_place(tile, wide, max_tiles)];
            const int units = (int) z2o::strip_units(t.key0, t.key1, wide, shift), cost = (int) z2o::strip_cost(units, cut.head);
            const int begin = t.begin + head * (int) z2o::strip_pitch(cost, cut);
            if (units && begin >= (b + 1) * cut.share) return false;
            const z2o::Piece p = z2o::strip_piece(begin, units, cut, b);
            const int g = head;
            if (units == 0 || ++head == nkv) { ++tile; head = 0; }
            if (p.u0 >= p.u1) continue;
            const int base = t.key0 & ~63, unit = z2o::unit_keys(wide) << shift;
            it = PlanItem{t.row0, t.rows, max(t.key0, base + p.u0 * unit), min(t.key1, base + p.u1 * unit), t.seq, g,
                          t.part0 + (g * z2o::max_pieces(cost, cut.share) + p.at) * t.rows * group, t.alone && p.n == 1};
            return true;
        }
        return false;
    }
};

// One block: a chain of scans and searches, bound by its barriers and dependent loads; 30 us for 64 sequences, 44 us for 256, once
// for all layers of a step. Everything is clamped to the tables' sizes, so that whatever the lengths say no entry leads outside the buffers; tables
// that are not ascending make no plan.
__global__ void __launch_bounds__(PLAN_T) k_paged_plan(PlanArgs a) {
    __shared__ int s_wave[PLAN_T / 64];
    __shared__ unsigned long long s_total;
    __shared__ int s_overlap;
    constexpr int LDS_TILES = 8192;
    __shared__ int s_begin[LDS_TILES];
    const int tid = threadIdx.x, group = a.n_head / a.nkv, tr = z2o::tile_rows(group);
    for (int t = tid; t < a.n_rows; t += PLAN_T) a.rows[t] = PlanRow{0, -1, 0, -1, 0, {0, 0, 0}};
    if (tid == 0) { s_total = 0; s_overlap = 0; }
    auto start_of = [&](int s) { return min(max(a.row_start[s], 0), a.n_rows); };
    auto len_of = [&](int s) { return min(max(a.kv_len[s], 0), a.cap); };
    auto first_of = [&](int g) { return min(max(a.group_start[g], 0), a.n_seq); };
    // ---- tiles of every span: the groups' prefixes, then the sequences' own keys. A span's tiles have tr rows each but for the last.
    int n_tiles[2] = {0, 0};                                     // narrow, wide
    unsigned long long units = 0;
    bool overlap = false;                                        // a table that goes back: a row could be in several spans of a kind
    for (int base = 0; base < a.n_group + a.n_seq; base += PLAN_T) {
        const int x = base + tid;
        int r0 = 0, r1 = 0, key0 = 0, key1 = 0, seq = 0, len = 0;
        const bool own = x >= a.n_group;
        if (x < a.n_group) {
            const int s0 = first_of(x), s1 = first_of(x + 1);
            overlap |= a.group_start[x + 1] < a.group_start[x];
            if (s0 < s1) {
                r0 = start_of(s0); r1 = start_of(s1); seq = s0;
                key1 = max(0, min(a.prefix_len[x], len_of(s0)));
            }
        } else if (x < a.n_group + a.n_seq) {
            seq = x - a.n_group;
            r0 = start_of(seq); r1 = start_of(seq + 1); len = key1 = len_of(seq);
            overlap |= a.row_start[seq + 1] < a.row_start[seq];
            const int g = z2o::group_of(a.group_start, a.n_group, seq);
            if (g >= 0) key0 = max(0, min(a.prefix_len[g], len_of(first_of(g))));
        }
        const bool some = r1 > r0 && (own || key1 > 0);
        const int n = some ? (r1 - r0 + tr - 1) / tr : 0, last = some ? r1 - r0 - (n - 1) * tr : 0;
        const int n_wide = !some ? 0 : z2o::is_wide(last * group) ? n : z2o::is_wide(tr * group) ? n - 1 : 0;
        int all;
        int at[2] = {n_tiles[0] + block_scan(n - n_wide, s_wave, all), 0};
        n_tiles[0] += all;
        at[1] = n_tiles[1] + block_scan(n_wide, s_wave, all);
        n_tiles[1] += all;
        for (int i = 0, r = r0; i < n; ++i, r += tr) {
            const int rows = min(tr, r1 - r), before = len - (r1 - r0) + (r - r0);
            const bool wide = z2o::is_wide(rows * group);
            const int place = tile_place(at[wide]++, wide, a.max_tiles);
            if (place < 0 || place >= a.max_tiles) continue;     // (cannot be, by the table's size)
            // own keys: up to what the tile's last row sees (`before`: cache rows before its first row's own)
            const int end = own ? max(key0, min(key1, before + rows)) : key1;
            a.tiles[place] = PlanTile{r, rows, key0, end, seq, own && key0 == 0, own ? before : 0, own};
            units += (unsigned long long) z2o::strip_units(key0, end, wide, 0) * a.nkv;
        }
    }
    atomicAdd(&s_total, units);                                  // integers: the order does not matter
    if (overlap) s_overlap = 1;
    __syncthreads();
    if (s_overlap) {                                             // places and sizes below count on a row's two tiles at most
        if (tid == 0) a.head[PH_MAGIC] = 0;
        return;
    }
    int shift = 0, n_parts = 0, n_wide_shares = 0;
    while (s_total >> shift >= 1ull << 28) ++shift;
#pragma unroll 1
    for (int kind = 1; kind >= 0; --kind) {
        const bool wide = kind;
        const int count = min(n_tiles[kind], a.max_tiles), max_shares = wide ? a.blocks : 4 * a.blocks, head = z2o::piece_cost(wide);
        auto tile = [&](int i) -> PlanTile & { return a.tiles[tile_place(i, wide, a.max_tiles)]; };
        auto units_of = [&](const PlanTile & t) { return (int) z2o::strip_units(t.key0, t.key1, wide, shift); };
        // ---- how to cut: what all strips cost in a row, and the smallest whole share that needs no more than there are
        int row_cost = 0, all;
        for (int i = tid; i < count; i += PLAN_T) row_cost += (int) z2o::strip_cost(units_of(tile(i)), head) * a.nkv;
        block_scan(row_cost, s_wave, all);
        const int in_row = z2o::row_share(all, max_shares, head);
        int whole = 0;
        if (count && (int64_t) count * a.nkv <= max_shares)      // (a share per strip at least)
            for (int j = 0; j < z2o::WHOLE_SHARES && !whole && z2o::whole_share(j) <= in_row + head; ++j) {
                const int share = z2o::whole_share(j);
                int n = 0;
                for (int i = tid; i < count; i += PLAN_T) n += (units_of(tile(i)) + share - 1) / share * a.nkv;
                block_scan(min(n, 1 << 20), s_wave, all);
                if (all <= max_shares) whole = share;
            }
        const z2o::Cut cut = z2o::choose_cut(in_row, whole, head);
        // ---- where every tile's strips begin, the places of their partial results, and the rows' entries
        int total = 0;
        for (int base = 0; base < count; base += PLAN_T) {
            const int i = base + tid;
            PlanTile t{};
            if (i < count) t = tile(i);
            const int before = t.begin, heads = t.rows * group;
            const bool own = t.part0;
            const int cost = i < count ? (int) z2o::strip_cost(units_of(t), cut.head) : 0;
            t.begin = total + block_scan((int) z2o::strip_pitch(cost, cut) * a.nkv, s_wave, all);
            total += all;
            t.part0 = n_parts + block_scan(z2o::max_pieces(cost, cut.share) * a.nkv * heads, s_wave, all);
            n_parts += all;
            if (i < count) {
                const int place = tile_place(i, wide, a.max_tiles);
                a.tiles[place] = t;
                if (i < LDS_TILES) s_begin[i] = t.begin;
                for (int r = 0; r < t.rows; ++r) {
                    PlanRow & p = a.rows[t.row0 + r];
                    if (own) { p.vis = max(0, before + r + 1); p.own_tile = cost ? place : -1; p.own_at = r * group; }
                    else { p.pre_tile = place; p.pre_at = r * group; }
                }
            }
        }
        __syncthreads();
        const PlanKind k{cut, count, shift, a.max_tiles, a.nkv, group, wide};
        // ---- of every strip, where its results are
        for (int64_t i = tid; i < (int64_t) count * a.nkv; i += PLAN_T) {
            const int place = tile_place((int) (i / a.nkv), wide, a.max_tiles), g = (int) (i % a.nkv);
            const PlanTile t = a.tiles[place];
            const int units = units_of(t), cost = (int) z2o::strip_cost(units, cut.head), heads = t.rows * group;
            const z2o::Piece p = z2o::strip_piece(t.begin + g * (int) z2o::strip_pitch(cost, cut), units, cut, 0);
            a.strips[(int64_t) place * a.nkv + g] = PlanStrip{t.part0 + g * z2o::max_pieces(cost, cut.share) * heads, (unsigned short) p.n,
                                                              (unsigned char) heads, (unsigned char) (t.alone && p.n == 1)};
        }
        // ---- every share's first piece. Narrow shares go first to the blocks that have no wide one, a wave on each of them, then
        // the next waves, and then to the others.
        const int shares = min((total + cut.share - 1) / cut.share, max_shares), free = a.blocks - n_wide_shares;
        for (int b = tid; b < max_shares; b += PLAN_T) {
            PlanShare sh{};
            sh.share = b;
            sh.tile = -1;
            if (b < shares) {
                const int at = b * cut.share;
                int lo = 0, hi = count;
                while (hi - lo > 1) {
                    const int m = (lo + hi) >> 1;
                    if ((m < LDS_TILES ? s_begin[m] : tile(m).begin) <= at) lo = m; else hi = m;
                }
                const PlanTile t = tile(lo);
                const int pitch = (int) z2o::strip_pitch(z2o::strip_cost(units_of(t), cut.head), cut);
                sh.tile = lo;
                sh.head = pitch ? min((at - t.begin) / pitch, a.nkv - 1) : 0;
                if (!k.next<false>(a.tiles, b, sh.tile, sh.head, sh.it)) sh.it.rows = 0;
                if (!cut.head || sh.it.rows == 0) sh.tile = -1;          // whole shares have one piece
            }
            if (wide) a.shares[b] = sh;
            else {
                int block, wave;
                if (b < 4 * free) { block = a.blocks - 1 - b % free; wave = b / free; }
                else { const int c = b - 4 * free; block = n_wide_shares - 1 - c % n_wide_shares; wave = c / n_wide_shares; }
                a.shares[a.blocks + 4 * block + wave] = sh;
            }
        }
        if (wide) n_wide_shares = shares;
        if (tid == 0) {
            int32_t * h = a.head + PH_KIND + 3 * kind;
            h[PK_TILES] = count; h[PK_SHARE] = cut.share; h[PK_HEAD] = cut.head;
        }
        __syncthreads();
    }
    if (tid == 0) {
        const bool fits = n_parts <= a.max_parts;                // (always, by the sizes' rule)
        a.head[PH_ROWS] = a.n_rows; a.head[PH_HEADS] = a.n_head; a.head[PH_GROUPS] = a.n_group; a.head[PH_SEQS] = a.n_seq;
        a.head[PH_KV_HEADS] = a.nkv; a.head[PH_SHIFT] = shift; a.head[PH_MAGIC] = fits ? PLAN_MAGIC : 0;
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
    const PlanTile * tiles;
    const PlanStrip * strips;
    const PlanShare * shares;
    int max_tiles, blocks;
    int64_t join0;                                               // first block of this launch of k_paged_join
    float2 * part_ml;
    float * part_o;
};

__device__ __forceinline__ bool plan_fits(const PagedArgs & args) {
    struct { const __attribute__((address_space(4))) int32_t * head; int n_rows, n_head, n_group, n_seq, nkv; } a{
        uniform(args.head), args.n_rows, args.n_head, args.n_group, args.n_seq, args.nkv};
    return a.head[PH_MAGIC] == PLAN_MAGIC && a.head[PH_ROWS] == a.n_rows && a.head[PH_HEADS] == a.n_head && a.head[PH_GROUPS] == a.n_group &&
           a.head[PH_SEQS] == a.n_seq && a.head[PH_KV_HEADS] == a.nkv;
}

// k_paged_attn: 4 waves. A wave holds the queries of 32 row-heads as the right operand of S^T = K Q^T and their O^T = V^T P^T:
// with v_mfma_f32_32x32x16 a lane then has one row-head's scores (16 of 32 keys, the lane 32 away the others), and a
// product's output registers 8 t .. 8 t + 7 are, in their order, the right operand of the next product's step t over the keys
// {16 t + 4 h + j, 16 t + 8 + 4 h + j} (h the lane's half, j < 4): P never moves between lanes. V^T's operand for these keys is two
// transposing LDS reads of 4 keys x 16 dims each from V rows stored as they are. K and V rows lie in LDS with their 16-byte
// pieces permuted by row, so that both reads take all banks (no conflict counted).
// A step of 64 keys takes a wave 4.6 thousand cycles beside the other block's wave: K Q with the requests of the next keys 1.2, the softmax
// and the weights' two parts 1.3, P V 1.2, the barrier 0.1, the rest masks and addresses. Operands read just before each product and
// all requests behind the barrier cost 6 us more over 16384 shared keys. Products take 41 % of the cycles, vector instructions 42 %. Two waves
// per SIMD are what the registers leave: 32 of queries, 64 of O, 32 of scores at head size 128. More row-heads per wave would halve the
// LDS reads per product, but not the exponentials, and leave one wave per SIMD. Scalar registers do not hold all sizes, strides and
// addresses of both walks: 97 (head size 128) to 264 (64) of them lie in lanes of vector registers.
template <typename T> struct CacheOf { typedef _Float16 type; };  // pages that queries of T go with
template <> struct CacheOf<__bf16> { typedef __bf16 type; };

template <int HD, typename T, typename TC>
struct AttnWave {
    typedef typename Vec8<TC>::type v8;
    static constexpr int KS = HD / 16, DT = HD / 32, BIAS = __is_same(TC, _Float16) ? 6 : 0;
    static constexpr bool SPLIT = __is_same(T, float);           // fp32 queries as two f16 each
    v8 q[KS], ql[SPLIT ? KS : 1];
    v16f_t o[DT];
    float m, l, c;                                               // m includes -BIAS: f16 weights up to 2^14, kept to 2^-24
    int vis;
    int k_place[KS], v_place[DT];                                // where the lane's operands lie in 16 keys' rows (elements)

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
        const int i16 = lane & 15, r = 4 * (lane >> 5) + (i16 >> 2);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) k_place[ks] = Tile<HD>::k_at(lane & 31, 2 * ks + (lane >> 5));
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const int d = 32 * dt + 16 * ((lane >> 4) & 1) + 4 * (i16 & 3);
            v_place[dt] = Tile<HD>::v_at(r, d >> 3) + (d & 7);
        }
        m = -__builtin_inff();
        l = 0.0f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[dt][i] = 0.0f;
    }

    // PRODUCTS products in order, whose LDS operands are requested AHEAD products before they are used; beside(i) is called behind product
    // i. The barriers keep the compiler from what it does by itself: to read, wait and multiply in turn.
    template <int PRODUCTS, typename READ, typename MUL, typename B>
    static __device__ __forceinline__ void products(READ read, MUL mul, B beside) {
        constexpr int MOST = SPLIT ? 2 : 4, AHEAD = PRODUCTS < MOST ? PRODUCTS : MOST;   // (fp32 queries leave registers for two)
        v8 f[AHEAD];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) f[i] = read(i);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < PRODUCTS; ++i) {
            mul(i, f[i % AHEAD]);
            if (i + AHEAD < PRODUCTS) f[i % AHEAD] = read(i + AHEAD);
            beside(i);
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    // scores of NT tiles of 32 keys whose rows lie at LDS rows r0, r0 + 32, ...
    template <int NT, typename B>
    __device__ __forceinline__ void scores(v16f_t (&s)[NT], const TC * sk, int r0, int lane, B beside) const {
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n] = v16f_t{};
        products<KS * NT>(
            [&](int i) __attribute__((always_inline)) { return *(const v8 *) (sk + k_place[i / NT] + (r0 + 32 * (i % NT)) * HD); },
            [&](int i, v8 kf) __attribute__((always_inline)) {
                s[i % NT] = mfma32<TC>(kf, q[i / NT], s[i % NT]);
                if constexpr (SPLIT) s[i % NT] = mfma32<TC>(kf, ql[i / NT], s[i % NT]);
            }, beside);
    }

    // keys key0 .. key0 + 32 NT, in the first rows of sk and sv; keys outside [from, min(to, vis)) are hidden. One body for all steps: a second
    // one for steps that hide something costs the compiler another set of accumulators (256 registers and 126 spilled against 237).
    // keys_done() is called when K has been read, values_ready() before V is.
    template <int NT, typename B, typename F, typename G>
    __device__ __forceinline__ void step(const TC * sk, const TC * sv, int key0, int from, int to, int lane, B beside, F keys_done, G values_ready) {
        // (the places stay one register each, to which every read adds a constant: left to itself the compiler keeps one for every buffer)
#pragma unroll
        for (int i = 0; i < KS; ++i) asm("" : "+v"(k_place[i]));
#pragma unroll
        for (int i = 0; i < DT; ++i) asm("" : "+v"(v_place[i]));
        const int end = min(to, vis), r0 = 0;
        v16f_t s[NT];
        scores<NT>(s, sk, r0, lane, beside);
        keys_done();
        __builtin_amdgcn_sched_barrier(0);                       // no V read ahead of the weights: registers
        if (__any(key0 < from || key0 + 32 * NT > end)) {
            const int h4 = 4 * (lane >> 5);
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
        const bool up = mx > m + (8.0f + BIAS);
        if (__any(up)) {
            const float mn = up ? mx - BIAS : m;
            const float w = mn == m || m == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(m - mn);   // (nothing to scale yet)
            m = mn;
            l *= w;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[dt][i] *= w;
        }
        const float mu = m == -__builtin_inff() ? 0.0f : m;
        // The weights meet the values as two numbers of the cache's type, the second carrying what the first's rounding leaves: off by 2^-22 of
        // them in f16, 2^-16 in bf16. One alone (2^-11, 2^-8) errs as much as the output's own rounding, over any number of keys: with
        // values of mean zero the output shrinks as the error does (1.3 times the rounding's rms in all; with one number 256 rows over 16384
        // shared keys take 103 us and 4 chunks of 333 rows 40, with two 129 and 49).
        v8 p[2 * NT], pl[2 * NT];
        float sum = 0.0f;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                typedef typename Pair<float>::type f2;
                typedef typename Pair<TC>::type c2;
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
        l += sum;
        __builtin_amdgcn_sched_barrier(0);
        values_ready();
        products<2 * NT * DT>([&](int i) __attribute__((always_inline)) { return __builtin_bit_cast(v8, values(sv, r0 + 16 * (i / DT), i % DT)); },
                              [&](int i, v8 vf) __attribute__((always_inline)) {
                                  o[i % DT] = mfma32<TC>(vf, p[i / DT], o[i % DT]);
                                  o[i % DT] = mfma32<TC>(vf, pl[i / DT], o[i % DT]);
                              }, [](int) {});
    }

    // V^T operand of 16 keys from LDS row r0 on, dims 32 dt ..: lanes 16 g + i read keys 4 (g / 2) + i / 4, dims 16 (g & 1) + 4 (i & 3)
    __device__ __forceinline__ s8_t values(const TC * sv, int r0, int dt) const {
        const TC * at = sv + v_place[dt] + r0 * HD;
        typedef __attribute__((address_space(3))) s4_t lds4;
        const s4_t x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *) at);
        const s4_t x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *) (at + 8 * HD));
        return __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    // What is not finite in the cache meets both parts of a number in two parts, which may differ in sign or be 0, and weights that are too
    // small for the cache's type: the product is then NaN where the definition has infinity (values) or a weight of 0 (keys), never
    // anything else that is wrong. So rows that hold NaN are formed once more, by k_paged_join (walk_row).
    __device__ __forceinline__ bool any_nan() const {
        bool nan = false;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) nan |= o[dt][i] != o[dt][i];
        return nan;
    }
    // Where some rows hide keys that others see (or that nobody has), a value that is not finite must not reach a row as 0 x inf. Such a
    // tile's values are set to 0 in LDS, and before that rows that see one get infinity (or both infinities: NaN): the product
    // of two numbers that are infinite together.
    template <int NT>
    __device__ __forceinline__ void infinite_values(const TC * sv, int r0, int key0, int from, int to, int lane) {
        typedef typename Vec8<__bf16>::type b8;
        const int end = min(to, vis), h4 = 4 * (lane >> 5);
        const __bf16 big = (__bf16) 3e38f, none = (__bf16) 0.0f;
#pragma unroll 1
        for (int t = 0; t < 2 * NT; ++t) {
            b8 seen;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int key = key0 + 16 * t + 8 * (j >> 2) + h4 + (j & 3);
                seen[j] = key >= from && key < end ? big : none;
            }
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const s8_t v = values(sv, r0 + 16 * t, dt);
                b8 up, down;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const unsigned x = (unsigned short) v[j];
                    const bool nan = (x & 0x7fffu) > EXP, neg = x & 0x8000u, bad = (x & EXP) == EXP;
                    up[j] = bad && (nan || !neg) ? big : none;
                    down[j] = bad && (nan || neg) ? -big : none;
                }
                o[dt] = mfma32<__bf16>(up, seen, o[dt]);
                o[dt] = mfma32<__bf16>(down, seen, o[dt]);
            }
        }
    }
    static constexpr unsigned EXP = __is_same(TC, _Float16) ? 0x7c00u : 0x7f80u;
};

// 16 rows of V in LDS: does one hold a value that is not finite; those values set to 0
template <int HD, typename TC>
__device__ __forceinline__ bool rows_not_finite(const TC * sv, int lane) {
    constexpr unsigned EXP = __is_same(TC, _Float16) ? 0x7c00u : 0x7f80u;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
        const u4_t x = *(const u4_t *) (sv + 8 * (lane + 64 * i));
#pragma unroll
        for (int j = 0; j < 4; ++j) bad |= (x[j] & EXP) == EXP || (x[j] & (EXP << 16)) == EXP << 16;
    }
    return bad;
}
template <int HD, typename TC>
__device__ __forceinline__ void clean_rows(TC * sv, int lane) {
    constexpr unsigned EXP = __is_same(TC, _Float16) ? 0x7c00u : 0x7f80u;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
        u4_t x = *(const u4_t *) (sv + 8 * (lane + 64 * i));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if ((x[j] & EXP) == EXP) x[j] &= 0xffff0000u;
            if ((x[j] & (EXP << 16)) == EXP << 16) x[j] &= 0xffffu;
        }
        *(u4_t *) (sv + 8 * (lane + 64 * i)) = x;
    }
}

// The lanes' places in the rows that a wave moves at a time: 64 / NC rows, row i's pieces permuted as Tile has them (the lane of
// LDS piece x reads piece x ^ permutation of its row).
template <int HD, typename TC>
struct Mover {
    static constexpr int NC = HD / 8, ROWS = 64 / NC;            // rows per instruction
    int k[16 / ROWS], v;                                         // element offsets within 16 rows, per instruction; V's differ by whole rows
    __device__ __forceinline__ explicit Mover(int lane) {
        const int row = lane / NC, x = lane % NC;
#pragma unroll
        for (int i = 0; i < 16 / ROWS; ++i) k[i] = Tile<HD>::k_at(i * ROWS + row, x);
        v = Tile<HD>::v_at(row, x);
    }
    static constexpr int N = 16 / ROWS;                          // instructions for 16 rows of K or V
    // 16 rows from `at` (elements from the start of k and v) to the rows of LDS at `to` (rows 16 apart are permuted alike)
    __device__ __forceinline__ void keys16(const PagedArgs & a, int64_t at, TC * to) const {
#pragma unroll
        for (int i = 0; i < N; ++i) to_lds((const TC *) a.k + at + k[i], to + i * ROWS * HD);
    }
    __device__ __forceinline__ void values16(const PagedArgs & a, int64_t at, TC * to) const {
#pragma unroll
        for (int i = 0; i < N; ++i) to_lds((const TC *) a.v + at + i * ROWS * HD + v, to + i * ROWS * HD);
    }
    // instruction i of these, K's before V's (none from 2 N on)
    __device__ __forceinline__ void rows16_part(const PagedArgs & a, int64_t at, TC * sk, TC * sv, int i) const {
        if (i < N) to_lds((const TC *) a.k + at + k[i], sk + i * ROWS * HD);
        else if (i < 2 * N) to_lds((const TC *) a.v + at + (i - N) * ROWS * HD + v, sv + (i - N) * ROWS * HD);
    }
    __device__ __forceinline__ void rows16(const PagedArgs & a, int64_t at, TC * sk, TC * sv) const {
        keys16(a, at, sk);
        values16(a, at, sv);
    }
};

template <int HD, typename T, typename TC>
struct PagedAttn {
    const PagedArgs & a;
    const Mover<HD, TC> mv;
    const int lane, wave, group;
    __device__ __forceinline__ PagedAttn(const PagedArgs & args, int lane_, int wave_)
        : a(args), mv(lane_), lane(lane_), wave(wave_), group(args.n_head / args.nkv) {}

    // the page that holds `key` >= 0, as the table has it: a scalar load that is requested a step ahead of its use, where no wait for LDS
    // follows soon (these loads come back in any order, so that such a wait is one for them too)
    __device__ __forceinline__ int entry_at(const PlanItem & it, int key) const {
        return uniform(a.table)[(int64_t) it.seq * a.table_len + min(key >> a.page_shift, a.table_len - 1)];
    }
    // elements from the start of k and v to the 16 rows that begin with `key` (one page holds them; any key and any page entry give
    // an address inside the cache)
    __device__ __forceinline__ int64_t rows_of(const PlanItem & it, int key, int entry) const {
        const int page = entry >= 0 && entry < a.n_pages ? entry : 0;
        return page * a.page_stride + (((int64_t) it.head << a.page_shift) + (key & ((1 << a.page_shift) - 1))) * HD;
    }
    // the row-heads first_rh .. first_rh + 31 of the piece: final, or partial. Final ones that hold NaN are left to k_paged_join (their
    // queries may lie where the results go), which finds them by a mark in the place of their maximum and sum.
    __device__ __forceinline__ void store(const PlanItem & it, AttnWave<HD, T, TC> & w, int first_rh) const {
        const int heads = it.rows * group, rh = first_rh + (lane & 31);
        w.l += other_half(w.l);
        float nan = it.direct && w.any_nan() ? 1.0f : 0.0f;
        nan = fmaxf(nan, other_half(nan));
        if (rh >= heads) return;
        if (lane < 32) a.part_ml[it.part0 + rh] = it.direct ? make_float2(0.0f, nan) : make_float2(w.m, w.l);
        if (nan != 0.0f) return;
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
    }

    // ---- narrow: the wave's own 32 rows of LDS (K at wk, V at wv), its own keys; nothing to wait for but its own loads. The next keys
    // are requested when this step's scores are formed, the next values when its values have been used.
    __device__ __forceinline__ void narrow(const PlanItem & it, TC * wk, TC * wv) const {
        int key = it.key0 & ~31;
        int e0 = entry_at(it, key), e1 = entry_at(it, key + 16);
        int64_t n0 = rows_of(it, key, e0), n1 = rows_of(it, key + 16, e1);
        e0 = entry_at(it, key + 32);
        e1 = entry_at(it, key + 48);
        mv.keys16(a, n0, wk);
        mv.keys16(a, n1, wk + 16 * HD);
        mv.values16(a, n0, wv);
        mv.values16(a, n1, wv + 16 * HD);
        AttnWave<HD, T, TC> w;
        w.init(a, it, 0, lane);
        for (; key < it.key1; key += 32) {
            const bool more = key + 32 < it.key1;
            wait_loads_but<2 * Mover<HD, TC>::N>();              // the values may still be on their way
            if (__any(key < it.key0 || key + 32 > min(it.key1, w.vis))) {
                wait_loads_but<0>();
                if (__any(rows_not_finite<HD>(wv, lane) || rows_not_finite<HD>(wv + 16 * HD, lane))) {
                    w.template infinite_values<1>(wv, 0, key, it.key0, it.key1, lane);
                    wait_lds();
                    clean_rows<HD>(wv, lane);
                    clean_rows<HD>(wv + 16 * HD, lane);
                    wait_lds();
                }
            }
            n0 = rows_of(it, key + 32, e0);
            n1 = rows_of(it, key + 48, e1);
            w.template step<1>(wk, wv, key, it.key0, it.key1, lane, [](int) {}, [&] {
                wait_lds();
                if (more) { mv.keys16(a, n0, wk); mv.keys16(a, n1, wk + 16 * HD); }
                e0 = entry_at(it, key + 64);
                e1 = entry_at(it, key + 80);
            }, [&] {
                if (more) wait_loads_but<2 * Mover<HD, TC>::N>();
                else wait_loads_but<0>();
            });
            wait_lds();
            if (more) { mv.values16(a, n0, wv); mv.values16(a, n1, wv + 16 * HD); }
        }
        store(it, w, 0);
    }

    // ---- wide: every wave takes 32 row-heads; 64 keys at a time in LDS for all, the next 64 on their way into the other buffer
    __device__ __forceinline__ void wide(const PlanItem & it, TC * s_k0, TC * s_v0, TC * s_k1, TC * s_v1, int * s_vis) const {
        static_assert(AttnWave<HD, T, TC>::KS == 2 * Mover<HD, TC>::N, "two requests beside every fourth of 2 KS products are all of them");
        const int mine = 16 * wave;
        int key = it.key0 & ~63;
        mv.rows16(a, rows_of(it, key + mine, entry_at(it, key + mine)), s_k0 + mine * HD, s_v0 + mine * HD);
        int entry = entry_at(it, key + 64 + mine);
        AttnWave<HD, T, TC> w;
        w.init(a, it, 32 * wave, lane);
        const bool live = 32 * wave < it.rows * group;
        int least = w.vis;                                       // the fewest cache rows that a row of the tile sees
#pragma unroll
        for (int o = 16; o; o >>= 1) least = min(least, __shfl_xor(least, o));
        if (lane == 0) s_vis[wave] = least;
        __syncthreads();
        least = min(min(s_vis[0], s_vis[1]), min(s_vis[2], s_vis[3]));
        const int whole = min(it.key1, __builtin_amdgcn_readfirstlane(least));         // steps up to here hide nothing behind them
        // one stage: its keys have arrived for every wave, and nobody reads the other buffer any more
        auto stage = [&](const TC * sk, TC * sv, TC * ok, TC * ov) __attribute__((always_inline)) {
            wait_loads_but<0>();                                 // (the barrier itself does not wait for loads to LDS)
            __syncthreads();
            const bool more = key + 64 < it.key1;
            if ((key < it.key0 || key + 64 > whole) && __syncthreads_or(rows_not_finite<HD>(sv + mine * HD, lane))) {
                if (live) w.template infinite_values<2>(sv, 0, key, it.key0, it.key1, lane);
                __syncthreads();
                clean_rows<HD>(sv + mine * HD, lane);
                __syncthreads();
            }
            // the next keys and values are requested two instructions at a time beside the products: all at once they hold the wave up
            // where the other block's narrow shares fill the queue
            const int64_t next = rows_of(it, key + 64 + mine, entry);
            if (live)
                w.template step<2>(sk, sv, key, it.key0, it.key1, lane, [&](int i) __attribute__((always_inline)) {
                    if (i % 4 == 0 && more) {
                        mv.rows16_part(a, next, ok + mine * HD, ov + mine * HD, i / 2);
                        mv.rows16_part(a, next, ok + mine * HD, ov + mine * HD, i / 2 + 1);
                    }
                }, [&] { entry = entry_at(it, key + 128 + mine); }, [] {});
            else {
                if (more) mv.rows16(a, next, ok + mine * HD, ov + mine * HD);
                entry = entry_at(it, key + 128 + mine);
            }
            key += 64;
        };
        __builtin_amdgcn_s_setprio(1);                           // before narrow shares, which wait for memory anyway (110 -> 107 us)
        while (key < it.key1) {
            stage(s_k0, s_v0, s_k1, s_v1);
            if (key >= it.key1) break;
            stage(s_k1, s_v1, s_k0, s_v0);
        }
        __builtin_amdgcn_s_setprio(0);
        store(it, w, 32 * wave);
        __syncthreads();                                         // LDS is free for the next piece
    }
};

template <int HD, typename T, typename TC>
__global__ void __launch_bounds__(256, 2) k_paged_attn(PagedArgs a) {
    // two buffers of 64 keys; arrays of their own, so that loads on their way to one do not hold up reads of the other
    __shared__ __attribute__((aligned(1024))) TC s_k0[64 * HD], s_k1[64 * HD], s_v0[64 * HD], s_v1[64 * HD];
    __shared__ int s_vis[4];
    const int wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6);
    if (!plan_fits(a)) return;
    const PagedAttn<HD, T, TC> p(a, threadIdx.x & 63, wave);
    PlanShare wide = uniform_copy(a.shares + blockIdx.x), narrow = uniform_copy(a.shares + a.blocks + 4 * blockIdx.x + wave);
    auto rest = [&](bool kind, PlanShare & s) __attribute__((always_inline)) {
        const auto * h = uniform(a.head) + PH_KIND + 3 * (int) kind;
        const PlanKind k{z2o::Cut{h[PK_SHARE], h[PK_HEAD]}, h[PK_TILES], uniform(a.head)[PH_SHIFT], a.max_tiles, a.nkv, p.group, kind};
        return s.tile >= 0 && k.template next<true>(a.tiles, s.share, s.tile, s.head, s.it);
    };
    // Half of the blocks (one of the two that a compute unit holds) begin with their narrow share: products and loads side by side.
    const int first = 2 * (int) blockIdx.x >= a.blocks;
#pragma unroll 1
    for (int phase = 0; phase < 2; ++phase) {
        if (phase == first) {
            if (wide.it.rows > 0)
                do p.wide(wide.it, s_k0, s_v0, s_k1, s_v1, s_vis); while (rest(true, wide));
        } else if (narrow.it.rows > 0) {
            // (a copy for each pair of arrays: loads on their way to one array do not hold up reads of the other)
            const int at = 32 * (wave & 1) * HD;
            if (wave & 2) { do p.narrow(narrow.it, s_k1 + at, s_v1 + at); while (rest(false, narrow)); }
            else { do p.narrow(narrow.it, s_k0 + at, s_v0 + at); while (rest(false, narrow)); }
        }
        __syncthreads();                                         // every wave is done with its part of LDS
    }
}

// A (row, head) in plain fp32, by one wave: 64 keys at a time, a lane each for the scores, then the dims over the lanes. A value that is
// not finite reaches the row whatever its weight. For rows whose results hold NaN (see AttnWave): 1.5 ms over 16384 keys, of chains of loads.
template <int HD, typename T, typename TC, int E>
__device__ __forceinline__ void walk_row(const PagedArgs & a, const PlanRow & r, int row, int head, float * s_q, float (&o)[E], float & l) {
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
    for (int part = 0; part < 2; ++part) {
        const int place = part ? r.own_tile : r.pre_tile;
        if (place < 0) continue;
        const PlanTile t = a.tiles[place];
        const int end = min(t.key1, r.vis);
        for (int key0 = t.key0; key0 < end; key0 += 64) {
            const int key = min(key0 + lane, end - 1), entry = a.table[(int64_t) t.seq * a.table_len + min(key >> a.page_shift, a.table_len - 1)];
            const int page = entry >= 0 && entry < a.n_pages ? entry : 0;
            const int64_t at = page * a.page_stride + (((int64_t) g << a.page_shift) + (key & ((1 << a.page_shift) - 1))) * HD;
            const typename Vec8<TC>::type * k = (const typename Vec8<TC>::type *) ((const TC *) a.k + at);
            float x[4] = {};
#pragma unroll 2                                                 // (64 registers at most, for the join's occupancy)
            for (int i = 0; i < HD / 8; ++i) {
                const typename Vec8<TC>::type kk = k[i];
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j & 3] = __builtin_fmaf(s_q[8 * i + j], (float) kk[j], x[j & 3]);
            }
            float s = ((x[0] + x[1]) + (x[2] + x[3])) * c;
            if (key0 + lane >= end) s = -__builtin_inff();
            if (__any(!(s < __builtin_inff()))) {                // infinity or no number: nor is any weight a number
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] = __builtin_nanf("");
                return;
            }
            const float mn = fmaxf(m, wave_max_f(s));
            const float w0 = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
            const float w = s == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(s - mn);
            m = mn;
            l = l * w0 + wave_tree_f(w);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = is_finite(o[e]) ? o[e] * w0 : o[e];
            const int n = min(64, end - key0), lo = (int) (uint64_t) at, hi = (int) ((uint64_t) at >> 32);
            for (int i0 = 0; i0 < n; i0 += 8) {                 // (lanes from n on have the last key, with no weight)
                float wi[8], v[8][E];
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    wi[u] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), i0 + u));
                    const uint64_t from = (uint64_t) (unsigned) __builtin_amdgcn_readlane(hi, i0 + u) << 32 | (unsigned) __builtin_amdgcn_readlane(lo, i0 + u);
#pragma unroll
                    for (int e = 0; e < E; ++e) v[u][e] = d < HD ? (float) ((const TC *) a.v)[from + d + e] : 0.0f;
                }
#pragma unroll
                for (int u = 0; u < 8; ++u)
#pragma unroll
                    for (int e = 0; e < E; ++e) o[e] = is_finite(v[u][e]) ? __builtin_fmaf(wi[u], v[u][e], o[e]) : o[e] + v[u][e];
            }
        }
    }
}

// One wave per (row, head), or with SHARED its block's four waves: weights of its partial results from their maxima (a lane each, 64 at a
// time), then the dims over the lanes. Bound by its chain of loads (row, strips, maxima, results), which four waves shorten, and with many
// rows by reading the results.
template <int HD, typename T, bool SHARED>
__global__ void __launch_bounds__(256) k_paged_join(PagedArgs a) {
    constexpr int STEP = SHARED ? 4 : 1;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6);
    const int id = SHARED ? (int) blockIdx.x : 4 * (int) (a.join0 + blockIdx.x) + wave, from = SHARED ? wave : 0;
    if (id >= a.n_rows * a.n_head) return;
    const int row = id / a.n_head, head = id % a.n_head, group = a.n_head / a.nkv, g = head / group;
    const PlanRow r = uniform_copy(a.rows + row);
    if (!plan_fits(a)) return;
    auto strip = [&](int tile) { return tile >= 0 ? uniform_copy(a.strips + (int64_t) tile * a.nkv + g) : PlanStrip{0, 0, 0, 0}; };
    const PlanStrip pre = strip(r.pre_tile), own = strip(r.own_tile);
    const int n_pre = pre.pieces, n_own = own.pieces, pre_step = pre.heads, own_step = own.heads;
    const int pre0 = pre.part0 + r.pre_at + head % group, own0 = own.part0 + r.own_at + head % group;
    // stored by its only piece, unless that one found NaN
    const bool again = own.stored && uniform(a.part_ml)[own0].y != 0.0f;
    if (own.stored && (!again || from)) return;
    const int n = again ? 0 : max(0, (n_pre + n_own - from + STEP - 1) / STEP);  // this wave's
    auto part = [&](int i) {
        i = i * STEP + from;
        return i < n_pre ? pre0 + i * pre_step : own0 + (i - n_pre) * own_step;
    };
    constexpr int E = HD >= 64 ? HD / 64 : 1;
    const int d = E * lane;
    constexpr int MB = 8;                                        // results on their way, the first of them with the maxima
    float m = -__builtin_inff(), l = 0.0f, o[E] = {}, x[MB][E];
    auto request = [&](int i0) {
#pragma unroll
        for (int u = 0; u < MB; ++u) {
            if (i0 + u >= n) break;
            const float * p = a.part_o + (int64_t) part(i0 + u) * HD + d;
#pragma unroll
            for (int e = 0; e < E; ++e) x[u][e] = d < HD ? p[e] : 0.0f;
        }
    };
    for (int i0 = 0; i0 < n; i0 += 64) {
        const float2 ml = i0 + lane < n ? a.part_ml[part(i0 + lane)] : make_float2(-__builtin_inff(), 0.0f);
        request(i0);
        const float mn = fmaxf(m, wave_max_f(ml.x));
        const float w = ml.x == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(ml.x - mn);
        const float w0 = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l = l * w0 + wave_tree_f(w * ml.y);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] *= w0;
        const int k = min(64, n - i0);
        for (int i = 0; i < k; i += MB) {
            if (i) request(i0 + i);
#pragma unroll
            for (int u = 0; u < MB; ++u) {
                if (i + u >= k) break;
                const float wi = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), i + u));
#pragma unroll
                    for (int e = 0; e < E; ++e) o[e] = __builtin_fmaf(wi, x[u][e], o[e]);
            }
        }
    }
    if constexpr (SHARED) if (!again) {
        __shared__ float s_o[4][64 * E], s_m[4], s_l[4];
        if (lane == 0) { s_m[wave] = m; s_l[wave] = l; }
#pragma unroll
        for (int e = 0; e < E; ++e) s_o[wave][d + e] = o[e];
        __syncthreads();
        if (wave) return;
        m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
        l = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float c = s_m[w] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(s_m[w] - m);
            l = __builtin_fmaf(c, s_l[w], l);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = __builtin_fmaf(c, s_o[w][d + e], o[e]);
        }
    }
    bool nan = again;
#pragma unroll
    for (int e = 0; e < E; ++e) nan |= o[e] != o[e];
    if (__any(nan)) {
        __shared__ float s_q[SHARED ? 1 : 4][HD];
        walk_row<HD, T, typename CacheOf<T>::type>(a, r, row, head, s_q[SHARED ? 0 : wave], o, l);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T * out = (T *) a.out + row * a.os + (int64_t) head * HD + d;
    if (d < HD)
#pragma unroll
        for (int e = 0; e < E; ++e) out[e] = (T) (o[e] * inv);
}

} // namespace z2d
