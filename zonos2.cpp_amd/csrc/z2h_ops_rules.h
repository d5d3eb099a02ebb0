// z2h_ops_rules.h — the argument checks, sizes and index rules of the operators on device tensors (z2h_ops.hip), as plain
// functions: the kernels use the index rules as they stand here, and a CPU test runs all of them without a GPU.
#pragma once
#include "z2h.h"
#include <cmath>
#include <cstdint>
#include <initializer_list>

#if defined(__HIPCC__)
#define Z2O_HD __host__ __device__ inline
#else
#define Z2O_HD inline
#endif

namespace z2o {

constexpr int MAX_GROUP = 64;                      // query heads per key head
constexpr int64_t MAX_ROW_HEADS = 1ll << 26;       // rows x heads of one attention call
constexpr int MAX_VOCAB = 1 << 20;
constexpr int MAX_ROPE_DIMS = 128;

// Blocks of `threads` that one launch may have (its threads are counted in 32 bits); calls of more launch several times.
constexpr int64_t launch_blocks(int threads) { return (1ll << 31) / threads; }

// ---- checks: nullptr, or what is wrong
inline const char * check_rope(const z2h_rope * r, int head_dim) {
    if (!r) return "null rope";
    if (head_dim <= 0 || head_dim > MAX_ROPE_DIMS || head_dim % 2) return "rope: head_dim must be even and at most 128";
    if (r->n_dims < 0 || r->n_dims > head_dim || r->n_dims % 2) return "rope: n_dims must be even, 0 .. head_dim";
    if (!(r->base > 0.0f) || !std::isfinite(r->base)) return "rope: base must be positive";
    if (!(r->factor > 0.0f) || !std::isfinite(r->factor)) return "rope: factor must be positive";
    if (!(r->mscale > 0.0f) || !std::isfinite(r->mscale)) return "rope: mscale must be positive";
    if (r->orig_ctx < 0) return "rope: orig_ctx must not be negative";
    if (r->orig_ctx > 0 && !(std::isfinite(r->low_turns) && std::isfinite(r->high_turns) && r->high_turns > r->low_turns))
        return "rope: high_turns must be above low_turns";
    return nullptr;
}

inline const char * check_pages(const z2h_pages * p) {
    if (!p) return "null pages";
    if (!p->k || !p->v || !p->table) return "pages: null buffer or table";
    if (p->type != Z2H_F16 && p->type != Z2H_BF16) return "pages: the cache must be F16 or BF16";
    if (p->head_dim != 32 && p->head_dim != 64 && p->head_dim != 128) return "pages: head_dim must be 32, 64 or 128";
    if (p->page_rows < 16 || p->page_rows > 4096 || (p->page_rows & (p->page_rows - 1))) return "pages: page_rows must be a power of two, 16 .. 4096";
    if (p->n_pages <= 0 || p->n_head_kv <= 0 || p->n_head_kv > 1024 || p->n_seq <= 0 || p->n_seq > (1 << 24) || p->table_len <= 0)
        return "pages: counts out of range";
    if ((int64_t) p->table_len * p->page_rows > (1ll << 30)) return "pages: a sequence of more than 2^30 rows";
    if (p->page_stride < (int64_t) p->n_head_kv * p->page_rows * p->head_dim) return "pages: page_stride below a page's size";
    if (p->page_stride % 8 || (uintptr_t) p->k % 16 || (uintptr_t) p->v % 16) return "pages: k, v and page_stride must be 16-byte aligned";
    return nullptr;
}

inline int type_size(int type) { return type == Z2H_F32 ? 4 : type == Z2H_F16 || type == Z2H_BF16 ? 2 : 0; }

// a row tensor of n_head heads: rows `stride` elements apart, elements aligned to their size (no rows: it may be null)
inline const char * check_rows(const void * p, int64_t stride, int n_head, int head_dim, int type, int n_rows = 1) {
    if (!type_size(type)) return "row type must be F32, F16 or BF16";
    if (!p && n_rows) return "null row tensor";
    if (stride < (int64_t) n_head * head_dim) return "row stride below a row's size";
    if ((uintptr_t) p % type_size(type)) return "row tensor not aligned to its elements";
    return nullptr;
}

inline const char * check_attn(const z2h_pages * p, int n_head, int n_rows, int n_group) {
    if (const char * e = check_pages(p)) return e;
    if (n_head <= 0 || n_head % p->n_head_kv || n_head / p->n_head_kv > MAX_GROUP) return "n_head must be 1 .. 64 times n_head_kv";
    if (n_rows < 0 || (int64_t) n_rows * n_head > MAX_ROW_HEADS) return "n_rows out of range";
    if (n_group < 0 || n_group > p->n_seq) return "n_group out of range (0 .. n_seq)";
    return nullptr;
}

inline const char * check_attn_type(int type, int cache) {
    if (type == Z2H_F32 || type == Z2H_F16) return cache == Z2H_F16 ? nullptr : "F32 and F16 queries need F16 pages";
    if (type == Z2H_BF16) return cache == Z2H_BF16 ? nullptr : "BF16 queries need BF16 pages";
    return "query type must be F32, F16 or BF16";
}

// ---- rotary frequencies: turns per position of every pair (theta' / 2 pi). theta_i by repeated multiplication in 80 bits: 64
// steps leave an error below 2^-57.
inline void rope_turns(const z2h_rope & r, double * turns) {
    const double two_pi = 6.283185307179586476925;
    const long double step = r.n_dims ? powl((long double) r.base, -2.0L / r.n_dims) : 1.0L;
    long double theta_i = 1.0L;
    for (int i = 0; i < r.n_dims / 2; ++i, theta_i *= step) {
        const double theta = (double) theta_i;
        double keep = 0.0;
        if (r.orig_ctx > 0) {
            keep = (r.orig_ctx * theta / two_pi - (double) r.low_turns) / ((double) r.high_turns - (double) r.low_turns);
            keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
        }
        turns[i] = theta * (keep + (1.0 - keep) / (double) r.factor) / two_pi;
    }
}

// ---- pages
// The page that holds row `pos` of sequence `seq`; -1 where the sequence, the position or the entry is out of range.
Z2O_HD int page_of(const int32_t * table, int n_seq, int table_len, int n_pages, int page_shift, int seq, int pos) {
    if (seq < 0 || seq >= n_seq || pos < 0 || (pos >> page_shift) >= table_len) return -1;
    const int page = table[(int64_t) seq * table_len + (pos >> page_shift)];
    return page >= 0 && page < n_pages ? page : -1;
}
inline int page_shift_of(int page_rows) { int s = 0; while ((1 << s) < page_rows) ++s; return s; }

// The group that sequence `seq` is in (start [n_group + 1] ascending); -1: none. No groups: `start` is not read.
Z2O_HD int group_of(const int32_t * start, int n_group, int seq) {
    if (n_group <= 0) return -1;
    int lo = -1, hi = n_group + 1;                                       // start[lo] <= seq < start[hi]
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (start[m] <= seq) lo = m; else hi = m;
    }
    return lo < n_group ? lo : -1;
}

// ---- attention: how the work is cut
// A span is a run of query rows over a run of cache rows: a group's rows over its shared prefix, a sequence's rows over the
// rest. Its rows are cut into tiles of at most TILE_RH row-heads of one key head. A tile of more than NARROW_RH row-heads is
// wide: the four waves of a block take 32 row-heads each of the same keys. Any other is narrow: one wave has all its row-heads.
// A strip is a tile with one of its key heads. All strips of a kind are dealt out in shares of equal work, one per block (wide) or
// per wave (narrow), whatever the sequences' lengths; so every block has as much of either kind as any other.
constexpr int TILE_RH = 128, NARROW_RH = 32;
Z2O_HD int tile_rows(int group) { return TILE_RH / group; }              // group <= MAX_GROUP: two rows at least
Z2O_HD bool is_wide(int row_heads) { return row_heads > NARROW_RH; }
// Keys of a strip are counted in units, the keys of one step (times 2^shift in calls of more than 2^28 units), from a multiple of 64 on.
Z2O_HD int unit_keys(bool wide) { return wide ? 64 : 32; }
Z2O_HD int64_t strip_units(int key0, int key1, bool wide, int shift) {
    const int64_t k = unit_keys(wide);
    return key1 > key0 ? (((int64_t) key1 - (key0 & ~63) + k - 1) / k + (1ll << shift) - 1) >> shift : 0;
}
// What it takes to begin and end a piece of a strip, in steps (query rows, page numbers, partial results: 6 us beside steps of
// about 2 and 3).
Z2O_HD int piece_cost(bool wide) { return wide ? 2 : 3; }
// Two ways to cut. Whole shares (`head` 0): every strip is cut into pieces of `share` units, the last one shorter; strips begin at
// multiples of the share, so that a share is a piece of one strip, and strips over the same keys have their pieces side by side. In a
// row (`head`: the cost of a piece): all strips one behind the other, cut into shares of equal cost, so that a share has the end of
// one strip, whole strips and the beginning of another; for batches of more or longer strips than there are shares.
struct Cut { int share, head; };
Z2O_HD int64_t strip_cost(int64_t units, int head) { return units ? head + units : 0; }
Z2O_HD int64_t strip_pitch(int64_t cost, Cut cut) { return cut.head ? cost : (cost + cut.share - 1) / cut.share * cut.share; }
Z2O_HD int row_share(int64_t cost, int max_shares, int head) {
    const int64_t s = (cost + max_shares - 1) / max_shares;
    return (int) (s <= head ? head + 1 : s);                             // a unit at least
}
constexpr int WHOLE_SHARES = 24;                                         // whole shares that are tried: 2, 3, 4, 6, 8, 12, ... units
Z2O_HD int whole_share(int i) { return (i & 1 ? 3 : 2) << i / 2; }
// Of a call whose strips in a row give shares of `in_row`, and whose smallest whole share that needs no more than there are is
// `whole` (0: none): whole ones where they take no longer (a share in a row usually has parts of two strips).
Z2O_HD Cut choose_cut(int in_row, int whole, int head) { return whole && whole <= in_row + head ? Cut{whole, 0} : Cut{in_row, head}; }

// The piece of a strip that share `b` has: units [u0, u1), the `at`-th of `n` pieces. The strip begins at `begin` of the row of strips.
struct Piece { int u0, u1, at, n; };
Z2O_HD int units_before(int cost, int units) { return cost <= 0 ? 0 : cost < units ? cost : units; }
Z2O_HD Piece strip_piece(int begin, int units, Cut cut, int b) {
    if (!units) return Piece{0, 0, 0, 0};
    const int share = cut.share, b0 = begin / share, b1 = (begin + cut.head + units - 1) / share, from = begin + cut.head;
    // a first piece may be too short for a unit; the others are not
    const int none = b1 > b0 && (b0 + 1) * share - from <= 0;
    Piece p;
    p.u0 = b <= b0 ? 0 : units_before(b * share - from, units);
    p.u1 = b >= b1 ? units : units_before((b + 1) * share - from, units);
    p.at = b - b0 - none;
    p.n = b1 - b0 + 1 - none;
    return p;
}
Z2O_HD int max_pieces(int cost, int share) { return cost ? cost / share + 2 : 0; }

// ---- attention workspace
struct AttnWs {
    int64_t rows = 0, tiles = 0, strips = 0, shares = 0, ml = 0, o = 0, bytes = 0;   // offsets in bytes; the header is at 0
    int64_t max_tiles = 0, max_parts = 0;
};
inline int64_t align256(int64_t n) { return (n + 255) & ~(int64_t) 255; }
// Every row is in at most one tile of its group's span and one of its sequence's, and a span's last tile may be partly filled.
// Pieces of a strip: at most cost / share + 2, so over all strips of a kind at most shares + 2 strips, of as many partial results as the
// tile has row-heads: blocks x min(TILE_RH, all rows' of one key head) + 4 blocks x min(NARROW_RH, ...) + 4 x rows x heads.
inline AttnWs attn_ws(const z2h_pages & p, int n_head, int n_rows, int n_group, int blocks) {
    AttnWs w;
    const int group = n_head / p.n_head_kv, tr = tile_rows(group);
    const int64_t by_span = (int64_t) p.n_seq + n_group + 2 * ((n_rows + tr - 1) / tr), by_row = 2 * (int64_t) n_rows;
    const int64_t rh = (int64_t) n_rows * group;
    w.max_tiles = by_span < by_row ? by_span : by_row;
    w.max_parts = n_rows ? blocks * ((rh < TILE_RH ? rh : TILE_RH) + 4 * (rh < NARROW_RH ? rh : NARROW_RH)) + 4 * (int64_t) n_rows * n_head : 0;
    w.rows = 256;
    w.tiles = w.rows + align256((int64_t) n_rows * 32);
    w.strips = w.tiles + align256(w.max_tiles * 32);
    w.shares = w.strips + align256(w.max_tiles * p.n_head_kv * 8);
    w.ml = w.shares + align256((int64_t) blocks * 5 * 64);
    w.o = w.ml + align256(w.max_parts * 8);
    w.bytes = w.o + align256(w.max_parts * p.head_dim * 4);
    return w;
}

// ---- attention over packed prompts
// A sequence's rows are cut into tiles of `rows` rows; tile j of sequence s is slot start[s] / rows + s + j, so that a slot's sequence is found by
// searching the row table alone. A sequence may have a slot too many.
Z2O_HD int64_t prompt_slot(int start, int seq, int rows) { return (int64_t) start / rows + seq; }
Z2O_HD int64_t prompt_slots(int n_rows, int n_seq, int rows) { return (int64_t) n_rows / rows + n_seq; }
// Rows of a tile of 16 row-heads (0: a group has more than these).
Z2O_HD int small_rows(int group) { return 16 / group; }
// How a call is cut, by its tiles of 128 row-heads. Few: 16 row-heads per block, whose keys four waves share (small). Up to a tile and a quarter per
// compute unit of long prompts: 128 row-heads and eight waves, each four over half of the keys (pair). Otherwise 128 row-heads and four waves
// (wide). Measured, small - pair - wide in us, 16 heads of 128 on 4 key heads, f16 and fp32:
//   1 x 300 rows,  37 tiles   9.0 - 13.9 - 13.5   16.2 - 48.2 - 48.9      8 x 224, 224 tiles   25.9 - 15.6 - 15.0   50.4 - 42.8 - 42.0
//   1 x 600,       75        15.9 - 19.0 - 20.6   32.5 - 87.1 - 92.2      8 x 256, 256         30.7 - 16.1 - 18.8   59.5 - 47.9 - 72.7
//   8 x 128,      128        15.4 - 11.9 - 10.7   25.5 - 29.4 - 28.1      4 x 512, 256         38.9 - 20.1 - 21.3   83.5 - 78.2 - 89.4
//   4 x 300,      150        20.6 - 15.9 - 15.4   40.1 - 52.4 - 53.5      1 x 2400, 300        97.9 - 55.7 - 65.5    284 -  316 -  365
//   8 x 192,      192        22.8 - 14.2 - 12.9   41.9 - 38.0 - 37.6      16 x 256, 512        54.0 - 27.5 - 21.4    108 - 83.6 - 75.0
// Heads of 64: 4 x 300 rows 11.1 - 10.5 - 11.0 and 23.0 - 29.7 - 31.8; 1 x 1200 19.0 - 20.9 - 25.4 and 43.1 - 91.3 - 103; 8 x 512, 512 tiles
// 31.9 - 23.7 - 21.0 and 68.9 - 75.6 - 76.3. Not met by the rule: 8 x 256 rows of heads of 64 (15.2 - 10.9 - 13.2, taken as wide), and long fp32 prompts
// (2000 rows, 250 tiles: 202 - 266 - 287, taken as pair; 4000, 500 tiles: 749 - 553 - 746, taken as wide).
enum PromptCut { PROMPT_WIDE, PROMPT_PAIR, PROMPT_SMALL };
inline PromptCut prompt_cut(int n_rows, int n_seq, int n_head, int n_head_kv, int head_dim, bool fp32, int n_cu) {
    const int64_t tiles = (int64_t) n_rows * n_head / TILE_RH;
    if (n_head / n_head_kv <= 16 && tiles * head_dim <= (fp32 ? 96ll : 42ll) * n_cu) return PROMPT_SMALL;
    return 4 * tiles <= 5ll * n_cu && (int64_t) n_rows * head_dim >= 32768ll * n_seq ? PROMPT_PAIR : PROMPT_WIDE;
}
constexpr int MAX_PROMPTS = 1 << 20;
inline const char * check_prompt(int n_seq, int n_rows, int n_head, int n_head_kv, int head_dim) {
    if (head_dim != 32 && head_dim != 64 && head_dim != 128) return "prompt: head_dim must be 32, 64 or 128";
    if (n_head_kv <= 0 || n_head_kv > 1024) return "prompt: n_head_kv out of range";
    if (n_head <= 0 || n_head % n_head_kv || n_head / n_head_kv > MAX_GROUP) return "n_head must be 1 .. 64 times n_head_kv";
    if (n_rows < 0 || (int64_t) n_rows * n_head > MAX_ROW_HEADS) return "n_rows out of range";
    if (n_seq < 0 || n_seq > MAX_PROMPTS) return "prompt: n_seq out of range";
    return nullptr;
}

// ---- mixture of experts for a few rows
constexpr int MOE_MAX_EXPERTS = 1024, MOE_MAX_TOP = 16, MOE_MAX_DIM = 65536, MOE_SHARES = 8;
inline const char * check_experts(const z2h_experts * x) {
    if (!x) return "null experts";
    if (!x->gate || !x->up || !x->down) return "experts: null weights";
    if (((uintptr_t) x->gate | (uintptr_t) x->up | (uintptr_t) x->down) % 16) return "experts: weights must be 16-byte aligned";
    if (x->type != Z2H_F16 && x->type != Z2H_BF16) return "experts: the weights must be F16 or BF16";
    if (x->n_expert <= 0 || x->n_expert > MOE_MAX_EXPERTS) return "experts: n_expert out of range";
    for (int32_t d : {x->n_ff, x->n_embd})
        if (d <= 0 || d % 8 || d > MOE_MAX_DIM) return "experts: n_ff and n_embd must be multiples of 8, at most 65536";
    return nullptr;
}
inline const char * check_moe(const z2h_experts * x, int n_rows, int top_k) {
    if (const char * e = check_experts(x)) return e;
    if (n_rows < 0 || n_rows > Z2H_MOE_ROWS_MAX) return "moe: n_rows out of range (0 .. 128)";
    if (top_k <= 0 || top_k > MOE_MAX_TOP || top_k > x->n_expert) return "moe: top_k must be 1 .. min(n_expert, 16)";
    return nullptr;
}
inline const char * check_moe_type(int type, int experts) {
    if (type == Z2H_F32 || type == Z2H_F16) return experts == Z2H_F16 ? nullptr : "F32 and F16 rows need F16 experts";
    if (type == Z2H_BF16) return experts == Z2H_BF16 ? nullptr : "BF16 rows need BF16 experts";
    return "row type must be F32, F16 or BF16";
}

// ---- a paged cache's upkeep
constexpr int MAX_POOL = 1 << 22, MAX_FORKS = 4096, POOL_SEG = 1024;
// What one block does by itself (k_fork_few, an item per wave, and k_moves_few), where a launch less is worth more than many blocks. In us, a row of
// calls, against the general kernels: 4 items on 110 pages 9.8 and 11.0, on 8000 10.2 and 11.9; 16 items on 180 pages 10.4 and 11.6, on 8000
// 12.4 and 11.9; 24 items, two to a wave, 13.0 and 12.0. Compaction of 4 layers, 300 pages: 7.7 and 9.2; 7000: 68.6 and 71.7; 14000:
// 130.1 and 129.5.
constexpr int FEW_PAGES = 8192, FEW_FORKS = 16;
inline const char * check_pool(const z2h_pages * p, int n) {
    if (const char * e = check_pages(p)) return e;
    if (p->n_pages > MAX_POOL) return "pages: n_pages above 2^22";
    if (n < 0 || n > MAX_FORKS) return "pages: more than 4096 items";
    return nullptr;
}
inline const char * check_layers(const z2h_pages * p, int n_layer, int64_t layer_stride) {
    if (n_layer <= 0 || n_layer > 65536) return "pages: n_layer out of range";
    if (n_layer > 1 && (layer_stride % 8 || layer_stride < p->n_pages * p->page_stride)) return "pages: layer_stride must be a multiple of 8, at least n_pages page_strides";
    if (n_layer * (int64_t) p->n_head_kv * p->page_rows * p->head_dim > 1ll << 32) return "pages: a page of more than 2^34 bytes in all layers";
    return nullptr;
}
// Rows that a fork keeps and has room for, of what the source holds and the table has; whole pages, pages in all.
struct ForkSize { int rows, room, whole, pages; };
Z2O_HD ForkSize fork_size(int rows, int room, int have_pages, int table_len, int page_shift) {
    const int held = have_pages << page_shift, most = table_len << page_shift;
    ForkSize f;
    f.rows = rows < 0 ? 0 : rows < held ? rows : held;
    f.room = room < f.rows ? f.rows : room < most ? room : most;
    f.whole = f.rows >> page_shift;
    f.pages = (int) (((int64_t) f.room + (1 << page_shift) - 1) >> page_shift);
    return f;
}
// Workspace: a bit per page, counts per 1024 pages, and per item 32 bytes (fork) or per page its new number and a move (compact).
struct PoolWs { int64_t bits = 0, counts = 0, items = 0, map = 0, moves = 0, bytes = 0; int segs = 0; };

// ---- verification
constexpr int VERIFY_PER_THREAD = 32;              // logits of a row per thread of k_verify_stats
constexpr int VERIFY_SHORT = 256 * VERIFY_PER_THREAD, VERIFY_CHUNK = 1024 * VERIFY_PER_THREAD;
// Longest rows that one block draws from. Behind it two launches, several blocks per row: 64 rows of 32000 probabilities 15.5 us in
// one launch of 1024 threads, 8.5 + 4.6 in two.
constexpr int VERIFY_ONE = 4096;
constexpr int VERIFY_STAT_BYTES = 24, VERIFY_DRAW_BYTES = 32;
inline int verify_chunks(int vocab) { return (vocab + VERIFY_CHUNK - 1) / VERIFY_CHUNK; }
constexpr int64_t MAX_VERIFY_BLOCKS = 1ll << 23;
inline const char * check_verify(int n_seq, int n_draft_max, int n_codebooks, int vocab) {
    if (n_seq < 0 || n_seq > (1 << 20) || n_draft_max < 0 || n_draft_max > 4096 || n_codebooks <= 0 || n_codebooks > 1024)
        return "verify: counts out of range";
    if (vocab <= 0 || vocab > MAX_VOCAB) return "verify: vocab out of range (1 .. 2^20)";
    if ((int64_t) n_seq * (n_draft_max + 1) * n_codebooks * verify_chunks(vocab) > MAX_VERIFY_BLOCKS) return "verify: too many rows";
    return nullptr;
}
inline int64_t verify_stats_bytes(int n_seq, int n_draft_max, int n_codebooks, int vocab) {
    return align256((int64_t) n_seq * (n_draft_max + 1) * n_codebooks * verify_chunks(vocab) * VERIFY_STAT_BYTES);
}
inline int64_t verify_ws_bytes(int n_seq, int n_draft_max, int n_codebooks, int vocab) {
    const int64_t draws = vocab > VERIFY_ONE ? (int64_t) n_seq * n_codebooks : 0;
    return 256 + verify_stats_bytes(n_seq, n_draft_max, n_codebooks, vocab) + align256(draws * VERIFY_DRAW_BYTES) +
           align256(draws * ((vocab + 255) / 256) * 8);
}

// Blocks that share 16 dims of the output: enough for about 768 blocks, three per compute unit, and at most 8, whose sums the join requests all
// at once (up to 16, one after the other: k_moe_down of 128 rows, 8 of 128 experts of 8 x 32, took 48 us in place of 25).
inline int moe_shares(int n_embd) {
    const int tiles = (n_embd + 15) / 16, s = (768 + tiles - 1) / tiles;
    return s < 1 ? 1 : s > MOE_SHARES ? MOE_SHARES : s;
}
inline int moe_h_stride(int n_ff) { return (n_ff + 31) / 32 * 32; }
struct MoeWs { int64_t touched = 0, w = 0, row_sel = 0, row_w = 0, tickets = 0, parts = 0, h = 0, bytes = 0; };
inline MoeWs moe_ws(const z2h_experts & x, int n_rows, int top_k) {
    MoeWs m;
    const int64_t routes = (int64_t) n_rows * top_k;
    const int shares = moe_shares(x.n_embd);
    m.touched = 256;
    m.w = m.touched + align256((routes < x.n_expert ? routes : x.n_expert) * 24);
    m.row_sel = m.w + align256(routes * 4);
    m.row_w = m.row_sel + align256(routes * 4);
    m.tickets = m.row_w + align256(routes * 4);
    m.parts = m.tickets + align256((int64_t) (x.n_embd + 15) / 16 * 4);
    m.h = m.parts + (shares > 1 ? align256((int64_t) shares * n_rows * x.n_embd * 4) : 0);
    m.bytes = m.h + align256(routes * 4 * moe_h_stride(x.n_ff));
    return m;
}

inline PoolWs pool_ws(int n_pages, int n) {
    PoolWs w;
    w.segs = (n_pages + POOL_SEG - 1) / POOL_SEG;
    w.counts = align256((int64_t) w.segs * (POOL_SEG / 8));
    w.items = w.counts + align256((int64_t) w.segs * 4);
    w.map = w.items + align256((int64_t) n * 32);
    w.moves = w.map + align256((int64_t) n_pages * 4);
    w.bytes = w.moves + 256 + align256((int64_t) n_pages * 4);           // (a move: two numbers, at most half of the pages)
    return w;
}

} // namespace z2o
