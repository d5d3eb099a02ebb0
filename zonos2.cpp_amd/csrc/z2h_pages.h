// z2h_pages.h — a paged cache's upkeep on the device: sequences that take over others' rows, room for more, the end of sequences, and moving
// the pages in use together.
//
// All state is the page table and a count per page (how many entries name it). Counts are sums, so that no order of the items matters; free
// pages are handed out lowest first by rank: a bit per page and a count per 1024 pages say which is the r-th, and every block finds its own.
//   k_pages_release   a block per item: is it sound, what does it give up and share
//   k_pages_scan      the bits and counts, and in one more block the items' needs and places among the free pages
//   k_pages_take      new pages into the table, and the rows of partly filled pages copied in all layers
//   k_pages_moves     (compact) every page's new number
//   k_pages_compact   pages moved in all layers, table and counts rewritten
// Few items on a small pool are latency alone: k_fork_few does the first three's work but the copies in one block, k_moves_few scan and moves.
// Copies are bound by memory: compaction of 24 layers of 1500 pages of 64 rows (1 GB read and written) 200 to 210 us, 5 TB/s; 64 forks of 2000 rows in
// 24 layers 32 to 52 us by how full the last pages are, of which release and scan take 9.
#pragma once
#include "z2h_common.h"
#include "z2h_ops_rules.h"
#include "z2h_tile.h"

namespace z2d {

struct PoolArgs {
    uint8_t * k, * v;
    int64_t page_bytes, layer_bytes;                             // apart
    int32_t * table, * refs;
    int n_pages, n_seq, table_len, page_shift, row_bytes, nkv, n_layer, segs;
    unsigned long long * bits;
    int * counts;
};
// of an item; ok: 1 and the pages that its source holds, 0 if it is not sound; keeps: the partly filled page stays its own
struct ForkItem { int ok, src, dst, part_page, keeps, need, base, spare; };
static_assert(sizeof(ForkItem) == 32, "workspace layout");
struct ForkArgs {
    PoolArgs p;
    int n;
    const int32_t * src, * dst, * rows, * room;
    int32_t * held;
    ForkItem * items;
};

// leading entries of a sequence that name a page, by the whole block of 256
__device__ __forceinline__ int held_pages(const PoolArgs & p, int seq, int * s_min) {
    const int32_t * row = p.table + (int64_t) seq * p.table_len;
    __syncthreads();
    if (threadIdx.x == 0) *s_min = p.table_len;
    __syncthreads();
    for (int e = threadIdx.x; e < p.table_len; e += 256)
        if ((unsigned) row[e] >= (unsigned) p.n_pages) { atomicMin(s_min, e); break; }
    __syncthreads();
    return *s_min;
}

__global__ void __launch_bounds__(256) k_pages_release(ForkArgs a) {
    __shared__ int s_min, s_bad;
    const int i = blockIdx.x, tid = threadIdx.x;
    const PoolArgs & p = a.p;
    const int src = a.src[i], dst = a.dst[i];
    if (tid == 0) s_bad = src < 0 || src >= p.n_seq || dst < 0 || dst >= p.n_seq;
    __syncthreads();
    bool bad = false;
    for (int j = tid; j < a.n; j += 256) {
        const int d = a.dst[j];
        bad |= (d == dst && j < i) || (d == src && src != dst);
    }
    if (bad) s_bad = 1;
    __syncthreads();
    if (s_bad) {
        if (tid == 0) a.items[i] = ForkItem{0, 0, 0, -1, 0, 0, 0, 0};
        return;
    }
    const int32_t * from = p.table + (int64_t) src * p.table_len, * own = p.table + (int64_t) dst * p.table_len;
    const int have = held_pages(p, src, &s_min), given = src == dst ? have : held_pages(p, dst, &s_min);
    const z2o::ForkSize f = z2o::fork_size(a.rows[i], a.room[i], have, p.table_len, p.page_shift);
    const int part = f.rows & ((1 << p.page_shift) - 1), stay = src == dst ? f.whole + (part > 0) : 0;
    for (int e = tid; e < given; e += 256)
        if (e >= stay) atomicSub(p.refs + own[e], 1);
    if (src != dst)
        for (int e = tid; e < f.whole; e += 256) atomicAdd(p.refs + from[e], 1);
    if (tid == 0) a.items[i] = ForkItem{1 + have, src, dst, part ? from[f.whole] : -1, 0, 0, 0, 0};
}

// which pages are free (FREE) or in use: a bit each, and counts per 1024. With a fork's items, one more block for these.
template <bool FREE>
__global__ void __launch_bounds__(256) k_pages_scan(ForkArgs a) {
    __shared__ int s_wave[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const PoolArgs & p = a.p;
    if ((int) blockIdx.x < p.segs) {
        int count = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int word = 4 * wave + j, page = (int) blockIdx.x * z2o::POOL_SEG + 64 * word + lane;
            const bool in = page < p.n_pages, used = in && p.refs[page] > 0;
            const unsigned long long b = __ballot(FREE ? in && !used : used);
            if (lane == 0) p.bits[(int64_t) blockIdx.x * (z2o::POOL_SEG / 64) + word] = b;
            count += __popcll(b);
        }
        if (lane == 0) s_wave[wave] = count;
        __syncthreads();
        if (tid == 0) p.counts[blockIdx.x] = s_wave[0] + s_wave[1] + s_wave[2] + s_wave[3];
        return;
    }
    int total = 0;
    for (int i0 = 0; i0 < a.n; i0 += 256) {
        const int i = i0 + tid;
        ForkItem it{};
        if (i < a.n) it = a.items[i];
        if (it.ok) {
            const z2o::ForkSize f = z2o::fork_size(a.rows[i], a.room[i], it.ok - 1, p.table_len, p.page_shift);
            it.keeps = it.part_page >= 0 && it.src == it.dst && p.refs[it.part_page] <= 1;
            it.need = min(f.pages - f.whole - it.keeps, p.n_pages);
        }
        int x = it.need;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(x, o);
            if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 63) s_wave[wave] = x;
        __syncthreads();
        int below = total;
        for (int w = 0; w < 4; ++w) {
            if (w < wave) below += s_wave[w];
            total += s_wave[w];
        }
        total = min(total, p.n_pages);                           // (256 needs and this are below 2^31)
        it.base = below + x - it.need;
        if (i < a.n) a.items[i] = it;
    }
}

// The bits' counts of all segments before each, in LDS (segs <= 4096), by a block of 256; entry segs: all of them.
__device__ __forceinline__ void seg_prefix(const PoolArgs & p, int * s_pre, int * s_wave) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int total = 0;
    for (int i0 = 0; i0 < p.segs; i0 += 256) {
        const int i = i0 + tid, c = i < p.segs ? p.counts[i] : 0;
        int x = c;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(x, o);
            if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 63) s_wave[wave] = x;
        __syncthreads();
        int below = total;
        for (int w = 0; w < 4; ++w) {
            if (w < wave) below += s_wave[w];
            total += s_wave[w];
        }
        if (i < p.segs) s_pre[i] = below + x - c;
    }
    if (tid == 0) s_pre[p.segs] = total;
    __syncthreads();
}
// Bits of a word of 64, in 32-bit operations: with a 64-bit shift by a lane's own amount, which lay in the last vector register that the kernel
// had (v_lshrrev_b64 by v31 of 32), about one call of a hundred had a wrong bit; so none after the change. That register is the only cause
// found, from the outside; no kernel of the library has such a shift, and a test of the built code keeps it so.
__device__ __forceinline__ bool bit_of(const unsigned long long * words, int n) { return ((const unsigned *) words)[n >> 5] >> (n & 31) & 1; }
// set bits below bit n (0 .. 63)
__device__ __forceinline__ int bits_below(unsigned long long w, int n) {
    const unsigned lo = (unsigned) w, hi = (unsigned) (w >> 32), below = (1u << (n & 31)) - 1;
    return n & 32 ? __popc(lo) + __popc(hi & below) : __popc(lo & below);
}
// the n-th set bit of w (it has more)
__device__ __forceinline__ int nth_bit(unsigned long long w, int n) {
    unsigned x = (unsigned) w;
    int at = 0, c = __popc(x);
    if (n >= c) { n -= c; x = (unsigned) (w >> 32); at = 32; }
#pragma unroll
    for (int half = 16; half; half >>= 1) {
        c = __popc(x & ((1u << half) - 1));
        if (n >= c) { n -= c; x >>= half; at += half; }
    }
    return at;
}
// the page of rank r among the pages whose bit is set (or not set, among the first `n`); r is below their number
template <bool SET>
__device__ __forceinline__ int page_of_rank(const PoolArgs & p, const int * s_pre, int r) {
    auto before = [&](int seg) { return SET ? s_pre[seg] : seg * z2o::POOL_SEG - s_pre[seg]; };
    int lo = 0, hi = p.segs;
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (before(m) <= r) lo = m; else hi = m;
    }
    r -= before(lo);
    const unsigned long long * w = p.bits + (int64_t) lo * (z2o::POOL_SEG / 64);
    for (int i = 0; i < z2o::POOL_SEG / 64; ++i) {
        const unsigned long long x = SET ? w[i] : ~w[i];
        const int c = __popcll(x);
        if (r < c) return lo * z2o::POOL_SEG + 64 * i + nth_bit(x, r);
        r -= c;
    }
    return -1;
}
// pages below `page` whose bit is set
__device__ __forceinline__ int set_before(const PoolArgs & p, const int * s_pre, int page) {
    const int seg = page / z2o::POOL_SEG, word = page / 64 % (z2o::POOL_SEG / 64);
    if (seg >= p.segs) return s_pre[p.segs];
    const unsigned long long * w = p.bits + (int64_t) seg * (z2o::POOL_SEG / 64);
    int n = s_pre[seg];
    for (int i = 0; i < word; ++i) n += __popcll(w[i]);
    return n + bits_below(w[word], page & 63);
}

typedef unsigned unit_t __attribute__((ext_vector_type(4)));
constexpr int COPY_UNITS = 8;                                    // units of 16 bytes that a thread has on their way

// `bytes` at the start of every head's run of a page (HEADS), or the whole page, to the same place of another, in all layers, by blocks of 256: block
// `part` of `parts`, 32 KB at a time. Whole pages, which nothing reads soon, go past the caches (compaction 210 us in place of 217); rows that forks
// copy do not, since items share sources and the new rows are read next (32 us in place of 53).
template <bool HEADS>
__device__ __forceinline__ void copy_page(const PoolArgs & p, int from, int to, int bytes, int part, int parts) {
    const int heads = HEADS ? p.nkv : 1, units = bytes / 16, total = p.n_layer * 2 * heads * units;
    const int run_bytes = p.row_bytes << p.page_shift;
    const int64_t src = from * p.page_bytes, ahead = to * p.page_bytes - src;
    constexpr int U = COPY_UNITS;
    for (int u0 = part * 256 * U + (int) threadIdx.x; u0 < total; u0 += parts * 256 * U) {
        unit_t x[U];
        uint8_t * at[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int u = u0 + i * 256, run = u / units, head = HEADS ? run % heads : 0, kv = HEADS ? run / heads : run;
            at[i] = (kv & 1 ? p.v : p.k) + src + (int64_t) (kv >> 1) * p.layer_bytes + (int64_t) head * run_bytes + (int64_t) (u - run * units) * 16;
            if (u < total) x[i] = HEADS ? *(const unit_t *) at[i] : __builtin_nontemporal_load((const unit_t *) at[i]);
        }
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (u0 + i * 256 < total) {
                if (HEADS) *(unit_t *) (at[i] + ahead) = x[i];
                else __builtin_nontemporal_store(x[i], (unit_t *) (at[i] + ahead));
            }
    }
}

__global__ void __launch_bounds__(256) k_pages_take(ForkArgs a) {
    __shared__ int s_pre[z2o::MAX_POOL / z2o::POOL_SEG + 1], s_wave[4];
    const int i = blockIdx.x, tid = threadIdx.x;
    const PoolArgs & p = a.p;
    const ForkItem it = a.items[i];
    if (!it.ok) {
        if (blockIdx.y == 0 && tid == 0 && a.held) a.held[i] = -1;
        return;
    }
    const z2o::ForkSize f = z2o::fork_size(a.rows[i], a.room[i], it.ok - 1, p.table_len, p.page_shift);
    const bool copy = it.part_page >= 0 && !it.keeps;
    if (blockIdx.y && !copy) return;
    seg_prefix(p, s_pre, s_wave);
    const int got = max(0, min(it.need, s_pre[p.segs] - it.base)), first = f.whole + it.keeps;
    if (blockIdx.y == 0) {
        const int32_t * from = p.table + (int64_t) it.src * p.table_len;
        int32_t * own = p.table + (int64_t) it.dst * p.table_len;
        if (it.src != it.dst)
            for (int e = tid; e < f.whole; e += 256) own[e] = from[e];
        for (int e = first + tid; e < p.table_len; e += 256) {
            int page = -1;
            if (e < first + got) {
                page = page_of_rank<true>(p, s_pre, it.base + e - first);
                p.refs[page] = 1;
            }
            own[e] = page;
        }
        if (tid == 0) {
            if (copy && it.src == it.dst) atomicSub(p.refs + it.part_page, 1);
            if (a.held) a.held[i] = min(f.room, (first + got) << p.page_shift);
        }
    }
    if (copy && got > 0)
        copy_page<true>(p, it.part_page, page_of_rank<true>(p, s_pre, it.base), (f.rows & ((1 << p.page_shift) - 1)) * p.row_bytes,
                        (int) blockIdx.y, (int) gridDim.y);
}

// ---- few items, a small pool: one block
constexpr int FEW_T = 1024, FEW_WORDS = z2o::FEW_PAGES / 64;
struct FewPool {
    unsigned long long bits[FEW_WORDS];
    int pre[FEW_WORDS + 1];                                      // set bits of all words before each
};
// The bits of the pages that are free (FREE) or in use, and their counts, by the whole block. Counts that this kernel has changed are read past the
// cache of the compute unit.
template <bool FREE>
__device__ __forceinline__ void few_scan(const PoolArgs & p, FewPool & s) {
    constexpr int PER = FEW_WORDS / (FEW_T / 64);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int refs[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int page = min(64 * (wave + FEW_T / 64 * i) + lane, p.n_pages - 1);
        refs[i] = __hip_atomic_load(p.refs + page, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int word = wave + FEW_T / 64 * i, page = 64 * word + lane;
        const unsigned long long b = __ballot(page < p.n_pages && (FREE ? refs[i] <= 0 : refs[i] > 0));
        if (lane == 0) s.bits[word] = b;
    }
    __syncthreads();
    if (wave == 0) {
        int total = 0;
        for (int w0 = 0; w0 < FEW_WORDS; w0 += 64) {
            const int c = __popcll(s.bits[w0 + lane]);
            int x = c;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int y = __shfl_up(x, o);
                if (lane >= o) x += y;
            }
            s.pre[w0 + lane] = total + x - c;
            total += __shfl(x, 63);
        }
        if (lane == 0) s.pre[FEW_WORDS] = total;
    }
    __syncthreads();
}
// the page of rank r among those whose bit is set (or not set); r is below their number
template <bool SET>
__device__ __forceinline__ int few_page(const FewPool & s, int r) {
    auto before = [&](int w) { return SET ? s.pre[w] : 64 * w - s.pre[w]; };
    int lo = 0, hi = FEW_WORDS;
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (before(m) <= r) lo = m; else hi = m;
    }
    return 64 * lo + nth_bit(SET ? s.bits[lo] : ~s.bits[lo], r - before(lo));
}
// leading entries of a sequence that name a page, by one wave, which has the first 64 of its table row in `first`
__device__ __forceinline__ int few_held(const PoolArgs & p, const int32_t * row, int first, int lane) {
    for (int e0 = 0;;) {
        const unsigned long long end = __ballot(e0 + lane >= p.table_len || (unsigned) first >= (unsigned) p.n_pages);
        if (end) return e0 + __builtin_ctzll(end);
        if ((e0 += 64) >= p.table_len) return p.table_len;
        first = row[min(e0 + lane, p.table_len - 1)];
    }
}

// A chain of dependent loads (items, table rows, counts, counts again) between barriers: 7 us for four items on 350 pages, and the copies 4; all
// of it 10.7 us one call behind the other, where the three kernels took 13.9.
__global__ void __launch_bounds__(FEW_T) k_fork_few(ForkArgs a) {
    __shared__ FewPool s;
    struct Item { int src, dst, rows, room, ok, keeps, need, base, part_page; z2o::ForkSize f; };
    __shared__ Item s_item[z2o::FEW_FORKS];
    const PoolArgs & p = a.p;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (tid < a.n) {
        const int src = a.src[tid], dst = a.dst[tid], rows = a.rows[tid], room = a.room[tid];
        s_item[tid].src = src; s_item[tid].dst = dst; s_item[tid].rows = rows; s_item[tid].room = room;
    }
    __syncthreads();
    for (int i = wave; i < a.n; i += FEW_T / 64) {
        Item & it = s_item[i];
        const int src = it.src, dst = it.dst;
        bool bad = src < 0 || src >= p.n_seq || dst < 0 || dst >= p.n_seq;
        if (lane < a.n) {
            const int d = s_item[lane].dst;
            bad |= (d == dst && lane < i) || (d == src && src != dst);
        }
        if (__any(bad)) {
            if (lane == 0) { it.ok = 0; it.need = 0; }
            continue;
        }
        const int32_t * from = p.table + (int64_t) src * p.table_len, * own = p.table + (int64_t) dst * p.table_len;
        const int at = min(lane, p.table_len - 1), from0 = from[at], own0 = own[at];
        const int have = few_held(p, from, from0, lane), given = src == dst ? have : few_held(p, own, own0, lane);
        const z2o::ForkSize f = z2o::fork_size(it.rows, it.room, have, p.table_len, p.page_shift);
        const int part = f.rows & ((1 << p.page_shift) - 1), stay = src == dst ? f.whole + (part > 0) : 0;
        for (int e = lane; e < given; e += 64)
            if (e >= stay) atomicSub(p.refs + (e < 64 ? own0 : own[e]), 1);
        if (src != dst)
            for (int e = lane; e < f.whole; e += 64) atomicAdd(p.refs + (e < 64 ? from0 : from[e]), 1);
        if (lane == 0) { it.ok = 1; it.f = f; it.part_page = part ? from[f.whole] : -1; }
    }
    static_assert(z2o::FEW_FORKS <= 64, "an item per lane");
    wait_loads_but<0>();                                         // every wave's counts have arrived
    __syncthreads();
    if (wave == FEW_T / 64 - 1) {
        int need = 0;
        if (lane < a.n && s_item[lane].ok) {
            Item & it = s_item[lane];
            it.keeps = it.part_page >= 0 && it.src == it.dst && __hip_atomic_load(p.refs + it.part_page, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) <= 1;
            it.need = need = min(it.f.pages - it.f.whole - it.keeps, p.n_pages);
        }
        int x = need;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(x, o);
            if (lane >= o) x += y;
        }
        if (lane < a.n) s_item[lane].base = x - need;
    }
    few_scan<true>(p, s);
    for (int i = wave; i < a.n; i += FEW_T / 64) {
        const Item it = s_item[i];
        if (!it.ok) {
            if (lane == 0) {
                a.items[i].ok = 0;
                if (a.held) a.held[i] = -1;
            }
            continue;
        }
        const bool copy = it.part_page >= 0 && !it.keeps;
        const int got = max(0, min(it.need, s.pre[FEW_WORDS] - it.base)), first = it.f.whole + it.keeps;
        const int32_t * from = p.table + (int64_t) it.src * p.table_len;
        int32_t * own = p.table + (int64_t) it.dst * p.table_len;
        if (it.src != it.dst)
            for (int e = lane; e < it.f.whole; e += 64) own[e] = from[e];
        for (int e = first + lane; e < p.table_len; e += 64) {
            int page = -1;
            if (e < first + got) {
                page = few_page<true>(s, it.base + e - first);
                p.refs[page] = 1;
            }
            own[e] = page;
        }
        if (lane == 0) {
            if (copy && it.src == it.dst) atomicSub(p.refs + it.part_page, 1);
            if (a.held) a.held[i] = min(it.f.room, (first + got) << p.page_shift);
            // (what is left to do: rows of one page to another)
            ForkItem to{};
            to.ok = copy && got > 0;
            to.part_page = it.part_page;
            to.base = to.ok ? few_page<true>(s, it.base) : 0;
            to.need = it.f.rows & ((1 << p.page_shift) - 1);
            a.items[i] = to;
        }
    }
}
__global__ void __launch_bounds__(256) k_fork_copy(ForkArgs a) {
    const ForkItem it = uniform_copy(a.items + blockIdx.x);
    if (it.ok) copy_page<true>(a.p, it.part_page, it.base, it.need * a.p.row_bytes, (int) blockIdx.y, (int) gridDim.y);
}

struct CompactArgs {
    PoolArgs p;
    int32_t * table_out, * refs_out, * n_used;
    int32_t * map;                                               // [n_pages] new numbers
    int32_t * n_moves;
    int2 * moves;
    int blocks;                                                  // that copy
};

__global__ void __launch_bounds__(256) k_pages_moves(CompactArgs a) {
    __shared__ int s_pre[z2o::MAX_POOL / z2o::POOL_SEG + 1], s_wave[4];
    const PoolArgs & p = a.p;
    seg_prefix(p, s_pre, s_wave);
    const int used = s_pre[p.segs], stay = set_before(p, s_pre, used), moves = used - stay;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        *a.n_moves = moves;
        if (a.n_used) *a.n_used = used;
    }
    const int page = blockIdx.x * 256 + threadIdx.x;
    if (page >= p.n_pages) return;
    const bool set = bit_of(p.bits, page);
    if (page < used) {
        a.map[page] = page;
        if (set) a.refs_out[page] = p.refs[page];
        return;
    }
    if (!set) {
        a.map[page] = -1;
        a.refs_out[page] = 0;
        return;
    }
    const int m = set_before(p, s_pre, page) - stay, to = page_of_rank<false>(p, s_pre, m), refs = p.refs[page];
    a.map[page] = to;
    a.moves[m] = make_int2(page, to);
    a.refs_out[page] = 0;
    a.refs_out[to] = refs;
}

__global__ void __launch_bounds__(FEW_T) k_moves_few(CompactArgs a) {
    __shared__ FewPool s;
    const PoolArgs & p = a.p;
    few_scan<false>(p, s);
    const int used = s.pre[FEW_WORDS], tid = threadIdx.x;
    auto before = [&](int page) { return s.pre[page >> 6] + (page & 63 ? bits_below(s.bits[page >> 6], page & 63) : 0); };
    const int stay = before(used);                               // (used <= FEW_PAGES: the last word's end has an entry of its own)
    if (tid == 0) {
        *a.n_moves = used - stay;
        if (a.n_used) *a.n_used = used;
    }
    for (int page = tid; page < p.n_pages; page += FEW_T) {
        const bool set = bit_of(s.bits, page);
        int to = page;
        if (page < used) {
            if (set) a.refs_out[page] = p.refs[page];
        } else {
            to = -1;
            if (set) {
                const int m = before(page) - stay, refs = p.refs[page];
                to = few_page<false>(s, m);
                a.moves[m] = make_int2(page, to);
                a.refs_out[to] = refs;
            }
            a.refs_out[page] = 0;
        }
        a.map[page] = to;
    }
}

__global__ void __launch_bounds__(256) k_pages_compact(CompactArgs a) {
    const PoolArgs & p = a.p;
    const int tid = threadIdx.x;
    if ((int) blockIdx.x >= a.blocks) {
        const int64_t n = (int64_t) p.n_seq * p.table_len, step = (int64_t) (gridDim.x - a.blocks) * 256;
        for (int64_t i = (int64_t) (blockIdx.x - a.blocks) * 256 + tid; i < n; i += step) {
            const int page = p.table[i];
            a.table_out[i] = (unsigned) page < (unsigned) p.n_pages ? a.map[page] : -1;
        }
        return;
    }
    const int moves = *a.n_moves, page_bytes = (p.nkv * p.row_bytes) << p.page_shift, units = page_bytes / 16 * 2 * p.n_layer;
    const int per = max(1, units / (256 * COPY_UNITS));                   // blocks that share a page
    for (int64_t w = blockIdx.x; w < (int64_t) moves * per; w += a.blocks) {
        const int2 m = a.moves[w / per];
        copy_page<false>(p, m.x, m.y, page_bytes, (int) (w % per), per);
    }
}

} // namespace z2d
