// z2h_pages.hip — the upkeep of a paged cache of include/z2h.h: forks (shares, room, ends) and compaction.
#include "z2h_ops_common.h"
#include "z2h_pages.h"

using namespace z2d;

namespace {

PoolArgs pool_args(const z2h_pages & pages, int n_layer, int64_t layer_stride, int32_t * refs, const z2o::PoolWs & w, uint8_t * ws) {
    PoolArgs p{};
    p.k = (uint8_t *) pages.k; p.v = (uint8_t *) pages.v;
    p.page_bytes = 2 * pages.page_stride; p.layer_bytes = 2 * layer_stride;
    p.table = const_cast<int32_t *>(pages.table); p.refs = refs;
    p.n_pages = pages.n_pages; p.n_seq = pages.n_seq; p.table_len = pages.table_len; p.page_shift = z2o::page_shift_of(pages.page_rows);
    p.row_bytes = 2 * pages.head_dim; p.nkv = pages.n_head_kv; p.n_layer = n_layer; p.segs = w.segs;
    p.bits = (unsigned long long *) ws; p.counts = (int *) (ws + w.counts);
    return p;
}

} // namespace

extern "C" {

int64_t z2h_pages_ws_bytes(z2h_ctx * ctx, const z2h_pages * pages, int n) {
    if (!ctx) return 0;
    if (const char * e = z2o::check_pool(pages, n)) { z2h_ctx_fail(ctx, Z2H_EINVAL, e); return 0; }
    return z2o::pool_ws(pages->n_pages, n).bytes;
}

int z2h_pages_fork(z2h_ctx * ctx, const z2h_pages * pages, int n_layer, int64_t layer_stride, int32_t * d_refs, int n, const int32_t * d_src,
                   const int32_t * d_dst, const int32_t * d_rows, const int32_t * d_room, int32_t * d_held, void * d_ws, int64_t ws_bytes,
                   void * stream) {
    if (!ctx) return Z2H_EINVAL;
    CHECK(z2o::check_pool(pages, n));
    CHECK(z2o::check_layers(pages, n_layer, layer_stride));
    if (n == 0) return Z2H_OK;
    REQUIRE(d_refs && d_src && d_dst && d_rows && d_room, "fork: null argument");
    const z2o::PoolWs w = z2o::pool_ws(pages->n_pages, n);
    CHECK(check_ws(d_ws, ws_bytes, w.bytes));
    ForkArgs a{};
    a.p = pool_args(*pages, n_layer, layer_stride, d_refs, w, (uint8_t *) d_ws);
    a.n = n; a.src = d_src; a.dst = d_dst; a.rows = d_rows; a.room = d_room; a.held = d_held;
    a.items = (ForkItem *) ((uint8_t *) d_ws + w.items);
    const hipStream_t st = (hipStream_t) stream;
    ON_DEVICE;
    // 8 units of 16 bytes per thread of what a page may have to copy
    const int64_t units = (int64_t) n_layer * 2 * pages->n_head_kv * pages->page_rows * pages->head_dim / 8;
    const int share = (int) std::min<int64_t>(std::max<int64_t>(1, units / (256 * COPY_UNITS)), std::max(1, 8192 / n));
    if (n <= z2o::FEW_FORKS && pages->n_pages <= z2o::FEW_PAGES) {
        hipLaunchKernelGGL(k_fork_few, dim3(1), dim3(FEW_T), 0, st, a);
        if (int rc = launched(ctx)) return rc;
        hipLaunchKernelGGL(k_fork_copy, dim3(n, share), dim3(256), 0, st, a);
        return launched(ctx);
    }
    hipLaunchKernelGGL(k_pages_release, dim3(n), dim3(256), 0, st, a);
    if (int rc = launched(ctx)) return rc;
    hipLaunchKernelGGL(k_pages_scan<true>, dim3(w.segs + 1), dim3(256), 0, st, a);
    if (int rc = launched(ctx)) return rc;
    hipLaunchKernelGGL(k_pages_take, dim3(n, share), dim3(256), 0, st, a);
    return launched(ctx);
}

int z2h_pages_compact(z2h_ctx * ctx, const z2h_pages * pages, int n_layer, int64_t layer_stride, int32_t * d_refs, int32_t * d_table_out,
                      int32_t * d_refs_out, int32_t * d_n_used, void * d_ws, int64_t ws_bytes, void * stream) {
    if (!ctx) return Z2H_EINVAL;
    CHECK(z2o::check_pool(pages, 0));
    CHECK(z2o::check_layers(pages, n_layer, layer_stride));
    REQUIRE(d_refs && d_table_out && d_refs_out, "compact: null argument");
    const z2o::PoolWs w = z2o::pool_ws(pages->n_pages, 0);
    CHECK(check_ws(d_ws, ws_bytes, w.bytes));
    uint8_t * ws = (uint8_t *) d_ws;
    ForkArgs s{};
    s.p = pool_args(*pages, n_layer, layer_stride, d_refs, w, ws);
    CompactArgs a{};
    a.p = s.p; a.table_out = d_table_out; a.refs_out = d_refs_out; a.n_used = d_n_used;
    a.map = (int32_t *) (ws + w.map); a.n_moves = (int32_t *) (ws + w.moves); a.moves = (int2 *) (ws + w.moves + 256);
    // eight units of 16 bytes per thread of what half of the pages have, 2048 blocks at most
    const int64_t units = (int64_t) n_layer * 2 * pages->n_head_kv * pages->page_rows * pages->head_dim / 8;
    a.blocks = (int) std::min<int64_t>(2048, std::max<int64_t>(1, pages->n_pages / 2 * std::max<int64_t>(1, units / (256 * COPY_UNITS))));
    const int64_t entries = (int64_t) pages->n_seq * pages->table_len;
    const hipStream_t st = (hipStream_t) stream;
    ON_DEVICE;
    if (pages->n_pages <= z2o::FEW_PAGES) hipLaunchKernelGGL(k_moves_few, dim3(1), dim3(FEW_T), 0, st, a);
    else {
        hipLaunchKernelGGL(k_pages_scan<false>, dim3(w.segs), dim3(256), 0, st, s);
        if (int rc = launched(ctx)) return rc;
        hipLaunchKernelGGL(k_pages_moves, dim3((pages->n_pages + 255) / 256), dim3(256), 0, st, a);
    }
    if (int rc = launched(ctx)) return rc;
    hipLaunchKernelGGL(k_pages_compact, dim3(a.blocks + (int) std::min<int64_t>((entries + 1023) / 1024, 1024)), dim3(256), 0, st, a);
    return launched(ctx);
}

} // extern "C"
