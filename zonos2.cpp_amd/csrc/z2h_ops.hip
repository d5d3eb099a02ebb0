// z2h_ops.hip — the operators on device tensors of include/z2h.h: rotary rows, paged append, attention over shared
// prefixes, draft verification. A translation unit of their own: z2h.hip's kernels keep their code layout.
#include "z2h.h"
#include "z2h_ctx_ops.h"
#include "z2h_ops_rules.h"
#include "z2h_rope.h"
#include "z2h_paged.h"
#include "z2h_verify.h"
#include "z2h_paged_step.h"

#include <algorithm>
#include <atomic>

using namespace z2d;

namespace {

// makes the context's device current for a scope and restores the caller's on every way out
struct OnDevice {
    int prev = -1;
    bool ok = false, moved = false;
    explicit OnDevice(const z2h_ctx * ctx) {
        const int device = z2h_ctx_device(ctx);
        if (hipGetDevice(&prev) != hipSuccess) return;
        moved = prev != device;
        ok = !moved || hipSetDevice(device) == hipSuccess;
    }
    ~OnDevice() { if (ok && moved) (void) hipSetDevice(prev); }
};

int launched(z2h_ctx * ctx) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? Z2H_OK : z2h_ctx_fail(ctx, Z2H_EDEVICE, hipGetErrorString(e));
}

#define CHECK(expr) do { if (const char * e_ = (expr)) return z2h_ctx_fail(ctx, Z2H_EINVAL, e_); } while (0)
#define REQUIRE(cond, what) do { if (!(cond)) return z2h_ctx_fail(ctx, Z2H_EINVAL, what); } while (0)
#define ON_DEVICE OnDevice on_(ctx); if (!on_.ok) return z2h_ctx_fail(ctx, Z2H_EDEVICE, "hipSetDevice failed")

template <typename T, typename TC>
void rope_launch(RopeArgs & a, int n_rows, bool halves, hipStream_t stream) {
    // 16-byte accesses where every row, head and unit of pairs allows them
    constexpr int N = 16 / (int) sizeof(T);
    const auto al = [](const void * p, int64_t stride) { return !p || ((uintptr_t) p % 16 == 0 && stride * (int64_t) sizeof(T) % 16 == 0); };
    const bool wide = a.hd % N == 0 && (a.n_dims / 2) % (halves ? N : N / 2) == 0 && (a.hd - a.n_dims) % N == 0 &&
                      al(a.q, a.qs) && al(a.q_out, a.qos) && al(a.k, a.ks) && al(a.v, a.vs);
    // few rows: their heads over several blocks, so that a row is one round of loads
    const int np = !wide ? 1 : halves ? N : N / 2, units = a.n_dims / 2 / np + (a.hd - a.n_dims) / (wide ? N : 1);
    const int rounds = (a.nh + a.nkv + 256 / units - 1) / (256 / units);
    for (a.row0 = 0; a.row0 < n_rows; a.row0 += z2o::launch_blocks(256)) {
        const dim3 grid(std::min<int64_t>(n_rows - a.row0, z2o::launch_blocks(256)), std::min(rounds, std::max(1, 1024 / n_rows)));
        if (halves && wide) hipLaunchKernelGGL((k_rope_append<T, TC, true, true>), grid, dim3(256), 0, stream, a);
        else if (halves) hipLaunchKernelGGL((k_rope_append<T, TC, true, false>), grid, dim3(256), 0, stream, a);
        else if (wide) hipLaunchKernelGGL((k_rope_append<T, TC, false, true>), grid, dim3(256), 0, stream, a);
        else hipLaunchKernelGGL((k_rope_append<T, TC, false, false>), grid, dim3(256), 0, stream, a);
    }
}
template <typename T>
void rope_launch(RopeArgs & a, int n_rows, bool halves, int cache, hipStream_t stream) {
    if (cache == Z2H_BF16) rope_launch<T, __bf16>(a, n_rows, halves, stream);
    else rope_launch<T, _Float16>(a, n_rows, halves, stream);
}
int rope_run(z2h_ctx * ctx, RopeArgs & a, const z2h_rope * rope, int n_rows, int type, int cache, void * stream) {
    a.mscale = rope->mscale;
    a.n_dims = rope->n_dims;
    z2o::rope_turns(*rope, a.turn);
    ON_DEVICE;
    const bool halves = rope->halves != 0;
    switch (type) {
        case Z2H_F32: rope_launch<float>(a, n_rows, halves, cache, (hipStream_t) stream); break;
        case Z2H_F16: rope_launch<_Float16>(a, n_rows, halves, cache, (hipStream_t) stream); break;
        default: rope_launch<__bf16>(a, n_rows, halves, cache, (hipStream_t) stream); break;
    }
    return launched(ctx);
}

int compute_units(int device) {
    static std::atomic<int> known[64] = {};
    const bool slot = device >= 0 && device < 64;
    int n = slot ? known[device].load(std::memory_order_relaxed) : 0;
    if (n <= 0) {
        if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || n <= 0) return 0;
        if (slot) known[device].store(n, std::memory_order_relaxed);
    }
    return n;
}
// blocks of k_paged_attn: as many as the device holds at once
int attn_blocks(int n_cu) { return 2 * n_cu; }

template <int HD, typename T, typename TC>
void attn_launch(PagedArgs & a, int blocks, hipStream_t stream) {
    hipLaunchKernelGGL((k_paged_attn<HD, T, TC>), dim3(blocks), dim3(256), 0, stream, a);
    // a block per (row, head) while the device holds all of them at once: 1024 of 24 partial results each 7.0 us against 5.3, 8192 of 10
    // each 9.4 against 14.9
    if (a.n_rows * a.n_head <= 4 * blocks) hipLaunchKernelGGL((k_paged_join<HD, T, true>), dim3(a.n_rows * a.n_head), dim3(256), 0, stream, a);
    else
        for (int64_t n = ((int64_t) a.n_rows * a.n_head + 3) / 4; a.join0 < n; a.join0 += z2o::launch_blocks(256))
            hipLaunchKernelGGL((k_paged_join<HD, T, false>), dim3(std::min(n - a.join0, z2o::launch_blocks(256))), dim3(256), 0, stream, a);
}
template <int HD>
void attn_launch(PagedArgs & a, int type, int blocks, hipStream_t stream) {
    switch (type) {
        case Z2H_F32: attn_launch<HD, float, _Float16>(a, blocks, stream); break;
        case Z2H_F16: attn_launch<HD, _Float16, _Float16>(a, blocks, stream); break;
        default: attn_launch<HD, __bf16, __bf16>(a, blocks, stream); break;
    }
}

const char * check_ws(const void * ws, int64_t have, int64_t need) {
    if (!ws || (uintptr_t) ws % 256) return "workspace must be 256-byte aligned";
    return have < need ? "workspace too small" : nullptr;
}

} // namespace

extern "C" {

int z2h_rope_rows(z2h_ctx * ctx, const z2h_rope * rope, int n_rows, int n_head, int head_dim, int type, const void * d_x,
                  int64_t x_stride, void * d_out, int64_t out_stride, const int32_t * d_pos, void * stream) {
    if (!ctx) return Z2H_EINVAL;
    CHECK(z2o::check_rope(rope, head_dim));
    REQUIRE(n_rows >= 0 && n_head > 0 && n_head <= 65536, "rope: row or head count out of range");
    CHECK(z2o::check_rows(d_x, x_stride, n_head, head_dim, type, n_rows));
    CHECK(z2o::check_rows(d_out, out_stride, n_head, head_dim, type, n_rows));
    if (n_rows == 0) return Z2H_OK;
    REQUIRE(d_x != d_out || x_stride == out_stride, "rope: in place with different strides");
    REQUIRE(d_pos, "null positions");
    RopeArgs a{};
    a.hd = head_dim; a.nh = n_head;
    a.pos = d_pos;
    a.q = d_x; a.qs = x_stride; a.q_out = d_out; a.qos = out_stride;
    return rope_run(ctx, a, rope, n_rows, type, Z2H_F16, stream);
}

int z2h_paged_append(z2h_ctx * ctx, const z2h_pages * pages, const z2h_rope * rope, int n_rows, const int32_t * d_seq,
                     const int32_t * d_pos, int type, const void * d_k, int64_t k_stride, const void * d_v, int64_t v_stride,
                     int n_head, const void * d_q, int64_t q_stride, void * d_q_out, int64_t q_out_stride, void * stream) {
    if (!ctx) return Z2H_EINVAL;
    CHECK(z2o::check_pages(pages));
    CHECK(z2o::check_rope(rope, pages->head_dim));
    REQUIRE(n_rows >= 0, "append: n_rows out of range");
    CHECK(z2o::check_rows(d_k, k_stride, pages->n_head_kv, pages->head_dim, type, n_rows));
    CHECK(z2o::check_rows(d_v, v_stride, pages->n_head_kv, pages->head_dim, type, n_rows));
    if (n_rows == 0) return Z2H_OK;
    REQUIRE(d_seq && d_pos, "append: null sequences or positions");
    if (d_q) {
        REQUIRE(n_head > 0 && n_head <= 65536, "append: n_head out of range");
        CHECK(z2o::check_rows(d_q, q_stride, n_head, pages->head_dim, type));
        CHECK(z2o::check_rows(d_q_out, q_out_stride, n_head, pages->head_dim, type));
        REQUIRE(d_q != d_q_out || q_stride == q_out_stride, "append: queries in place with different strides");
    }
    RopeArgs a{};
    a.hd = pages->head_dim; a.nh = d_q ? n_head : 0; a.nkv = pages->n_head_kv;
    a.seq = d_seq; a.pos = d_pos;
    a.q = d_q; a.qs = q_stride; a.q_out = d_q_out; a.qos = q_out_stride;
    a.k = d_k; a.ks = k_stride; a.v = d_v; a.vs = v_stride;
    a.kc = pages->k; a.vc = pages->v; a.page_stride = pages->page_stride;
    a.table = pages->table; a.n_seq = pages->n_seq; a.table_len = pages->table_len; a.n_pages = pages->n_pages;
    a.page_shift = z2o::page_shift_of(pages->page_rows);
    return rope_run(ctx, a, rope, n_rows, type, pages->type, stream);
}

int64_t z2h_paged_ws_bytes(z2h_ctx * ctx, const z2h_pages * pages, int n_head, int n_rows, int n_group) {
    int64_t bytes;
    return ctx && z2h_paged_ws(ctx, pages, n_head, n_rows, n_group, &bytes) == Z2H_OK ? bytes : 0;
}

int z2h_paged_plan(z2h_ctx * ctx, const z2h_pages * pages, int n_head, int n_rows, const int32_t * d_row_start,
                   const int32_t * d_kv_len, int n_group, const int32_t * d_group_start, const int32_t * d_prefix_len,
                   void * d_ws, int64_t ws_bytes, void * stream) {
    if (!ctx) return Z2H_EINVAL;
    CHECK(z2o::check_attn(pages, n_head, n_rows, n_group));
    REQUIRE(d_row_start && d_kv_len && (n_group == 0 || (d_group_start && d_prefix_len)), "plan: null table");
    const int n_cu = compute_units(z2h_ctx_device(ctx));
    if (!n_cu) return z2h_ctx_fail(ctx, Z2H_EDEVICE, "compute-unit count query failed");
    const z2o::AttnWs w = z2o::attn_ws(*pages, n_head, n_rows, n_group, attn_blocks(n_cu));
    CHECK(check_ws(d_ws, ws_bytes, w.bytes));
    PlanArgs a{};
    a.row_start = d_row_start; a.kv_len = d_kv_len; a.group_start = d_group_start; a.prefix_len = d_prefix_len;
    a.n_seq = pages->n_seq; a.n_rows = n_rows; a.n_group = n_group; a.n_head = n_head; a.nkv = pages->n_head_kv;
    a.cap = pages->table_len * pages->page_rows;
    a.blocks = attn_blocks(n_cu);
    uint8_t * ws = (uint8_t *) d_ws;
    a.head = (int32_t *) ws; a.rows = (PlanRow *) (ws + w.rows); a.tiles = (PlanTile *) (ws + w.tiles); a.strips = (PlanStrip *) (ws + w.strips);
    a.shares = (PlanShare *) (ws + w.shares);
    a.max_tiles = (int) w.max_tiles; a.max_parts = (int) w.max_parts;
    ON_DEVICE;
    hipLaunchKernelGGL(k_paged_plan, dim3(1), dim3(PLAN_T), 0, (hipStream_t) stream, a);
    return launched(ctx);
}

int z2h_paged_attn(z2h_ctx * ctx, const z2h_pages * pages, int n_head, int n_rows, int n_group, float scale, int type,
                   const void * d_q, int64_t q_stride, void * d_out, int64_t out_stride, void * d_ws, int64_t ws_bytes,
                   void * stream) {
    if (!ctx) return Z2H_EINVAL;
    CHECK(z2o::check_attn(pages, n_head, n_rows, n_group));
    CHECK(z2o::check_attn_type(type, pages->type));
    CHECK(z2o::check_rows(d_q, q_stride, n_head, pages->head_dim, type, n_rows));
    CHECK(z2o::check_rows(d_out, out_stride, n_head, pages->head_dim, type, n_rows));
    REQUIRE(n_rows == 0 || d_q != d_out || q_stride == out_stride, "attention: in place with different strides");
    REQUIRE(std::isfinite(scale), "attention: scale must be finite");
    const int n_cu = compute_units(z2h_ctx_device(ctx));
    if (!n_cu) return z2h_ctx_fail(ctx, Z2H_EDEVICE, "compute-unit count query failed");
    const z2o::AttnWs w = z2o::attn_ws(*pages, n_head, n_rows, n_group, attn_blocks(n_cu));
    CHECK(check_ws(d_ws, ws_bytes, w.bytes));
    if (n_rows == 0) return Z2H_OK;
    PagedArgs a{};
    a.k = pages->k; a.v = pages->v; a.page_stride = pages->page_stride; a.qs = q_stride; a.os = out_stride;
    a.table = pages->table; a.n_seq = pages->n_seq; a.table_len = pages->table_len; a.n_pages = pages->n_pages;
    a.page_shift = z2o::page_shift_of(pages->page_rows);
    a.nkv = pages->n_head_kv; a.n_head = n_head; a.n_rows = n_rows; a.n_group = n_group; a.scale = scale;
    a.q = d_q; a.out = d_out;
    uint8_t * ws = (uint8_t *) d_ws;
    a.head = (const int32_t *) ws; a.rows = (const PlanRow *) (ws + w.rows); a.tiles = (const PlanTile *) (ws + w.tiles);
    a.strips = (const PlanStrip *) (ws + w.strips); a.shares = (const PlanShare *) (ws + w.shares);
    a.part_ml = (float2 *) (ws + w.ml); a.part_o = (float *) (ws + w.o);
    const int blocks = attn_blocks(n_cu);
    a.max_tiles = (int) w.max_tiles;
    a.blocks = blocks;
    ON_DEVICE;
    switch (pages->head_dim) {
        case 32: attn_launch<32>(a, type, blocks, (hipStream_t) stream); break;
        case 64: attn_launch<64>(a, type, blocks, (hipStream_t) stream); break;
        default: attn_launch<128>(a, type, blocks, (hipStream_t) stream); break;
    }
    return launched(ctx);
}

int64_t z2h_verify_ws_bytes(int n_seq, int n_draft_max, int n_codebooks, int vocab) {
    return z2o::check_verify(n_seq, n_draft_max, n_codebooks, vocab) ? 0 : z2o::verify_ws_bytes(n_seq, n_draft_max, n_codebooks, vocab);
}

int z2h_verify(z2h_ctx * ctx, int n_seq, int n_draft_max, int n_codebooks, int vocab, const int32_t * d_draft,
               const int32_t * d_n_draft, const float * d_target, const float * d_temperature, const float * d_draft_probs,
               const double * d_u_accept, const double * d_u_draw, int32_t * d_n_accept, int32_t * d_codes, void * d_ws,
               int64_t ws_bytes, void * stream) {
    if (!ctx) return Z2H_EINVAL;
    CHECK(z2o::check_verify(n_seq, n_draft_max, n_codebooks, vocab));
    if (n_seq == 0) return Z2H_OK;
    REQUIRE(d_target && d_u_draw && d_n_accept && d_codes && (n_draft_max == 0 || (d_draft && d_u_accept)), "verify: null argument");
    CHECK(check_ws(d_ws, ws_bytes, z2o::verify_ws_bytes(n_seq, n_draft_max, n_codebooks, vocab)));
    VerifyArgs a{};
    a.n_seq = n_seq; a.K = n_draft_max; a.C = n_codebooks; a.V = vocab;
    a.draft = d_draft; a.n_draft = d_n_draft; a.target = d_target; a.temperature = d_temperature; a.draft_probs = d_draft_probs;
    a.u_accept = d_u_accept; a.u_draw = d_u_draw; a.n_accept = d_n_accept; a.codes = d_codes;
    a.n_chunk = z2o::verify_chunks(vocab);
    a.stats = (VerifyStat *) d_ws;
    uint8_t * draws_at = (uint8_t *) d_ws + z2o::verify_stats_bytes(n_seq, n_draft_max, n_codebooks, vocab);
    a.draws = (VerifyDraw *) draws_at;
    a.sums = (double *) (draws_at + z2o::align256((int64_t) n_seq * n_codebooks * z2o::VERIFY_DRAW_BYTES));
    const hipStream_t st = (hipStream_t) stream;
    const int draws = n_seq * n_codebooks;
    ON_DEVICE;
    const int rows = n_seq * (n_draft_max + 1) * n_codebooks;
    if (d_temperature) {
        const int threads = vocab <= z2o::VERIFY_SHORT ? 256 : 1024;
        const int64_t blocks = (int64_t) rows * a.n_chunk;       // (a row of at most VERIFY_SHORT logits is one chunk)
        for (; a.block0 < blocks; a.block0 += z2o::launch_blocks(threads)) {
            const dim3 grid(std::min(blocks - a.block0, z2o::launch_blocks(threads)));
            if (threads == 256) hipLaunchKernelGGL(k_verify_stats<256>, grid, dim3(256), 0, st, a);
            else hipLaunchKernelGGL(k_verify_stats<1024>, grid, dim3(1024), 0, st, a);
        }
        if (int rc = launched(ctx)) return rc;                   // (no draws from statistics that nobody formed)
    }
    if (vocab <= z2o::VERIFY_ONE) hipLaunchKernelGGL(k_verify, dim3(draws), dim3(256), 0, st, a);
    else {
        // shares of 1024 codes (a round of the block's loads) or more, about 512 blocks in all
        a.n_share = std::min((vocab + 1023) / 1024, std::max(1, 512 / draws));
        hipLaunchKernelGGL(k_verify_sums, dim3(draws * a.n_share), dim3(256), 0, st, a);
        hipLaunchKernelGGL(k_verify_pick, dim3(draws), dim3(256), 0, st, a);
    }
    return launched(ctx);
}

} // extern "C"

int z2h_paged_ws(z2h_ctx * ctx, const z2h_pages * pages, int n_head, int n_rows, int n_group, int64_t * bytes) {
    CHECK(z2o::check_attn(pages, n_head, n_rows, n_group));
    const int n_cu = compute_units(z2h_ctx_device(ctx));
    if (!n_cu) return z2h_ctx_fail(ctx, Z2H_EDEVICE, "compute-unit count query failed");
    *bytes = z2o::attn_ws(*pages, n_head, n_rows, n_group, attn_blocks(n_cu)).bytes;
    return Z2H_OK;
}

int z2h_paged_layer(z2h_ctx * ctx, const Z2hPagedPass & s, int layer, float * qkvg, const float * temp, float * out, void * stream) {
    z2h_pages pages = s.pages;
    const int64_t at = 2 * layer * s.layer_stride;
    pages.k = (uint8_t *) pages.k + at;
    pages.v = (uint8_t *) pages.v + at;
    const int nh = s.n_head, nkv = pages.n_head_kv, hd = pages.head_dim;
    const HeadRows h{qkvg, s.R, s.n_rows, nh, nkv, hd, temp, s.qk_eps, out};
    float * k = qkvg + nh * hd, * v = k + nkv * hd;
    {
        ON_DEVICE;
        hipLaunchKernelGGL(k_head_norm, dim3((s.n_rows * (nh + nkv) + 3) / 4), dim3(256), 0, (hipStream_t) stream, h);
        if (int rc = launched(ctx)) return rc;
    }
    if (int rc = z2h_paged_append(ctx, &pages, &s.rope, s.n_rows, s.d_seq, s.d_pos, Z2H_F32, k, s.R, v, s.R, nh, qkvg, s.R, qkvg, s.R, stream))
        return rc;
    if (int rc = z2h_paged_attn(ctx, &pages, nh, s.n_rows, s.n_group, s.scale, Z2H_F32, qkvg, s.R, out, (int64_t) nh * hd, s.d_ws, s.ws_bytes, stream))
        return rc;
    ON_DEVICE;
    hipLaunchKernelGGL(k_head_gate, dim3(s.n_rows, (nh * hd + 1023) / 1024), dim3(256), 0, (hipStream_t) stream, h);
    return launched(ctx);
}
