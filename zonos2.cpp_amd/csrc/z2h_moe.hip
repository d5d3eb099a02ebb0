// z2h_moe.hip — z2h_moe_rows of include/z2h.h: a mixture-of-experts layer for a few rows on the caller's tensors.
#include "z2h_ops_common.h"
#include "z2h_moe.h"

using namespace z2d;

namespace {

// Rows up to which every block of k_moe_gate_up routes for itself, a wave per row, which saves a launch: 5 rows, 1 of 16 experts of 4096 x 2048, 57.8 us
// in place of 59.7, 8 rows 73.4 and 75.4; with 16 rows, two to a wave, it is even at last (4 of 32 of 1536 x 2048: 124.3 and 123.3; 128 rows of
// 128 experts of 8 x 32: 116 and 52).
constexpr int MOE_OWN_ROWS = 8;

template <typename T, typename TW, int NT>
void gate_up_launch(const MoeArgs & a, int n_cu, hipStream_t st) {
    const int64_t tiles = (int64_t) std::min(a.E, a.n * a.k) * (a.F / 8);
    hipLaunchKernelGGL((k_moe_gate_up<T, TW, NT>), dim3(std::min<int64_t>(n_cu * moe_per_cu<T, NT>(), tiles)), dim3(MOE_T), 0, st, a);
}
// (each kernel takes its bounds and places from what the one before leaves in the workspace: none is launched behind one that could not be)
template <typename T, typename TW>
int moe_launch(z2h_ctx * ctx, const MoeArgs & a, int n_cu, hipStream_t st) {
    if (a.row_sel) {
        hipLaunchKernelGGL(k_moe_route, dim3(a.n), dim3(64), 0, st, a);
        if (int rc = launched(ctx)) return rc;
    }
    // One tile of 16 rows leaves registers for two blocks per compute unit, two read the weights of an expert with more rows once. From 17 rows
    // on, two: 32 rows most of which take the same 8 of 64 experts 61 us in place of 76, 64 rows the same 6 of 64 81 and 110, 128 rows, 2 of 8, 95 and
    // 111. Spread evenly over many experts, of whom few have more than 16 rows, one would be a little faster (32 rows, 8 of 64: 174 to 188 in
    // place of 177 to 195; 64 rows, 6 of 64: 200 in place of 207); the host does not know the spread.
    if (a.n <= 16) gate_up_launch<T, TW, 1>(a, n_cu, st);
    else gate_up_launch<T, TW, 2>(a, n_cu, st);
    if (int rc = launched(ctx)) return rc;
    hipLaunchKernelGGL((k_moe_down<T, TW>), dim3(a.tiles, a.shares), dim3(MOE_DT), MOE_DW * a.n * 64, st, a);
    return launched(ctx);
}

} // namespace

extern "C" {

int64_t z2h_moe_rows_ws_bytes(const z2h_experts * experts, int n_rows, int top_k) {
    return z2o::check_moe(experts, n_rows, top_k) ? 0 : z2o::moe_ws(*experts, n_rows, top_k).bytes;
}

int z2h_moe_rows(z2h_ctx * ctx, const z2h_experts * experts, int n_rows, int top_k, int renorm, const float * d_logits,
                 const float * d_bias, int type, const void * d_x, int64_t x_stride, void * d_out, int64_t out_stride, int32_t * d_sel,
                 float * d_weights, void * d_ws, int64_t ws_bytes, void * stream) {
    if (!ctx) return Z2H_EINVAL;
    CHECK(z2o::check_moe(experts, n_rows, top_k));
    CHECK(z2o::check_moe_type(type, experts->type));
    CHECK(z2o::check_rows(d_x, x_stride, 1, experts->n_embd, type, n_rows));
    CHECK(z2o::check_rows(d_out, out_stride, 1, experts->n_embd, type, n_rows));
    if (n_rows == 0) return Z2H_OK;
    REQUIRE(d_x != d_out || x_stride == out_stride, "moe: in place with different strides");
    REQUIRE(d_logits, "moe: null logits");
    const z2o::MoeWs w = z2o::moe_ws(*experts, n_rows, top_k);
    CHECK(check_ws(d_ws, ws_bytes, w.bytes));
    uint8_t * ws = (uint8_t *) d_ws;
    MoeArgs a{};
    a.gate = experts->gate; a.up = experts->up; a.down = experts->down;
    a.E = experts->n_expert; a.F = experts->n_ff; a.D = experts->n_embd; a.n = n_rows; a.k = top_k; a.renorm = renorm;
    a.logits = d_logits; a.bias = d_bias; a.x = d_x; a.xs = x_stride; a.out = d_out; a.os = out_stride;
    a.sel = d_sel; a.weights = d_weights;
    a.shares = z2o::moe_shares(a.D); a.tiles = (a.D + 15) / 16;
    a.table = (MoeTable *) ws; a.touched = (MoeTouched *) (ws + w.touched); a.w = (float *) (ws + w.w);
    if (n_rows > MOE_OWN_ROWS || a.E > MOE_OWN_EXPERTS) { a.row_sel = (int32_t *) (ws + w.row_sel); a.row_w = (float *) (ws + w.row_w); }
    a.tickets = (int32_t *) (ws + w.tickets); a.parts = (float *) (ws + w.parts); a.h = (float *) (ws + w.h); a.hs = z2o::moe_h_stride(a.F);
    const int n_cu = compute_units(z2h_ctx_device(ctx));
    if (!n_cu) return z2h_ctx_fail(ctx, Z2H_EDEVICE, "compute-unit count query failed");
    ON_DEVICE;
    switch (type) {
        case Z2H_F32: return moe_launch<float, _Float16>(ctx, a, n_cu, (hipStream_t) stream);
        case Z2H_F16: return moe_launch<_Float16, _Float16>(ctx, a, n_cu, (hipStream_t) stream);
        default: return moe_launch<__bf16, __bf16>(ctx, a, n_cu, (hipStream_t) stream);
    }
}

} // extern "C"
