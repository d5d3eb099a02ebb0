// z2h_prompt.hip — z2h_prompt_attn of include/z2h.h: causal attention of packed prompts.
#include "z2h_ops_common.h"
#include "z2h_prompt.h"

using namespace z2d;

namespace {

template <int HD, typename T>
void prompt_launch(PromptArgs & a, int n_cu, hipStream_t st) {
    const auto al = [](const void * p, int64_t stride) { return (uintptr_t) p % 16 == 0 && stride * (int64_t) sizeof(T) % 16 == 0; };
    const bool aligned = al(a.k, a.ks) && al(a.v, a.vs);
    const int group = a.n_head / a.nkv;
    const z2o::PromptCut cut = z2o::prompt_cut(a.n_rows, a.n_seq, a.n_head, a.nkv, HD, sizeof(T) == 4, n_cu);
    const bool small = cut == z2o::PROMPT_SMALL, pair = cut == z2o::PROMPT_PAIR;
    for (int64_t n = z2o::prompt_slots(a.n_rows, a.n_seq, small ? z2o::small_rows(group) : z2o::tile_rows(group)) * a.nkv; a.block0 < n;
         a.block0 += z2o::launch_blocks(256)) {
        const dim3 grid(std::min(n - a.block0, z2o::launch_blocks(256)));
        if (small && aligned) hipLaunchKernelGGL((k_prompt_small<HD, T, true>), grid, dim3(256), 0, st, a);
        else if (small) hipLaunchKernelGGL((k_prompt_small<HD, T, false>), grid, dim3(256), 0, st, a);
        else if (pair && aligned) hipLaunchKernelGGL((k_prompt<HD, T, true, 2>), grid, dim3(512), 0, st, a);
        else if (pair) hipLaunchKernelGGL((k_prompt<HD, T, false, 2>), grid, dim3(512), 0, st, a);
        else if (aligned) hipLaunchKernelGGL((k_prompt<HD, T, true, 1>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((k_prompt<HD, T, false, 1>), grid, dim3(256), 0, st, a);
    }
}
template <int HD>
void prompt_launch(PromptArgs & a, int type, int n_cu, hipStream_t st) {
    switch (type) {
        case Z2H_F32: prompt_launch<HD, float>(a, n_cu, st); break;
        case Z2H_F16: prompt_launch<HD, _Float16>(a, n_cu, st); break;
        default: prompt_launch<HD, __bf16>(a, n_cu, st); break;
    }
}

} // namespace

extern "C" {

int z2h_prompt_attn(z2h_ctx * ctx, int n_seq, const int32_t * d_row_start, int n_rows, int n_head, int n_head_kv, int head_dim,
                    float scale, int type, const void * d_q, int64_t q_stride, const void * d_k, int64_t k_stride, const void * d_v,
                    int64_t v_stride, void * d_out, int64_t out_stride, void * stream) {
    if (!ctx) return Z2H_EINVAL;
    CHECK(z2o::check_prompt(n_seq, n_rows, n_head, n_head_kv, head_dim));
    CHECK(z2o::check_rows(d_q, q_stride, n_head, head_dim, type, n_rows));
    CHECK(z2o::check_rows(d_k, k_stride, n_head_kv, head_dim, type, n_rows));
    CHECK(z2o::check_rows(d_v, v_stride, n_head_kv, head_dim, type, n_rows));
    CHECK(z2o::check_rows(d_out, out_stride, n_head, head_dim, type, n_rows));
    REQUIRE(std::isfinite(scale), "prompt: scale must be finite");
    if (n_rows == 0 || n_seq == 0) return Z2H_OK;
    REQUIRE(d_q != d_out || q_stride == out_stride, "prompt: in place with different strides");
    REQUIRE(d_row_start, "prompt: null row table");
    PromptArgs a{};
    a.start = d_row_start; a.n_seq = n_seq; a.n_rows = n_rows; a.n_head = n_head; a.nkv = n_head_kv;
    a.q = d_q; a.k = d_k; a.v = d_v; a.out = d_out;
    a.qs = q_stride; a.ks = k_stride; a.vs = v_stride; a.os = out_stride;
    a.scale = scale;
    const int n_cu = compute_units(z2h_ctx_device(ctx));
    if (!n_cu) return z2h_ctx_fail(ctx, Z2H_EDEVICE, "compute-unit count query failed");
    ON_DEVICE;
    switch (head_dim) {
        case 32: prompt_launch<32>(a, type, n_cu, (hipStream_t) stream); break;
        case 64: prompt_launch<64>(a, type, n_cu, (hipStream_t) stream); break;
        default: prompt_launch<128>(a, type, n_cu, (hipStream_t) stream); break;
    }
    return launched(ctx);
}

} // extern "C"
