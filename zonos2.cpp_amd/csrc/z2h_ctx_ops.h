// z2h_ctx_ops.h — what the operators on device tensors (z2h_ops.hip) need of a context, defined beside it in z2h.hip.
#pragma once
#include "z2h.h"

#define Z2H_LOCAL __attribute__((visibility("hidden")))

Z2H_LOCAL int z2h_ctx_fail(z2h_ctx * ctx, int code, const char * what) noexcept;   // sets the error string, returns code
Z2H_LOCAL int z2h_ctx_device(const z2h_ctx * ctx) noexcept;

// z2h_paged_ws_bytes with the reason of a refusal
Z2H_LOCAL int z2h_paged_ws(z2h_ctx * ctx, const z2h_pages * pages, int n_head, int n_rows, int n_group, int64_t * bytes);

// One layer's attention of z2h_step_paged on the context's fused projection rows qkvg [n_rows][R] (query heads, key heads, value
// heads, a gate per query head): norms, append, attention, gates; out is [n_rows][n_head head_dim].
struct Z2hPagedPass {
    z2h_pages pages;                                     // of layer 0
    int64_t layer_stride, ws_bytes;
    z2h_rope rope;
    int n_rows, n_head, n_group, R;
    float qk_eps, scale;
    const int32_t * d_seq, * d_pos;
    void * d_ws;                                         // of z2h_paged_ws_bytes, with the pass's plan
};
Z2H_LOCAL int z2h_paged_layer(z2h_ctx * ctx, const Z2hPagedPass & pass, int layer, float * qkvg, const float * temp, float * out,
                              void * stream);
