// z2h_ctx_ops.h — what the operators on device tensors (z2h_ops.hip) need of a context, defined beside it in z2h.hip.
#pragma once
#include "z2h.h"

#define Z2H_LOCAL __attribute__((visibility("hidden")))

Z2H_LOCAL int z2h_ctx_fail(z2h_ctx * ctx, int code, const char * what) noexcept;   // sets the error string, returns code
Z2H_LOCAL int z2h_ctx_device(const z2h_ctx * ctx) noexcept;
