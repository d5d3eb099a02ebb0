// z2h_ops_common.h — what the entry points of the operators on device tensors share: the context's device for a call, errors, checks.
#pragma once
#include "z2h.h"
#include "z2h_ctx_ops.h"
#include "z2h_ops_rules.h"
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>

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

const char * check_ws(const void * ws, int64_t have, int64_t need) {
    if (!ws || (uintptr_t) ws % 256) return "workspace must be 256-byte aligned";
    return have < need ? "workspace too small" : nullptr;
}

} // namespace
