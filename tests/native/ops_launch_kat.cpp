// ops_launch_kat.cpp — the operators' entry points when a kernel cannot be launched, on the CPU: linked with the host side of their
// translation units and, in place of the runtime, functions that count launches and let one of them fail. A call whose kernel could not be
// launched says so and launches nothing that would read what it left out.
#include "z2h.h"
#include <hip/hip_runtime.h>
#include <cstdint>
#include <cstdio>
#include <cstdlib>

struct z2h_ctx { int failed; };
__attribute__((visibility("hidden"))) int z2h_ctx_fail(z2h_ctx * ctx, int code, const char *) noexcept { ctx->failed = code; return code; }
__attribute__((visibility("hidden"))) int z2h_ctx_device(const z2h_ctx *) noexcept { return 0; }

static int n_launched, fail_at;                                  // the launch that fails, from 1 on (0: none)
static hipError_t pending = hipSuccess;

extern "C" {
hipError_t hipGetDevice(int * d) { *d = 0; return hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipDeviceGetAttribute(int * v, hipDeviceAttribute_t, int) { *v = 256; return hipSuccess; }
hipError_t hipGetLastError() { const hipError_t e = pending; pending = hipSuccess; return e; }
const char * hipGetErrorString(hipError_t) { return "not launched"; }
hipError_t hipLaunchKernel(const void *, dim3, dim3, void **, size_t, hipStream_t) {
    if (++n_launched != fail_at) return hipSuccess;
    return pending = hipErrorLaunchFailure;
}
hipError_t __hipPushCallConfiguration(dim3, dim3, size_t, hipStream_t) { return hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3 * g, dim3 * b, size_t * n, hipStream_t * s) { *g = *b = dim3(1); *n = 0; *s = nullptr; return hipSuccess; }
void ** __hipRegisterFatBinary(const void *) { static void * none; return &none; }
void __hipRegisterFunction(void **, const void *, char *, const char *, unsigned, void *, void *, void *, void *, int *) {}
void __hipRegisterVar(void **, void *, char *, char *, int, size_t, int, int) {}
void __hipUnregisterFatBinary(void **) {}
}

static int bad = 0;
// all launches succeed: `want` of them; the k-th fails: an error, and none behind it
template <typename F>
static void check(const char * what, int want, F call) {
    for (int k = 0; k <= want; ++k) {
        z2h_ctx ctx{0};
        n_launched = 0; fail_at = k; pending = hipSuccess;
        const int rc = call(&ctx), n = k ? k : want;
        if (rc != (k ? Z2H_EDEVICE : Z2H_OK) || n_launched != n) {
            std::printf("%s: launch %d of %d fails: returned %d after %d launches\n", what, k, want, rc, n_launched);
            ++bad;
        }
    }
}

int main() {
    // (addresses that nothing reads)
    void * const p = (void *) (uintptr_t) 0x10000;
    float * const f = (float *) p;
    int32_t * const i = (int32_t *) p;
    double * const d = (double *) p;
    const auto moe = [&](int n_rows, int n_expert) {
        return [=](z2h_ctx * c) {
            const z2h_experts x{p, p, p, Z2H_F16, n_expert, 64, 64};
            return z2h_moe_rows(c, &x, n_rows, 2, 0, f, nullptr, Z2H_F32, p, 64, p, 64, i, f, p, 1ll << 40, nullptr);
        };
    };
    check("moe, 1 row", 2, moe(1, 16));
    check("moe, 8 rows", 2, moe(8, 256));
    check("moe, 9 rows", 3, moe(9, 16));
    check("moe, 128 rows", 3, moe(128, 16));
    check("moe, 1 row of 300 experts", 3, moe(1, 300));
    const auto pages = [&](int n_pages) { z2h_pages g{}; g.k = p; g.v = p; g.page_stride = 4 * 16 * 64; g.type = Z2H_F16; g.n_pages = n_pages; g.page_rows = 16;
                                          g.n_head_kv = 4; g.head_dim = 64; g.n_seq = 64; g.table_len = 16; g.table = i; return g; };
    for (int few = 0; few < 2; ++few) {
        const z2h_pages g = pages(few ? 100 : 100000);
        check("fork", few ? 2 : 3, [&](z2h_ctx * c) { return z2h_pages_fork(c, &g, 1, 0, i, 4, i, i, i, i, i, p, 1ll << 40, nullptr); });
        check("compact", few ? 2 : 3, [&](z2h_ctx * c) { return z2h_pages_compact(c, &g, 1, 0, i, i, i, i, p, 1ll << 40, nullptr); });
    }
    const auto prompt = [&](z2h_ctx * c) { return z2h_prompt_attn(c, 2, i, 600, 8, 2, 64, 0.125f, Z2H_F16, p, 512, p, 128, p, 128, p, 512, nullptr); };
    check("prompt", 1, prompt);
    for (int vocab : {1025, 131072})
        for (int logits = 0; logits < 2; ++logits)
            check("verify", logits + (vocab > 100000 ? 2 : 1), [&](z2h_ctx * c) {
                return z2h_verify(c, 4, 3, 2, vocab, i, i, f, logits ? f : nullptr, nullptr, d, d, i, i, p, 1ll << 40, nullptr);
            });
    std::puts(bad ? "failed" : "ok");
    return bad != 0;
}
