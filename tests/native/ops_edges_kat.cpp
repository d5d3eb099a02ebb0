// Index rules of the operators on device tensors at their edges (csrc/z2h_ops_rules.h), without a GPU: prints "ok" or the first thing that
// is wrong.
#include "../../zonos2.cpp_amd/csrc/z2h_ops_rules.h"
#include <cstdio>
#include <cstdlib>
#include <initializer_list>

#define EXPECT(cond) do { if (!(cond)) { std::printf("line %d: %s\n", __LINE__, #cond); std::exit(1); } } while (0)

static void groups() {
    EXPECT(z2o::group_of(nullptr, 0, 0) == -1 && z2o::group_of(nullptr, 0, 1 << 24) == -1);      // no groups: no table
    const int32_t one[2] = {2, 5};
    EXPECT(z2o::group_of(one, 1, 1) == -1 && z2o::group_of(one, 1, 2) == 0 && z2o::group_of(one, 1, 4) == 0 && z2o::group_of(one, 1, 5) == -1);
    const int32_t some[5] = {0, 0, 3, 3, 7};                                                   // empty groups among them
    EXPECT(z2o::group_of(some, 4, 0) == 1 && z2o::group_of(some, 4, 2) == 1 && z2o::group_of(some, 4, 3) == 3 && z2o::group_of(some, 4, 6) == 3);
    EXPECT(z2o::group_of(some, 4, 7) == -1);
}

static void launches() {
    for (int threads : {64, 256, 1024}) {
        EXPECT(z2o::launch_blocks(threads) >= 1 << 20 && z2o::launch_blocks(threads) * threads < 1ll << 32);
        EXPECT(z2o::launch_blocks(threads) <= 0x7fffffff);
    }
    // the largest calls' counts: 32-bit numbers of their own
    EXPECT(4 * (z2o::MAX_ROW_HEADS / 4) <= 0x7fffffff - 4 * 256 && z2o::MAX_VERIFY_BLOCKS <= 0x7fffffff);
}

static void no_rows() {
    EXPECT(!z2o::check_rows(nullptr, 128, 2, 64, Z2H_F16, 0) && z2o::check_rows(nullptr, 128, 2, 64, Z2H_F16, 1));
    EXPECT(z2o::check_rows(nullptr, 127, 2, 64, Z2H_F16, 0) && z2o::check_rows(nullptr, 128, 2, 64, Z2H_Q8_0, 0));
}

int main() {
    no_rows();
    launches();
    groups();
    std::puts("ok");
}
