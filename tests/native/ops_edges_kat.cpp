// Index rules of the operators on device tensors at their edges (csrc/z2h_ops_rules.h), without a GPU: prints "ok" or the first thing that
// is wrong.
#include "../../zonos2.cpp_amd/csrc/z2h_ops_rules.h"
#include <cstdio>
#include <cstdlib>

#define EXPECT(cond) do { if (!(cond)) { std::printf("line %d: %s\n", __LINE__, #cond); std::exit(1); } } while (0)

static void groups() {
    EXPECT(z2o::group_of(nullptr, 0, 0) == -1 && z2o::group_of(nullptr, 0, 1 << 24) == -1);      // no groups: no table
    const int32_t one[2] = {2, 5};
    EXPECT(z2o::group_of(one, 1, 1) == -1 && z2o::group_of(one, 1, 2) == 0 && z2o::group_of(one, 1, 4) == 0 && z2o::group_of(one, 1, 5) == -1);
    const int32_t some[5] = {0, 0, 3, 3, 7};                                                   // empty groups among them
    EXPECT(z2o::group_of(some, 4, 0) == 1 && z2o::group_of(some, 4, 2) == 1 && z2o::group_of(some, 4, 3) == 3 && z2o::group_of(some, 4, 6) == 3);
    EXPECT(z2o::group_of(some, 4, 7) == -1);
}

int main() {
    groups();
    std::puts("ok");
}
