// z2h_paged_step.h — what a layer of z2h_step_paged does around the append and the attention: per-head RMSNorm of q and k
// (times the head's temperature for q) before, the heads' sigmoid gates behind (src/zonos2-graph.cpp:96-107, 173). Both pass over the rows once,
// in fp32, and are a few microseconds of launch at the widths of a step.
#pragma once
#include "z2h_common.h"

namespace z2d {

struct HeadRows { float * x; int64_t ld; int n_rows, nh, nkv, hd; const float * temp; float eps; float * out; };

// one wave per (row, query or key head), in place; the sum of squares in 64 bits like the band kernels'
__global__ void __launch_bounds__(256) k_head_norm(HeadRows a) {
    const int lane = threadIdx.x & 63, per = a.nh + a.nkv, id = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= a.n_rows * per) return;
    const int row = id / per, h = id % per, np = a.hd / 2;
    float * p = a.x + row * a.ld + (int64_t) h * a.hd + 2 * lane;
    const float x0 = lane < np ? p[0] : 0.0f, x1 = lane < np ? p[1] : 0.0f;
    const double ss = wave_tree_d((double) (x0 * x0) + (double) (x1 * x1));
    const float sc = 1.0f / sqrtf((float) (ss / (double) a.hd) + a.eps), mul = h < a.nh ? a.temp[h] : 1.0f;
    if (lane < np) { p[0] = x0 * sc * mul; p[1] = x1 * sc * mul; }
}

// out [row][nh hd] times its head's sigmoid(gate), the gates behind the row's value heads
__global__ void __launch_bounds__(256) k_head_gate(HeadRows a) {
    const int width = a.nh * a.hd, row = blockIdx.x;
    const float * gate = a.x + row * a.ld + (int64_t) (a.nh + 2 * a.nkv) * a.hd;
    for (int i = blockIdx.y * 256 + threadIdx.x; i < width; i += 256 * gridDim.y) a.out[(int64_t) row * width + i] *= z_sigmoid(gate[i / a.hd]);
}

} // namespace z2d
