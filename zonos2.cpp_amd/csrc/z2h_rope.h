// z2h_rope.h — rotary positions of rows of heads, and appending rotated rows to a paged cache.
//
//   (x, y) -> (x cos a - y sin a, x sin a + y cos a),  a = position * theta'
// theta' is formed on the host in 64 bits (rope_turns) and travels with the kernel's arguments; the angle is reduced in 64 bits, so
// positions up to 2^31 keep it to 4e-8 turns. A block's threads form the cosines and sines of their pairs once per row and
// use them for all its heads. Bound by reading and writing the rows once; single tokens by the launch.
#pragma once
#include "z2h_common.h"
#include "z2h_ops_rules.h"

namespace z2d {

// cos and sin of `turn` turns (any double): reduced to the nearest quarter turn in 64 bits, then the Taylor polynomials
// of z_sincos on [-pi/4, pi/4].
__device__ __forceinline__ void turn_sincos(double turn, float & s, float & c) {
    const double f = turn - rint(turn);
    const double q = rint(4.0 * f);
    const float r = (float) ((f - 0.25 * q) * 6.28318530717958647692);
    const float r2 = r * r;
    float sp = 2.75573192e-6f;                                           // 1/9!
    sp = __builtin_fmaf(sp, r2, -1.98412698e-4f);
    sp = __builtin_fmaf(sp, r2, 8.33333333e-3f);
    sp = __builtin_fmaf(sp, r2, -1.66666667e-1f);
    const float sr = __builtin_fmaf(sp * r2, r, r);
    float cp = 2.48015873e-5f;                                           // 1/8!
    cp = __builtin_fmaf(cp, r2, -1.38888889e-3f);
    cp = __builtin_fmaf(cp, r2, 4.16666667e-2f);
    cp = __builtin_fmaf(cp, r2, -0.5f);
    const float cr = __builtin_fmaf(cp, r2, 1.0f);
    const int qi = ((int) q) & 3;
    s = qi == 0 ? sr : qi == 1 ? cr : qi == 2 ? -sr : -cr;
    c = qi == 0 ? cr : qi == 1 ? -sr : qi == 2 ? -cr : sr;
}

struct RopeArgs {
    double turn[z2o::MAX_ROPE_DIMS / 2];           // turns per position of each pair
    float mscale;
    int n_dims, hd, nh, nkv;
    int64_t row0;                                  // of this launch
    const int32_t * seq, * pos;                    // seq NULL: rows of queries only
    const void * q, * k, * v;
    void * q_out, * kc, * vc;
    int64_t qs, qos, ks, vs, page_stride;
    const int32_t * table;
    int n_seq, table_len, n_pages, page_shift;
};

template <int N, typename T> struct VecOf { typedef T type __attribute__((ext_vector_type(N))); };
template <typename T> struct VecOf<1, T> { struct type { T x; __device__ T & operator[](int) { return x; } __device__ const T & operator[](int) const { return x; } }; };
template <int N, typename T>
__device__ __forceinline__ void load_f32(float (&o)[N], const T * p) {
    const typename VecOf<N, T>::type x = *(const typename VecOf<N, T>::type *) p;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = (float) x[i];
}
template <int N, typename T>
__device__ __forceinline__ void store_as(T * p, const float (&o)[N]) {
    typename VecOf<N, T>::type x;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = (T) o[i];
    *(typename VecOf<N, T>::type *) p = x;
}

// values a thread takes of a row at a time: 16 bytes of T, or one pair
template <typename T, bool WIDE> struct RopeUnit { static constexpr int N = WIDE ? 16 / (int) sizeof(T) : 1; };

// grid (rows, shares of the heads). A thread keeps one unit of a head (pairs, or dims behind them) and walks the heads: rotated
// query heads, then rotated key heads and copied value heads. WIDE: rows, strides and pairs allow 16-byte accesses. With both kinds of
// pairs a thread reads and writes whole 16-byte units, so the rows pass once at the rate of a copy: 4099 rows of 32 heads of 128 in
// bf16 (67 MB) 13.8 us, 2088 rows of queries, keys and values into bf16 pages (51 MB) 12.2 us, 16 fp32 rows 3.8 us (launch).
template <typename T, typename TC, bool HALVES, bool WIDE>
__global__ void __launch_bounds__(256) k_rope_append(RopeArgs a) {
    constexpr int N = RopeUnit<T, WIDE>::N, NP = HALVES ? N : WIDE ? N / 2 : 1;      // values behind the pairs; pairs per unit
    const int64_t t = a.row0 + blockIdx.x;
    const int tid = threadIdx.x;
    const int seq = a.seq ? a.seq[t] : 0, pos = a.pos[t];
    if (a.seq && (seq < 0 || seq >= a.n_seq)) return;
    const int half = a.n_dims / 2, up = half / NP, U = up + (a.hd - a.n_dims) / N, HL = 256 / U;
    const int u = tid % U, hl = tid / U;
    int page = -1;
    if (a.k) page = z2o::page_of(a.table, a.n_seq, a.table_len, a.n_pages, a.page_shift, seq, pos);
    const int64_t cell = page < 0 ? 0 : page * a.page_stride + (int64_t) (pos & ((1 << a.page_shift) - 1)) * a.hd;
    const int64_t head_step = (int64_t) a.hd << a.page_shift;
    // the row's cosines and sines once for all heads: a thread's own would take more time than its loads (8 pairs of a bf16
    // unit, 4099 rows of 32 heads: 20.5 us against 14.0)
    __shared__ float s_c[z2o::MAX_ROPE_DIMS / 2], s_s[z2o::MAX_ROPE_DIMS / 2];
    if (tid < half) {
        float c, s;
        turn_sincos((double) pos * a.turn[tid], s, c);
        s_c[tid] = c * a.mscale;
        s_s[tid] = s * a.mscale;
    }
    lds_sync();
    if (hl < HL) {
        if (u < up) {
            float c[NP], s[NP];
#pragma unroll
            for (int i = 0; i < NP; ++i) { c[i] = s_c[u * NP + i]; s[i] = s_s[u * NP + i]; }
            auto turn = [&](const T * x, auto * y) {
                if constexpr (HALVES) {
                    float p[NP], q[NP], r[NP], w[NP];
                    load_f32(p, x + u * NP); load_f32(q, x + half + u * NP);
#pragma unroll
                    for (int i = 0; i < NP; ++i) { r[i] = p[i] * c[i] - q[i] * s[i]; w[i] = p[i] * s[i] + q[i] * c[i]; }
                    store_as(y + u * NP, r); store_as(y + half + u * NP, w);
                } else if constexpr (WIDE) {
                    float p[2 * NP], r[2 * NP];
                    load_f32(p, x + 2 * NP * u);
#pragma unroll
                    for (int i = 0; i < NP; ++i) {
                        r[2 * i] = p[2 * i] * c[i] - p[2 * i + 1] * s[i];
                        r[2 * i + 1] = p[2 * i] * s[i] + p[2 * i + 1] * c[i];
                    }
                    store_as(y + 2 * NP * u, r);
                } else {
                    const float p = (float) x[2 * u], q = (float) x[2 * u + 1];
                    typedef __remove_reference_t(decltype(*y)) O;
                    y[2 * u] = (O) (p * c[0] - q * s[0]);
                    y[2 * u + 1] = (O) (p * s[0] + q * c[0]);
                }
            };
            for (int h = hl + blockIdx.y * HL; h < a.nh + a.nkv; h += HL * gridDim.y) {
                if (h < a.nh) turn((const T *) a.q + t * a.qs + (int64_t) h * a.hd, (T *) a.q_out + t * a.qos + (int64_t) h * a.hd);
                else if (page >= 0) turn((const T *) a.k + t * a.ks + (int64_t) (h - a.nh) * a.hd, (TC *) a.kc + cell + (h - a.nh) * head_step);
            }
        } else {
            const int d = a.n_dims + (u - up) * N;
            float x[N];
            for (int h = hl + blockIdx.y * HL; h < a.nh + a.nkv; h += HL * gridDim.y) {
                if (h < a.nh) {
                    load_f32(x, (const T *) a.q + t * a.qs + (int64_t) h * a.hd + d);
                    store_as((T *) a.q_out + t * a.qos + (int64_t) h * a.hd + d, x);
                } else if (page >= 0) {
                    load_f32(x, (const T *) a.k + t * a.ks + (int64_t) (h - a.nh) * a.hd + d);
                    store_as((TC *) a.kc + cell + (h - a.nh) * head_step + d, x);
                }
            }
        }
    }
    if (page < 0) return;
    const int uv = a.hd / N;
    for (int i = tid + 256 * blockIdx.y; i < a.nkv * uv; i += 256 * gridDim.y) {
        const int g = i / uv, d = i % uv * N;
        float x[N];
        load_f32(x, (const T *) a.v + t * a.vs + (int64_t) g * a.hd + d);
        store_as((TC *) a.vc + cell + g * head_step + d, x);
    }
}

} // namespace z2d
