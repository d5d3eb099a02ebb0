// z2h_tile.h — what the attention kernels on matrix instructions share: operand types and products, rows of keys and values in LDS,
// loads that go straight there, scalar reads.
#pragma once
#include "z2h_common.h"

namespace z2d {

// What a kernel only reads and a whole wave agrees on is read through the constant address space: as scalar loads, which do not queue behind
// the wave's other loads (a page number read as a vector load waits for all K and V on their way: steps of 2.6 us against 1.6).
template <typename T>
__device__ __forceinline__ const __attribute__((address_space(4))) T * uniform(const T * p) { return (const __attribute__((address_space(4))) T *) p; }
template <typename T>
__device__ __forceinline__ T uniform_copy(const T * p) {
    static_assert(sizeof(T) % 4 == 0, "");
    struct { int w[sizeof(T) / 4]; } x;
#pragma unroll
    for (int i = 0; i < (int) (sizeof(T) / 4); ++i) x.w[i] = uniform((const int *) p)[i];
    return __builtin_bit_cast(T, x);
}

typedef float v16f_t __attribute__((ext_vector_type(16)));
typedef unsigned u4_t __attribute__((ext_vector_type(4)));
typedef short s4_t __attribute__((ext_vector_type(4)));
typedef short s8_t __attribute__((ext_vector_type(8)));
template <typename T> struct Pair { typedef T type __attribute__((ext_vector_type(2))); };
template <typename TC> struct Vec8 { typedef TC type __attribute__((ext_vector_type(8))); };

template <typename TC>
__device__ __forceinline__ v16f_t mfma32(typename Vec8<TC>::type a, typename Vec8<TC>::type b, v16f_t c) {
    if constexpr (__is_same(TC, _Float16)) return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ bool is_finite(float v) { return fabsf(v) < __builtin_inff(); }
// the value of the lane 32 away
__device__ __forceinline__ float other_half(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    const unsigned r0 = r[0], r1 = r[1];
    return __builtin_bit_cast(float, (threadIdx.x & 32) ? r0 : r1);
}

// Rows of keys and values in LDS, stored as they are with their 16-byte pieces permuted by row, so that row-wise reads (keys) and transposing
// reads (values) both take all banks (no conflict counted).
template <int HD>
struct Tile {
    static constexpr int NC = HD / 8, RP = 128 / HD;             // 16-byte pieces of a row, rows per 256 bytes
    // (rows of the same place in 32 are permuted alike)
    static __device__ __forceinline__ int k_at(int row, int piece) { return row * HD + ((piece ^ ((row / RP) & (NC - 1))) * 8); }
    static __device__ __forceinline__ int v_at(int row, int piece) { return row * HD + ((piece ^ (4 * ((row / RP) & (NC / 4 - 1)))) * 8); }
};

// w - hi of two numbers, whose halves are taken out of the pair as it is converted (each by itself they are converted twice over: 27.9
// million vector instructions against 25.6 in 256 rows over 16384 keys)
template <typename F2, typename C2>
__device__ __forceinline__ F2 two_rest(F2 w, C2 hi) {
    if constexpr (__is_same(C2, Pair<__bf16>::type)) {
        const unsigned x = __builtin_bit_cast(unsigned, hi);
        return F2{w[0] - __builtin_bit_cast(float, x << 16), w[1] - __builtin_bit_cast(float, x & 0xffff0000u)};
    } else return F2{w[0] - (float) hi[0], w[1] - (float) hi[1]};
}

// all of the wave's own loads but the last N have arrived; its own LDS reads have been answered
template <int N>
__device__ __forceinline__ void wait_loads_but() { static_assert(N < 16, ""); __builtin_amdgcn_s_waitcnt(0x0f70 | N); asm volatile("" ::: "memory"); }
__device__ __forceinline__ void wait_lds() { asm volatile("" ::: "memory"); __builtin_amdgcn_s_waitcnt(0xc07f); }

template <typename T>
__device__ __forceinline__ void store4(T * p, float x0, float x1, float x2, float x3) {
    typedef T tv __attribute__((ext_vector_type(4)));
    if (((uintptr_t) p & (4 * sizeof(T) - 1)) == 0) {
        tv v = {(T) x0, (T) x1, (T) x2, (T) x3};
        *(tv *) p = v;
    } else {
        p[0] = (T) x0; p[1] = (T) x1; p[2] = (T) x2; p[3] = (T) x3;
    }
}

// 16 bytes per lane from global memory to the 1024 bytes of LDS at `to` (of one mind over the wave), in lane order, in flight until the
// wave waits for its loads
template <typename TC>
__device__ __forceinline__ void to_lds(const TC * from, TC * to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *) from, (__attribute__((address_space(3))) void *) to, 16, 0, 0);
}

} // namespace z2d
