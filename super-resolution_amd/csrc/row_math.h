// Device helpers of the operators that work on rows of channels (residual_norm.hip) and on long vectors (grad_clip.hip):
// 16-byte loads and stores of fp32 / bf16 / fp16 at any element alignment, and sums over a group of lanes.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace sr {

using bf16_t = __bf16;
using f16_t = _Float16;

// A vector access of N elements at the alignment of ONE element: gfx950 takes global accesses at any byte address, so rows and
// views that start at odd elements need no peeling (an access that straddles a cache line costs a second line).
template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Vec {
    T v[N];
};

template <typename T, int N>
__device__ __forceinline__ void load_vec(const T* p, float (&o)[N]) {
    const Vec<T, N> x = *reinterpret_cast<const Vec<T, N>*>(p);
#pragma unroll
    for (int k = 0; k < N; ++k) o[k] = (float)x.v[k];
}

template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[N]) {
    Vec<T, N> x;
#pragma unroll
    for (int k = 0; k < N; ++k) x.v[k] = (T)v[k];   // round to nearest even
    *reinterpret_cast<Vec<T, N>*>(p) = x;
}

// ... a 16-byte store that passes the caches by
template <typename T, int N>
__device__ __forceinline__ void store_vec_nt(T* p, const float (&v)[N]) {
    static_assert(N * sizeof(T) == 16, "one vector");
    typedef unsigned U4 __attribute__((ext_vector_type(4), aligned(2)));
    Vec<T, N> x;
#pragma unroll
    for (int k = 0; k < N; ++k) x.v[k] = (T)v[k];
    U4 b;
    __builtin_memcpy(&b, &x, 16);
    __builtin_nontemporal_store(b, reinterpret_cast<U4*>(p));
}

template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, 0xF, 0xF, true));
}

// Sum over aligned groups of 1 << tl lanes (tl <= 6, the same in every lane); every lane of a group ends with the same bits: each
// step adds two values that are already the same in both halves, and a + b == b + a.
__device__ __forceinline__ float lanes_sum(float v, int tl) {
    if (tl >= 1) v = dpp_add<0xB1>(v);    // quad_perm [1,0,3,2]
    if (tl >= 2) v = dpp_add<0x4E>(v);    // quad_perm [2,3,0,1]
    if (tl >= 3) v = dpp_add<0x141>(v);   // row_half_mirror: the other quad of 8 lanes
    if (tl >= 4) v = dpp_add<0x140>(v);   // row_mirror: the other half of 16 lanes
    if (tl >= 5) {                        // rows 0 <-> 1, 2 <-> 3
        const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    }
    if (tl >= 6) {                        // lanes 0..31 <-> 32..63
        const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    }
    return v;
}

}  // namespace sr
