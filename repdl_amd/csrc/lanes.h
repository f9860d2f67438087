// Reductions over the lanes of a wave without LDS, and a barrier that orders LDS alone.
#pragma once

#include <hip/hip_runtime.h>

// Value of a partner lane for step `off` of a butterfly in which every lane of a group of `off` lanes already holds the group's
// result (so any lane of the neighbouring group will do): quad permutations and mirrors inside a row of 16 lanes, as operands
// of the vector instruction that uses them.
template <int CTRL>
__device__ __forceinline__ float lane_partner(float v)
{
    return __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(v), CTRL, 0xF, 0xF, true));
}

// v combined over W = 4 .. 64 neighbouring lanes, in every one of them.  The order is that of the butterfly v op v[lane ^ 1],
// ^ 2, ^ 4, ...; op has to be commutative.  Steps of 16 and 32 lanes swap rows between two copies of the register.  Against six
// ds_bpermute round trips (about 100 clocks each): about 10 clocks a step, which is what a row's two reductions cost when
// few waves share a SIMD.
template <int W, typename Op>
__device__ __forceinline__ float lanes_reduce(float v, Op op)
{
    static_assert(W == 4 || W == 8 || W == 16 || W == 32 || W == 64, "whole groups of lanes");
    v = op(v, lane_partner<0xB1>(v)); // quad_perm [1,0,3,2]
    v = op(v, lane_partner<0x4E>(v)); // quad_perm [2,3,0,1]
    if (W >= 8)
        v = op(v, lane_partner<0x141>(v)); // row_half_mirror
    if (W >= 16)
        v = op(v, lane_partner<0x140>(v)); // row_mirror
    if (W >= 32)
    {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    if (W >= 64)
    {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    return v;
}

template <int W>
__device__ __forceinline__ float lanes_sum(float v)
{
    return lanes_reduce<W>(v, [](float a, float b) { return a + b; });
}

// (NaN passes through)
template <int W>
__device__ __forceinline__ float lanes_max(float v)
{
    return lanes_reduce<W>(v, [](float a, float b) { return __builtin_elementwise_maximum(a, b); });
}

// Barrier of the workgroup that orders LDS accesses only: loads from global memory stay under way across it (__syncthreads
// waits for them).
__device__ __forceinline__ void lds_barrier()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}
