// Tensors of binary32, bfloat16 or binary16 elements that are computed on in binary32: loads widen exactly, stores
// round once (to nearest even).  Shared by the kernels of layer normalisation, dropout and the preference loss.
#pragma once

#include "common.h"

// Widening and rounding of one element, by the type's code in the C ABI.
template <int DT>
struct LowpType;

template <>
struct LowpType<REPDL_F32>
{
    typedef float T;
    __device__ static __forceinline__ float widen(float v) { return v; }
    __device__ static __forceinline__ float narrow(float v) { return v; }
};

template <>
struct LowpType<REPDL_BF16>
{
    typedef __bf16 T;
    __device__ static __forceinline__ float widen(__bf16 v) { return (float)v; }
    __device__ static __forceinline__ __bf16 narrow(float v) { return (__bf16)v; }
};

template <>
struct LowpType<REPDL_F16>
{
    typedef _Float16 T;
    __device__ static __forceinline__ float widen(_Float16 v) { return (float)v; }
    __device__ static __forceinline__ _Float16 narrow(float v)
    {
        // The value as binary32 has it, then the conversion: left to itself the compiler makes one v_fma_mixlo_f16 of a product and the
        // conversion where it packs no pair, which rounds once -- and the same element differs with its place in the tensor.
        asm("" : "+v"(v));
        return (_Float16)v;
    }
};

// Tensors of this size and more are read and written past the caches (non-temporal accesses): what a kernel leaves of a smaller
// one in the 256 MB that sit before the memory, the next kernel finds there.  Measured, dropout of bfloat16 and a copy that
// reads its result: at 64 MB 0.0499 ms against 0.0528 past the caches, at 128 MB 0.0916 / 0.0952, at 256 MB 0.202 / 0.195; dropout alone at
// 256 MB 0.102 / 0.091, the loss's forward pass over 2.1 GB of logits 0.288 / 0.275.  Stores only where rows start on 16-byte boundaries
// (partial lines past the caches: the loss's gradient on rows of 50257 bfloat16 0.038 -> 0.045 ms).
constexpr int64_t REPDL_STREAM_BYTES = 256LL << 20;

// 16 bytes of a tensor, the unit that a lane moves: `G` elements.
template <int DT>
struct Lowp
{
    typedef typename LowpType<DT>::T T;
    static constexpr int G = 16 / (int)sizeof(T);
    typedef uint32_t Raw __attribute__((ext_vector_type(4)));

    // Rows may start at any element (an odd row length in a 16-bit type): the hardware takes a 16-byte access on any
    // boundary, so there is one path for aligned and unaligned rows, and the order of a sum never depends on an address.
    typedef Raw RawAnywhere __attribute__((aligned(2)));
    template <bool STREAM = false>
    __device__ static __forceinline__ Raw load_raw(const T *p)
    {
        if (STREAM)
            return __builtin_nontemporal_load(reinterpret_cast<const RawAnywhere *>(p));
        Raw r;
        __builtin_memcpy(&r, p, 16);
        return r;
    }
    template <bool STREAM = false>
    __device__ static __forceinline__ void store_raw(T *p, const Raw &r)
    {
        if (STREAM)
            __builtin_nontemporal_store(r, reinterpret_cast<RawAnywhere *>(p));
        else
            __builtin_memcpy(p, &r, 16);
    }
    __device__ static __forceinline__ void unpack(const Raw &r, float *v)
    {
        T t[G];
        __builtin_memcpy(t, &r, 16);
#pragma unroll
        for (int k = 0; k < G; k++)
            v[k] = LowpType<DT>::widen(t[k]);
    }
    __device__ static __forceinline__ Raw pack(const float *v)
    {
        T t[G];
#pragma unroll
        for (int k = 0; k < G; k++)
            t[k] = LowpType<DT>::narrow(v[k]);
        Raw r;
        __builtin_memcpy(&r, t, 16);
        return r;
    }

    // elements c .. c+G-1 of a row of n; those past the end come as `fill`
    template <bool STREAM = false>
    __device__ static __forceinline__ void load(const T *row, int64_t c, int64_t n, float fill, float *v)
    {
        if (c + G <= n)
            unpack(load_raw<STREAM>(row + c), v);
        else
        {
#pragma unroll
            for (int k = 0; k < G; k++)
                v[k] = c + k < n ? LowpType<DT>::widen(row[c + k]) : fill;
        }
    }
    template <bool STREAM = false>
    __device__ static __forceinline__ void store(T *row, int64_t c, int64_t n, const float *v)
    {
        if (c + G <= n)
            store_raw<STREAM>(row + c, pack(v));
        else
        {
#pragma unroll
            for (int k = 0; k < G; k++)
                if (c + k < n)
                    row[c + k] = LowpType<DT>::narrow(v[k]);
        }
    }
};

// A launch counts its threads in 32 bits.  f(first, count) launches workgroups first .. first + count - 1 of `blocks`; rows of a
// few elements pass that bound long before they fill the memory.
template <typename F>
int repdl_launch_slices(int64_t blocks, int threads, F f)
{
    const int64_t most = 0xffffffffLL / threads;
    int rc = REPDL_OK;
    for (int64_t first = 0; first < blocks && rc == REPDL_OK; first += most)
    {
        f(first, (unsigned)(blocks - first < most ? blocks - first : most));
        rc = repdl_launch_status();
    }
    return rc;
}

static inline bool repdl_known_dtype(int dtype) { return dtype == REPDL_F32 || dtype == REPDL_BF16 || dtype == REPDL_F16; }
static inline int64_t repdl_dtype_bytes(int dtype) { return dtype == REPDL_F32 ? 4 : 2; }
