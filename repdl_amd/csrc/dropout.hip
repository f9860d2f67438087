// Dropout from a counter-based generator.
//
//   word_j = philox(key = seed, counter = (j / 4, call)) [j % 4]
//   keep_j = word_j >= threshold,  threshold = round(p 2^32)
//   y_j    = keep_j ? x_j * scale : 0,                      scale = float(1 / (1 - p))
//            keep_j ? residual_j + x_j * scale : residual_j   (two roundings in binary32, one to the tensor's type)
//
// The generator is Philox4x32 with ten rounds (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011):
// a block of four 32-bit words is a function of a 128-bit counter and a 64-bit key.  The low half of the counter is the
// number of the block in the tensor, the high half the number of the call, so two calls never share a word, and a mask is a
// function of (seed, call, position, p) alone -- not of the device, the launch or the tensor's type.  It is never stored: the
// backward pass is the same call on the incoming gradient.
//
// Bound: HBM, 8 B per element in binary32 (12 with a residual), 4 (6) in 16 bits.  The ten rounds are 20 products of 32 by 32
// to 64 bits (a quarter of the vector rate each) and about 20 three-operand exclusive ors for four elements, 25 issue slots per
// element: 39.3e12 / 25 = 1.6e12 elements/s, which at 16 bits is 6.3 TB/s, what a copy reaches.  Measured (a non-temporal copy of 1 GiB moves 6.3 TB/s):
// 2^26 f32 0.086 ms = 6.2 TB/s, with a residual 0.127 = 6.4; 2^27 bf16 0.096 = 5.6, f16 0.097, with a residual 0.135 = 6.0, 0.136; 64000 f32 2.9 us.
#include "lowp.h"

namespace
{
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ u4 philox(uint64_t block, uint64_t call, uint64_t seed)
{
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = (uint32_t)call, c3 = (uint32_t)(call >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; r++)
    {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        const uint32_t n0 = (uint32_t)(b >> 32) ^ c1 ^ k0, n2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c1 = (uint32_t)b;
        c3 = (uint32_t)a;
        c0 = n0;
        c2 = n2;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return u4{c0, c1, c2, c3};
}

struct DropoutArgs
{
    uint32_t threshold; // kept: word >= threshold
    int all;            // everything is dropped (p == 1)
    float scale;
};

// A thread takes DROP_GRANULES 16-byte granules, a workgroup's span apart.  One / two / four / eight, ms: 2^27 bf16 0.093 / 0.091 / 0.096 / 0.107, with a
// residual 0.132 / 0.133 / 0.135 / 0.226; 2^26 f32 0.086 / 0.086 / 0.086 / 0.090; 2^26 bf16 0.042 / 0.043 / 0.051 / 0.050; 12345677 f32 with a residual 0.0224 / 0.0222 /
// 0.0232 / 0.0234, bf16 0.0146 / 0.0162 / 0.0172 / 0.0204; 64000 f32 0.0024 / 0.0025 / 0.0029 / 0.0041.  Fewer would do as well or better, with the same bits.
constexpr int DROP_THREADS = 256, DROP_GRANULES = 4;

template <int DT, bool RES, bool STREAM>
__global__ __launch_bounds__(DROP_THREADS) void dropout_kernel(const typename LowpType<DT>::T *__restrict__ x,
                                                               const typename LowpType<DT>::T *__restrict__ residual,
                                                               typename LowpType<DT>::T *__restrict__ y, int64_t n, DropoutArgs d,
                                                               const int64_t *__restrict__ state, uint64_t seed, uint64_t call)
{
    typedef Lowp<DT> L;
    constexpr int G = L::G;
    if (state != nullptr)
    {
        seed = (uint64_t)state[0];
        call = (uint64_t)state[1];
    }
    const int64_t base = (int64_t)blockIdx.x * (DROP_THREADS * DROP_GRANULES) + threadIdx.x; // in granules
    float v[DROP_GRANULES][G], r[DROP_GRANULES][G];
#pragma unroll
    for (int i = 0; i < DROP_GRANULES; i++)
    {
        const int64_t c = (base + i * DROP_THREADS) * G;
        L::template load<STREAM>(x, c, n, 0.0f, v[i]);
        if (RES)
            L::template load<STREAM>(residual, c, n, 0.0f, r[i]);
    }
#pragma unroll
    for (int i = 0; i < DROP_GRANULES; i++)
    {
        const int64_t c = (base + i * DROP_THREADS) * G;
        if (c >= n)
            break;
#pragma unroll
        for (int q = 0; q < G / 4; q++)
        {
            const u4 w = philox((uint64_t)c / 4 + q, call, seed);
#pragma unroll
            for (int k = 0; k < 4; k++)
            {
                const bool keep = w[k] >= d.threshold && !d.all;
                const float t = v[i][4 * q + k] * d.scale;
                if (RES)
                    v[i][4 * q + k] = keep ? r[i][4 * q + k] + t : r[i][4 * q + k];
                else
                    v[i][4 * q + k] = keep ? t : 0.0f;
            }
        }
        L::template store<STREAM>(y, c, n, v[i]);
    }
}

__global__ void dropout_next_call_kernel(int64_t *state, int64_t *used)
{
    used[0] = state[0];
    used[1] = state[1];
    state[1] = (int64_t)((uint64_t)state[1] + 1);
}

template <int DT, bool RES, bool STREAM>
int launch_dropout(const void *x, const void *residual, void *y, int64_t n, DropoutArgs d, const int64_t *state, uint64_t seed,
                   uint64_t call, hipStream_t s)
{
    typedef typename LowpType<DT>::T T;
    const int64_t blocks = repdl_cdiv(n, (int64_t)Lowp<DT>::G * DROP_THREADS * DROP_GRANULES);
    REPDL_REQUIRE(blocks <= 0xffffffffLL / DROP_THREADS); // (2^36 elements: more than the memory holds)
    REPDL_LAUNCH((dropout_kernel<DT, RES, STREAM>), dim3((unsigned)blocks), dim3(DROP_THREADS), 0, s, static_cast<const T *>(x),
                 static_cast<const T *>(residual), static_cast<T *>(y), n, d, state, seed, call);
    return repdl_launch_status();
}

template <int DT>
int dropout_typed(const void *x, const void *residual, void *y, int64_t n, DropoutArgs d, const int64_t *state, uint64_t seed,
                  uint64_t call, hipStream_t s)
{
    const bool stream = n >= REPDL_STREAM_BYTES / repdl_dtype_bytes(DT) && (reinterpret_cast<uintptr_t>(y) & 15) == 0;
    if (residual != nullptr)
        return stream ? launch_dropout<DT, true, true>(x, residual, y, n, d, state, seed, call, s)
                      : launch_dropout<DT, true, false>(x, residual, y, n, d, state, seed, call, s);
    return stream ? launch_dropout<DT, false, true>(x, residual, y, n, d, state, seed, call, s)
                  : launch_dropout<DT, false, false>(x, residual, y, n, d, state, seed, call, s);
}
} // namespace

REPDL_API int repdl_hip_dropout(const void *x, const void *residual, void *y, int64_t n, double p, const int64_t *state, uint64_t seed,
                                uint64_t call, int dtype, void *stream)
{
    REPDL_REQUIRE(n >= 0 && p >= 0.0 && p <= 1.0 && repdl_known_dtype(dtype)); // (a NaN p fails here)
    if (n == 0)
        return REPDL_OK;
    REPDL_REQUIRE(x != nullptr && y != nullptr);
    const double t = p * 4294967296.0 + 0.5;
    DropoutArgs d;
    d.all = t >= 4294967296.0;
    d.threshold = d.all ? 0u : (uint32_t)t;
    d.scale = d.all ? 0.0f : (float)(1.0 / (1.0 - p));
    hipStream_t s = repdl_stream(stream);
    return dtype == REPDL_F32    ? dropout_typed<REPDL_F32>(x, residual, y, n, d, state, seed, call, s)
           : dtype == REPDL_BF16 ? dropout_typed<REPDL_BF16>(x, residual, y, n, d, state, seed, call, s)
                                 : dropout_typed<REPDL_F16>(x, residual, y, n, d, state, seed, call, s);
}

REPDL_API int repdl_hip_dropout_next_call(int64_t *state, int64_t *used, void *stream)
{
    REPDL_REQUIRE(state != nullptr && used != nullptr);
    REPDL_LAUNCH(dropout_next_call_kernel, dim3(1), dim3(1), 0, repdl_stream(stream), state, used);
    return repdl_launch_status();
}
