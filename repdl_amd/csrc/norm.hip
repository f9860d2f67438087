// Layer normalisation, forward and backward.
//
//   mean = (1/N) sum_j x_j,  var = (1/N) sum_j (x_j - mean)^2,  rstd = 1 / sqrt(var + eps)
//   xh_j = (x_j - mean) rstd,  y_j = xh_j w_j + b_j
//   g_j = gy_j w_j,  gx_j = rstd ((g_j - mean(g)) - xh_j mean(g xh))
//   gw_j = sum_i gy_ij xh_ij,  gb_j = sum_i gy_ij
//
// Offset rows.  A binary32 mean is off by a few roundings of the row's level: harmless where the level is near the spread, ruin where
// it is a thousand times above it (a constant row came out as y = -1 instead of 0).  A row with |mean| > 16 spreads is therefore centred in
// two numbers: the mean corrected by S(x_j - mean) / N, then rest = S(x_j - mean) / N, and x_j - mean - rest stands for the centred
// x_j.  The backward pass has the corrected mean and makes `rest` again.  Such a row costs two more sums over its registers and the squares
// again forward, one sum backward; any other (off by at most 17 spreads' worth of its sum's roundings) a comparison.  No row / every row offset:
// 8192 x 1024 f32 forward 0.0124 / 0.0129 ms, backward 0.0219 / 0.0221; 8192 x 4096 bf16 0.0243 / 0.0276, 0.0421 / 0.0434; 32768 x 2056 f16 0.0536 /
// 0.0648, 0.092 / 0.094.  (Sixteen: at that level the mean's error is what a row of no offset has in a sum of its length anyway.)
//
// Every operation above is one IEEE binary32 operation (nothing is fused; the square root and the reciprocal are the
// correctly rounded ones of crmath.h; "(1/N)" is one multiplication by float(1/N), as in the library's averages), so a
// result is a function of the inputs and of the order of the sums alone.  That order is fixed by the row length, the type
// and -- for gw and gb -- the number of rows; the device, the stream, the addresses and the other rows have no part in it:
//   over a row   a granule's elements in pairs, pairs of pairs, ...; a thread's granules in turn; the threads of a wave as a
//                butterfly; the waves in turn;
//   over rows    a workgroup's run of rows, each of its teams taking every (number of teams)-th one in turn; the teams in turn; sixteen
//                sums of every sixteenth run; those in turn.  At most 256 rows: 16 to 64 sums of every 16th to 64th row, those in turn.
//
// The two passes over a row (mean, then centred squares) read it from registers: one thread holds E = 16 or 24 of its elements, as
// 16-byte granules TPR granules apart, TPR threads a row.  Bound: HBM, 2 passes over the tensor forward and 3 backward.  Measured
// (a non-temporal copy of 1 GiB moves 6.3 TB/s): forward 16384 x 8192 bf16 0.096 ms = 5.6 TB/s, 8192 x 1024 f32 0.0124 = 5.4, 65536 x 256 f32
// 0.024 = 5.6; backward with both launches 0.170 ms = 4.7 TB/s, 0.0219 = 4.6, 0.038 = 5.3.
#include <type_traits>

#include "lowp.h"
#include "crmath.h"
#include "lanes.h"

namespace
{
// Threads per row: the smallest power of two, at least 4, that holds the row in E elements per thread.
__host__ __device__ constexpr int ln_threads_per_row(int64_t N, int E)
{
    int t = 4;
    while ((int64_t)t * E < N)
        t *= 2;
    return t;
}
constexpr int ln_grad_threads(int tpr) { return tpr < 256 ? 256 : tpr; }
constexpr int64_t LN_FEW_ROWS = 256; // (up to here one launch makes all gradients, see ln_few_rows)
constexpr int64_t LN_MAX_ONCHIP = 16384; // (1024 threads of 16 elements; longer rows are read from memory for every pass)

// Elements per thread: 16, or 24 in a 16-bit type whose row would leave many of 16 elements' threads without any (half the threads
// then hold it).  Forward wherever that pads the row less, rows of up to 1.5 powers of two: 32768 x 2056 f16 0.0696 -> 0.0535 ms,
// 32768 x 1280 bf16 0.0389 -> 0.0351, 32768 x 1536 0.0405 -> 0.0401.  Backward, where a thread's sums of gw and gb grow with its elements,
// for rows of up to 1.125 powers of two: 2056 0.111 -> 0.090, 1280 0.0604 -> 0.0581, but 8192 x 5120 0.0561 -> 0.0604.
int ln_elements(int64_t N, int dtype, bool backward)
{
    const int64_t padded = 16 * (int64_t)ln_threads_per_row(N, 16);
    if (dtype == REPDL_F32 || padded <= 64 || N > LN_MAX_ONCHIP)
        return 16;
    return backward ? (16 * N <= 9 * padded ? 24 : 16) : (4 * N <= 3 * padded ? 24 : 16);
}

// Sum over the TPR threads of a row of K values each, in every thread of the row: a butterfly inside the wave, then the
// waves' sums in order.  `scratch`: K * (TPR / 64) floats of LDS per row team, free again at the next call's second barrier;
// callers alternate between two halves.
template <int TPR, int K>
__device__ __forceinline__ void team_sum(float (&v)[K], float *scratch, int j)
{
    constexpr int W = TPR < 64 ? TPR : 64;
#pragma unroll
    for (int k = 0; k < K; k++)
        v[k] = lanes_sum<W>(v[k]);
    if (TPR > 64)
    {
        constexpr int NW = TPR / 64;
        if ((j & 63) == 0)
        {
#pragma unroll
            for (int k = 0; k < K; k++)
                scratch[k * NW + (j >> 6)] = v[k];
        }
        lds_barrier();
#pragma unroll
        for (int k = 0; k < K; k++)
        {
            float s = scratch[k * NW];
#pragma unroll
            for (int w = 1; w < NW; w++)
                s = s + scratch[k * NW + w];
            v[k] = s;
        }
    }
}

// A value that the whole wave shares, in scalar registers (rows of 64 threads and more: a wave works on one).
template <int TPR>
__device__ __forceinline__ int64_t wave_value(int64_t v)
{
    if (TPR < 64)
        return v;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return (int64_t)(((uint64_t)hi << 32) | lo);
}

// Sum of a granule's elements: pairs, pairs of pairs.
template <int G>
__device__ __forceinline__ float granule_sum(const float *v)
{
    float t[G];
#pragma unroll
    for (int k = 0; k < G; k++)
        t[k] = v[k];
#pragma unroll
    for (int step = 1; step < G; step <<= 1)
    {
#pragma unroll
        for (int k = 0; k + step < G; k += 2 * step)
            t[k] = t[k] + t[k + step];
    }
    return t[0];
}

__device__ __forceinline__ float ln_rstd(float var, float eps) { return crm_div(1.0f, crm_sqrt(var + eps)); }

// An offset row (see the top), from what the forward pass has and from what the backward pass has.
constexpr float LN_OFFSET = 16.0f;
__device__ __forceinline__ bool ln_offset(float mean, float var) { return mean * mean > LN_OFFSET * LN_OFFSET * var; }
__device__ __forceinline__ bool ln_offset_saved(float mean, float rstd) { return __builtin_fabsf(mean) * rstd > LN_OFFSET; }

// Does any of the rows that have to go through a row sum together have `offset` set: those of a wave, and where a row's
// threads are two of a workgroup's four waves (their sums meet at a barrier) those of the workgroup: `other` says so of the other row.
template <int TPR>
__device__ __forceinline__ bool ln_any(bool offset, bool other)
{
    return TPR <= 64 ? __any(offset) : TPR == 128 ? offset || other : offset;
}

// Parameters are read in granules of the activation's element count, whatever their own type.
template <int G, int PDT>
__device__ __forceinline__ void load_param(const typename LowpType<PDT>::T *p, int64_t c, int64_t n, float fill, float *v)
{
    typedef Lowp<PDT> P;
    if (p == nullptr)
    {
#pragma unroll
        for (int k = 0; k < G; k++)
            v[k] = fill;
        return;
    }
    if (P::G == G)
        P::load(p, c, n, 0.0f, v);
    else // binary32 parameters of a 16-bit activation: two granules
    {
        P::load(p, c, n, 0.0f, v);
        P::load(p, c + P::G, n, 0.0f, v + G - P::G);
    }
}

// The granules of one thread in a row of N elements.  The granule that would cross the row's end starts G elements before it
// instead: all its accesses are whole 16-byte ones, its first `skip` elements are the previous granule's, computed here a second
// time with the same result and left out of the row's sums.  A granule that lies behind the row's end repeats the last one
// whole (skip = G) and stores nothing.  Rows shorter than a granule (TINY) are read element by element.
template <int DT, int TPR, int E, bool TINY>
struct RowGranules
{
    typedef Lowp<DT> L;
    static constexpr int G = L::G, GPT = E / G;
    uint32_t at[GPT];
    int skip[GPT];
    __device__ __forceinline__ RowGranules(int N, int j)
    {
#pragma unroll
        for (int i = 0; i < GPT; i++)
        {
            const int c = (i * TPR + j) * G, last = TINY ? 0 : N - G;
            at[i] = c < last ? c : last;
            skip[i] = c - (int)at[i] < G ? c - (int)at[i] : G;
        }
    }
    __device__ __forceinline__ bool stores(int i) const { return skip[i] < G; }
    template <bool STREAM>
    __device__ __forceinline__ typename L::Raw load(const typename L::T *row, int i, int N) const
    {
        if (!TINY)
            return L::template load_raw<STREAM>(row + at[i]);
        typename L::Raw r = {0u, 0u, 0u, 0u};
        typename L::T t[G];
        __builtin_memcpy(t, &r, 16);
#pragma unroll
        for (int k = 0; k < G; k++)
            if (k < N)
                t[k] = row[k];
        __builtin_memcpy(&r, t, 16);
        return r;
    }
    template <bool STREAM>
    __device__ __forceinline__ void store(typename L::T *row, int i, int N, const float *v) const
    {
        if (!TINY)
            L::template store_raw<STREAM>(row + at[i], L::pack(v));
        else
        {
#pragma unroll
            for (int k = 0; k < G; k++)
                if (k < N)
                    row[k] = LowpType<DT>::narrow(v[k]);
        }
    }
    // what granule i adds to a sum over the row
    __device__ __forceinline__ float sum(const float *v, int i, int N) const
    {
        float t[G];
#pragma unroll
        for (int k = 0; k < G; k++)
            t[k] = v[k];
        if (skip[i] > 0 || TINY)
        {
#pragma unroll
            for (int k = 0; k < G; k++)
                t[k] = k >= skip[i] && (!TINY || k < N) ? t[k] : 0.0f;
        }
        return granule_sum<G>(t);
    }
    // weight or bias at the granule's columns
    template <int PDT>
    __device__ __forceinline__ void param(const typename LowpType<PDT>::T *p, int i, int N, float *v) const
    {
        typedef Lowp<PDT> P;
#pragma unroll
        for (int h = 0; h < G; h += P::G)
        {
            if (!TINY)
                P::unpack(P::load_raw(p + at[i] + h), v + h);
            else
                P::load(p, h, N, 0.0f, v + h);
        }
    }
};

template <int DT, int PDT, int TPR, int E, bool TINY, bool STREAM>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR, 8) void layer_norm_kernel(
    const typename LowpType<DT>::T *__restrict__ x, const typename LowpType<PDT>::T *__restrict__ w,
    const typename LowpType<PDT>::T *__restrict__ b, typename LowpType<DT>::T *__restrict__ y, float *__restrict__ mean_out,
    float *__restrict__ rstd_out, int64_t M, int N, float inv_n, float eps)
{
    typedef Lowp<DT> L;
    constexpr int G = L::G, GPT = E / G;
    constexpr int THREADS = TPR < 256 ? 256 : TPR, TEAMS = THREADS / TPR;
    __shared__ float scratch[2][TEAMS][TPR / 64 + 1];
    __shared__ int offsets[TEAMS];
    const int tid = threadIdx.x, team = tid / TPR, j = tid % TPR;
    const int64_t row = wave_value<TPR>((int64_t)blockIdx.x * TEAMS + team);
    const bool live = row < M;
    const typename L::T *xr = x + (live ? row : M - 1) * N;
    const RowGranules<DT, TPR, E, TINY> rg(N, j);

    typename L::Raw raw[GPT];
#pragma unroll
    for (int i = 0; i < GPT; i++)
        raw[i] = rg.template load<STREAM>(xr, i, N);
    float v[GPT][G];
    float s[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < GPT; i++)
    {
        L::unpack(raw[i], v[i]);
        s[0] = s[0] + rg.sum(v[i], i, N);
    }
    team_sum<TPR, 1>(s, scratch[0][team], j);
    float mean = s[0] * inv_n;
    // v - by, squared and summed: by the mean, then (in an offset row) by what the mean leaves
    float q[1];
    auto centre = [&](float by) {
        q[0] = 0.0f;
#pragma unroll
        for (int i = 0; i < GPT; i++)
        {
            float sq[G];
#pragma unroll
            for (int k = 0; k < G; k++)
            {
                v[i][k] = v[i][k] - by;
                sq[k] = v[i][k] * v[i][k];
            }
            q[0] = q[0] + rg.sum(sq, i, N);
        }
    };
    centre(mean);
    team_sum<TPR, 1>(q, scratch[1][team], j);
    const bool offset = ln_offset(mean, q[0] * inv_n);
    bool other = false;
    if (TPR == 128)
    {
        if (j == 0)
            offsets[team] = offset;
        lds_barrier();
        other = offsets[TEAMS - 1 - team];
    }
    if (__builtin_expect(ln_any<TPR>(offset, other), 0)) // (a row that is not offset but goes along ends with the bits it had)
    {
        s[0] = 0.0f;
#pragma unroll
        for (int i = 0; i < GPT; i++)
            s[0] = s[0] + rg.sum(v[i], i, N);
        team_sum<TPR, 1>(s, scratch[0][team], j);
        const float better = mean + s[0] * inv_n, by = offset ? better - mean : 0.0f; // (exact)
        mean = offset ? better : mean;
        s[0] = 0.0f;
#pragma unroll
        for (int i = 0; i < GPT; i++)
        {
#pragma unroll
            for (int k = 0; k < G; k++)
                v[i][k] = v[i][k] - by;
            s[0] = s[0] + rg.sum(v[i], i, N);
        }
        team_sum<TPR, 1>(s, scratch[1][team], j);
        centre(offset ? s[0] * inv_n : 0.0f);
        team_sum<TPR, 1>(q, scratch[0][team], j);
    }
    const float rstd = ln_rstd(q[0] * inv_n, eps);
    if (!live)
        return;
    if (mean_out != nullptr && j == 0)
    {
        mean_out[row] = mean;
        rstd_out[row] = rstd;
    }
    typename L::T *yr = y + row * N;
#pragma unroll
    for (int i = 0; i < GPT; i++)
    {
        if (rg.stores(i))
        {
            float p[G];
#pragma unroll
            for (int k = 0; k < G; k++)
                v[i][k] = v[i][k] * rstd;
            if (w != nullptr)
            {
                rg.template param<PDT>(w, i, N, p);
#pragma unroll
                for (int k = 0; k < G; k++)
                    v[i][k] = v[i][k] * p[k];
            }
            if (b != nullptr)
            {
                rg.template param<PDT>(b, i, N, p);
#pragma unroll
                for (int k = 0; k < G; k++)
                    v[i][k] = v[i][k] + p[k];
            }
            rg.template store<STREAM>(yr, i, N, v[i]);
        }
    }
}

// Rows too long for the registers of a workgroup: 1024 threads, three passes over the row (the second and third out of the caches).
template <int DT, int PDT>
__global__ __launch_bounds__(1024) void layer_norm_long_kernel(
    const typename LowpType<DT>::T *__restrict__ x, const typename LowpType<PDT>::T *__restrict__ w,
    const typename LowpType<PDT>::T *__restrict__ b, typename LowpType<DT>::T *__restrict__ y, float *__restrict__ mean_out,
    float *__restrict__ rstd_out, int64_t M, int64_t N, float inv_n, float eps)
{
    typedef Lowp<DT> L;
    constexpr int G = L::G, TPR = 1024;
    __shared__ float scratch[2][TPR / 64];
    const int j = threadIdx.x;
    const int64_t row = blockIdx.x;
    const typename L::T *xr = x + row * N;
    float v[G];
    float s[1] = {0.0f};
    for (int64_t c = (int64_t)j * G; c < N; c += TPR * G)
    {
        L::load(xr, c, N, 0.0f, v);
        s[0] = s[0] + granule_sum<G>(v);
    }
    team_sum<TPR, 1>(s, scratch[0], j);
    const float mean = s[0] * inv_n;
    float better = 0.0f, rest = 0.0f; // of an offset row
    // S(x_j - mean - better - rest), or of its square
    auto centred = [&](bool square) {
        float t = 0.0f;
        for (int64_t c = (int64_t)j * G; c < N; c += TPR * G)
        {
            L::load(xr, c, N, mean, v);
#pragma unroll
            for (int k = 0; k < G; k++)
            {
                v[k] = c + k < N ? ((v[k] - mean) - better) - rest : 0.0f;
                v[k] = square ? v[k] * v[k] : v[k];
            }
            t = t + granule_sum<G>(v);
        }
        return t;
    };
    float q[1] = {centred(true)};
    team_sum<TPR, 1>(q, scratch[1], j);
    if (ln_offset(mean, q[0] * inv_n)) // (the whole workgroup's)
    {
        s[0] = centred(false);
        team_sum<TPR, 1>(s, scratch[0], j);
        better = (mean + s[0] * inv_n) - mean; // (exact)
        s[0] = centred(false);
        team_sum<TPR, 1>(s, scratch[1], j);
        rest = s[0] * inv_n;
        q[0] = centred(true);
        team_sum<TPR, 1>(q, scratch[0], j);
    }
    const float rstd = ln_rstd(q[0] * inv_n, eps);
    if (mean_out != nullptr && j == 0)
    {
        mean_out[row] = mean + better;
        rstd_out[row] = rstd;
    }
    typename L::T *yr = y + row * N;
    for (int64_t c = (int64_t)j * G; c < N; c += TPR * G)
    {
        float wv[G], bv[G];
        L::load(xr, c, N, 0.0f, v);
        load_param<G, PDT>(w, c, N, 1.0f, wv);
        load_param<G, PDT>(b, c, N, 0.0f, bv);
#pragma unroll
        for (int k = 0; k < G; k++)
        {
            v[k] = (((v[k] - mean) - better) - rest) * rstd;
            if (w != nullptr)
                v[k] = v[k] * wv[k];
            if (b != nullptr)
                v[k] = v[k] + bv[k];
        }
        L::store(yr, c, N, v);
    }
}

// ---- backward ---------------------------------------------------------------------------------
// An offset row's centred values once more (those of a row that goes along stay as they are).
template <int TPR, typename Granules, int GPT, int G>
__device__ __forceinline__ void ln_centre_again(const Granules &rg, float (&xv)[GPT][G], bool offset, float *scratch, int j, int N, float inv_n)
{
    float t[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < GPT; i++)
        t[0] = t[0] + rg.sum(xv[i], i, N);
    team_sum<TPR, 1>(t, scratch, j);
    const float rest = offset ? t[0] * inv_n : 0.0f;
#pragma unroll
    for (int i = 0; i < GPT; i++)
#pragma unroll
        for (int k = 0; k < G; k++)
            xv[i][k] = xv[i][k] - rest;
}

// A workgroup owns a run of consecutive rows, its teams taking them in turn; a thread meets the same columns in every row and
// adds up their gw and gb in registers.  At the end the teams' sums are added in order through LDS and written as one row of
// `partial` [blocks][2][N]; layer_norm_param_kernel adds the blocks.  x and gy are read once, gx is written once.
// The next row's x, gy, mean and rstd are under way while a row is worked on (two to four rows ahead changed nothing: what
// bounds a small call is a row's latency of about a microsecond and the second launch, what bounds a large one is HBM).  A
// workgroup's 8 waves of up to 256 registers are all that its share of a CU holds: with registers for twice the waves the loop
// spilled and ran 10-40 % slower (8192 x 4096 bf16 0.0537 -> 0.0503 ms, 100000 x 64 0.0205 -> 0.0148).
template <int DT, int PDT, int TPR, int E, bool TINY, bool STREAM>
__global__ __launch_bounds__(ln_grad_threads(TPR), TPR < 1024 ? 2 : 4) void layer_norm_grad_kernel(
    const typename LowpType<DT>::T *__restrict__ gy, const typename LowpType<DT>::T *__restrict__ x,
    const typename LowpType<PDT>::T *__restrict__ w, const float *__restrict__ mean_in, const float *__restrict__ rstd_in,
    typename LowpType<DT>::T *__restrict__ gx, float *__restrict__ partial, int64_t M, int N, int64_t rows_per_block, float inv_n)
{
    typedef Lowp<DT> L;
    constexpr int G = L::G, GPT = E / G;
    constexpr int THREADS = ln_grad_threads(TPR), TEAMS = THREADS / TPR;
    __shared__ float scratch[2][TEAMS][2 * (TPR / 64) + 1];
    __shared__ float fold[TEAMS > 1 ? THREADS * E : 1];
    __shared__ int some;
    const int tid = threadIdx.x, team = tid / TPR, j = tid % TPR;
    const int64_t r0 = (int64_t)blockIdx.x * rows_per_block;
    const int64_t r1 = r0 + rows_per_block < M ? r0 + rows_per_block : M;
    const RowGranules<DT, TPR, E, TINY> rg(N, j);

    float aw[GPT][G], ab[GPT][G];
#pragma unroll
    for (int i = 0; i < GPT; i++)
#pragma unroll
        for (int k = 0; k < G; k++)
            aw[i][k] = ab[i][k] = 0.0f;
    typedef Lowp<PDT> P;
    constexpr int WPG = G / P::G; // granules of w per granule of x
    constexpr bool KEEP_W = !TINY && (DT != REPDL_F32 || TPR < 1024);
    typename P::Raw wr[KEEP_W ? GPT * WPG : 1];
    if (KEEP_W && w != nullptr)
    {
#pragma unroll
        for (int i = 0; i < GPT * WPG; i++)
            wr[i] = P::load_raw(w + rg.at[i / WPG] + i % WPG * P::G);
    }
    typename L::Raw nx[GPT], ng[GPT];
    float next_mean, next_rstd;
    auto fetch = [&](int64_t at) {
        const int64_t rr = wave_value<TPR>(at < r1 ? at : r1 - 1);
#pragma unroll
        for (int i = 0; i < GPT; i++)
        {
            nx[i] = rg.template load<STREAM>(x + rr * N, i, N);
            ng[i] = rg.template load<STREAM>(gy + rr * N, i, N);
        }
        next_mean = mean_in[rr];
        next_rstd = rstd_in[rr];
    };
    fetch(r0 + team);
    bool other = false;
    if (TPR == 128) // (any row of the run, asked once: asking for the other team's row at every step took 100 ns a step)
    {
        bool found = false;
        for (int64_t r = r0 + tid; r < r1; r += THREADS)
            found = found || ln_offset_saved(mean_in[r], rstd_in[r]);
        if (tid == 0)
            some = 0;
        lds_barrier();
        if (found)
            some = 1;
        lds_barrier();
        other = some;
    }
    int half = 0;
    for (int64_t base = r0; base < r1; base += TEAMS)
    {
        const int64_t row = wave_value<TPR>(base + team);
        const bool live = row < r1;
        float xv[GPT][G], gv[GPT][G];
#pragma unroll
        for (int i = 0; i < GPT; i++)
        {
            L::unpack(nx[i], xv[i]);
            L::unpack(ng[i], gv[i]);
        }
        const float mean = next_mean, rstd = next_rstd;
        const bool offset = ln_offset_saved(mean, rstd), any = ln_any<TPR>(offset, other);
        if (base + TEAMS < r1)
            fetch(row + TEAMS);
#pragma unroll
        for (int i = 0; i < GPT; i++)
#pragma unroll
            for (int k = 0; k < G; k++)
                xv[i][k] = xv[i][k] - mean;
        if (__builtin_expect(any, 0)) // (out of the loop's way: 4096 x 16384 f32 0.174 -> 0.168 ms)
        {
            ln_centre_again<TPR>(rg, xv, offset, scratch[half][team], j, N, inv_n);
            half ^= 1;
        }
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < GPT; i++)
        {
            float p[G];
#pragma unroll
            for (int k = 0; k < G; k++)
                xv[i][k] = xv[i][k] * rstd;
            if (live && partial != nullptr)
            {
#pragma unroll
                for (int k = 0; k < G; k++)
                {
                    aw[i][k] = aw[i][k] + gv[i][k] * xv[i][k];
                    ab[i][k] = ab[i][k] + gv[i][k];
                }
            }
            if (w != nullptr)
            {
                if (KEEP_W)
                {
#pragma unroll
                    for (int h = 0; h < WPG; h++)
                    {
                        asm("" : "+v"(wr[i * WPG + h])); // (not widened ahead of the loop: that would take twice the registers)
                        P::unpack(wr[i * WPG + h], p + h * P::G);
                    }
                }
                else
                    rg.template param<PDT>(w, i, N, p);
#pragma unroll
                for (int k = 0; k < G; k++)
                    gv[i][k] = gv[i][k] * p[k];
            }
#pragma unroll
            for (int k = 0; k < G; k++)
                p[k] = gv[i][k] * xv[i][k];
            s[0] = s[0] + rg.sum(gv[i], i, N);
            s[1] = s[1] + rg.sum(p, i, N);
        }
        if (gx == nullptr)
            continue;
        team_sum<TPR, 2>(s, scratch[half][team], j);
        half ^= 1; // (the next row's sums go to the other half: a wave still reading this one is not overtaken by two rows)
        const float m1 = s[0] * inv_n, m2 = s[1] * inv_n;
        if (live)
        {
#pragma unroll
            for (int i = 0; i < GPT; i++)
            {
                if (rg.stores(i))
                {
                    float o[G];
#pragma unroll
                    for (int k = 0; k < G; k++)
                        o[k] = rstd * ((gv[i][k] - m1) - xv[i][k] * m2);
                    rg.template store<STREAM>(gx + row * N, i, N, o);
                }
            }
        }
    }
    if (partial == nullptr)
        return;
    float *out = partial + (int64_t)blockIdx.x * 2 * N;
#pragma unroll
    for (int which = 0; which < 2; which++)
    {
        if (TEAMS > 1)
        {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < GPT; i++)
                if (rg.stores(i))
                {
#pragma unroll
                    for (int k = 0; k < G; k++)
                        fold[team * TPR * E + rg.at[i] + k] = which == 0 ? aw[i][k] : ab[i][k];
                }
            __syncthreads();
            for (int c = tid; c < N; c += THREADS)
            {
                float s = fold[c];
                for (int t = 1; t < TEAMS; t++)
                    s = s + fold[t * TPR * E + c];
                out[which * N + c] = s;
            }
        }
        else
        {
#pragma unroll
            for (int i = 0; i < GPT; i++)
                if (rg.stores(i))
                {
#pragma unroll
                    for (int h = 0; h < G; h += 4)
                    {
                        const Lowp<REPDL_F32>::Raw r = Lowp<REPDL_F32>::pack((which == 0 ? aw[i] : ab[i]) + h);
                        __builtin_memcpy(out + which * N + rg.at[i] + h, &r, 16);
                    }
                }
        }
    }
}

// Few rows: one launch for all three gradients.  The first `row_blocks` workgroups make gx, a row per team; the others make gw and gb
// straight from x, gy and the rows' statistics, 16 granules of columns a workgroup, every 16 threads taking every
// (threads / 16)-th row in turn and their sums added in order through LDS.  x and gy are read twice, the second time out of
// the caches, and there are no partial sums, no second launch and no scratch.  Where rows are offset, each of these workgroups sums them
// all for itself (every row: 64 x 1024 f32 0.018 ms instead of 0.003, 256 x 16384 f32 0.153 instead of 0.014).
template <int DT, int PDT, int TPR, int E, bool TINY>
__global__ __launch_bounds__(ln_grad_threads(TPR), TPR == 1024 && DT == REPDL_F32 ? 8 : 1) void layer_norm_grad_few_kernel(
    const typename LowpType<DT>::T *__restrict__ gy, const typename LowpType<DT>::T *__restrict__ x,
    const typename LowpType<PDT>::T *__restrict__ w, const float *__restrict__ mean_in, const float *__restrict__ rstd_in,
    typename LowpType<DT>::T *__restrict__ gx, typename LowpType<PDT>::T *__restrict__ gw, typename LowpType<PDT>::T *__restrict__ gb,
    int M, int N, int row_blocks, float inv_n)
{
    typedef Lowp<DT> L;
    constexpr int G = L::G, GPT = E / G;
    constexpr int THREADS = ln_grad_threads(TPR), TEAMS = THREADS / TPR, GROUPS = THREADS / 16;
    __shared__ float scratch[2][TEAMS][2 * (TPR / 64) + 1];
    __shared__ float fold[GROUPS][16 * G];
    __shared__ float rest[LN_FEW_ROWS];
    __shared__ int some;
    const int tid = threadIdx.x, team = tid / TPR, j = tid % TPR;
    if ((int)blockIdx.x < row_blocks)
    {
        const int64_t row = wave_value<TPR>((int64_t)blockIdx.x * TEAMS + team);
        const bool live = row < M;
        const int64_t rr = live ? row : M - 1;
        const RowGranules<DT, TPR, E, TINY> rg(N, j);
        typename L::Raw rx[GPT], rgy[GPT];
#pragma unroll
        for (int i = 0; i < GPT; i++)
        {
            rx[i] = rg.template load<false>(x + rr * N, i, N);
            rgy[i] = rg.template load<false>(gy + rr * N, i, N);
        }
        const float mean = mean_in[rr], rstd = rstd_in[rr];
        const bool offset = ln_offset_saved(mean, rstd);
        bool other = false;
        if (TPR == 128)
        {
            const int64_t ro = wave_value<TPR>(row + 1 - 2 * team < M ? row + 1 - 2 * team : M - 1);
            other = ln_offset_saved(mean_in[ro], rstd_in[ro]);
        }
        float xv[GPT][G], gv[GPT][G];
#pragma unroll
        for (int i = 0; i < GPT; i++)
        {
            L::unpack(rx[i], xv[i]);
            L::unpack(rgy[i], gv[i]);
#pragma unroll
            for (int k = 0; k < G; k++)
                xv[i][k] = xv[i][k] - mean;
        }
        if (ln_any<TPR>(offset, other))
            ln_centre_again<TPR>(rg, xv, offset, scratch[1][team], j, N, inv_n);
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < GPT; i++)
        {
            float p[G];
            if (w != nullptr)
            {
                rg.template param<PDT>(w, i, N, p);
#pragma unroll
                for (int k = 0; k < G; k++)
                    gv[i][k] = gv[i][k] * p[k];
            }
#pragma unroll
            for (int k = 0; k < G; k++)
            {
                xv[i][k] = xv[i][k] * rstd;
                p[k] = gv[i][k] * xv[i][k];
            }
            s[0] = s[0] + rg.sum(gv[i], i, N);
            s[1] = s[1] + rg.sum(p, i, N);
        }
        team_sum<TPR, 2>(s, scratch[0][team], j);
        const float m1 = s[0] * inv_n, m2 = s[1] * inv_n;
        if (live)
        {
#pragma unroll
            for (int i = 0; i < GPT; i++)
                if (rg.stores(i))
                {
                    float o[G];
#pragma unroll
                    for (int k = 0; k < G; k++)
                        o[k] = rstd * ((gv[i][k] - m1) - xv[i][k] * m2);
                    rg.template store<false>(gx + row * N, i, N, o);
                }
        }
        return;
    }
    // columns c .. c+G-1 (the last granule of the row starts earlier where it would cross the end, see RowGranules)
    const int lane = tid % 16, group = tid / 16;
    const int wanted = (((int)blockIdx.x - row_blocks) * 16 + lane) * G;
    const int c = TINY ? 0 : (wanted < N - G ? wanted : N - G);
    float aw[G], ab[G];
    bool found = false;
    auto accumulate = [&](auto with_rest) {
        constexpr bool REST = decltype(with_rest)::value;
#pragma unroll
        for (int k = 0; k < G; k++)
            aw[k] = ab[k] = 0.0f;
        constexpr int AHEAD = 4; // rows under way at once
        for (int base = group; base < M; base += AHEAD * GROUPS)
        {
            typename L::Raw rx[AHEAD], rgy[AHEAD];
            float mean[AHEAD], rstd[AHEAD];
#pragma unroll
            for (int u = 0; u < AHEAD; u++)
            {
                const int row = base + u * GROUPS < M ? base + u * GROUPS : M - 1;
                const int64_t at = (int64_t)row * N + c;
                if (!TINY)
                {
                    rx[u] = L::load_raw(x + at);
                    rgy[u] = L::load_raw(gy + at);
                }
                else
                {
                    float v[G];
                    L::load(x + at, 0, N, 0.0f, v);
                    rx[u] = L::pack(v);
                    L::load(gy + at, 0, N, 0.0f, v);
                    rgy[u] = L::pack(v);
                }
                mean[u] = mean_in[row];
                rstd[u] = rstd_in[row];
            }
#pragma unroll
            for (int u = 0; u < AHEAD; u++)
            {
                float xv[G], gv[G];
                L::unpack(rx[u], xv);
                L::unpack(rgy[u], gv);
                found = found || ln_offset_saved(mean[u], rstd[u]);
                if (base + u * GROUPS < M)
                {
#pragma unroll
                    for (int k = 0; k < G; k++)
                    {
                        const float d = REST ? (xv[k] - mean[u]) - rest[base + u * GROUPS] : xv[k] - mean[u];
                        aw[k] = aw[k] + gv[k] * (d * rstd[u]);
                        ab[k] = ab[k] + gv[k];
                    }
                }
            }
        }
    };
    if (tid == 0)
        some = 0;
    lds_barrier();
    accumulate(std::false_type());
    if (found)
        some = 1;
    lds_barrier();
    if (some) // offset rows: what their means leave, a wave a row (a lane's granules in turn, a butterfly), and the sums again
    {
        constexpr int WAVES = THREADS / 64;
        static_assert(64 * WAVES >= LN_FEW_ROWS, "a lane for every row");
        const int wave = __builtin_amdgcn_readfirstlane(tid / 64), at = tid % 64, mine = wave + WAVES * at;
        const float mean = mine < M ? mean_in[mine] : 0.0f;
        const bool offset = mine < M && ln_offset_saved(mean, rstd_in[mine]);
        if (mine < M && !offset)
            rest[mine] = 0.0f;
        for (uint64_t left = __ballot(offset); left != 0; left &= left - 1)
        {
            const int from = __builtin_ctzll(left), row = wave + WAVES * from;
            const float m = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(mean), from));
            const typename L::T *xr = x + (int64_t)row * N;
            float t = 0.0f, v[G];
            int c = at * G;
            constexpr int AHEAD = 8;
            for (int to = AHEAD * 64 * G; to <= N; to += AHEAD * 64 * G, c += AHEAD * 64 * G) // whole rounds of the wave
            {
                typename L::Raw raw[AHEAD];
#pragma unroll
                for (int u = 0; u < AHEAD; u++)
                    raw[u] = L::load_raw(xr + c + u * 64 * G);
#pragma unroll
                for (int u = 0; u < AHEAD; u++)
                {
                    L::unpack(raw[u], v);
#pragma unroll
                    for (int k = 0; k < G; k++)
                        v[k] = v[k] - m;
                    t = t + granule_sum<G>(v);
                }
            }
            for (; c < N; c += 64 * G)
            {
                L::load(xr, c, N, m, v);
#pragma unroll
                for (int k = 0; k < G; k++)
                    v[k] = v[k] - m;
                t = t + granule_sum<G>(v);
            }
            t = lanes_sum<64>(t);
            if (at == 0)
                rest[row] = t * inv_n;
        }
        lds_barrier();
        accumulate(std::true_type());
    }
#pragma unroll
    for (int which = 0; which < 2; which++)
    {
        typename LowpType<PDT>::T *out = which == 0 ? gw : gb;
        if (out == nullptr)
            continue;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < G; k++)
            fold[group][lane * G + k] = which == 0 ? aw[k] : ab[k];
        __syncthreads();
        if (tid < 16 * G)
        {
            float s = fold[0][tid];
#pragma unroll 8
            for (int g = 1; g < GROUPS; g++)
                s = s + fold[g][tid];
            // this thread's column: granule tid / G of the workgroup, whose start may have been moved
            const int start = (((int)blockIdx.x - row_blocks) * 16 + tid / G) * G;
            const int col = (TINY ? 0 : (start < N - G ? start : N - G)) + tid % G;
            if (start < N && col < N)
                out[col] = LowpType<PDT>::narrow(s);
        }
    }
}

// The same for rows too long for the registers: gx by a workgroup per row that reads it twice (an offset row three times), and what the
// row's mean leaves ...
template <int DT, int PDT>
__global__ __launch_bounds__(1024) void layer_norm_grad_long_kernel(
    const typename LowpType<DT>::T *__restrict__ gy, const typename LowpType<DT>::T *__restrict__ x,
    const typename LowpType<PDT>::T *__restrict__ w, const float *__restrict__ mean_in, const float *__restrict__ rstd_in,
    typename LowpType<DT>::T *__restrict__ gx, float *__restrict__ rest_out, int64_t N, float inv_n)
{
    typedef Lowp<DT> L;
    constexpr int G = L::G, TPR = 1024;
    __shared__ float scratch[2 * (TPR / 64)], rest_scratch[TPR / 64];
    const int j = threadIdx.x;
    const int64_t row = blockIdx.x;
    const float mean = mean_in[row], rstd = rstd_in[row];
    float xv[G], gv[G], wv[G];
    float rest = 0.0f;
    if (ln_offset_saved(mean, rstd)) // (the whole workgroup's)
    {
        float t[1] = {0.0f};
        for (int64_t c = (int64_t)j * G; c < N; c += TPR * G)
        {
            L::load(x + row * N, c, N, mean, xv);
#pragma unroll
            for (int k = 0; k < G; k++)
                xv[k] = xv[k] - mean;
            t[0] = t[0] + granule_sum<G>(xv);
        }
        team_sum<TPR, 1>(t, rest_scratch, j);
        rest = t[0] * inv_n;
    }
    if (rest_out != nullptr && j == 0)
        rest_out[row] = rest;
    if (gx == nullptr)
        return;
    float s[2] = {0.0f, 0.0f};
    for (int64_t c = (int64_t)j * G; c < N; c += TPR * G)
    {
        L::load(x + row * N, c, N, 0.0f, xv);
        L::load(gy + row * N, c, N, 0.0f, gv);
        load_param<G, PDT>(w, c, N, 1.0f, wv);
#pragma unroll
        for (int k = 0; k < G; k++)
        {
            const float xh = c + k < N ? ((xv[k] - mean) - rest) * rstd : 0.0f;
            if (w != nullptr)
                gv[k] = gv[k] * wv[k];
            xv[k] = gv[k] * xh;
        }
        s[0] = s[0] + granule_sum<G>(gv);
        s[1] = s[1] + granule_sum<G>(xv);
    }
    team_sum<TPR, 2>(s, scratch, j);
    const float m1 = s[0] * inv_n, m2 = s[1] * inv_n;
    for (int64_t c = (int64_t)j * G; c < N; c += TPR * G)
    {
        L::load(x + row * N, c, N, 0.0f, xv);
        L::load(gy + row * N, c, N, 0.0f, gv);
        load_param<G, PDT>(w, c, N, 1.0f, wv);
#pragma unroll
        for (int k = 0; k < G; k++)
        {
            const float xh = ((xv[k] - mean) - rest) * rstd;
            if (w != nullptr)
                gv[k] = gv[k] * wv[k];
            gv[k] = rstd * ((gv[k] - m1) - xh * m2);
        }
        L::store(gx + row * N, c, N, gv);
    }
}

// ... and the partial sums of gw and gb by a thread per granule of columns and block of rows.
template <int DT>
__global__ __launch_bounds__(256) void layer_norm_param_long_kernel(const typename LowpType<DT>::T *__restrict__ gy,
                                                                    const typename LowpType<DT>::T *__restrict__ x,
                                                                    const float *__restrict__ mean_in,
                                                                    const float *__restrict__ rstd_in,
                                                                    const float *__restrict__ rest_in, float *__restrict__ partial,
                                                                    int64_t M, int64_t N, int64_t rows_per_block)
{
    typedef Lowp<DT> L;
    constexpr int G = L::G;
    const int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * G;
    if (c >= N)
        return;
    const int64_t r0 = (int64_t)blockIdx.y * rows_per_block;
    const int64_t r1 = r0 + rows_per_block < M ? r0 + rows_per_block : M;
    float aw[G], ab[G];
#pragma unroll
    for (int k = 0; k < G; k++)
        aw[k] = ab[k] = 0.0f;
    for (int64_t row = r0; row < r1; row++)
    {
        float xv[G], gv[G];
        L::load(x + row * N, c, N, 0.0f, xv);
        L::load(gy + row * N, c, N, 0.0f, gv);
        const float mean = mean_in[row], rstd = rstd_in[row], rest = rest_in[row];
#pragma unroll
        for (int k = 0; k < G; k++)
        {
            aw[k] = aw[k] + gv[k] * (((xv[k] - mean) - rest) * rstd);
            ab[k] = ab[k] + gv[k];
        }
    }
    float *out = partial + (int64_t)blockIdx.y * 2 * N;
#pragma unroll
    for (int k = 0; k < G; k++)
        if (c + k < N)
        {
            out[c + k] = aw[k];
            out[N + c + k] = ab[k];
        }
}

// gw and gb from `blocks` rows of partial sums: 16 threads of a column add every sixteenth block, then their sums in order.
constexpr int LN_FOLD = 16;
template <int PDT>
__global__ __launch_bounds__(64 * LN_FOLD) void layer_norm_param_kernel(const float *__restrict__ partial,
                                                                        typename LowpType<PDT>::T *__restrict__ gw,
                                                                        typename LowpType<PDT>::T *__restrict__ gb, int64_t N,
                                                                        int blocks, int64_t first)
{
    __shared__ float sums[LN_FOLD][64];
    const int lane = threadIdx.x & 63, part = threadIdx.x >> 6;
    const int64_t col = (first + blockIdx.x) * 64 + lane;
    float s = 0.0f;
    if (col < 2 * N)
    {
#pragma unroll 8
        for (int b = part; b < blocks; b += LN_FOLD)
            s = s + partial[(int64_t)b * 2 * N + col];
    }
    sums[part][lane] = s;
    __syncthreads();
    if (part == 0 && col < 2 * N)
    {
#pragma unroll
        for (int p = 1; p < LN_FOLD; p++)
            s = s + sums[p][lane];
        typename LowpType<PDT>::T *out = col < N ? gw : gb;
        if (out != nullptr)
            out[col < N ? col : col - N] = LowpType<PDT>::narrow(s);
    }
}

// ---- host -------------------------------------------------------------------------------------
// Large tensors go past the caches (4096 x 16384 f32 forward 0.103 -> 0.096 ms, backward 0.181 -> 0.162): rows that a wave or more
// shares, on 16-byte boundaries.
template <int DT>
bool ln_streams(int64_t M, int64_t N, const void *out)
{
    return M * N >= REPDL_STREAM_BYTES / repdl_dtype_bytes(DT) && N % Lowp<DT>::G == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
}

// f(threads per row as a constant) for rows of `tpr` threads
template <typename F>
int ln_with_threads(int tpr, F f)
{
    switch (tpr)
    {
    case 4: return f(std::integral_constant<int, 4>());
    case 8: return f(std::integral_constant<int, 8>());
    case 16: return f(std::integral_constant<int, 16>());
    case 32: return f(std::integral_constant<int, 32>());
    case 64: return f(std::integral_constant<int, 64>());
    case 128: return f(std::integral_constant<int, 128>());
    case 256: return f(std::integral_constant<int, 256>());
    case 512: return f(std::integral_constant<int, 512>());
    default: return f(std::integral_constant<int, 1024>());
    }
}

template <int DT, int PDT, int TPR, int E, bool TINY>
int launch_layer_norm(const void *x, const void *w, const void *b, void *y, float *mean, float *rstd, int64_t M, int64_t N, float eps,
                      hipStream_t s)
{
    typedef typename LowpType<DT>::T T;
    typedef typename LowpType<PDT>::T P;
    constexpr int THREADS = TPR < 256 ? 256 : TPR, TEAMS = THREADS / TPR;
    const bool streams = TPR >= 64 && ln_streams<DT>(M, N, y);
    return repdl_launch_slices(repdl_cdiv(M, TEAMS), THREADS, [&](int64_t first, unsigned count) {
        const int64_t row = first * TEAMS;
        const T *xs = static_cast<const T *>(x) + row * N;
        T *ys = static_cast<T *>(y) + row * N;
        float *ms = mean == nullptr ? nullptr : mean + row, *rs = rstd == nullptr ? nullptr : rstd + row;
        if (streams)
            REPDL_LAUNCH((layer_norm_kernel<DT, PDT, TPR, E, TINY, (TPR >= 64)>), dim3(count), dim3(THREADS), 0, s, xs,
                         static_cast<const P *>(w), static_cast<const P *>(b), ys, ms, rs, M - row, (int)N, (float)(1.0 / (double)N), eps);
        else
            REPDL_LAUNCH((layer_norm_kernel<DT, PDT, TPR, E, TINY, false>), dim3(count), dim3(THREADS), 0, s, xs,
                         static_cast<const P *>(w), static_cast<const P *>(b), ys, ms, rs, M - row, (int)N, (float)(1.0 / (double)N), eps);
    });
}

template <int DT, int PDT>
int layer_norm_typed(const void *x, const void *w, const void *b, void *y, float *mean, float *rstd, int64_t M, int64_t N, float eps,
                     hipStream_t s)
{
    if (N > LN_MAX_ONCHIP)
    {
        typedef typename LowpType<DT>::T T;
        typedef typename LowpType<PDT>::T P;
        return repdl_launch_slices(M, 1024, [&](int64_t row, unsigned count) {
            REPDL_LAUNCH((layer_norm_long_kernel<DT, PDT>), dim3(count), dim3(1024), 0, s, static_cast<const T *>(x) + row * N,
                         static_cast<const P *>(w), static_cast<const P *>(b), static_cast<T *>(y) + row * N,
                         mean == nullptr ? nullptr : mean + row, rstd == nullptr ? nullptr : rstd + row, M - row, N,
                         (float)(1.0 / (double)N), eps);
        });
    }
    if (N < Lowp<DT>::G)
        return launch_layer_norm<DT, PDT, 4, 16, true>(x, w, b, y, mean, rstd, M, N, eps, s);
    const int E = ln_elements(N, DT, false);
    return ln_with_threads(ln_threads_per_row(N, E), [&](auto threads) {
        constexpr int TPR = decltype(threads)::value;
        constexpr int E24 = DT == REPDL_F32 || TPR == 1024 ? 16 : 24; // (no such rows of binary32, nor of 1024 threads)
        return E == 24 ? launch_layer_norm<DT, PDT, TPR, E24, false>(x, w, b, y, mean, rstd, M, N, eps, s)
                       : launch_layer_norm<DT, PDT, TPR, 16, false>(x, w, b, y, mean, rstd, M, N, eps, s);
    });
}

// Runs of rows of the backward pass, each of at least four rows and a multiple of the workgroup's teams: 256 runs, one to a CU,
// or 512 of 256 threads from 4096 rows on.  More runs write and read more partial sums, fewer leave a row's latency uncovered
// (512 x 4096 bf16 in runs of 1 / 4 / 8 rows 0.0159 / 0.0116 / 0.0152 ms; 2048 x 2048 in 512 / 256 runs 0.0160 / 0.0135; 4096 x 16384
// 0.114 / 0.101; 8192 x 4096 0.050 / 0.062).
int64_t ln_rows_per_block(int64_t M, int64_t N, int dtype)
{
    const int tpr = N > LN_MAX_ONCHIP ? 1024 : ln_threads_per_row(N, ln_elements(N, dtype, true));
    const int64_t teams = ln_grad_threads(tpr) / tpr;
    const int64_t rows = repdl_cdiv(M, tpr < 512 && M >= 4096 ? 512 : 256);
    return repdl_cdiv(rows < 4 ? 4 : rows, teams) * teams;
}

int64_t ln_partial_floats(int64_t M, int64_t N, int dtype) { return repdl_cdiv(M, ln_rows_per_block(M, N, dtype)) * 2 * N; }

// Rows up to which one launch makes all gradients (layer_norm_grad_few_kernel).  Both sides, two launches against one: 64 x 1024 f32
// 0.0081 / 0.0054 ms, 256 x 1024 0.0081 / 0.0058, 256 x 8192 0.0167 / 0.0090, 256 x 4096 bf16 0.0109 / 0.0076; 512 x 1024 f32 0.0081 / 0.0089,
// 1024 x 4096 bf16 0.0177 / 0.0244.
bool ln_few_rows(int64_t M, int64_t N) { return M <= LN_FEW_ROWS && N <= LN_MAX_ONCHIP; }

template <int DT, int PDT, int TPR, int E, bool TINY>
int launch_layer_norm_grad(const void *gy, const void *x, const void *w, const float *mean, const float *rstd, void *gx, void *gw, void *gb,
                           float *partial, int64_t M, int64_t N, hipStream_t s)
{
    typedef typename LowpType<DT>::T T;
    typedef typename LowpType<PDT>::T P;
    if (ln_few_rows(M, N))
    {
        const int rows = gx != nullptr ? (int)repdl_cdiv(M, ln_grad_threads(TPR) / TPR) : 0;
        const int cols = gw != nullptr || gb != nullptr ? (int)repdl_cdiv(N, 16 * Lowp<DT>::G) : 0;
        REPDL_LAUNCH((layer_norm_grad_few_kernel<DT, PDT, TPR, E, TINY>), dim3((unsigned)(rows + cols)), dim3(ln_grad_threads(TPR)), 0, s,
                     static_cast<const T *>(gy), static_cast<const T *>(x), static_cast<const P *>(w), mean, rstd, static_cast<T *>(gx),
                     static_cast<P *>(gw), static_cast<P *>(gb), (int)M, (int)N, rows, (float)(1.0 / (double)N));
        return repdl_launch_status();
    }
    const int64_t rpb = ln_rows_per_block(M, N, DT);
    const dim3 grid((unsigned)repdl_cdiv(M, rpb)), block(ln_grad_threads(TPR));
    if (TPR >= 64 && ln_streams<DT>(M, N, gx))
        REPDL_LAUNCH((layer_norm_grad_kernel<DT, PDT, TPR, E, TINY, (TPR >= 64)>), grid, block, 0, s, static_cast<const T *>(gy),
                     static_cast<const T *>(x), static_cast<const P *>(w), mean, rstd, static_cast<T *>(gx), partial, M, (int)N, rpb,
                     (float)(1.0 / (double)N));
    else
        REPDL_LAUNCH((layer_norm_grad_kernel<DT, PDT, TPR, E, TINY, false>), grid, block, 0, s, static_cast<const T *>(gy),
                     static_cast<const T *>(x), static_cast<const P *>(w), mean, rstd, static_cast<T *>(gx), partial, M, (int)N, rpb,
                     (float)(1.0 / (double)N));
    return repdl_launch_status();
}

template <int DT, int PDT>
int layer_norm_grad_typed(const void *gy, const void *x, const void *w, const float *mean, const float *rstd, void *gx, void *gw, void *gb,
                          float *partial, int64_t M, int64_t N, hipStream_t s)
{
    typedef typename LowpType<DT>::T T;
    typedef typename LowpType<PDT>::T P;
    if (N > LN_MAX_ONCHIP)
    {
        float *rest = partial == nullptr ? nullptr : partial + ln_partial_floats(M, N, DT); // (behind the partial sums)
        const int rc = repdl_launch_slices(M, 1024, [&](int64_t row, unsigned count) {
            REPDL_LAUNCH((layer_norm_grad_long_kernel<DT, PDT>), dim3(count), dim3(1024), 0, s, static_cast<const T *>(gy) + row * N,
                         static_cast<const T *>(x) + row * N, static_cast<const P *>(w), mean + row, rstd + row,
                         gx == nullptr ? nullptr : static_cast<T *>(gx) + row * N, rest == nullptr ? nullptr : rest + row, N,
                         (float)(1.0 / (double)N));
        });
        if (rc != REPDL_OK)
            return rc;
        if (partial != nullptr)
        {
            const int64_t rpb = ln_rows_per_block(M, N, DT);
            REPDL_LAUNCH((layer_norm_param_long_kernel<DT>),
                         dim3((unsigned)repdl_cdiv(N, 256 * Lowp<DT>::G), (unsigned)repdl_cdiv(M, rpb)), dim3(256), 0, s,
                         static_cast<const T *>(gy), static_cast<const T *>(x), mean, rstd, rest, partial, M, N, rpb);
        }
        return repdl_launch_status();
    }
    if (N < Lowp<DT>::G)
        return launch_layer_norm_grad<DT, PDT, 4, 16, true>(gy, x, w, mean, rstd, gx, gw, gb, partial, M, N, s);
    const int E = ln_elements(N, DT, true);
    return ln_with_threads(ln_threads_per_row(N, E), [&](auto threads) {
        constexpr int TPR = decltype(threads)::value;
        constexpr int E24 = DT == REPDL_F32 || TPR == 1024 ? 16 : 24;
        return E == 24 ? launch_layer_norm_grad<DT, PDT, TPR, E24, false>(gy, x, w, mean, rstd, gx, gw, gb, partial, M, N, s)
                       : launch_layer_norm_grad<DT, PDT, TPR, 16, false>(gy, x, w, mean, rstd, gx, gw, gb, partial, M, N, s);
    });
}

template <int PDT>
int layer_norm_params(const float *partial, void *gw, void *gb, int64_t M, int64_t N, int dtype, hipStream_t s)
{
    typedef typename LowpType<PDT>::T P;
    // (no rows: no blocks, the sums of nothing)
    const int blocks = M == 0 ? 0 : (int)repdl_cdiv(M, ln_rows_per_block(M, N, dtype));
    return repdl_launch_slices(repdl_cdiv(2 * N, 64), 64 * LN_FOLD, [&](int64_t first, unsigned count) {
        REPDL_LAUNCH((layer_norm_param_kernel<PDT>), dim3(count), dim3(64 * LN_FOLD), 0, s, partial, static_cast<P *>(gw),
                     static_cast<P *>(gb), N, blocks, first);
    });
}

bool ln_shape_ok(int64_t M, int64_t N, int dtype, int param_dtype)
{
    return M >= 0 && N >= 0 && M <= REPDL_I32_MAX && N <= REPDL_I32_MAX / 4 && repdl_known_dtype(dtype) &&
           (param_dtype == dtype || param_dtype == REPDL_F32);
}

// f(DT, PDT) for the pairs the library has: parameters of the activation's type, or binary32
#define LN_DISPATCH(dtype, param_dtype, f, ...)                                    \
    ((dtype) == REPDL_F32                 ? f<REPDL_F32, REPDL_F32>(__VA_ARGS__)   \
     : (dtype) == REPDL_BF16                                                       \
         ? ((param_dtype) == REPDL_F32 ? f<REPDL_BF16, REPDL_F32>(__VA_ARGS__)     \
                                       : f<REPDL_BF16, REPDL_BF16>(__VA_ARGS__))   \
         : ((param_dtype) == REPDL_F32 ? f<REPDL_F16, REPDL_F32>(__VA_ARGS__)      \
                                       : f<REPDL_F16, REPDL_F16>(__VA_ARGS__)))
} // namespace

REPDL_API int repdl_hip_layer_norm(const void *x, const void *weight, const void *bias, void *y, float *mean, float *rstd, int64_t M,
                                   int64_t N, float eps, int dtype, int param_dtype, void *stream)
{
    REPDL_REQUIRE(ln_shape_ok(M, N, dtype, param_dtype));
    REPDL_REQUIRE((mean == nullptr) == (rstd == nullptr));
    if (M == 0 || N == 0)
        return REPDL_OK;
    REPDL_REQUIRE(x != nullptr && y != nullptr);
    return LN_DISPATCH(dtype, param_dtype, layer_norm_typed, x, weight, bias, y, mean, rstd, M, N, eps, repdl_stream(stream));
}

REPDL_API int repdl_hip_layer_norm_grad(const void *grad_y, const void *x, const void *weight, const float *mean, const float *rstd,
                                        void *grad_x, void *grad_weight, void *grad_bias, int64_t M, int64_t N, int dtype,
                                        int param_dtype, void *stream)
{
    REPDL_REQUIRE(ln_shape_ok(M, N, dtype, param_dtype));
    const bool params = grad_weight != nullptr || grad_bias != nullptr;
    if (N == 0 || (grad_x == nullptr && !params) || (M == 0 && !params))
        return REPDL_OK;
    REPDL_REQUIRE(M == 0 || (grad_y != nullptr && x != nullptr && mean != nullptr && rstd != nullptr));
    hipStream_t s = repdl_stream(stream);
    float *partial = nullptr;
    const bool one_launch = M > 0 && ln_few_rows(M, N);
    if (params && M > 0 && !one_launch)
    {
        hipError_t e = repdl_ws_acquire(reinterpret_cast<void **>(&partial),
                                        (size_t)(ln_partial_floats(M, N, dtype) + (N > LN_MAX_ONCHIP ? M : 0)) * sizeof(float), s);
        if (e != hipSuccess)
            return (int)e;
    }
    int rc = REPDL_OK;
    if (M > 0)
        rc = LN_DISPATCH(dtype, param_dtype, layer_norm_grad_typed, grad_y, x, weight, mean, rstd, grad_x, grad_weight, grad_bias, partial, M, N, s);
    if (rc == REPDL_OK && params && !one_launch)
        rc = param_dtype == REPDL_F32    ? layer_norm_params<REPDL_F32>(partial, grad_weight, grad_bias, M, N, dtype, s)
             : param_dtype == REPDL_BF16 ? layer_norm_params<REPDL_BF16>(partial, grad_weight, grad_bias, M, N, dtype, s)
                                         : layer_norm_params<REPDL_F16>(partial, grad_weight, grad_bias, M, N, dtype, s);
    if (partial != nullptr)
    {
        const hipError_t e = repdl_ws_release(partial, s);
        if (rc == REPDL_OK && e != hipSuccess)
            rc = (int)e;
    }
    return rc;
}

REPDL_API size_t repdl_hip_layer_norm_grad_workspace_bytes(int64_t M, int64_t N)
{
    if (!ln_shape_ok(M, N, REPDL_F32, REPDL_F32) || M == 0 || N == 0)
        return 0;
    float *fake = const_cast<float *>(repdl_ws_fake_pointer(true));
    size_t need = 0; // (for any type: the runs of rows of binary32 and of 16 bits may differ)
    for (int dtype : {REPDL_F32, REPDL_BF16})
    {
        const size_t bytes =
            repdl_ws_query([&]() { return repdl_hip_layer_norm_grad(fake, fake, fake, fake, fake, fake, fake, fake, M, N, dtype, REPDL_F32, nullptr); });
        need = bytes > need ? bytes : need;
    }
    return need;
}

REPDL_API int repdl_hip_layer_norm_grad_ws(const void *grad_y, const void *x, const void *weight, const float *mean, const float *rstd,
                                           void *grad_x, void *grad_weight, void *grad_bias, int64_t M, int64_t N, int dtype,
                                           int param_dtype, void *workspace, size_t workspace_bytes, void *stream)
{
    RepdlWorkspace ws(workspace, workspace_bytes);
    return repdl_hip_layer_norm_grad(grad_y, x, weight, mean, rstd, grad_x, grad_weight, grad_bias, M, N, dtype, param_dtype, stream);
}
