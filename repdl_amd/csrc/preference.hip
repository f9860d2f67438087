// Preference loss of paired answers, from token logits.
//
// Sequences 0 .. P-1 are the preferred answers, P .. 2P-1 the others; r are a reference model's log probabilities.
//   lp_t = x[target_t] - m - log(sum_v exp(x_v - m)),  m = max_v x_v        every token whose target is not ignore_index
//   L_i  = sum_t lp_t
//   z_p  = beta ((L_p - L_{P+p}) - (r_p - r_{P+p}))
//   loss = (1/P) sum_p [(1 - eps) softplus(-z_p) + eps softplus(z_p)]
//   c_p  = d loss / d L_p = (beta / P) (eps sigma(z_p) - (1 - eps) sigma(-z_p)),  c_{P+p} = -c_p
//   d loss / d x_{t,v} = c (1[v = target_t] - exp(x_v - m) / sum)               0 on tokens that are not counted
//
// preference_rows_kernel reads the counted rows once and leaves (m, sum) per row and chunk of columns;
// preference_pairs_kernel, a workgroup per pair, joins a row's chunks, adds up the sequences and makes the pair's loss and c
// (and the last of them the mean); preference_grad_kernel reads the logits again and writes the gradient.  (c of a row needs
// every row of its pair: the second read cannot be saved.)
//
// Bound: HBM, and for 16-bit logits level with it the vector ALU.  A column of the forward pass is 13 instructions -- widen, half
// a maximum, clamp, 9 of crm_exp_term, an addition -- so 39.3e12 / 13 = 3e12 columns/s are 6 TB/s of 16-bit ones.  Measured, three
// quarters of the tokens counted: 8192 x 131072 bf16 forward 0.281 ms = 5.7 TB/s read (0.351 with the exponential as
// crm_exp_neg of a difference, 16 instructions; degree 6 here 0.304), backward 0.670 ms = 5.6 TB/s; 8192 x 32000 f32 forward 0.120 ms =
// 6.5, backward 0.340 = 5.4; a pair of 12 tokens x 1000 4 + 3 us, backward 4.
//
// The row sum is in binary32 in a fixed order (a thread's granules in turn, a butterfly over the wave, the waves, the chunks),
// which the vocabulary and the type determine alone.  Everything per token and per pair after it is in binary64: L is a sum
// of hundreds of terms of size ten whose differences of a tenth decide the loss.
#include "lowp.h"
#include "crmath.h"
#include "lanes.h"

namespace
{
__device__ const uint64_t g_exp_tab3[256] = CRM_EXP_TAB_INIT;
__device__ const float g_log_invc3[128] = CRM_LOG_INVC_INIT;
__device__ const double g_log_hi3[128] = CRM_LOG_HI_INIT;
__device__ const float g_log_lo3[128] = CRM_LOG_LO_INIT;

struct PrefShape
{
    int64_t seq_stride, step_stride; // elements between sequences and between steps of the logits
    int64_t vocab;
    int64_t width;  // columns of a chunk
    int64_t ignore; // target of a token that is not counted
    int32_t steps, rows, chunks;
    uint32_t first; // workgroup of the call that the launch begins with
};

// Row of logits `row` (0 .. 2 P steps - 1)
template <typename T>
__device__ __forceinline__ const T *pref_row(const T *x, const PrefShape &p, uint32_t row)
{
    const uint32_t seq = row / (uint32_t)p.steps, step = row - seq * (uint32_t)p.steps;
    return x + (int64_t)seq * p.seq_stride + (int64_t)step * p.step_stride;
}

// TPR threads share the E * TPR columns (at most) of one chunk of a row: 64 where a wave holds the whole row, else a workgroup.
template <int DT, int TPR, int E, bool STREAM>
__global__ __launch_bounds__(256) void preference_rows_kernel(const typename LowpType<DT>::T *__restrict__ x,
                                                              const int64_t *__restrict__ target, float2 *__restrict__ part,
                                                              float *__restrict__ picked, int *__restrict__ counter, PrefShape p)
{
    typedef Lowp<DT> L;
    constexpr int G = L::G, GPT = E / G, TEAMS = 256 / TPR;
    constexpr int DEGREE = DT == REPDL_F32 ? 6 : 5; // of the terms' polynomial
    __shared__ float wave_m[4], wave_s[4];
    const int tid = threadIdx.x, j = tid % TPR;
    if (p.first + blockIdx.x == 0 && tid == 0)
        *counter = 0; // (of the pairs kernel, which the stream orders after this one)
    const uint32_t item = __builtin_amdgcn_readfirstlane((p.first + blockIdx.x) * TEAMS + tid / TPR); // (row, chunk): the wave's
    const uint32_t row = TPR == 64 ? item : item / (uint32_t)p.chunks;
    const uint32_t chunk = TPR == 64 ? 0 : item - row * (uint32_t)p.chunks;
    if (row >= (uint32_t)p.rows)
        return;
    const int64_t t = target[row];
    if (t == p.ignore)
        return; // (the whole team: nothing of such a row is read or written)
    const typename L::T *xr = pref_row(x, p, row);
    const int64_t c0 = (int64_t)chunk * p.width;
    const int64_t c1 = c0 + p.width < p.vocab ? c0 + p.width : p.vocab;
    const int width = (int)(c1 - c0);
    if (chunk == 0 && j == 0)
        picked[row] = t >= 0 && t < p.vocab ? LowpType<DT>::widen(xr[t]) : __builtin_nanf("");

    typename L::Raw raw[GPT];
    const float none = -__builtin_inff();
    float v[GPT][G];
#pragma unroll
    for (int i = 0; i < GPT; i++)
    {
        const int c = (i * TPR + j) * G;
        if (c + G <= width)
            raw[i] = L::template load_raw<STREAM>(xr + c0 + c);
    }
    float m = none;
#pragma unroll
    for (int i = 0; i < GPT; i++)
    {
        const int c = (i * TPR + j) * G;
        if (c + G <= width)
            L::unpack(raw[i], v[i]);
        else
        {
#pragma unroll
            for (int k = 0; k < G; k++)
                v[i][k] = c + k < width ? LowpType<DT>::widen(xr[c0 + c + k]) : none;
        }
#pragma unroll
        for (int k = 0; k < G; k += 2) // (the maximum that a NaN passes through)
            m = __builtin_elementwise_maximum(__builtin_elementwise_maximum(v[i][k], v[i][k + 1]), m);
    }
    m = lanes_max<64>(m);
    if (TPR > 64)
    {
        if ((tid & 63) == 0)
            wave_m[tid >> 6] = m;
        __syncthreads();
        m = __builtin_elementwise_maximum(__builtin_elementwise_maximum(wave_m[0], wave_m[1]),
                                          __builtin_elementwise_maximum(wave_m[2], wave_m[3]));
    }
    // (a maximum too large for the terms' integers, or no number: it is subtracted first)
    float top = m;
    if (!(__builtin_fabsf(m) <= 0x1p21f))
    {
#pragma unroll
        for (int i = 0; i < GPT; i++)
#pragma unroll
            for (int k = 0; k < G; k++)
                v[i][k] = v[i][k] - m;
        top = 0.0f;
    }
    // (the clamp as a median of three: as a maximum it would take a second instruction that quiets NaNs)
    const float shift = crm_exp_shift(top), least = top - 86.0f;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < GPT; i++)
    {
        if (i * TPR * G < width) // (uniform: whole rounds past the row's end)
        {
            float e[G];
#pragma unroll
            for (int k = 0; k < G; k++)
                e[k] = crm_exp_term(__builtin_amdgcn_fmed3f(v[i][k], least, top), shift, DEGREE);
#pragma unroll
            for (int step = 1; step < G; step <<= 1)
#pragma unroll
                for (int k = 0; k + step < G; k += 2 * step)
                    e[k] = e[k] + e[k + step];
            s = s + e[0];
        }
    }
    s = lanes_sum<64>(s);
    if (TPR > 64)
    {
        if ((tid & 63) == 0)
            wave_s[tid >> 6] = s;
        __syncthreads();
        s = ((wave_s[0] + wave_s[1]) + wave_s[2]) + wave_s[3];
    }
    if (j == 0)
    {
        const float base = crm_exp_base(top, shift);
        float sum = s * base;
        // A row that one token owns: the maximum's own term times the base is 1 but for an error of up to 2.2e-7 (degree 6: 1.2e-7), so the
        // token's log probability would come out as that, of either sign, instead of 0, and 1 - p in the gradient likewise.  Below 1 + 2^-16
        // (seventy times the error: no such row is missed) that term counts as exactly 1.  s is at least it: rounded sums of positive
        // terms do not fall below one of them.  (A vocabulary of a single token keeps its one term as the sum has it.)
        if (sum > 0.5f && sum < 1.0f + 0x1p-16f && p.vocab > 1)
            sum = 1.0f + (s - crm_exp_term(top, shift, DEGREE)) * base;
        part[(int64_t)row * p.chunks + chunk] = make_float2(m, sum);
    }
}

constexpr int PAIR_THREADS = 1024;

__device__ __forceinline__ double wave_sum(double v)
{
#pragma unroll
    for (int off = 1; off < 64; off <<= 1)
        v = v + __shfl_xor(v, off, 64);
    return v;
}

// The tables of crm_exp64_core and crm_log64_core, in LDS.
struct PairTables
{
    uint64_t exp_tab[256];
    double log_hi[128];
    float log_invc[128], log_lo[128];
    __device__ crm_log_tables log_tables() const
    {
        crm_log_tables t;
        t.invc = log_invc;
        t.logc_hi = log_hi;
        t.logc_lo = log_lo;
        return t;
    }
};

// One pair: z -> its loss and d loss / d L of the preferred answer.  e = exp(-|z|) gives both sigmas without cancellation;
// log(1 + e) from its series where 1 + e would round e away.  |z| is capped at 700, where every term is its limit in binary32.
__device__ __forceinline__ void pair_terms(double z, double beta, double smoothing, double pairs, const PairTables &tables, double &loss,
                                           double &coef)
{
    const double a = __builtin_fabs(z);
    const double e = crm_exp64_core(a < 700.0 ? -a : -700.0, tables.exp_tab);
    const double l1 = e < 0x1p-20 ? crm_fma(-0.5 * e, e, e) : crm_log64_core(1.0 + e, tables.log_tables());
    const double near = 1.0 / (1.0 + e), far = e / (1.0 + e); // sigma(|z|), sigma(-|z|)
    const double sp = z >= 0 ? near : far, sn = z >= 0 ? far : near; // sigma(z), sigma(-z)
    loss = (1.0 - smoothing) * (l1 + (z < 0 ? a : 0.0)) + smoothing * (l1 + (z > 0 ? a : 0.0));
    if (smoothing == 0.0) // (0 times an infinite term is not wanted)
        loss = l1 + (z < 0 ? a : 0.0);
    coef = beta / pairs * (smoothing * sp - (1.0 - smoothing) * sn);
    if (!(a == a))
        loss = coef = a;
}

__global__ __launch_bounds__(PAIR_THREADS) void preference_pairs_kernel(const int64_t *__restrict__ target, const float2 *__restrict__ part,
                                                                        const float *__restrict__ picked,
                                                                        const float *__restrict__ ref, double *pair_loss, int *counter,
                                                                        float *__restrict__ loss, float *__restrict__ logps,
                                                                        float2 *__restrict__ row_stats, float *__restrict__ coef_out,
                                                                        PrefShape p, int pairs, double beta, double smoothing)
{
    __shared__ double scratch[PAIR_THREADS / 64];
    __shared__ int last;
    __shared__ PairTables tables;
    const int tid = threadIdx.x, pair = (int)(p.first + blockIdx.x);
    // the first half of the workgroup takes the preferred answer's tokens, the second half the other's
    constexpr int HALF = PAIR_THREADS / 2;
    const int side = tid / HALF;
    const int64_t row0 = (int64_t)(side == 0 ? pair : pairs + pair) * p.steps;
    if (tid < 256)
        tables.exp_tab[tid] = g_exp_tab3[tid];
    if (tid < 128)
    {
        tables.log_hi[tid] = g_log_hi3[tid];
        tables.log_invc[tid] = g_log_invc3[tid];
        tables.log_lo[tid] = g_log_lo3[tid];
    }
    double acc = 0.0;
    for (int base = 0; base < p.steps; base += HALF)
    {
        const int step = base + tid % HALF;
        const bool live = step < p.steps;
        const int64_t row = row0 + (live ? step : 0);
        // (read ahead of what decides whether they count: one trip to memory instead of three)
        const int64_t t = target[row];
        const float x = picked[row];
        float2 v = part[row * p.chunks];
        float m = v.x, s = v.y;
        for (int c = 1; c < p.chunks; c++)
        {
            v = part[row * p.chunks + c];
            const float top = __builtin_elementwise_maximum(m, v.x);
            s = s * crm_exp_neg(m - top) + v.y * crm_exp_neg(v.x - top);
            m = top;
        }
        if (base == 0)
            lds_barrier(); // (the tables)
        if (live && t != p.ignore)
        {
            // s >= 1 (a single token's vocabulary: 1 - 2^-22) unless the row holds a NaN, +inf or nothing but -inf
            const double lp = s > 0.5f ? ((double)x - (double)m) - crm_log64_core((double)s, tables.log_tables()) : __builtin_nan("");
            acc = acc + lp;
            if (row_stats != nullptr)
                row_stats[row] = make_float2(m, crm_div(1.0f, s));
        }
    }
    acc = wave_sum(acc);
    if ((tid & 63) == 0)
        scratch[tid >> 6] = acc;
    __syncthreads();
    double value = 0.0, coef = 0.0;
    if (tid == 0)
    {
        double L[2];
#pragma unroll
        for (int i = 0; i < 2; i++)
        {
            L[i] = scratch[i * (HALF / 64)];
            for (int w = 1; w < HALF / 64; w++)
                L[i] = L[i] + scratch[i * (HALF / 64) + w];
        }
        double z = L[0] - L[1];
        if (ref != nullptr)
            z = z - ((double)ref[pair] - (double)ref[pairs + pair]);
        pair_terms(beta * z, beta, smoothing, (double)pairs, tables, value, coef);
        logps[pair] = (float)L[0];
        logps[pairs + pair] = (float)L[1];
        if (coef_out != nullptr)
        {
            coef_out[pair] = (float)coef;
            coef_out[pairs + pair] = (float)-coef;
        }
    }
    if (pairs == 1)
    {
        if (tid == 0)
            *loss = (float)value;
        return;
    }
    // The workgroup that ends last adds the pairs' losses.  They and the counter are atomics of device scope, which go past the
    // L2s of the XCDs; the wait orders a workgroup's loss before its count.  (A release fence would also write back the whole L2:
    // 5 us here; a launch of its own for the mean takes 4.)
    if (tid == 0)
    {
        __hip_atomic_store(&pair_loss[pair], value, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == pairs - 1;
    }
    __syncthreads();
    if (!last)
        return;
    acc = 0.0;
    for (int i = tid; i < pairs; i += PAIR_THREADS)
        acc = acc + __hip_atomic_load(&pair_loss[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    acc = wave_sum(acc);
    if ((tid & 63) == 0) // (scratch: the first thread read the sequences' sums before the barrier above)
        scratch[tid >> 6] = acc;
    __syncthreads();
    if (tid == 0)
    {
        for (int w = 1; w < PAIR_THREADS / 64; w++)
            acc = acc + scratch[w];
        *loss = (float)(acc / (double)pairs);
    }
}

// d loss / d x: k e^(x - m) with k = -c / sum, and c more at the target.
template <int DT, int TPR, int E, bool STREAM>
__global__ __launch_bounds__(256, 4) void preference_grad_kernel(const typename LowpType<DT>::T *__restrict__ x,
                                                              const int64_t *__restrict__ target,
                                                              const float2 *__restrict__ row_stats, const float *__restrict__ coef,
                                                              const float *__restrict__ grad_loss,
                                                              typename LowpType<DT>::T *__restrict__ gx, PrefShape p)
{
    typedef Lowp<DT> L;
    constexpr int G = L::G, GPT = E / G, TEAMS = 256 / TPR;
    const int tid = threadIdx.x, j = tid % TPR;
    const uint32_t item = __builtin_amdgcn_readfirstlane((p.first + blockIdx.x) * TEAMS + tid / TPR);
    const uint32_t row = TPR == 64 ? item : item / (uint32_t)p.chunks;
    const uint32_t chunk = TPR == 64 ? 0 : item - row * (uint32_t)p.chunks;
    if (row >= (uint32_t)p.rows)
        return;
    const int64_t c0 = (int64_t)chunk * p.width;
    const int64_t c1 = c0 + p.width < p.vocab ? c0 + p.width : p.vocab;
    const int width = (int)(c1 - c0);
    typename L::T *gr = gx + (int64_t)row * p.vocab + c0;
    // (read beside the target that decides whether they count: one trip to memory instead of two)
    const float2 st = row_stats[row];
    const float cc = coef[row / (uint32_t)p.steps] * *grad_loss;
    const int64_t t = target[row];
    float v[G];
    if (t == p.ignore)
    {
#pragma unroll
        for (int k = 0; k < G; k++)
            v[k] = 0.0f;
#pragma unroll
        for (int i = 0; i < GPT; i++)
        {
            const int c = (i * TPR + j) * G;
            if (c < width)
                L::template store<STREAM>(gr, c, width, v);
        }
        return;
    }
    const typename L::T *xr = pref_row(x, p, row) + c0;
    typename L::Raw raw[GPT];
#pragma unroll
    for (int i = 0; i < GPT; i++)
    {
        const int c = (i * TPR + j) * G;
        if (c + G <= width)
            raw[i] = L::template load_raw<STREAM>(xr + c);
    }
    const float k0 = -(cc * st.y);
    const int64_t at = t - c0; // the target's column in this chunk, if it has it
#pragma unroll
    for (int i = 0; i < GPT; i++)
    {
        const int c = (i * TPR + j) * G;
        if (c < width)
        {
            if (c + G <= width)
                L::unpack(raw[i], v);
            else
            {
#pragma unroll
                for (int k = 0; k < G; k++)
                    v[k] = c + k < width ? LowpType<DT>::widen(xr[c + k]) : 0.0f;
            }
#pragma unroll
            for (int k = 0; k < G; k++)
                v[k] = k0 * crm_exp_neg(v[k] - st.x);
            if (at >= c && at < c + G)
            {
#pragma unroll
                for (int k = 0; k < G; k++)
                    v[k] = at == c + k ? v[k] + cc : v[k];
            }
            L::template store<STREAM>(gr, c, width, v);
        }
    }
}

// ---- host -------------------------------------------------------------------------------------
// Vocabularies of up to 1024 and 4096 columns go to a wave, 16 or 64 columns a lane, longer ones to workgroups of up to 16384.  Both sides, ms, every
// token counted, rows x vocabulary (f32 | bf16):
//   16 / 64 a lane      8192 x 100   0.0106 / 0.0146 | 0.0109 / 0.0148     8192 x 1000  0.0134 / 0.0161 | 0.0113 / 0.0150     131072 x 1000  0.125 / 0.132 | 0.070 / 0.107
//   wave / workgroup    8192 x 1100  0.0170 / 0.0414 | 0.0166 / 0.0313     8192 x 4096  0.0283 / 0.0425 | 0.0207 / 0.0317     24 x 4000      0.0077 / 0.0081 | 0.0078 / 0.0079
//   16384 / 8192 columns a workgroup   8192 x 32000 0.164 / 0.481 | 0.101 / 0.110     8192 x 131072 bf16 0.371 / 0.439     1288 x 50257 0.0465 / 0.107 | 0.0330 / 0.0309
constexpr int PREF_E = 64, PREF_SMALL_E = 16;
constexpr int64_t PREF_WAVE_SMALL = 64 * PREF_SMALL_E;
constexpr int64_t PREF_WAVE = 64 * PREF_E;
constexpr int64_t PREF_CHUNK = 256 * PREF_E;

// Chunks of about equal width, in whole rounds of a workgroup's granules (2048 columns are one of 16-bit elements, two of binary32):
// all rounds but a row's last are full.
void pref_chunks(int64_t vocab, int64_t most, int32_t &chunks, int64_t &width)
{
    chunks = (int32_t)repdl_cdiv(vocab, most);
    width = repdl_cdiv(repdl_cdiv(vocab, chunks), 2048) * 2048;
    chunks = (int32_t)repdl_cdiv(vocab, width);
}

bool pref_shape_ok(int64_t pairs, int64_t steps, int64_t vocab, int64_t seq_stride, int64_t step_stride, int dtype)
{
    if (pairs < 1 || steps < 0 || vocab < 1 || seq_stride < 0 || step_stride < 0 || !repdl_known_dtype(dtype))
        return false;
    if (pairs > REPDL_I32_MAX / 2 || steps > REPDL_I32_MAX || vocab > REPDL_I32_MAX / 4)
        return false;
    return steps == 0 || (2 * pairs <= REPDL_I32_MAX / steps && 2 * pairs * steps <= REPDL_I32_MAX / (repdl_cdiv(vocab, PREF_CHUNK / 2) + 1));
}

PrefShape pref_shape(int64_t pairs, int64_t steps, int64_t vocab, int64_t seq_stride, int64_t step_stride, int64_t ignore, int64_t most)
{
    PrefShape p;
    p.seq_stride = seq_stride;
    p.step_stride = step_stride;
    p.vocab = vocab;
    p.ignore = ignore;
    p.steps = (int32_t)steps;
    p.rows = (int32_t)(2 * pairs * steps);
    p.first = 0;
    pref_chunks(vocab, most, p.chunks, p.width);
    return p;
}

template <int DT>
bool pref_streams(const PrefShape &p)
{
    return (int64_t)p.rows * p.vocab >= REPDL_STREAM_BYTES / repdl_dtype_bytes(DT);
}

template <int DT>
int launch_pref_rows(const void *logits, const int64_t *target, float2 *part, float *picked, int *counter, PrefShape p, hipStream_t s)
{
    const auto *x = static_cast<const typename LowpType<DT>::T *>(logits);
    const bool by_wave = p.vocab <= PREF_WAVE, streams = pref_streams<DT>(p);
    // (one workgroup at least: it clears the counter)
    const int64_t blocks = p.rows == 0 ? 1 : by_wave ? repdl_cdiv(p.rows, 4) : (int64_t)p.rows * p.chunks;
    return repdl_launch_slices(blocks, 256, [&](int64_t first, unsigned count) {
        p.first = (uint32_t)first;
        if (p.vocab <= PREF_WAVE_SMALL)
            REPDL_LAUNCH((preference_rows_kernel<DT, 64, PREF_SMALL_E, false>), dim3(count), dim3(256), 0, s, x, target, part, picked, counter, p);
        else if (by_wave)
            REPDL_LAUNCH((preference_rows_kernel<DT, 64, PREF_E, false>), dim3(count), dim3(256), 0, s, x, target, part, picked, counter, p);
        else if (streams)
            REPDL_LAUNCH((preference_rows_kernel<DT, 256, PREF_E, true>), dim3(count), dim3(256), 0, s, x, target, part, picked, counter, p);
        else
            REPDL_LAUNCH((preference_rows_kernel<DT, 256, PREF_E, false>), dim3(count), dim3(256), 0, s, x, target, part, picked, counter, p);
    });
}

// The gradient of up to 1024 columns by a wave, 16 a lane; against a workgroup, as above: 8192 x 100 0.0044 / 0.0102 | 0.0055 / 0.0107, 8192 x 1000 0.0119 / 0.0152 |
// 0.0078 / 0.0121, 131072 x 1000 0.213 / 0.206 | 0.099 / 0.164.  Longer ones by workgroups of 32 columns a thread; 16 / 32 / 64: 8192 x 5000 0.0750 / 0.0612 / 0.0749 |
// 0.0333 / 0.0295 / 0.0291, 8192 x 10000 0.113 / 0.129 / 0.127 | 0.057 / 0.067 / 0.065, 8192 x 32000 0.366 / 0.384 / 0.403 | 0.180 / 0.196 / 0.193, 8192 x 131072 bf16 0.712 / 0.721 /
// 0.742, 1288 x 50257 0.099 / 0.100 / 0.115 | 0.042 / 0.043 / 0.047, 24 x 32000 0.0045 / 0.0054 / 0.0092 | 0.0033 / 0.0041 / 0.0061.
constexpr int PREF_GRAD_E = 32;

template <int DT>
int launch_pref_grad(const void *logits, const int64_t *target, const float2 *row_stats, const float *coef, const float *grad_loss,
                     void *grad_logits, PrefShape p, hipStream_t s)
{
    typedef typename LowpType<DT>::T T;
    const T *x = static_cast<const T *>(logits);
    T *gx = static_cast<T *>(grad_logits);
    const bool by_wave = p.vocab <= PREF_WAVE_SMALL;
    const bool streams = pref_streams<DT>(p) && p.vocab % Lowp<DT>::G == 0 && (reinterpret_cast<uintptr_t>(gx) & 15) == 0;
    return repdl_launch_slices(by_wave ? repdl_cdiv(p.rows, 4) : (int64_t)p.rows * p.chunks, 256, [&](int64_t first, unsigned count) {
        p.first = (uint32_t)first;
        if (by_wave)
            REPDL_LAUNCH((preference_grad_kernel<DT, 64, PREF_SMALL_E, false>), dim3(count), dim3(256), 0, s, x, target, row_stats, coef,
                         grad_loss, gx, p);
        else if (streams)
            REPDL_LAUNCH((preference_grad_kernel<DT, 256, PREF_GRAD_E, true>), dim3(count), dim3(256), 0, s, x, target, row_stats, coef,
                         grad_loss, gx, p);
        else
            REPDL_LAUNCH((preference_grad_kernel<DT, 256, PREF_GRAD_E, false>), dim3(count), dim3(256), 0, s, x, target, row_stats, coef,
                         grad_loss, gx, p);
    });
}
} // namespace

REPDL_API int repdl_hip_preference_loss(const void *logits, const int64_t *target, const float *ref_logps, float *loss, float *logps,
                                        float *row_stats, float *coef, int64_t pairs, int64_t steps, int64_t vocab, int64_t seq_stride,
                                        int64_t step_stride, double beta, double label_smoothing, int64_t ignore_index, int dtype,
                                        void *stream)
{
    REPDL_REQUIRE(pref_shape_ok(pairs, steps, vocab, seq_stride, step_stride, dtype));
    REPDL_REQUIRE(loss != nullptr && logps != nullptr && (steps == 0 || (logits != nullptr && target != nullptr)));
    REPDL_REQUIRE((row_stats != nullptr) == (coef != nullptr) || (steps == 0 && coef != nullptr)); // (no rows: no statistics)
    hipStream_t s = repdl_stream(stream);
    PrefShape p = pref_shape(pairs, steps, vocab, seq_stride, step_stride, ignore_index, PREF_CHUNK);
    // scratch: (m, sum) per row and chunk, the pairs' losses, the target's logit per row, a counter
    const size_t parts = (size_t)p.rows * (size_t)p.chunks;
    char *work = nullptr;
    hipError_t e = repdl_ws_acquire(reinterpret_cast<void **>(&work), parts * sizeof(float2) + (size_t)pairs * sizeof(double) +
                                                                          (size_t)p.rows * sizeof(float) + sizeof(int), s);
    if (e != hipSuccess)
        return (int)e;
    float2 *part = reinterpret_cast<float2 *>(work);
    double *pair_loss = reinterpret_cast<double *>(part + parts);
    float *picked = reinterpret_cast<float *>(pair_loss + pairs);
    int *counter = reinterpret_cast<int *>(picked + p.rows);
    int rc = dtype == REPDL_F32    ? launch_pref_rows<REPDL_F32>(logits, target, part, picked, counter, p, s)
             : dtype == REPDL_BF16 ? launch_pref_rows<REPDL_BF16>(logits, target, part, picked, counter, p, s)
                                   : launch_pref_rows<REPDL_F16>(logits, target, part, picked, counter, p, s);
    if (rc == REPDL_OK)
        rc = repdl_launch_slices(pairs, PAIR_THREADS, [&](int64_t first, unsigned count) { // (the counter goes on from slice to slice)
            p.first = (uint32_t)first;
            REPDL_LAUNCH(preference_pairs_kernel, dim3(count), dim3(PAIR_THREADS), 0, s, target, part, picked, ref_logps, pair_loss,
                         counter, loss, logps, reinterpret_cast<float2 *>(row_stats), coef, p, (int)pairs, beta, label_smoothing);
        });
    e = repdl_ws_release(work, s);
    return rc != REPDL_OK ? rc : (int)e;
}

REPDL_API size_t repdl_hip_preference_loss_workspace_bytes(int64_t pairs, int64_t steps, int64_t vocab)
{
    if (!pref_shape_ok(pairs, steps, vocab, 0, 0, REPDL_F32))
        return 0;
    float *fake = const_cast<float *>(repdl_ws_fake_pointer(true));
    return repdl_ws_query([&]() {
        return repdl_hip_preference_loss(fake, reinterpret_cast<const int64_t *>(fake), fake, fake, fake, fake, fake, pairs, steps, vocab, 0, 0,
                                         1.0, 0.0, 0, REPDL_F32, nullptr);
    });
}

REPDL_API int repdl_hip_preference_loss_ws(const void *logits, const int64_t *target, const float *ref_logps, float *loss, float *logps,
                                           float *row_stats, float *coef, int64_t pairs, int64_t steps, int64_t vocab,
                                           int64_t seq_stride, int64_t step_stride, double beta, double label_smoothing,
                                           int64_t ignore_index, int dtype, void *workspace, size_t workspace_bytes, void *stream)
{
    RepdlWorkspace ws(workspace, workspace_bytes);
    return repdl_hip_preference_loss(logits, target, ref_logps, loss, logps, row_stats, coef, pairs, steps, vocab, seq_stride, step_stride,
                                     beta, label_smoothing, ignore_index, dtype, stream);
}

REPDL_API int repdl_hip_preference_loss_grad(const void *logits, const int64_t *target, const float *row_stats, const float *coef,
                                             const float *grad_loss, void *grad_logits, int64_t pairs, int64_t steps, int64_t vocab,
                                             int64_t seq_stride, int64_t step_stride, int64_t ignore_index, int dtype, void *stream)
{
    REPDL_REQUIRE(pref_shape_ok(pairs, steps, vocab, seq_stride, step_stride, dtype));
    if (steps == 0)
        return REPDL_OK;
    REPDL_REQUIRE(logits != nullptr && target != nullptr && row_stats != nullptr && coef != nullptr && grad_loss != nullptr && grad_logits != nullptr);
    hipStream_t s = repdl_stream(stream);
    const PrefShape p = pref_shape(pairs, steps, vocab, seq_stride, step_stride, ignore_index, 256 * PREF_GRAD_E);
    const float2 *stats = reinterpret_cast<const float2 *>(row_stats);
    return dtype == REPDL_F32    ? launch_pref_grad<REPDL_F32>(logits, target, stats, coef, grad_loss, grad_logits, p, s)
           : dtype == REPDL_BF16 ? launch_pref_grad<REPDL_BF16>(logits, target, stats, coef, grad_loss, grad_logits, p, s)
                                 : launch_pref_grad<REPDL_F16>(logits, target, stats, coef, grad_loss, grad_logits, p, s);
}
