/* The preference loss of csrc/preference.hip, operation by operation and in the order of its sums, on the CPU: what the tests hold
 * the kernels' loss, log probabilities, row statistics and coefficients to, every bit.  Finite logits, at least one counted token per
 * sequence or none; x is [2 pairs * steps][vocab], widened to binary32.  Compiled with contraction off. */
#include <stdlib.h>

#include "crmath.h"

static const uint64_t exp_tab[256] = CRM_EXP_TAB_INIT;
static const float log_invc[128] = CRM_LOG_INVC_INIT;
static const double log_hi[128] = CRM_LOG_HI_INIT;
static const float log_lo[128] = CRM_LOG_LO_INIT;

static float pairs_of(float *v, int n) /* neighbours, pairs of neighbours, ... */
{
    for (int step = 1; step < n; step *= 2)
        for (int k = 0; k + step < n; k += 2 * step)
            v[k] = v[k] + v[k + step];
    return v[0];
}

static double pairs_of_d(double *v, int n)
{
    for (int step = 1; step < n; step *= 2)
        for (int k = 0; k + step < n; k += 2 * step)
            v[k] = v[k] + v[k + step];
    return v[0];
}

/* (m, sum) of `width` columns by `threads` threads of `each` elements in granules of g */
static void chunk_sum(const float *x, int64_t width, int threads, int each, int g, float *m_out, float *s_out)
{
    float m = -INFINITY;
    for (int64_t c = 0; c < width; c++)
        m = x[c] > m ? x[c] : m;
    const int large = !(fabsf(m) <= 0x1p21f);
    const float top = large ? 0.0f : m, shift = crm_exp_shift(top), least = top - 86.0f;
    float waves[4], lanes[64];
    for (int w = 0; w < threads / 64; w++)
    {
        for (int l = 0; l < 64; l++)
        {
            const int j = 64 * w + l;
            float s = 0.0f;
            for (int i = 0; i < each / g; i++)
                if ((int64_t)i * threads * g < width)
                {
                    float e[8];
                    for (int k = 0; k < g; k++)
                    {
                        const int64_t c = ((int64_t)i * threads + j) * g + k;
                        float v = c < width ? x[c] : -INFINITY;
                        if (large)
                            v = v - m;
                        v = v < least ? least : v;
                        e[k] = crm_exp_term(v, shift, g == 4 ? 6 : 5);
                    }
                    s = s + pairs_of(e, g);
                }
            lanes[l] = s;
        }
        waves[w] = pairs_of(lanes, 64);
    }
    float s = waves[0];
    for (int w = 1; w < threads / 64; w++)
        s = s + waves[w];
    *m_out = m;
    *s_out = s * crm_exp_base(top, shift);
}

static void row(const float *x, int64_t vocab, int g, float *m_out, float *s_out)
{
    if (vocab <= 4096)
    {
        chunk_sum(x, vocab, 64, vocab <= 1024 ? 16 : 64, g, m_out, s_out);
        return;
    }
    int64_t chunks = (vocab + 16383) / 16384, width = (vocab + chunks - 1) / chunks;
    width = (width + 2047) / 2048 * 2048;
    float m = 0.0f, s = 0.0f;
    for (int64_t c0 = 0; c0 < vocab; c0 += width)
    {
        float cm, cs;
        chunk_sum(x + c0, c0 + width < vocab ? width : vocab - c0, 256, 64, g, &cm, &cs);
        if (c0 == 0)
            m = cm, s = cs;
        else
        {
            const float top = m > cm ? m : cm;
            s = s * crm_exp_neg(m - top) + cs * crm_exp_neg(cm - top);
            m = top;
        }
    }
    *m_out = m;
    *s_out = s;
}

void preference_model(const float *x, const int64_t *target, const float *ref, int64_t pairs, int64_t steps, int64_t vocab, int g, double beta,
                      double smoothing, int64_t ignore, float *loss, float *logps, float *stats, float *coef)
{
    const crm_log_tables lt = {log_invc, log_hi, log_lo};
    double *L = malloc(2 * pairs * sizeof(double)), *terms = malloc(pairs * sizeof(double));
    for (int64_t q = 0; q < 2 * pairs; q++)
    {
        double acc[512] = {0.0};
        for (int64_t t = 0; t < steps; t++)
        {
            const int64_t r = q * steps + t;
            if (target[r] == ignore)
                continue;
            float m, s;
            row(x + r * vocab, vocab, g, &m, &s);
            stats[2 * r] = m;
            stats[2 * r + 1] = crm_div(1.0f, s);
            acc[t % 512] = acc[t % 512] + (((double)x[r * vocab + target[r]] - (double)m) - crm_log64_core((double)s, lt));
        }
        L[q] = pairs_of_d(acc, 64);
        for (int w = 1; w < 8; w++)
            L[q] = L[q] + pairs_of_d(acc + 64 * w, 64);
        logps[q] = (float)L[q];
    }
    for (int64_t p = 0; p < pairs; p++)
    {
        double z = L[p] - L[pairs + p];
        if (ref)
            z = z - ((double)ref[p] - (double)ref[pairs + p]);
        z = beta * z;
        const double a = fabs(z), e = crm_exp64_core(a < 700.0 ? -a : -700.0, exp_tab);
        const double l1 = e < 0x1p-20 ? crm_fma(-0.5 * e, e, e) : crm_log64_core(1.0 + e, lt);
        const double near = 1.0 / (1.0 + e), far = e / (1.0 + e), sp = z >= 0 ? near : far, sn = z >= 0 ? far : near;
        terms[p] = smoothing == 0.0 ? l1 + (z < 0 ? a : 0.0)
                                    : (1.0 - smoothing) * (l1 + (z < 0 ? a : 0.0)) + smoothing * (l1 + (z > 0 ? a : 0.0));
        const double c = beta / (double)pairs * (smoothing * sp - (1.0 - smoothing) * sn);
        coef[p] = (float)c;
        coef[pairs + p] = (float)-c;
    }
    if (pairs == 1)
        *loss = (float)terms[0];
    else
    {
        double acc[1024] = {0.0};
        for (int64_t p = 0; p < pairs; p++)
            acc[p % 1024] = acc[p % 1024] + terms[p];
        double sum = pairs_of_d(acc, 64);
        for (int w = 1; w < 16; w++)
            sum = sum + pairs_of_d(acc + 64 * w, 64);
        *loss = (float)(sum / (double)pairs);
    }
    free(L);
    free(terms);
}
