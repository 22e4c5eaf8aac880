// gridgcn_gnorm.hip -- group normalisation with an activation on channels-last rows, forward and backward.
//
//   x [B, N, C], G groups of cg = C / G channels, statistics of a (cloud, group) over its rows n < count_b and its channels:
//     d = x - mean,  t = d * rstd * gamma_c + beta_c,  y = act(t);       rows n >= count_b: y = 0, dx = 0, never read
//   backward, x^ = x or the 8-bit form the forward kept (gridgcn_act8.h), d = x^ - mean, xh = d * rstd:
//     g = dy * act'(t);  dbeta_c = sum g;  dgamma_c = sum g xh;
//     dx = rstd (gamma g - S1 - xh S2),  S1 = sum_group(gamma g) / M,  S2 = sum_group(gamma g xh) / M,  M = count_b * cg
//
// All of it is streaming: a thread keeps one column chunk of 16 bytes (its channels' constants sit in registers) and walks
// rows.  The statistics are a reduction over a whole cloud, so a pass over the data has to end before the next begins: two
// passes with a small launch between them that turns the workgroups' partial sums into statistics, or -- where the rows of a
// few groups of one cloud fit a workgroup's registers -- ONE launch that reads them once.
//
// Numerics.  Sums of the statistics run in 64 bits on x - x[first row, first channel of the group] (64-bit vector adds run at
// the rate of 32-bit ones here, the passes wait for memory): the variance needs no second look at the data even when the mean is
// large against it.  The mean is subtracted as two floats, so d is x - mean to 32 bits whatever the mean.  Sums of the backward:
// 32 bits over UNROLL rows, then 64.  No atomics: every sum has one order.
#include "../../include/gridgcn.h"
#include "gridgcn_act8.h"
#include <type_traits>

namespace {
constexpr int THREADS = 256;
constexpr int UNROLL = 4;
constexpr int FEW = 512;                   // threads of the one-launch form, which keeps its values in registers
template <class T> constexpr int KEEP = sizeof(T) == 4 ? 16 : 8;     // chunks a thread keeps
constexpr float SQRT1_2 = 0.70710678118654752f, INV_SQRT_2PI = 0.39894228040143268f;

typedef double f64x2 __attribute__((ext_vector_type(2)));

struct Lay { int nq, tpr, rpb; };          // chunks of a slab row, threads per row, rows per step
Lay lay_of(int nq, int threads = THREADS)
{
    Lay l;
    l.nq = nq;
    l.tpr = nq < threads ? nq : threads;
    l.rpb = threads / l.tpr;
    return l;
}

struct Args {
    const void *x, *dy;
    const uint8_t *codes, *scales;
    uint8_t *codes_out, *scales_out;
    void *y;                               // y or dx, contiguous [B, N, C]
    long long N, xb, xn, gb, gn;           // strides of x and dy in elements
    int B, C, G, cg, ptype;
    const void *gamma, *beta;
    void *dgamma, *dbeta;
    const int *counts;
    float eps;
    double *stats;                         // [B, G, 2] mean, rstd
    double *part;                          // [B, chunks, C, 2] partial sums of the workgroups
    double *tot;                           // [B, C, 2] sums of g and g * xh
    float2 *coef;                          // [B, G] rstd S1, rstd S2
    long long rpc;                         // rows of a chunk
    bool past;                             // y or dx around the caches
    int chunks;
};

__device__ __forceinline__ long long count_of(const Args &a, int b)
{
    if (!a.counts) return a.N;
    const long long n = a.counts[b];
    return n < 0 ? 0 : (n < a.N ? n : a.N);
}

// Phi(t) = (1 + erf(t / sqrt 2)) / 2 and e = exp(-t^2 / 2), which its derivative wants as well.  Phi(-a) = e R(a), and R falls slowly,
// from 1/2 as 1 / (a sqrt(2 pi)): a polynomial in k = 1 / (1 + p a), fitted for the least relative error over 0 <= a <= 14.5 (beyond,
// e is 0).
//   32-bit rows: R = k Q(1 - k), Q of degree 9, error 2e-9: t Phi(t) is off by 3.5e-8 of its norm for normal t (0.5 t (1 + erf), erf
//   to a step: 3.7e-8) and keeps its digits where Phi(t) is small (4e-6 of the value at t = -9, the exponential's);
//   16-bit rows: degree 6 in k, error 1e-7 at 0, growing to 2e-4 (half of fp16's half step) from |t| = 5 on.  (Degree 9 for them too:
//   backward of 16 x 65536 x 64 bf16 from codes 159 us, not 146.)
template <class T> __device__ __forceinline__ float normal_cdf(float t, float &e)
{
    e = __builtin_amdgcn_exp2f(t * t * -0.72134752f);
    float q;
    if constexpr (GGRowT<T>::id == GG_T_F32) {
        const float pa = 0.2375f * fminf(fabsf(t), 16.f), k = __builtin_amdgcn_rcpf(1.f + pa), m = pa * k;      // m = 1 - k
        q = fmaf(m, -0.0271149112f, 0.105926423f);
        q = fmaf(m, q, -0.114639388f);
        q = fmaf(m, q, -0.0758714394f);
        q = fmaf(m, q, 0.169976482f);
        q = fmaf(m, q, 0.313199016f);
        q = fmaf(m, q, -1.1696099f);
        q = fmaf(m, q, 1.57263014f);
        q = fmaf(m, q, -1.17975722f);
        q = fmaf(m, q, 0.500000001f) * (k * e);
    } else {
        const float k = __builtin_amdgcn_rcpf(fmaf(fabsf(t), 0.2875f, 1.f));
        q = fmaf(k, -0.0921373988f, 0.305879399f);
        q = fmaf(k, q, -0.11953044f);
        q = fmaf(k, q, 0.19386526f);
        q = fmaf(k, q, 0.0956545484f);
        q = fmaf(k, q, 0.116268678f) * (k * e);
    }
    return t < 0.f ? q : 1.f - q;           // (q = Phi(-|t|): no cancellation on the side where it is small)
}
// (the reciprocal instruction is good to one step: far below the activation's own rounding budget)
__device__ __forceinline__ float sigmoid(float t) { return __builtin_amdgcn_rcpf(1.f + __expf(-t)); }

template <int ACT, class T> __device__ __forceinline__ float act_of(float t)
{
    if constexpr (ACT == GRIDGCN_ACT_RELU) return t > 0.f ? t : (t != t ? t : 0.f);     // (NaN stays NaN)
    if constexpr (ACT == GRIDGCN_ACT_SILU) return t * sigmoid(t);
    if constexpr (ACT == GRIDGCN_ACT_GELU) {
        float e;
        return t * normal_cdf<T>(t, e);
    }
    return t;
}
template <int ACT, class T> __device__ __forceinline__ float act_grad(float t)
{
    if constexpr (ACT == GRIDGCN_ACT_SILU) {
        const float s = sigmoid(t);
        return s * fmaf(t, 1.f - s, 1.f);
    }
    if constexpr (ACT == GRIDGCN_ACT_GELU) {
        float e;
        const float c = normal_cdf<T>(t, e);
        return fmaf(t * INV_SQRT_2PI, e, c);
    }
    return 1.f;
}

// the largest float that is not above v
__device__ __forceinline__ float float_below(double v)
{
    const float f = (float)v;
    if (!((double)f > v)) return f;                        // (NaN stays NaN)
    const unsigned u = __float_as_uint(f);
    return __uint_as_float(u == 0u ? 0x80000001u : (u >> 31 ? u + 1 : u - 1));
}

// constants of one channel
struct Chan {
    float mh, ml, a;                        // mean in two parts, rstd * gamma
    float beta;                             // forward, and the backward of the smooth activations
    float rstd;                             // backward
    float thr;                              // ReLU backward: t > 0 exactly where `flip`ped x > thr
    unsigned flip;
};
// The sign of t = (x - mean) rstd gamma + beta decides a whole gradient under ReLU, and 32 bits get it wrong where the two terms
// cancel.  t > 0 is x > mean - beta / (rstd gamma), or < where gamma is negative: that border is formed once per channel in 64 bits
// and rounded down to a float, which loses nothing against an x that is a float.
template <int ACT, bool BACKWARD> __device__ __forceinline__ Chan chan_of(const Args &a, double mean, double rstd, int c)
{
    Chan k;
    k.mh = (float)mean;
    k.ml = (float)(mean - (double)k.mh);
    k.beta = gg_ld_param(a.beta, a.ptype, c, 0.f);
    const double m = rstd * (double)gg_ld_param(a.gamma, a.ptype, c, 1.f);
    k.a = (float)m;
    k.rstd = (float)rstd;
    k.thr = 0.f;
    k.flip = 0u;
    if constexpr (BACKWARD && ACT == GRIDGCN_ACT_RELU) {
        const double t = mean - (double)k.beta / m;
        k.flip = m < 0.0 ? 0x80000000u : 0u;
        k.thr = float_below(m < 0.0 ? -t : t);
        if (m == 0.0) k.thr = k.beta > 0.f ? -INFINITY : INFINITY;
    }
    return k;
}
// ... of the V channels of a thread, from the statistics in memory
template <int ACT, bool BACKWARD, int V, class P> __device__ __forceinline__ void chans(const Args &a, const P &p, Chan (&k)[V])
{
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int c = p.c + i < a.C ? p.c + i : a.C - 1;
        const double *st = a.stats + ((size_t)p.b * a.G + c / a.cg) * 2;
        k[i] = chan_of<ACT, BACKWARD>(a, st[0], st[1], c);
    }
}
__device__ __forceinline__ float dev_of(const Chan &k, float x) { return (x - k.mh) - k.ml; }

// where the workgroup's threads stand
template <int V> struct Pos {
    int tr, q, c, b;
    bool on;
    __device__ __forceinline__ Pos(const Lay &l, int q0, int b_)
    {
        tr = (int)threadIdx.x / l.tpr;
        q = q0 + (int)threadIdx.x % l.tpr;
        c = q * V;
        b = b_;
        on = tr < l.rpb && q < q0 + l.tpr && q < l.nq;
    }
};

// Sums s[V][2] of the threads of a column over the workgroup's row lanes: LDS red[rpb][tpr * V][2]; afterwards red[0] holds them.
// All threads take part: strips of rows first, then the strips (a thread per sum alone walks up to 512 rows of LDS one after
// the other).
template <int V, int NT> __device__ __forceinline__ void reduce_rows(double *red, const Lay &l, int tr, int qi, const double (&s)[V][2])
{
    const int w = l.tpr * V * 2;
    if (tr < l.rpb) {
#pragma unroll
        for (int i = 0; i < V; i++) {
            red[(size_t)tr * w + (qi * V + i) * 2] = s[i][0];
            red[(size_t)tr * w + (qi * V + i) * 2 + 1] = s[i][1];
        }
    }
    __syncthreads();
    const int strips = NT / w, per = strips > 1 ? (l.rpb + strips - 1) / strips : 1;
    if (per > 1) {
        const int k = (int)threadIdx.x / w, r0 = k * per, r1 = r0 + per < l.rpb ? r0 + per : l.rpb;
        if (k < strips && r0 < r1) {
            double *q = red + (size_t)threadIdx.x % w;
            double v = q[(size_t)r0 * w];
            for (int r = r0 + 1; r < r1; r++) v += q[(size_t)r * w];
            q[(size_t)r0 * w] = v;         // (this thread's alone)
        }
        __syncthreads();
    }
    for (int j = threadIdx.x; j < w; j += NT) {
        double v = red[j];
        for (int r = per; r < l.rpb; r += per) v += red[(size_t)r * w + j];
        red[j] = v;                        // (entry j of row 0 is this thread's alone)
    }
    __syncthreads();
}

// the values that the sums of a thread's channels are taken from: x[first row, first channel of the group]
template <class T>
__device__ __forceinline__ void base_of(const Args &a, const Pos<GGRowT<T>::V> &p, const T *x, double (&base)[GGRowT<T>::V])
{
    T w[GGRowT<T>::V];
#pragma unroll
    for (int i = 0; i < GGRowT<T>::V; i++) w[i] = x[((p.c + i < a.C ? p.c + i : a.C - 1) / a.cg) * a.cg];
#pragma unroll
    for (int i = 0; i < GGRowT<T>::V; i++) base[i] = (double)GGRowT<T>::get(w + i);
}

// first pass over the rows r0 <= n < r1 of cloud b: sums of x - base and its square per channel, and (SAVE8) the 8-bit form
template <class T, bool SAVE8>
__device__ __forceinline__ void rows_stats(const Args &a, const Lay &l, const Pos<GGRowT<T>::V> &p, long long r0, long long r1,
                                           double (&s)[GGRowT<T>::V][2], double (&base)[GGRowT<T>::V])
{
    constexpr int V = GGRowT<T>::V;
    const T *x = (const T *)a.x + (size_t)p.b * a.xb;
    const int Cp = gg_a8_cp(a.C), nb = Cp / GG_A8_BLOCK;
    const GGCol<T> col(p.on ? p.c : 0, a.C);
    base_of<T>(a, p, x, base);                             // (row 0 is valid where any row is)
#pragma unroll
    for (int i = 0; i < V; i++) s[i][0] = s[i][1] = 0.0;
    constexpr int U = SAVE8 ? UNROLL : 2 * UNROLL;
    for (long long n0 = r0; n0 < r1; n0 += (long long)l.rpb * U) {
        GGChunk<T> r[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const long long n = n0 + (long long)u * l.rpb + p.tr;
            r[u].load(x + (size_t)(n < r1 ? n : r1 - 1) * a.xn, col, a.C);        // (rows past the end: in no sum, not stored)
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const long long n = n0 + (long long)u * l.rpb + p.tr;
            const bool in = p.on && n < r1;
            float v[V];
            r[u].align(col);
            r[u].get(v);
            if (in) {
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const double d = (double)v[i] - base[i];
                    s[i][0] += d;
                    s[i][1] = fma(d, d, s[i][1]);
                }
            }
            if constexpr (SAVE8) {
                bool clean;
                const unsigned byte = gg_a8_block_byte<V>(v, clean);
                unsigned w[V / 4];
                gg_a8_encode<V>(v, byte, clean, w);
                if (in) {
                    const size_t row = (size_t)p.b * a.N + n;
                    gg_a8_st_codes<V>(a.codes_out + row * Cp + p.c, w);
                    if (p.c % GG_A8_BLOCK == 0) a.scales_out[row * nb + p.c / GG_A8_BLOCK] = (uint8_t)byte;
                }
            }
        }
    }
}

// mean and rstd of a group from the sums of its channels (all on the same base)
__device__ __forceinline__ void finish_stats(double s, double q, double base, double m, float eps, double *mean, double *rstd)
{
    m = m < 1.0 ? 1.0 : m;
    const double e = s / m;
    double var = q / m - e * e;
    var = var < 0.0 ? 0.0 : var;           // (NaN stays NaN)
    *mean = base + e;
    *rstd = 1.0 / sqrt(var + (double)eps);
}

// second pass: y of the rows r0 <= n < r1; rows from `count` on are zero
template <class T, int ACT>
__device__ __forceinline__ void rows_apply(const Args &a, const Lay &l, const Pos<GGRowT<T>::V> &p, long long r0, long long r1,
                                           long long count, const Chan (&k)[GGRowT<T>::V])
{
    constexpr int V = GGRowT<T>::V;
    const T *x = (const T *)a.x + (size_t)p.b * a.xb;
    T *y = (T *)a.y + (size_t)p.b * a.N * a.C;
    if (!p.on) return;
    const GGCol<T> col(p.c, a.C);
    const long long rv = r1 < count ? r1 : count;          // rows with values
    long long n0 = r0 + p.tr;
    for (; n0 < rv; n0 += (long long)l.rpb * UNROLL) {
        GGChunk<T> r[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            const long long n = n0 + (long long)u * l.rpb;
            r[u].load(x + (size_t)(n < rv ? n : n0) * a.xn, col, a.C);
        }
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            const long long n = n0 + (long long)u * l.rpb;
            if (n >= r1) continue;
            float v[V], o[V];
            r[u].align(col);
            r[u].get(v);
#pragma unroll
            for (int i = 0; i < V; i++) o[i] = n < rv ? act_of<ACT, T>(fmaf(dev_of(k[i], v[i]), k[i].a, k[i].beta)) : 0.f;
            gg_st_chunk(y + (size_t)n * a.C, p.c, a.C, o, a.past);
        }
    }
    float z[V];
#pragma unroll
    for (int i = 0; i < V; i++) z[i] = 0.f;
    for (; n0 < r1; n0 += l.rpb) gg_st_chunk(y + (size_t)n0 * a.C, p.c, a.C, z, a.past);
}

// x^ of one chunk as it stands in memory: the input itself or its 8-bit form (whose rows are whole chunks)
template <class T, bool Q8> struct Xhat {
    typename std::conditional<Q8, GGCodes<GGRowT<T>::V>, GGChunk<T>>::type r;
    __device__ __forceinline__ void load(const Args &a, const Pos<GGRowT<T>::V> &p, const GGCol<T> &col, long long n)
    {
        if constexpr (Q8) {
            const int Cp = gg_a8_cp(a.C);
            const size_t row = (size_t)p.b * a.N + n;
            r.load(a.codes + row * Cp + p.c, a.scales + row * (Cp / GG_A8_BLOCK) + p.c / GG_A8_BLOCK);
        } else {
            r.load((const T *)a.x + (size_t)p.b * a.xb + (size_t)n * a.xn, col, a.C);
        }
    }
    __device__ __forceinline__ void get(const GGCol<T> &col, float (&v)[GGRowT<T>::V])
    {
        if constexpr (!Q8) r.align(col);
        r.get(v);
    }
};

// g = dy act'(t) of one value
template <int ACT, class T> __device__ __forceinline__ float gate(const Chan &k, float dy, float d, float x)
{
    if constexpr (ACT == GRIDGCN_ACT_NONE) return dy;
    if constexpr (ACT == GRIDGCN_ACT_RELU) return __uint_as_float(__float_as_uint(x) ^ k.flip) > k.thr ? dy : 0.f;
    return dy * act_grad<ACT, T>(fmaf(d, k.a, k.beta));
}

// backward, first pass over r0 <= n < r1 (all below count): s = sums of g and g * xh per channel
template <class T, int ACT, bool Q8>
__device__ __forceinline__ void rows_bwd_sums(const Args &a, const Lay &l, const Pos<GGRowT<T>::V> &p, long long r0, long long r1,
                                              const Chan (&k)[GGRowT<T>::V], double (&s)[GGRowT<T>::V][2])
{
    constexpr int V = GGRowT<T>::V;
    const T *dy = (const T *)a.dy + (size_t)p.b * a.gb;
#pragma unroll
    for (int i = 0; i < V; i++) s[i][0] = s[i][1] = 0.0;
    if (!p.on) return;
    const GGCol<T> col(p.c, a.C);
    for (long long n0 = r0 + p.tr; n0 < r1; n0 += (long long)l.rpb * UNROLL) {
        GGChunk<T> re[UNROLL];
        Xhat<T, Q8> rx[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            const long long n = n0 + (long long)u * l.rpb, nn = n < r1 ? n : n0;
            re[u].load(dy + (size_t)nn * a.gn, col, a.C);
            rx[u].load(a, p, col, nn);
        }
        float s0[V], s1[V];
#pragma unroll
        for (int i = 0; i < V; i++) s0[i] = s1[i] = 0.f;
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            if (n0 + (long long)u * l.rpb >= r1) continue;
            float e[V], v[V];
            re[u].align(col);
            re[u].get(e);
            rx[u].get(col, v);
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float d = dev_of(k[i], v[i]);
                const float g = gate<ACT, T>(k[i], e[i], d, v[i]);
                s0[i] += g;
                s1[i] = fmaf(g, d * k[i].rstd, s1[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < V; i++) {
            s[i][0] += (double)s0[i];
            s[i][1] += (double)s1[i];
        }
    }
}

// backward, second pass: dx of the rows r0 <= n < r1; rows from `count` on are zero
template <class T, int ACT, bool Q8>
__device__ __forceinline__ void rows_bwd_dx(const Args &a, const Lay &l, const Pos<GGRowT<T>::V> &p, long long r0, long long r1,
                                            long long count, const Chan (&k)[GGRowT<T>::V], const float2 (&f)[GGRowT<T>::V])
{
    constexpr int V = GGRowT<T>::V;
    const T *dy = (const T *)a.dy + (size_t)p.b * a.gb;
    T *dx = (T *)a.y + (size_t)p.b * a.N * a.C;
    if (!p.on) return;
    const GGCol<T> col(p.c, a.C);
    const long long rv = r1 < count ? r1 : count;          // rows with values
    long long n0 = r0 + p.tr;
    for (; n0 < rv; n0 += (long long)l.rpb * UNROLL) {
        GGChunk<T> re[UNROLL];
        Xhat<T, Q8> rx[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            const long long n = n0 + (long long)u * l.rpb, nn = n < rv ? n : n0;
            re[u].load(dy + (size_t)nn * a.gn, col, a.C);
            rx[u].load(a, p, col, nn);
        }
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            const long long n = n0 + (long long)u * l.rpb;
            if (n >= r1) continue;
            float e[V], v[V], o[V];
            re[u].align(col);
            re[u].get(e);
            rx[u].get(col, v);
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float d = dev_of(k[i], v[i]);
                const float g = gate<ACT, T>(k[i], e[i], d, v[i]);
                o[i] = n < rv ? fmaf(k[i].a, g, -fmaf(d * k[i].rstd, f[i].y, f[i].x)) : 0.f;
            }
            gg_st_chunk(dx + (size_t)n * a.C, p.c, a.C, o, a.past);
        }
    }
    float z[V];
#pragma unroll
    for (int i = 0; i < V; i++) z[i] = 0.f;
    for (; n0 < r1; n0 += l.rpb) gg_st_chunk(dx + (size_t)n0 * a.C, p.c, a.C, z, a.past);
}

// Average (least) of ten calls, us.  8 x 81920 x 128 fp32 (336 MB a tensor), SiLU: stats 67 (60), apply 117 (114), backward sums 116 (112), dx
// 180 (176): memory, at 5.0 - 5.8 TB/s; the forward reads x twice, the backward x and dy twice.  16 x 65536 x 64 bf16, GELU, x kept in 8
// bits: stats 48 (46, the codes written), apply 55 (53), sums 78 (74), dx 76 (73): the last three bound by arithmetic (GELU and the codes
// keep the vector pipes busy all the time).
// ---- many rows: pass, small launch, pass ----------------------------------------------------------------------------
template <class T, bool SAVE8>
__global__ __launch_bounds__(THREADS, 4) void gg_k_gn_stats(Args a, Lay l)
{
    constexpr int V = GGRowT<T>::V;
    __shared__ double red[THREADS * V * 2];
    const Pos<V> p(l, blockIdx.y * l.tpr, blockIdx.z);
    const long long count = count_of(a, p.b);
    const long long r0 = (long long)blockIdx.x * a.rpc;
    const long long r1 = r0 + a.rpc < count ? r0 + a.rpc : count;
    double s[V][2], base[V];
    rows_stats<T, SAVE8>(a, l, p, r0, r1, s, base);
    reduce_rows<V, THREADS>(red, l, p.tr, (int)threadIdx.x % l.tpr, s);
    double *out = a.part + ((size_t)p.b * a.chunks + blockIdx.x) * a.C * 2;
    const int c0 = blockIdx.y * l.tpr * V;
    for (int j = threadIdx.x; j < l.tpr * V * 2; j += THREADS)
        if (c0 + j / 2 < a.C) out[(size_t)c0 * 2 + j] = red[j];
}

// sums over the chunks of one cloud for the n channels from c0 on: f(channel, sum 0, sum 1), each channel once, by the thread
// that owns it.  red: LDS [THREADS * 2].  Every thread calls.
template <class F> __device__ __forceinline__ void sum_chunks(const Args &a, int b, int c0, int n, double *red, F f)
{
    const int cw = n < THREADS ? n : THREADS, nl = THREADS / cw;
    const int cl = threadIdx.x % cw, kl = threadIdx.x / cw;       // (kl >= nl: idle)
    for (int o = 0; o < n; o += cw) {
        double s0 = 0.0, s1 = 0.0;
        if (kl < nl && o + cl < n) {
            const f64x2 *p = (const f64x2 *)a.part + (size_t)b * a.chunks * a.C + c0 + o + cl;
            constexpr int U = 8;           // (loads in flight: with one at a time a group of 131 channels took 66 us, not 7)
            for (int k = kl; k < a.chunks; k += nl * U) {
                f64x2 v[U];
#pragma unroll
                for (int u = 0; u < U; u++) v[u] = p[(size_t)(k + u * nl < a.chunks ? k + u * nl : k) * a.C];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (k + u * nl >= a.chunks) continue;
                    s0 += v[u].x;
                    s1 += v[u].y;
                }
            }
        }
        red[threadIdx.x * 2] = s0;
        red[threadIdx.x * 2 + 1] = s1;
        for (int d = 128; d > 0; d /= 2) {          // (nl <= 256)
            if (d >= nl) continue;
            __syncthreads();
            if (kl < d && kl + d < nl) {
                s0 += red[(threadIdx.x + d * cw) * 2];
                s1 += red[(threadIdx.x + d * cw) * 2 + 1];
                red[threadIdx.x * 2] = s0;
                red[threadIdx.x * 2 + 1] = s1;
            }
        }
        if (kl == 0 && o + cl < n) f(c0 + o + cl, s0, s1);
        __syncthreads();
    }
}

// the workgroup's sums of (s, q), in one order; every thread calls, all get them
__device__ __forceinline__ void sum_block(double *red, double &s, double &q)
{
    red[threadIdx.x * 2] = s;
    red[threadIdx.x * 2 + 1] = q;
    for (int d = THREADS / 2; d > 0; d /= 2) {
        __syncthreads();
        if ((int)threadIdx.x < d) {
            red[threadIdx.x * 2] += red[(threadIdx.x + d) * 2];
            red[threadIdx.x * 2 + 1] += red[(threadIdx.x + d) * 2 + 1];
        }
    }
    __syncthreads();
    s = red[0];
    q = red[1];
}

// for each of ng groups of cg values in LDS: the sums of get(value index) -> (s, q), then done(group, s, q) by one thread.
// Many channels: a wave per group; few: a thread per group.
template <int NT, class G, class D> __device__ __forceinline__ void for_groups(int cg, int ng, G get, D done)
{
    if (cg >= 32) {
        const int lane = threadIdx.x & 63;
        for (int j = threadIdx.x >> 6; j < ng; j += NT / 64) {
            double s = 0.0, q = 0.0;
            for (int c = lane; c < cg; c += 64) get(j * cg + c, s, q);
#pragma unroll
            for (int d = 32; d > 0; d /= 2) {
                s += __shfl_xor(s, d);
                q += __shfl_xor(q, d);
            }
            if (lane == 0) done(j, s, q);
        }
    } else {
        for (int j = threadIdx.x; j < ng; j += NT) {
            double s = 0.0, q = 0.0;
            for (int c = 0; c < cg; c++) get(j * cg + c, s, q);
            done(j, s, q);
        }
    }
}

template <class T>
__global__ __launch_bounds__(THREADS) void gg_k_gn_stats_fin(Args a)
{
    __shared__ double red[THREADS * 2];
    const int g = blockIdx.x, b = blockIdx.y;
    double s = 0.0, q = 0.0;
    sum_chunks(a, b, g * a.cg, a.cg, red, [&](int, double s0, double s1) { s += s0; q += s1; });
    sum_block(red, s, q);
    if (threadIdx.x == 0) {
        const long long count = count_of(a, b);
        const double base = count > 0 ? (double)GGRowT<T>::get((const T *)a.x + (size_t)b * a.xb + g * a.cg) : 0.0;
        double *o = a.stats + ((size_t)b * a.G + g) * 2;
        finish_stats(s, q, base, (double)count * a.cg, a.eps, o, o + 1);
    }
}

template <class T, int ACT>
__global__ __launch_bounds__(THREADS) void gg_k_gn_apply(Args a, Lay l)
{
    constexpr int V = GGRowT<T>::V;
    const Pos<V> p(l, blockIdx.y * l.tpr, a.B - 1 - (int)blockIdx.z);
    // (last rows first: they are what the pass before left in the caches)
    const long long r0 = (long long)(gridDim.x - 1 - blockIdx.x) * a.rpc;
    const long long r1 = r0 + a.rpc < a.N ? r0 + a.rpc : a.N;
    Chan k[V];
    chans<ACT, false, V>(a, p, k);
    rows_apply<T, ACT>(a, l, p, r0, r1, count_of(a, p.b), k);
}

template <class T, int ACT, bool Q8>
__global__ __launch_bounds__(THREADS, sizeof(T) == 4 ? 4 : 3) void gg_k_gn_bwd_sums(Args a, Lay l)
{
    constexpr int V = GGRowT<T>::V;
    __shared__ double red[THREADS * V * 2];
    const Pos<V> p(l, blockIdx.y * l.tpr, blockIdx.z);
    const long long count = count_of(a, p.b);
    const long long r0 = (long long)blockIdx.x * a.rpc;
    const long long r1 = r0 + a.rpc < count ? r0 + a.rpc : count;
    Chan k[V];
    chans<ACT, true, V>(a, p, k);
    double s[V][2];
    rows_bwd_sums<T, ACT, Q8>(a, l, p, r0, r1, k, s);
    reduce_rows<V, THREADS>(red, l, p.tr, (int)threadIdx.x % l.tpr, s);
    double *out = a.part + ((size_t)p.b * a.chunks + blockIdx.x) * a.C * 2;
    const int c0 = blockIdx.y * l.tpr * V;
    for (int j = threadIdx.x; j < l.tpr * V * 2; j += THREADS)
        if (c0 + j / 2 < a.C) out[(size_t)c0 * 2 + j] = red[j];
}

// What dx needs of a group, from the sums of gamma g and gamma g xh over it:  dx = (rstd gamma) g - (rstd S1 + xh rstd S2).  (One
// factor rstd each: its square leaves float32 where the standard deviation is beyond 1e19 or below 1e-19.)
__device__ __forceinline__ float2 coef_of(const Args &a, int b, int g, double s1, double s2)
{
    const long long count = count_of(a, b);
    if (count < 1) return make_float2(0.f, 0.f);
    const double m = (double)count * a.cg, rstd = a.stats[((size_t)b * a.G + g) * 2 + 1];
    return make_float2((float)(rstd * s1 / m), (float)(rstd * s2 / m));
}

__global__ __launch_bounds__(THREADS) void gg_k_gn_bwd_fin(Args a)
{
    __shared__ double red[THREADS * 2];
    const int g = blockIdx.x, b = blockIdx.y;
    double s = 0.0, q = 0.0;
    sum_chunks(a, b, g * a.cg, a.cg, red, [&](int c, double s0, double s1) {
        double *t = a.tot + ((size_t)b * a.C + c) * 2;
        t[0] = s0;
        t[1] = s1;
        const double w = (double)gg_ld_param(a.gamma, a.ptype, c, 1.f);
        s += w * s0;
        q += w * s1;
    });
    sum_block(red, s, q);
    if (threadIdx.x == 0) a.coef[(size_t)b * a.G + g] = coef_of(a, b, g, s, q);
}

// dgamma, dbeta of the channels c0 <= c < c1 (at most PAR of them): the clouds' totals, PARL lanes' strided sums, then the lanes.
// red: LDS [THREADS * 2]; every thread calls.
constexpr int PAR = 16, PARL = THREADS / PAR;
__device__ __forceinline__ void params_of(const Args &a, int c0, int c1, double *red)
{
    const int c = c0 + (int)threadIdx.x % PAR, k0 = (int)threadIdx.x / PAR;
    double db = 0.0, dg = 0.0;
    if (c < c1) {
        for (int b = k0; b < a.B; b += PARL) {
            const double *t = a.tot + ((size_t)b * a.C + c) * 2;
            db += t[0];
            dg += t[1];
        }
    }
    red[threadIdx.x * 2] = db;
    red[threadIdx.x * 2 + 1] = dg;
    __syncthreads();
    if (k0 == 0 && c < c1) {
        for (int k = 1; k < PARL; k++) {
            db += red[(threadIdx.x + k * PAR) * 2];
            dg += red[(threadIdx.x + k * PAR) * 2 + 1];
        }
        if (a.dbeta) gg_st_param(a.dbeta, a.ptype, c, (float)db);
        if (a.dgamma) gg_st_param(a.dgamma, a.ptype, c, (float)dg);
    }
    __syncthreads();
}

// (16-bit rows, eight channels a thread: three waves, as at four their constants spill.  Backward of 16 x 65536 x 64 bf16 from codes,
// GELU 150 | 170 us, ReLU 114 | 154)
template <class T, int ACT, bool Q8>
__global__ __launch_bounds__(THREADS, sizeof(T) == 4 ? 4 : 3) void gg_k_gn_bwd_dx(Args a, Lay l)
{
    constexpr int V = GGRowT<T>::V;
    // (the workgroups take some channels' parameters along)
    __shared__ double red[THREADS * 2];
    if (a.dgamma || a.dbeta) {
        const long long nth = ((long long)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
        const long long all = (long long)gridDim.z * gridDim.y * gridDim.x;
        for (long long c = nth * PAR; c < a.C; c += all * PAR) params_of(a, (int)c, c + PAR < a.C ? (int)c + PAR : a.C, red);
    }
    const Pos<V> p(l, blockIdx.y * l.tpr, a.B - 1 - (int)blockIdx.z);
    const long long r0 = (long long)(gridDim.x - 1 - blockIdx.x) * a.rpc;
    const long long r1 = r0 + a.rpc < a.N ? r0 + a.rpc : a.N;
    Chan k[V];
    chans<ACT, true, V>(a, p, k);
    float2 f[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int c = p.c + i < a.C ? p.c + i : a.C - 1;
        f[i] = a.coef[(size_t)p.b * a.G + c / a.cg];
    }
    rows_bwd_dx<T, ACT, Q8>(a, l, p, r0, r1, count_of(a, p.b), k, f);
}

__global__ __launch_bounds__(THREADS) void gg_k_gn_params(Args a)
{
    __shared__ double red[THREADS * 2];
    const int c0 = blockIdx.x * PAR;
    params_of(a, c0, c0 + PAR < a.C ? c0 + PAR : a.C, red);
}

// ---- few rows: one launch, a workgroup = whole groups of one cloud (l.nq chunks from channel slab * slab_c on), every value read
// once and kept in registers: the time is one trip to memory, a reduction and the stores: 16 ragged clouds of 1024 rows, 128
// channels, fp32, average (least) of ten: forward with the codes 19 us (17), backward 15 (14); 32 rows of 512: 8 (7) and 10 (9) --------
template <class T, int ACT, bool SAVE8>
__global__ __launch_bounds__(FEW) void gg_k_gn_small(Args a, Lay l, int slab_c)
{
    constexpr int V = GGRowT<T>::V, K = KEEP<T>;
    __shared__ double red[FEW * V * 2];
    const int c0 = blockIdx.x * slab_c, c1 = c0 + slab_c < a.C ? c0 + slab_c : a.C;
    Pos<V> p(l, c0 / V, blockIdx.y);
    p.on = p.tr < l.rpb && p.c < (SAVE8 && c1 == a.C ? gg_a8_cp(a.C) : c1);
    const long long count = count_of(a, p.b);
    const T *x = (const T *)a.x + (size_t)p.b * a.xb;
    const GGCol<T> col(p.on ? p.c : 0, a.C);
    GGChunk<T> r[K];
#pragma unroll
    for (int u = 0; u < K; u++) {
        if ((long long)u * l.rpb >= a.N) continue;
        const long long n = (long long)u * l.rpb + p.tr;
        r[u].load(x + (size_t)(n < count ? n : 0) * a.xn, col, a.C);               // (rows past the end: in no sum, not stored)
    }
    double s[V][2], base[V];
    base_of<T>(a, p, x, base);
#pragma unroll
    for (int i = 0; i < V; i++) s[i][0] = s[i][1] = 0.0;
    const int Cp = gg_a8_cp(a.C), nb = Cp / GG_A8_BLOCK;
#pragma unroll
    for (int u = 0; u < K; u++) {
        const long long n = (long long)u * l.rpb + p.tr;
        const bool in = p.on && n < count;
        if ((long long)u * l.rpb >= a.N) continue;
        float v[V];
        r[u].align(col);
        r[u].get(v);
        if (in) {
#pragma unroll
            for (int i = 0; i < V; i++) {
                const double d = (double)v[i] - base[i];
                s[i][0] += d;
                s[i][1] = fma(d, d, s[i][1]);
            }
        }
        if constexpr (SAVE8) {
            bool clean;
            const unsigned byte = gg_a8_block_byte<V>(v, clean);
            unsigned w[V / 4];
            gg_a8_encode<V>(v, byte, clean, w);
            if (in) {
                const size_t row = (size_t)p.b * a.N + n;
                gg_a8_st_codes<V>(a.codes_out + row * Cp + p.c, w);
                if (p.c % GG_A8_BLOCK == 0) a.scales_out[row * nb + p.c / GG_A8_BLOCK] = (uint8_t)byte;
            }
        }
    }
    reduce_rows<V, FEW>(red, l, p.tr, (int)threadIdx.x % l.tpr, s);
    // (a group's statistics take the place of its first channel's sums, once the group is summed)
    for_groups<FEW>(a.cg, (c1 - c0) / a.cg, [&](int c, double &t, double &q) { t += red[c * 2]; q += red[c * 2 + 1]; },
                    [&](int j, double t, double q) {
        const int g = c0 / a.cg + j;
        const double b0 = count > 0 ? (double)GGRowT<T>::get(x + g * a.cg) : 0.0;
        double mean, rstd;
        finish_stats(t, q, b0, (double)count * a.cg, a.eps, &mean, &rstd);
        red[j * a.cg * 2] = mean;
        red[j * a.cg * 2 + 1] = rstd;
        if (a.stats) {
            a.stats[((size_t)p.b * a.G + g) * 2] = mean;
            a.stats[((size_t)p.b * a.G + g) * 2 + 1] = rstd;
        }
    });
    __syncthreads();
    if (!p.on || p.c >= c1) return;
    Chan k[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int c = p.c + i < c1 ? p.c + i : c1 - 1;
        const double *st = red + ((c - c0) / a.cg) * a.cg * 2;
        k[i] = chan_of<ACT, false>(a, st[0], st[1], c);
    }
    T *y = (T *)a.y + (size_t)p.b * a.N * a.C;
#pragma unroll
    for (int u = 0; u < K; u++) {
        const long long n = (long long)u * l.rpb + p.tr;
        if (n >= a.N) continue;
        float v[V], o[V];
        r[u].get(v);
#pragma unroll
        for (int i = 0; i < V; i++) o[i] = n < count ? act_of<ACT, T>(fmaf(dev_of(k[i], v[i]), k[i].a, k[i].beta)) : 0.f;
        gg_st_chunk(y + (size_t)n * a.C, p.c, a.C, o, false);
    }
}

template <class T, int ACT, bool Q8>
__global__ __launch_bounds__(FEW) void gg_k_gn_small_bwd(Args a, Lay l, int slab_c)
{
    constexpr int V = GGRowT<T>::V, K = KEEP<T>;
    __shared__ double red[FEW * V * 2];
    const int c0 = blockIdx.x * slab_c, c1 = c0 + slab_c < a.C ? c0 + slab_c : a.C;
    Pos<V> p(l, c0 / V, blockIdx.y);
    p.on = p.tr < l.rpb && p.c < c1;
    const long long count = count_of(a, p.b);
    const T *dy = (const T *)a.dy + (size_t)p.b * a.gb;
    Pos<V> at = p;
    if (!p.on) at.c = c0;
    const GGCol<T> col(at.c, a.C);
    GGChunk<T> rg[K];
    Xhat<T, Q8> rx[K];
#pragma unroll
    for (int u = 0; u < K; u++) {
        if ((long long)u * l.rpb >= a.N) continue;
        const long long n = (long long)u * l.rpb + p.tr, nn = n < count ? n : 0;    // (rows past the end: in no sum, not stored)
        rg[u].load(dy + (size_t)nn * a.gn, col, a.C);
        rx[u].load(a, at, col, nn);
    }
    Chan k[V];
    chans<ACT, true, V>(a, p, k);
    double s[V][2];
#pragma unroll
    for (int i = 0; i < V; i++) s[i][0] = s[i][1] = 0.0;
#pragma unroll
    for (int u = 0; u < K; u++) {
        if (!(p.on && (long long)u * l.rpb + p.tr < count)) continue;
        float e[V], v[V];
        rg[u].align(col);
        rg[u].get(e);
        rx[u].get(col, v);
#pragma unroll
        for (int i = 0; i < V; i++) {
            const float d = dev_of(k[i], v[i]);
            const float g = gate<ACT, T>(k[i], e[i], d, v[i]);
            s[i][0] += (double)g;
            s[i][1] = fma((double)g, (double)(d * k[i].rstd), s[i][1]);
        }
    }
    reduce_rows<V, FEW>(red, l, p.tr, (int)threadIdx.x % l.tpr, s);
    for (int j = threadIdx.x; j < c1 - c0; j += FEW) {
        const int c = c0 + j;
        const double db = red[j * 2], dg = red[j * 2 + 1];
        if (a.B == 1) {
            if (a.dbeta) gg_st_param(a.dbeta, a.ptype, c, (float)db);
            if (a.dgamma) gg_st_param(a.dgamma, a.ptype, c, (float)dg);
        } else {
            a.tot[((size_t)p.b * a.C + c) * 2] = db;
            a.tot[((size_t)p.b * a.C + c) * 2 + 1] = dg;
        }
    }
    if (!a.y) return;
    __syncthreads();
    // (a group's coefficients take the place of its first channel's sums)
    for_groups<FEW>(a.cg, (c1 - c0) / a.cg, [&](int c, double &t, double &q) {
        const double w = (double)gg_ld_param(a.gamma, a.ptype, c0 + c, 1.f);
        t += w * red[c * 2];
        q += w * red[c * 2 + 1];
    }, [&](int j, double t, double q) {
        const float2 f = coef_of(a, p.b, c0 / a.cg + j, t, q);
        red[j * a.cg * 2] = (double)f.x;
        red[j * a.cg * 2 + 1] = (double)f.y;
    });
    __syncthreads();
    if (!p.on) return;
    float2 f[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int c = p.c + i < c1 ? p.c + i : c1 - 1;
        const double *q = red + ((c - c0) / a.cg) * a.cg * 2;
        f[i] = make_float2((float)q[0], (float)q[1]);
    }
    T *dx = (T *)a.y + (size_t)p.b * a.N * a.C;
#pragma unroll
    for (int u = 0; u < K; u++) {
        const long long n = (long long)u * l.rpb + p.tr;
        if (n >= a.N) continue;
        float e[V], v[V], o[V];
        rg[u].get(e);
        rx[u].r.get(v);
#pragma unroll
        for (int i = 0; i < V; i++) {
            const float d = dev_of(k[i], v[i]);
            const float g = gate<ACT, T>(k[i], e[i], d, v[i]);
            o[i] = n < count ? fmaf(k[i].a, g, -fmaf(d * k[i].rstd, f[i].y, f[i].x)) : 0.f;
        }
        gg_st_chunk(dx + (size_t)n * a.C, p.c, a.C, o, false);
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------
struct Plan {
    bool small;
    int slab_c, slabs;      // small: channels of a workgroup
    Lay l;                  // of a pass (small: of a slab)
    int nq;                 // chunks of a row
    long long rpc;
    int chunks;
    size_t off_part, off_tot, off_coef, off_stats, bytes;
};

long long gcd_ll(long long a, long long b) { return b ? gcd_ll(b, a % b) : a; }

// One launch wherever a workgroup's registers hold the rows of at least 64 bytes' worth of whole groups (32768 values);
// rows beyond that: two passes.  Measured (forward + backward, us; one launch | two passes):  fp32, 32 groups of 128 channels,
// 16 x 1024 rows 27 | 35,  16 x 2048 rows (the most that fit) 41 | 48,  64 x 2048 rows 112 | 112;  one group, 256 x 256 rows 49 | 72;
// 256 x 1 rows of 512 channels 24 | 58;  bf16 16 x 1024 rows 33 | 38.
Plan plan_of(int B, long long N, int C, int G, int dtype, bool save8, bool stats, bool backward)
{
    Plan p = {};
    const int V = dtype == GRIDGCN_F32 ? 4 : 8, cg = C / G, keep = dtype == GRIDGCN_F32 ? KEEP<float> : KEEP<gg_bf16>;
    p.nq = save8 ? gg_a8_cp(C) / V : (C + V - 1) / V;
    // whole groups, whole chunks (whole blocks of the 8-bit form)
    const long long unit = save8 ? GG_A8_BLOCK : V;
    long long slab = (long long)cg / gcd_ll(cg, unit) * unit;
    const long long least = 64 / (dtype == GRIDGCN_F32 ? 4 : 2);
    if (slab < least) slab = (least + slab - 1) / slab * slab;
    if (slab > C) slab = C;
    auto quads = [&](long long s) { return save8 ? (s + GG_A8_BLOCK - 1) / GG_A8_BLOCK * (GG_A8_BLOCK / V) : (s + V - 1) / V; };
    auto fits = [&](long long s) { return quads(s) <= FEW && N <= (long long)keep * (FEW / quads(s)); };
    p.small = fits(slab);
    if (p.small) {
        // short rows are taken whole: a workgroup for 16 channels of one row would be all start-up (32 rows of 512 fp32 channels,
        // forward + backward 18 us, not 60; 256 rows 24, not 420)
        while (slab < C && N * slab * 2 <= 2048 && fits(slab * 2)) slab *= 2;
        if (slab > C) slab = C;
        p.slab_c = (int)slab;
        p.slabs = (int)((C + slab - 1) / slab);
        p.l = lay_of((int)quads(slab), FEW);
    } else {
        p.l = lay_of(p.nq);
        const long long slabs = (p.nq + p.l.tpr - 1) / p.l.tpr, step = (long long)p.l.rpb * UNROLL;
        long long want = (2048 + B * slabs - 1) / (B * slabs);
        long long chunks = (N + step - 1) / step;
        if (chunks > want) chunks = want;
        p.rpc = ((N + chunks - 1) / chunks + step - 1) / step * step;
        p.chunks = (int)((N + p.rpc - 1) / p.rpc);
    }
    size_t o = 0;
    auto take = [&o](size_t n) { const size_t at = o; o += (n + 255) & ~(size_t)255; return at; };
    p.off_part = take(p.small ? 0 : (size_t)B * p.chunks * C * 16);
    p.off_tot = take(backward && (!p.small || B > 1) ? (size_t)B * C * 16 : 0);
    p.off_coef = take(backward && !p.small ? (size_t)B * G * 8 : 0);
    p.off_stats = take(backward || stats || p.small ? 0 : (size_t)B * G * 16);
    p.bytes = o;
    return p;
}

// f((T *)nullptr) for the type
template <class F> int with_type(int dtype, F f)
{
    if (dtype == GRIDGCN_F32) { f((float *)nullptr); return 0; }
    if (dtype == GRIDGCN_BF16) { f((gg_bf16 *)nullptr); return 0; }
    if (dtype == GRIDGCN_F16) { f((gg_f16 *)nullptr); return 0; }
    return GRIDGCN_EINVAL;
}

template <class T, int ACT, bool SAVE8> void launch_fwd(Args &a, const Plan &p, hipStream_t st)
{
    if (p.small) {
        gg_k_gn_small<T, ACT, SAVE8><<<dim3(p.slabs, a.B), FEW, 0, st>>>(a, p.l, p.slab_c);
        return;
    }
    const unsigned slabs = (p.nq + p.l.tpr - 1) / p.l.tpr;
    gg_k_gn_stats<T, SAVE8><<<dim3(p.chunks, slabs, a.B), THREADS, 0, st>>>(a, p.l);
    gg_k_gn_stats_fin<T><<<dim3(a.G, a.B), THREADS, 0, st>>>(a);
    const Lay l = lay_of((a.C + GGRowT<T>::V - 1) / GGRowT<T>::V);
    const unsigned sl = (l.nq + l.tpr - 1) / l.tpr;
    gg_k_gn_apply<T, ACT><<<dim3(p.chunks, sl, a.B), THREADS, 0, st>>>(a, l);
}

template <class T, int ACT, bool Q8> void launch_bwd(Args &a, const Plan &p, hipStream_t st)
{
    if (p.small) {
        gg_k_gn_small_bwd<T, ACT, Q8><<<dim3(p.slabs, a.B), FEW, 0, st>>>(a, p.l, p.slab_c);
        if (a.B > 1 && (a.dgamma || a.dbeta)) gg_k_gn_params<<<dim3((a.C + PAR - 1) / PAR), THREADS, 0, st>>>(a);
        return;
    }
    const unsigned slabs = (p.l.nq + p.l.tpr - 1) / p.l.tpr;
    gg_k_gn_bwd_sums<T, ACT, Q8><<<dim3(p.chunks, slabs, a.B), THREADS, 0, st>>>(a, p.l);
    gg_k_gn_bwd_fin<<<dim3(a.G, a.B), THREADS, 0, st>>>(a);
    if (a.y) gg_k_gn_bwd_dx<T, ACT, Q8><<<dim3(p.chunks, slabs, a.B), THREADS, 0, st>>>(a, p.l);
    else gg_k_gn_params<<<dim3((a.C + PAR - 1) / PAR), THREADS, 0, st>>>(a);
}

template <class T, bool Q> void fwd_act(Args &a, const Plan &p, int act, hipStream_t st)
{
    if (act == GRIDGCN_ACT_NONE) launch_fwd<T, GRIDGCN_ACT_NONE, Q>(a, p, st);
    else if (act == GRIDGCN_ACT_RELU) launch_fwd<T, GRIDGCN_ACT_RELU, Q>(a, p, st);
    else if (act == GRIDGCN_ACT_SILU) launch_fwd<T, GRIDGCN_ACT_SILU, Q>(a, p, st);
    else launch_fwd<T, GRIDGCN_ACT_GELU, Q>(a, p, st);
}
template <class T, bool Q> void bwd_act(Args &a, const Plan &p, int act, hipStream_t st)
{
    if (act == GRIDGCN_ACT_NONE) launch_bwd<T, GRIDGCN_ACT_NONE, Q>(a, p, st);
    else if (act == GRIDGCN_ACT_RELU) launch_bwd<T, GRIDGCN_ACT_RELU, Q>(a, p, st);
    else if (act == GRIDGCN_ACT_SILU) launch_bwd<T, GRIDGCN_ACT_SILU, Q>(a, p, st);
    else launch_bwd<T, GRIDGCN_ACT_GELU, Q>(a, p, st);
}

bool sizes_ok(int B, long long N, int C, int G)
{
    // (grid.y and grid.z are 16-bit)
    return B >= 1 && B <= 65535 && N >= 1 && C >= 1 && C <= GRIDGCN_GN_MAX_C && G >= 1 && G <= C && C % G == 0;
}
bool type_ok(int t) { return t == GRIDGCN_F32 || t == GRIDGCN_BF16 || t == GRIDGCN_F16; }
}  // namespace

extern "C" {

int gridgcn_group_norm_act_workspace_bytes(int B, long long N, int C, int G, int dtype, int save8, int stats, int backward,
                                           size_t *bytes)
{
    if (!bytes || !sizes_ok(B, N, C, G) || !type_ok(dtype)) return GRIDGCN_EINVAL;
    *bytes = plan_of(B, N, C, G, dtype, save8 && !backward, stats != 0, backward != 0).bytes;
    return GRIDGCN_OK;
}

int gridgcn_group_norm_act_fwd(const void *x, int dtype, int B, long long N, int C, long long ldb, long long ldn, int G,
                               const void *gamma, const void *beta, int ptype, const int32_t *counts, float eps, int act,
                               void *y, double *stats, uint8_t *codes, uint8_t *scales, void *ws, size_t ws_bytes, void *stream)
{
    if (!x || !y || !sizes_ok(B, N, C, G) || !type_ok(dtype) || !type_ok(ptype) || ldn < C || ldn > GRIDGCN_MAX_LD || (B > 1 && ldb < 0) ||
        !(eps >= 0.f) || act < GRIDGCN_ACT_NONE || act > GRIDGCN_ACT_GELU || !codes != !scales || ((uintptr_t)codes & 15))
        return GRIDGCN_EINVAL;
    const Plan p = plan_of(B, N, C, G, dtype, codes != nullptr, stats != nullptr, false);
    if (p.bytes && (!ws || ws_bytes < p.bytes || ((uintptr_t)ws & 15))) return GRIDGCN_EWORKSPACE;
    Args a = {};
    a.x = x; a.y = y; a.N = N; a.xb = ldb; a.xn = ldn; a.B = B; a.C = C; a.G = G; a.cg = C / G; a.ptype = ptype;
    a.gamma = gamma; a.beta = beta; a.counts = counts; a.eps = eps; a.codes_out = codes; a.scales_out = scales;
    a.part = (double *)((char *)ws + p.off_part);
    a.stats = stats || p.small ? stats : (double *)((char *)ws + p.off_stats);
    a.rpc = p.rpc; a.chunks = p.chunks; a.past = gg_past_caches(B * N, C, dtype);
    const hipStream_t st = (hipStream_t)stream;
    const int rc = with_type(dtype, [&](auto *t) {
        typedef typename std::remove_pointer<decltype(t)>::type T;
        if (codes) fwd_act<T, true>(a, p, act, st);
        else fwd_act<T, false>(a, p, act, st);
    });
    if (rc) return rc;
    return hipGetLastError() == hipSuccess ? GRIDGCN_OK : GRIDGCN_ELAUNCH;
}

int gridgcn_group_norm_act_bwd(const void *dy, long long ldgb, long long ldgn, const void *x, long long ldb, long long ldn,
                               const uint8_t *codes, const uint8_t *scales, int dtype, int B, long long N, int C, int G,
                               const double *stats, const void *gamma, const void *beta, int ptype, const int32_t *counts,
                               int act, void *dx, void *dgamma, void *dbeta, void *ws, size_t ws_bytes, void *stream)
{
    if (!dy || !stats || !codes != !scales || (!x && !codes) || !sizes_ok(B, N, C, G) || !type_ok(dtype) || !type_ok(ptype) ||
        ldgn < C || ldgn > GRIDGCN_MAX_LD || (B > 1 && ldgb < 0) ||
        (x && !codes && (ldn < C || ldn > GRIDGCN_MAX_LD || (B > 1 && ldb < 0))) || act < GRIDGCN_ACT_NONE || act > GRIDGCN_ACT_GELU || ((uintptr_t)codes & 15))
        return GRIDGCN_EINVAL;
    if (!dx && !dgamma && !dbeta) return GRIDGCN_OK;
    const Plan p = plan_of(B, N, C, G, dtype, false, true, true);
    if (p.bytes && (!ws || ws_bytes < p.bytes || ((uintptr_t)ws & 15))) return GRIDGCN_EWORKSPACE;
    Args a = {};
    a.dy = dy; a.gb = ldgb; a.gn = ldgn; a.x = x; a.xb = ldb; a.xn = ldn; a.codes = codes; a.scales = scales;
    a.y = dx; a.N = N; a.B = B; a.C = C; a.G = G; a.cg = C / G; a.ptype = ptype; a.gamma = gamma; a.beta = beta;
    a.dgamma = dgamma; a.dbeta = dbeta; a.counts = counts; a.stats = (double *)stats;
    a.part = (double *)((char *)ws + p.off_part);
    a.tot = (double *)((char *)ws + p.off_tot);
    a.coef = (float2 *)((char *)ws + p.off_coef);
    a.rpc = p.rpc; a.chunks = p.chunks; a.past = gg_past_caches(B * N, C, dtype);
    const hipStream_t st = (hipStream_t)stream;
    const int rc = with_type(dtype, [&](auto *t) {
        typedef typename std::remove_pointer<decltype(t)>::type T;
        if (codes) bwd_act<T, true>(a, p, act, st);
        else bwd_act<T, false>(a, p, act, st);
    });
    if (rc) return rc;
    return hipGetLastError() == hipSuccess ? GRIDGCN_OK : GRIDGCN_ELAUNCH;
}

}  // extern "C"
