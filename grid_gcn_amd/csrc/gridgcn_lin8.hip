// gridgcn_lin8.hip -- the linear layer that keeps its input in 8 bits (gridgcn_act8.h) between forward and backward.
//
//   forward   y [R, N] = x [R, K] W^T + b, and in the same pass over x its 8-bit form
//   backward  dx [R, K] = dy W;   dW [N, K] = dy^T x^, x^ the values of the 8-bit form;   db = sum of dy's rows
//
// Rows are many (one per point or edge), K and N a few hundred: with 16-bit rows all three products wait for memory, with
// 32-bit rows they would wait for the fp32 matrix instruction (1/16 of the bf16 rate).  So a 32-bit operand enters as three bf16
// numbers, x = hi + mid + lo (to nearest each: the remainder has 16, then 8 bits: nothing is lost), and a product keeps the
// six partial products down to 2^-18 of the largest; what is dropped is below 2^-26, under the rounding of the fp32 sums.
// A value of the 8-bit form is exact in bf16 as it is: dW needs three.
#include "../../include/gridgcn.h"
#include "gridgcn_act8.h"
#include "gridgcn_mma.h"
#include "gridgcn_once.h"
#include <type_traits>

namespace {
typedef ggm_f32x16 F16;
typedef gg_bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef gg_f16 f16x8 __attribute__((ext_vector_type(8)));

template <class T> struct Ty {                       // 16-bit rows: the operand as it is
    static constexpr int P = 1;
    static __device__ __forceinline__ F16 mfma(gg_u32x4 a, gg_u32x4 b, F16 c)
    {
        if constexpr (std::is_same<T, gg_f16>::value)
            return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <> struct Ty<float> {
    static constexpr int P = 3;
    static __device__ __forceinline__ F16 mfma(gg_u32x4 a, gg_u32x4 b, F16 c) { return Ty<gg_bf16>::mfma(a, b, c); }
};

__device__ __forceinline__ F16 zero16()
{
    F16 z;
#pragma unroll
    for (int r = 0; r < 16; r++) z[r] = 0.f;
    return z;
}

// the low (c = 0) or high 16 bits of two registers as one
__device__ __forceinline__ unsigned gg_pair16(unsigned a, unsigned b, int c)
{
    return (unsigned)__builtin_amdgcn_perm(b, a, c ? 0x07060302u : 0x05040100u);
}

// two floats as three bf16 pairs
__device__ __forceinline__ void split2(float a, float b, unsigned &h, unsigned &m, unsigned &l)
{
    h = gg_cvt_bf16(a, b);
    a -= gg_lo16f(h); b -= gg_hi16f(h);
    m = gg_cvt_bf16(a, b);
    a -= gg_lo16f(m); b -= gg_hi16f(m);
    l = gg_cvt_bf16(a, b);
}

// acc[t] += A B[t] from the pieces of both, the smallest partial products first; neighbouring instructions on different tiles
template <class T, int NT, int PA, int PB>
__device__ __forceinline__ void mul(const gg_u32x4 (&a)[PA], const gg_u32x4 (&b)[NT][PB], F16 (&c)[NT])
{
    auto one = [&](int i, int j) {
#pragma unroll
        for (int t = 0; t < NT; t++) c[t] = Ty<T>::mfma(a[i], b[t][j], c[t]);
    };
    if constexpr (PA == 3 && PB == 3) { one(2, 0); one(1, 1); one(0, 2); one(1, 0); one(0, 1); }
    else if constexpr (PA == 3) { one(2, 0); one(1, 0); }
    one(0, 0);
}

// ---- 64 bytes of a row: a lane's share of a contraction step.  A step is KS channels (128 bytes of a row: a line), the half-wave h
// takes the KS / 2 from KS / 2 * h on -- any order serves a contraction, as long as both operands have it -- so a lane's loads are
// neighbours and the two halves share a line. ----------------------------------------------------------------------------
template <class T> constexpr int KS = 128 / (int)sizeof(T);
template <class T> constexpr int SS = KS<T> / 16;        // matrix instructions of a step: 8 channels of each half
template <class T> struct Block {
    static constexpr int VW = 16 / (int)sizeof(T), CH = 4 * VW;
    gg_u32x4 w[4];
    __device__ __forceinline__ void load_full(const T *q)
    {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (sizeof(T) == 4) w[i] = *(const gg_u32x4_a4 *)(q + i * VW);
            else w[i] = *(const gg_u32x4_a2 *)(q + i * VW);
        }
    }
    // channels k0 .. k0 + CH - 1 of a row of K, zeros behind it
    __device__ __forceinline__ void load(const T *row, int k0, int K)
    {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            GGChunk<T> c;
            c.zero();
            if (k0 + i * VW < K) c.load(row, k0 + i * VW, K);
            w[i] = c.w;
        }
    }
    // channels 8 s .. 8 s + 7 as a matrix operand
    __device__ __forceinline__ void frag(int s, gg_u32x4 (&f)[Ty<T>::P]) const
    {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                unsigned h, m, l;
                split2(__uint_as_float(w[2 * s + j / 2][2 * (j & 1)]), __uint_as_float(w[2 * s + j / 2][2 * (j & 1) + 1]), h, m, l);
                f[0][j] = h; f[1][j] = m; f[2][j] = l;
            }
        } else {
            f[0] = w[s];
        }
    }
    __device__ __forceinline__ float get(int i) const
    {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i / 4][i % 4]);
        else if constexpr (std::is_same<T, gg_bf16>::value) return (i & 1) ? gg_hi16f(w[i / 8][(i % 8) / 2]) : gg_lo16f(w[i / 8][(i % 8) / 2]);
        else return gg_f16of(w[i / 8][(i % 8) / 2], i & 1);
    }
    // the 8-bit form: 16-bit rows, the lane holds a block of 32; 32-bit rows, the two halves hold one together (every lane of
    // the wave calls; `on`: this lane stores).  k: first channel of the lane's share, in a row of Cp padded channels
    __device__ __forceinline__ void save(uint8_t *codes, uint8_t *scales, int k, bool on) const
    {
        auto top = [&](bool finite) {
            unsigned m = 0;
#pragma unroll
            for (int i = 0; i < CH; i++) {
                const unsigned u = finite ? gg_a8_mag(get(i)) : __float_as_uint(get(i)) & 0x7fffffffu;
                m = m > u ? m : u;
            }
            if constexpr (CH == 16) {
                const unsigned o = (unsigned)__shfl_xor((int)m, 32);
                m = m > o ? m : o;
            }
            return m;
        };
        unsigned m = top(false);
        const bool clean = !__any(m >= 0x7f800000u);                  // (as gg_a8_block_byte)
        if (!clean) m = top(true);
        const unsigned byte = gg_a8_byte(m);
        const float s = gg_a8_unscale(byte);
        Block b = *this;
#pragma unroll
        for (int i = 0; i < 4; i++) asm volatile("" : "+v"(b.w[i]));  // (16-bit rows: unpacked again, not held unpacked)
        if (!on) return;
#pragma unroll
        for (int i = 0; i < CH / 16; i++) {
            gg_u32x4 o;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float v[4];
                unsigned w[1];
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = b.get(16 * i + 4 * j + e);
                gg_a8_encode<4>(v, byte, clean, w);
                o[j] = w[0];
            }
            *(gg_u32x4 *)(codes + k + 16 * i) = o;
        }
        if (k % 32 == 0) scales[k / 32] = (uint8_t)byte;
    }
};

struct Mm {
    const void *a;             // [R][K] rows, stride lda
    const void *w;             // TRANS ? [K][N] : [N][K], contiguous
    const void *bias;
    void *y;                   // [R][N] contiguous
    uint8_t *codes, *scales;
    long long R, lda;
    int K, N;
    unsigned ncol;             // column blocks
    unsigned nrow;             // row blocks
};

// Workgroup -> (row block, column block): workgroups of consecutive numbers go to different XCDs; the column blocks of one row
// block read the same rows, so they get numbers that are 8 apart and share an L2.
__device__ __forceinline__ bool place(const Mm &p, unsigned &row, unsigned &col)
{
    const unsigned id = blockIdx.x, xcd = id & 7, slot = id >> 3;
    col = slot % p.ncol;
    row = (slot / p.ncol) * 8 + xcd;
    return row < p.nrow;
}
unsigned place_grid(unsigned nrow, unsigned ncol) { return (nrow + 7) / 8 * 8 * ncol; }

// W of a contraction step in LDS, in operand order: [tile of 32 columns][s][piece][lane], 16 bytes each; the lanes 32.. start one
// slot later, so that the k-groups of a column land on different banks when they are written.
// Tile nt holds the columns NT * j + nt: a lane's NT results of a row are then neighbours in memory.
constexpr int FRAG = 66 * 16;

template <class T, bool TRANS, int NT, int THREADS> struct Wstage {
    static constexpr int P = Ty<T>::P, S = SS<T>, G = 2 * S;          // G groups of 8 consecutive channels in a step
    static constexpr int ITEMS_ALL = TRANS ? G * NT * 16 : G * NT * 32;
    static constexpr int ITEMS = (ITEMS_ALL + THREADS - 1) / THREADS;
    static constexpr int BYTES = NT * S * P * FRAG;
    // not TRANS: 8 consecutive k of a column; TRANS: 8 consecutive k (rows of w) of two neighbouring columns
    static constexpr int WORDS = TRANS ? (sizeof(T) == 4 ? 16 : 8) : (sizeof(T) == 4 ? 8 : 4);
    unsigned r[ITEMS][WORDS];
    static_assert(ITEMS_ALL % THREADS == 0, "every thread has the same number of items");

    // A step whose channels all exist.  Columns behind the last are other columns: nobody stores their results.  (TRANS: N >= 2)
    __device__ __forceinline__ void load_full(const Mm &p, int n0, int k0)
    {
        const T *w = (const T *)p.w;
#pragma unroll
        for (int i = 0; i < ITEMS; i++) {
            const int e = (int)threadIdx.x + i * THREADS;
            if constexpr (!TRANS) {
                const int n = n0 + e / G;
                const T *q = w + (size_t)(n < p.N ? n : p.N - 1) * p.K + k0 + 8 * (e % G);
#pragma unroll
                for (int j = 0; j < WORDS / 4; j++) {
                    gg_u32x4 u;
                    if constexpr (sizeof(T) == 4) u = *(const gg_u32x4_a4 *)(q + 4 * j);
                    else u = *(const gg_u32x4_a2 *)q;
#pragma unroll
                    for (int t = 0; t < 4; t++) r[i][4 * j + t] = u[t];
                }
            } else {
                const int n = n0 + 2 * (e % (NT * 16));
                const bool last = n + 1 >= p.N;                      // (the pair in front; its second is column N - 1)
                const T *q = w + (size_t)(k0 + 8 * (e / (NT * 16))) * p.N + (last ? p.N - 2 : n);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    if constexpr (sizeof(T) == 4) {
                        const gg_u32x2 u = *(const gg_u32x2_a4 *)(q + (size_t)j * p.N);
                        r[i][2 * j] = last ? u[1] : u[0];
                        r[i][2 * j + 1] = u[1];
                    } else {
                        const unsigned u = *(const gg_u32_a2 *)(q + (size_t)j * p.N);
                        r[i][j] = last ? u >> 16 : u;
                    }
                }
            }
        }
    }
    // the last step, from channel k0 on: zeros behind K
    __device__ __forceinline__ void load_tail(const Mm &p, int n0, int k0)
    {
        const T *w = (const T *)p.w;
#pragma unroll
        for (int i = 0; i < ITEMS; i++) {
            const int e = (int)threadIdx.x + i * THREADS;
            const int n = n0 + (TRANS ? 2 * (e % (NT * 16)) : e / G), k = k0 + 8 * (TRANS ? e / (NT * 16) : e % G);
#pragma unroll
            for (int j = 0; j < WORDS; j++) r[i][j] = 0u;
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
                for (int c = 0; c < (TRANS ? 2 : 1); c++) {
                    if (k + j >= p.K || n + c >= p.N) continue;
                    const T *q = w + (TRANS ? (size_t)(k + j) * p.N + n + c : (size_t)n * p.K + k + j);
                    const int at = TRANS ? 2 * j + c : j;            // element of the item
                    if constexpr (sizeof(T) == 4) r[i][at] = *(const unsigned *)q;
                    else r[i][at / 2] |= (unsigned)*(const unsigned short *)q << (16 * (at & 1));
                }
        }
    }

    static __device__ __forceinline__ void put(char *lds, int nl, int k8, const gg_u32x4 (&f)[P])
    {
        const int nt = nl % NT, j = nl / NT, h = k8 / S, s = k8 % S;
#pragma unroll
        for (int q = 0; q < P; q++) *(gg_u32x4 *)(lds + ((nt * S + s) * P + q) * FRAG + (h * 33 + j) * 16) = f[q];
    }

    __device__ __forceinline__ void store(char *lds) const
    {
#pragma unroll
        for (int i = 0; i < ITEMS; i++) {
            const int e = (int)threadIdx.x + i * THREADS;
            if constexpr (!TRANS) {
                gg_u32x4 f[P];
                if constexpr (sizeof(T) == 4) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        unsigned h, m, l;
                        split2(__uint_as_float(r[i][2 * j]), __uint_as_float(r[i][2 * j + 1]), h, m, l);
                        f[0][j] = h; f[1][j] = m; f[2][j] = l;
                    }
                } else {
                    f[0] = gg_u32x4{r[i][0], r[i][1], r[i][2], r[i][3]};
                }
                put(lds, e / G, e % G, f);
            } else {
                const int nl = 2 * (e % (NT * 16)), k8 = e / (NT * 16);
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    gg_u32x4 f[P];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        if constexpr (sizeof(T) == 4) {
                            unsigned h, m, l;
                            split2(__uint_as_float(r[i][4 * j + c]), __uint_as_float(r[i][4 * j + 2 + c]), h, m, l);
                            f[0][j] = h; f[1][j] = m; f[2][j] = l;
                        } else {
                            f[0][j] = gg_pair16(r[i][2 * j], r[i][2 * j + 1], c);
                        }
                    }
                    put(lds, nl + c, k8, f);
                }
            }
        }
    }
};

// y of one row for NT neighbouring columns
template <class T, int NT> __device__ __forceinline__ void put_row(T *y, long long row, int n, int N, const float (&v)[NT])
{
    T *q = y + (size_t)row * N + n;
    if (NT == 4 && n + 4 <= N) {
        if constexpr (sizeof(T) == 4) {
            *(gg_u32x4_a4 *)q = gg_u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
        } else if constexpr (std::is_same<T, gg_bf16>::value) {
            *(gg_u32x2_a2 *)q = gg_u32x2{gg_cvt_bf16(v[0], v[1]), gg_cvt_bf16(v[2], v[3])};
        } else {
            *(gg_u32x2_a2 *)q = gg_u32x2{gg_cvt_f16(v[0], v[1]), gg_cvt_f16(v[2], v[3])};
        }
    } else {
#pragma unroll
        for (int t = 0; t < NT; t++)
            if (n + t < N) GGRowT<T>::put(q + t, v[t]);
    }
}

// ---- many rows: a wave owns 32 rows and 32 NT columns, its rows straight from memory into registers (each row is read by one wave
// only), W through LDS, the next step of both in flight while this one is multiplied; three or four workgroups per CU, so that
// one's barriers and stores are another's matrix instructions ----------------------------------------------------------------
constexpr int MW = 4;             // waves
template <class T, bool TRANS, bool SAVE, int NT>
__global__ __launch_bounds__(MW * 64, 3) void gg_k_lin8(Mm p)
{
    constexpr int P = Ty<T>::P, S = SS<T>;
    typedef Wstage<T, TRANS, NT, MW * 64> W;
    extern __shared__ __attribute__((aligned(16))) char lds8[];
    unsigned brow, bcol;
    if (!place(p, brow, bcol)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, j = lane & 31;
    const int n0 = (int)bcol * 32 * NT;
    const long long m0 = (long long)brow * (MW * 32) + wave * 32, r = m0 + j;
    const bool live = r < p.R;
    const int Cp = gg_a8_cp(p.K), steps = (p.K + KS<T> - 1) / KS<T>, kh = KS<T> / 2 * h;
    const T *row = (const T *)p.a + (size_t)(live ? r : p.R - 1) * p.lda;
    F16 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) acc[t] = zero16();

    auto keep = [&](const Block<T> &b, int st) {
        if (SAVE && bcol == 0) {
            const int k = st * KS<T> + kh;
            b.save(p.codes + (size_t)r * Cp, p.scales + (size_t)r * (Cp / 32), k, live && k < Cp);
        }
    };
    auto multiply = [&](const Block<T> &b, const char *cur) {
#pragma unroll
        for (int s = 0; s < S; s++) {
            gg_u32x4 fa[P];
            b.frag(s, fa);
#pragma unroll
            for (int t = 0; t < NT; t += 2) {                     // (two tiles at a time: independent neighbours, few registers)
                gg_u32x4 fb[2][P];
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int q = 0; q < P; q++) fb[u][q] = *(const gg_u32x4 *)(cur + (((t + u) * S + s) * P + q) * FRAG + (h * 33 + j) * 16);
                F16(&two)[2] = *(F16(*)[2])&acc[t];
                mul<T>(fa, fb, two);
            }
        }
    };
    const int full = p.K / KS<T>;
    if (full) {
        W ws;
        Block<T> a, nx;
        ws.load_full(p, n0, 0);
        a.load_full(row + kh);
        ws.store(lds8);
        __syncthreads();
        for (int st = 0; st < full; st++) {
            const bool more = st + 1 < full;
            if (more) {
                ws.load_full(p, n0, (st + 1) * KS<T>);
                nx.load_full(row + (st + 1) * KS<T> + kh);
            }
            keep(a, st);
            multiply(a, lds8 + (st & 1) * W::BYTES);
            if (more) {
                ws.store(lds8 + ((st + 1) & 1) * W::BYTES);
                a = nx;
            }
            __syncthreads();
        }
    }
    if (full < steps) {
        W ws;
        Block<T> a;
        ws.load_tail(p, n0, full * KS<T>);
        a.load(row, full * KS<T> + kh, p.K);
        ws.store(lds8 + (full & 1) * W::BYTES);
        __syncthreads();
        keep(a, full);
        multiply(a, lds8 + (full & 1) * W::BYTES);
    }
    const int n = n0 + NT * j;
    float b[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) b[t] = n + t < p.N ? gg_ld_param(p.bias, GGRowT<T>::id, n + t, 0.f) : 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const long long o = m0 + ggm_row(i, lane);
        if (o >= p.R) continue;
        float v[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) v[t] = acc[t][i] + b[t];
        put_row<T, NT>((T *)p.y, o, n, p.N, v);
    }
}

// ---- few rows: a workgroup owns 32 x 32 results, its waves share the contraction (a step of 64 each in turn) and add up in LDS;
// both operands straight from memory ------------------------------------------------------------------------------------------
constexpr int SW = 8;
template <class T, bool TRANS, bool SAVE>
__global__ __launch_bounds__(SW * 64) void gg_k_lin8_few(Mm p)
{
    constexpr int P = Ty<T>::P;
    __shared__ float part[SW][16][64];
    unsigned brow, bcol;
    if (!place(p, brow, bcol)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, j = lane & 31;
    const int n = (int)bcol * 32 + j;
    const long long r = (long long)brow * 32 + j;
    const int Cp = gg_a8_cp(p.K), steps = (p.K + KS<T> - 1) / KS<T>;
    const T *row = (const T *)p.a + (size_t)(r < p.R ? r : p.R - 1) * p.lda;
    const T *w = (const T *)p.w;
    const int nn = n < p.N ? n : p.N - 1;
    F16 acc[1] = {zero16()};
    for (int st = wave; st < steps; st += SW) {
        const int k0 = KS<T> * st + KS<T> / 2 * h;
        Block<T> a, b;
        a.load(row, k0, p.K);
        if constexpr (!TRANS) {
            b.load(w + (size_t)nn * p.K, k0, p.K);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) b.w[i] = gg_u32x4{0u, 0u, 0u, 0u};
#pragma unroll
            for (int i = 0; i < Block<T>::CH; i++) {
                if (k0 + i >= p.K) continue;
                const T *q = w + (size_t)(k0 + i) * p.N + nn;
                if constexpr (sizeof(T) == 4) b.w[i / 4][i % 4] = *(const unsigned *)q;
                else b.w[i / 8][(i % 8) / 2] |= (unsigned)*(const unsigned short *)q << (16 * (i & 1));
            }
        }
        if (SAVE && bcol == 0) a.save(p.codes + (size_t)r * Cp, p.scales + (size_t)r * (Cp / 32), k0, r < p.R && k0 < Cp);
#pragma unroll
        for (int s = 0; s < SS<T>; s++) {
            gg_u32x4 fa[P], fb[1][P];
            a.frag(s, fa);
            b.frag(s, fb[0]);
            mul<T>(fa, fb, acc);
        }
    }
#pragma unroll
    for (int i = 0; i < 16; i++) part[wave][i][lane] = acc[0][i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16 / SW; i++) {
        const int reg = wave * (16 / SW) + i;
        float v[1] = {part[0][reg][lane]};
#pragma unroll
        for (int q = 1; q < SW; q++) v[0] += part[q][reg][lane];
        const long long rr = (long long)brow * 32 + ggm_row(reg, lane);
        if (rr < p.R && n < p.N) {
            v[0] += gg_ld_param(p.bias, GGRowT<T>::id, n, 0.f);
            put_row<T, 1>((T *)p.y, rr, n, p.N, v);
        }
    }
}

// ---- dW, db: the contraction runs over the rows.  A lane loads four neighbouring columns of a row (dy: 16 or 8 bytes, codes: 4)
// for eight rows: the values of one column are then the 8 consecutive contraction elements an operand wants -- no transposition --
// and the four columns are four tiles (tile i holds the columns 4 j + i).  A wave owns 128 x 128 results in 256 registers and
// strips of 16 rows; the waves of a workgroup add up in LDS, the workgroups of a tile through memory in one order. -------------
constexpr int GT = 128;           // results of a tile per side
constexpr int GW = 4;             // waves
struct Wg {
    const void *dy;               // [R][N], stride ldy
    const uint8_t *codes, *scales; // without dw (tk = 1): any readable bytes, Cp = 0
    void *dw, *db;                // [N][K], [N]
    float *part, *dbpart;         // splits > 1: [split][tile][128][128], [split][tiles_n * 128]
    long long R, ldy;
    int N, K, Cp;
    unsigned tn, tk, splits;
};

template <class T> struct Strip {
    static constexpr int DW = sizeof(T) == 4 ? 4 : 2;
    unsigned d[8][DW];
    unsigned c[8], s[8];
    // rows 8 h + 0..7 of a strip that lies inside: `dy`, `codes`, `scales` are the strip's first row (uniform), od / oc / os the lane's
    // byte offsets: no arithmetic per load
    __device__ __forceinline__ void load_full(const Wg &p, const char *dy, const char *codes, const char *scales, unsigned od, unsigned oc,
                                              unsigned os)
    {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const char *q = dy + (size_t)i * p.ldy * sizeof(T);
            if constexpr (sizeof(T) == 4) {
                const gg_u32x4 u = *(const gg_u32x4_a4 *)(q + od);
#pragma unroll
                for (int t = 0; t < 4; t++) d[i][t] = u[t];
            } else {
                const gg_u32x2 u = *(const gg_u32x2_a2 *)(q + od);
                d[i][0] = u[0]; d[i][1] = u[1];
            }
            c[i] = *(const unsigned *)(codes + (size_t)i * p.Cp + oc);
            s[i] = *(const uint8_t *)(scales + (size_t)i * (p.Cp / 32) + os);
        }
    }
    // ... of a strip that may end behind the last row or column
    __device__ __forceinline__ void load_tail(const Wg &p, long long r0, int n, int k)
    {
        const int nb = p.Cp / 32;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const long long r = r0 + i;
            const bool in = r < p.R;
            const T *q = (const T *)p.dy + (size_t)(in ? r : 0) * p.ldy + n;
#pragma unroll
            for (int t = 0; t < DW; t++) d[i][t] = 0u;
            c[i] = 0u;
            s[i] = GG_A8_MIN_BYTE;
#pragma unroll
            for (int t = 0; t < 4; t++) {
                if (!in || n + t >= p.N) continue;
                if constexpr (sizeof(T) == 4) d[i][t] = ((const unsigned *)q)[t];
                else d[i][t / 2] |= (unsigned)((const unsigned short *)q)[t] << (16 * (t & 1));
            }
            if (in && k < p.Cp) {
                c[i] = *(const unsigned *)(p.codes + (size_t)r * p.Cp + k);
                s[i] = p.scales[(size_t)r * nb + k / 32];
            }
        }
    }
    __device__ __forceinline__ float dyv(int i, int t) const
    {
        if constexpr (sizeof(T) == 4) return __uint_as_float(d[i][t]);
        else if constexpr (std::is_same<T, gg_bf16>::value) return (t & 1) ? gg_hi16f(d[i][t / 2]) : gg_lo16f(d[i][t / 2]);
        else return gg_f16of(d[i][t / 2], t & 1);
    }
    // column t of dy as an operand
    __device__ __forceinline__ void frag_dy(int t, gg_u32x4 (&f)[Ty<T>::P]) const
    {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            if constexpr (sizeof(T) == 4) {
                unsigned h, m, l;
                split2(__uint_as_float(d[2 * q][t]), __uint_as_float(d[2 * q + 1][t]), h, m, l);
                f[0][q] = h; f[1][q] = m; f[2][q] = l;
            } else {
                f[0][q] = gg_pair16(d[2 * q][t / 2], d[2 * q + 1][t / 2], t & 1);
            }
        }
    }
    // the four columns of x^ as operands (exact in 16 bits)
    __device__ __forceinline__ void frag_x(gg_u32x4 (&f)[4][1]) const
    {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            float u[4], v[4];
            gg_a8_dec4(c[2 * q], u[0], u[1], u[2], u[3]);
            gg_a8_dec4(c[2 * q + 1], v[0], v[1], v[2], v[3]);
            const float su = gg_a8_scale(s[2 * q]), sv = gg_a8_scale(s[2 * q + 1]);
#pragma unroll
            for (int t = 0; t < 4; t++) {
                if constexpr (std::is_same<T, gg_f16>::value) f[t][0][q] = gg_cvt_f16(u[t] * su, v[t] * sv);
                else f[t][0][q] = gg_pair16(__float_as_uint(u[t] * su), __float_as_uint(v[t] * sv), 1);
            }
        }
    }
};

template <class T>
__global__ __launch_bounds__(GW * 64, 1) void gg_k_lin8_wgrad(Wg p)
{
    constexpr int P = Ty<T>::P;
    constexpr int D = 3;              // strips in flight (a wave's own: there is one per SIMD)
    extern __shared__ __attribute__((aligned(16))) float ldsf[];    // [GW][4][16][64]
    // (the tiles of one split read the same rows: same XCD, as in place())
    const unsigned tiles = p.tn * p.tk, id = blockIdx.x, xcd = id & 7, slot = id >> 3;
    const unsigned tile = slot % tiles, split = (slot / tiles) * 8 + xcd;
    if (split >= p.splits) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), h = lane >> 5, j = lane & 31;
    const int n0 = (int)(tile / p.tk) * GT, k0 = (int)(tile % p.tk) * GT, n = n0 + 4 * j, k = k0 + 4 * j;
    const bool first = tile % p.tk == 0;
    const long long strips = (p.R + 15) / 16, stride = (long long)p.splits * GW;
    // Strips that are loaded unchecked.  What a lane reads behind the last column belongs to results that nobody stores (such lanes
    // read the columns from 0 on, and at most 3 values behind a row's end: the rows of these strips have 4 more behind them).
    const long long whole = p.R > 4 ? (p.R - 4) / 16 : 0;
    const unsigned od = (unsigned)((8 * h * p.ldy + (n < p.N ? n : 0)) * (long long)sizeof(T));
    const int kc = k < p.Cp ? k : 0;
    const unsigned oc = (unsigned)(8 * h * p.Cp + kc), os = (unsigned)(8 * h * (p.Cp / 32) + kc / 32);
    F16 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int t = 0; t < 4; t++) acc[i][t] = zero16();
    float dbs[4] = {0.f, 0.f, 0.f, 0.f};
    Strip<T> q[D];
    auto fetch = [&](long long g, Strip<T> &s) {
        if (g < whole)
            s.load_full(p, (const char *)p.dy + (size_t)g * 16 * p.ldy * sizeof(T), (const char *)p.codes + (size_t)g * 16 * p.Cp,
                        (const char *)p.scales + (size_t)g * 16 * (p.Cp / 32), od, oc, os);
    };
    auto use = [&](const Strip<T> &s) {
        gg_u32x4 fx[4][1];
        s.frag_x(fx);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            gg_u32x4 fd[P];
            s.frag_dy(i, fd);
            mul<T>(fd, fx, acc[i]);
        }
        if (first) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float v = s.dyv(0, i);
#pragma unroll
                for (int e = 1; e < 8; e++) v += s.dyv(e, i);
                dbs[i] += v;
            }
        }
    };
    long long g = (long long)split * GW + wave;
#pragma unroll
    for (int d = 0; d < D - 1; d++) fetch(g + d * stride, q[d]);
    while (g < whole) {
#pragma unroll
        for (int d = 0; d < D; d++) {
            if (g < whole) {
                fetch(g + (D - 1) * stride, q[(d + D - 1) % D]);
                use(q[d]);
                g += stride;
            }
        }
    }
    for (; g < strips; g += stride) {                             // (the last one or two strips of all)
        Strip<T> s;
        s.load_tail(p, g * 16 + 8 * h, n, k);
        use(s);
    }
    // the waves' sums: a quarter of the tile's rows at a time
    float *pt = p.part ? p.part + ((size_t)split * tiles + tile) * GT * GT : nullptr;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        __syncthreads();
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) ldsf[((wave * 4 + t) * 16 + r) * 64 + lane] = acc[i][t][r];
        __syncthreads();
#pragma unroll
        for (int q = 0; q < 16 / GW; q++) {
            const int r = wave * (16 / GW) + q;
            float v[4];
#pragma unroll
            for (int t = 0; t < 4; t++) {
                v[t] = ldsf[(t * 16 + r) * 64 + lane];
#pragma unroll
                for (int w = 1; w < GW; w++) v[t] += ldsf[((w * 4 + t) * 16 + r) * 64 + lane];
            }
            const int nl = 4 * ggm_row(r, lane) + i;
            if (pt) *(float4 *)(pt + (size_t)nl * GT + 4 * j) = make_float4(v[0], v[1], v[2], v[3]);
            else if (p.dw && n0 + nl < p.N) put_row<T, 4>((T *)p.dw, n0 + nl, k, p.K, v);
        }
    }
    if (!first || !p.db) return;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; i++) ldsf[(wave * 4 + i) * 64 + lane] = dbs[i];
    __syncthreads();
    if ((int)threadIdx.x < GT) {
        const int jj = threadIdx.x / 4, i = threadIdx.x % 4;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < GW; w++) v += ldsf[(w * 4 + i) * 64 + jj] + ldsf[(w * 4 + i) * 64 + jj + 32];
        const int nn = n0 + (int)threadIdx.x;
        if (p.part) p.dbpart[(size_t)split * p.tn * GT + nn] = v;
        else if (nn < p.N) GGRowT<T>::put((T *)p.db + nn, v);
    }
}

// sums of the splits: a workgroup = 32 groups of 4 results x 8 lanes over the splits
template <class T>
__global__ __launch_bounds__(256) void gg_k_lin8_wsum(Wg p, unsigned nw)
{
    __shared__ float4 red[8][32];
    const unsigned tiles = p.tn * p.tk;
    const int e = threadIdx.x & 31, l = threadIdx.x >> 5;
    const bool isdb = blockIdx.x >= nw;
    const size_t at = ((size_t)(isdb ? blockIdx.x - nw : blockIdx.x) * 32 + e) * 4;
    const size_t stride = isdb ? (size_t)p.tn * GT : (size_t)tiles * GT * GT;
    const float *src = (isdb ? p.dbpart : p.part) + at;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (unsigned q = l; q < p.splits; q += 8) {
        const float4 v = *(const float4 *)(src + q * stride);
        s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    red[l][e] = s;
    __syncthreads();
    if (l) return;
#pragma unroll
    for (int q = 1; q < 8; q++) {
        const float4 v = red[q][e];
        s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    const float v[4] = {s.x, s.y, s.z, s.w};
    if (isdb) {
#pragma unroll
        for (int t = 0; t < 4; t++)
            if ((int)at + t < p.N) GGRowT<T>::put((T *)p.db + at + t, v[t]);
    } else {
        const unsigned tile = (unsigned)(at / (GT * GT));
        const int rem = (int)(at % (GT * GT)), n = (int)(tile / p.tk) * GT + rem / GT, k = (int)(tile % p.tk) * GT + rem % GT;
        if (n < p.N) put_row<T, 4>((T *)p.dw, n, k, p.K, v);
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------
template <class T, bool TRANS, bool SAVE> int launch_mm(Mm &p, hipStream_t st)
{
    constexpr int NT = 4;
    const long long blocks = (p.R + MW * 32 - 1) / (MW * 32) * ((p.N + 32 * NT - 1) / (32 * NT));
    // fewer workgroups than half the CUs: smaller ones, their waves on the contraction.  (One column: the pairs of W's columns that
    // the other kernel loads do not exist.)
    if (blocks < 128 || (TRANS && p.N < 2)) {
        p.nrow = (unsigned)((p.R + 31) / 32);
        p.ncol = (unsigned)((p.N + 31) / 32);
        gg_k_lin8_few<T, TRANS, SAVE><<<place_grid(p.nrow, p.ncol), SW * 64, 0, st>>>(p);
        return 0;
    }
    constexpr int LDS = 2 * Wstage<T, TRANS, NT, MW * 64>::BYTES;
    static GGDevOnce done;
    if (!done) {
        if (hipFuncSetAttribute((const void *)gg_k_lin8<T, TRANS, SAVE, NT>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS) != hipSuccess)
            return GRIDGCN_ELAUNCH;
        done = true;
    }
    p.nrow = (unsigned)((p.R + MW * 32 - 1) / (MW * 32));
    p.ncol = (unsigned)((p.N + 32 * NT - 1) / (32 * NT));
    gg_k_lin8<T, TRANS, SAVE, NT><<<place_grid(p.nrow, p.ncol), MW * 64, LDS, st>>>(p);
    return 0;
}

unsigned splits_of(long long R, unsigned tiles)
{
    // one generation of workgroups (one per CU: they use all its registers), at least four strips for each wave
    long long s = 256 / tiles;
    const long long most = (R + 16 * GW * 4 - 1) / (16 * GW * 4);
    if (s > most) s = most;
    return (unsigned)(s < 1 ? 1 : s);
}

size_t wgrad_bytes(long long R, unsigned tn, unsigned tk)
{
    const unsigned s = splits_of(R, tn * tk);
    return s > 1 ? (size_t)s * ((size_t)tn * tk * GT * GT + (size_t)tn * GT) * 4 : 256;
}

template <class T> int launch_wgrad(Wg &p, hipStream_t st)
{
    static GGDevOnce done;
    constexpr int LDS = GW * 4 * 16 * 64 * 4;
    if (!done) {
        if (hipFuncSetAttribute((const void *)gg_k_lin8_wgrad<T>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS) != hipSuccess)
            return GRIDGCN_ELAUNCH;
        done = true;
    }
    const unsigned tiles = p.tn * p.tk;
    gg_k_lin8_wgrad<T><<<(p.splits + 7) / 8 * 8 * tiles, GW * 64, LDS, st>>>(p);
    if (p.splits > 1) {
        const unsigned nw = p.dw ? tiles * (GT * GT / 128) : 0, nd = p.db ? p.tn : 0;
        gg_k_lin8_wsum<T><<<nw + nd, 256, 0, st>>>(p, nw);
    }
    return 0;
}

bool type_ok(int t) { return t == GRIDGCN_F32 || t == GRIDGCN_BF16 || t == GRIDGCN_F16; }
bool sizes_ok(long long R, int K, int N)
{
    // (grids stay below 2^31 workgroups)
    return R >= 1 && R <= (1ll << 36) && K >= 1 && K <= GRIDGCN_ACT8_MAX_C && N >= 1 && N <= GRIDGCN_ACT8_MAX_C &&
           (R + 31) / 32 * ((N + 31) / 32) < (1ll << 30) && (R + 31) / 32 * ((K + 31) / 32) < (1ll << 30);
}
template <class F> int with_type(int dtype, F f)
{
    if (dtype == GRIDGCN_F32) return f((float *)nullptr);
    if (dtype == GRIDGCN_BF16) return f((gg_bf16 *)nullptr);
    return f((gg_f16 *)nullptr);
}
}  // namespace

extern "C" {

int gridgcn_linear_act8_fwd(const void *x, int dtype, long long R, int K, long long ldx, const void *W, const void *bias,
                            int N, void *y, uint8_t *codes, uint8_t *scales, void *stream)
{
    if (!x || !W || !y || !type_ok(dtype) || !sizes_ok(R, K, N) || ldx < K || ldx > GRIDGCN_MAX_LD || !codes != !scales || ((uintptr_t)codes & 15))
        return GRIDGCN_EINVAL;
    Mm p = {};
    p.a = x; p.w = W; p.bias = bias; p.y = y; p.codes = codes; p.scales = scales; p.R = R; p.lda = ldx; p.K = K; p.N = N;
    const hipStream_t st = (hipStream_t)stream;
    const int rc = with_type(dtype, [&](auto *t) {
        typedef typename std::remove_pointer<decltype(t)>::type T;
        return codes ? launch_mm<T, false, true>(p, st) : launch_mm<T, false, false>(p, st);
    });
    if (rc) return rc;
    return hipGetLastError() == hipSuccess ? GRIDGCN_OK : GRIDGCN_ELAUNCH;
}

int gridgcn_linear_act8_bwd_workspace_bytes(long long R, int K, int N, size_t *bytes)
{
    if (!bytes || !sizes_ok(R, K, N)) return GRIDGCN_EINVAL;
    const size_t w = wgrad_bytes(R, (N + GT - 1) / GT, (K + GT - 1) / GT), b = wgrad_bytes(R, (N + GT - 1) / GT, 1);
    *bytes = w > b ? w : b;
    return GRIDGCN_OK;
}

int gridgcn_linear_act8_bwd(const void *dy, int dtype, long long R, int N, long long ldy, const void *W, int K,
                            const uint8_t *codes, const uint8_t *scales, void *dx, void *dW, void *dbias, void *ws,
                            size_t ws_bytes, void *stream)
{
    if (!dy || !type_ok(dtype) || !sizes_ok(R, K, N) || ldy < N || ldy > GRIDGCN_MAX_LD || (dx && !W) || (dW && (!codes || !scales)) ||
        ((uintptr_t)codes & 15))
        return GRIDGCN_EINVAL;
    Wg g = {};
    g.dy = dy; g.dw = dW; g.db = dbias; g.R = R; g.ldy = ldy; g.N = N; g.K = K; g.Cp = gg_a8_cp(K);
    g.codes = dW ? codes : (const uint8_t *)dy;
    g.scales = dW ? scales : (const uint8_t *)dy;
    if (!dW) g.Cp = 0;
    g.tn = (N + GT - 1) / GT;
    g.tk = dW ? (K + GT - 1) / GT : 1;
    g.splits = splits_of(R, g.tn * g.tk);
    if ((dW || dbias) && g.splits > 1) {
        if (!ws || ws_bytes < wgrad_bytes(R, g.tn, g.tk) || ((uintptr_t)ws & 15)) return GRIDGCN_EWORKSPACE;
        g.part = (float *)ws;
        g.dbpart = g.part + (size_t)g.splits * g.tn * g.tk * GT * GT;
    }
    const hipStream_t st = (hipStream_t)stream;
    const int rc = with_type(dtype, [&](auto *t) {
        typedef typename std::remove_pointer<decltype(t)>::type T;
        if (dx) {
            Mm p = {};
            p.a = dy; p.w = W; p.y = dx; p.R = R; p.lda = ldy; p.K = N; p.N = K;
            const int e = launch_mm<T, true, false>(p, st);
            if (e) return e;
        }
        return dW || dbias ? launch_wgrad<T>(g, st) : 0;
    });
    if (rc) return rc;
    return hipGetLastError() == hipSuccess ? GRIDGCN_OK : GRIDGCN_ELAUNCH;
}

}  // extern "C"
