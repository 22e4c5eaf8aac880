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

// two floats as three bf16 pairs
__device__ __forceinline__ void split2(float a, float b, unsigned &h, unsigned &m, unsigned &l)
{
    h = gg_cvt_bf16(a, b);
    a -= gg_lo16f(h); b -= gg_hi16f(h);
    m = gg_cvt_bf16(a, b);
    a -= gg_lo16f(m); b -= gg_hi16f(m);
    l = gg_cvt_bf16(a, b);
}

// acc += A B from the pieces of both, the smallest partial products first
template <class T, int PA, int PB>
__device__ __forceinline__ F16 mul(const gg_u32x4 (&a)[PA], const gg_u32x4 (&b)[PB], F16 c)
{
    if constexpr (PA == 3 && PB == 3) {
        c = Ty<T>::mfma(a[2], b[0], c);
        c = Ty<T>::mfma(a[1], b[1], c);
        c = Ty<T>::mfma(a[0], b[2], c);
        c = Ty<T>::mfma(a[1], b[0], c);
        c = Ty<T>::mfma(a[0], b[1], c);
        return Ty<T>::mfma(a[0], b[0], c);
    } else if constexpr (PA == 3) {
        c = Ty<T>::mfma(a[2], b[0], c);
        c = Ty<T>::mfma(a[1], b[0], c);
        return Ty<T>::mfma(a[0], b[0], c);
    } else {
        return Ty<T>::mfma(a[0], b[0], c);
    }
}

// ---- 32 consecutive channels of a row: a lane's share of a contraction step of 64 -----------------------------------
template <class T> struct Block {
    static constexpr int NW = 2 * (int)sizeof(T);    // 16-byte words
    static constexpr int VW = 16 / (int)sizeof(T);
    gg_u32x4 w[NW];
    __device__ __forceinline__ void load(const T *row, int k0, int K)
    {
#pragma unroll
        for (int i = 0; i < NW; i++) {
            const int k = k0 + i * VW;
            if (k + VW <= K) {
                if constexpr (sizeof(T) == 4) w[i] = *(const gg_u32x4_a4 *)(row + k);
                else w[i] = *(const gg_u32x4_a2 *)(row + k);
            } else {
                gg_u32x4 u = {0u, 0u, 0u, 0u};
                if (k < K) {
                    if constexpr (sizeof(T) == 4) {
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            if (k + j < K) u[j] = ((const unsigned *)row)[k + j];
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            if (k + j < K) u[j / 2] |= (unsigned)((const unsigned short *)row)[k + j] << (16 * (j & 1));
                    }
                }
                w[i] = u;
            }
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
    // the 8-bit form of the 32: the lane holds the whole block, no lane is asked
    __device__ __forceinline__ void save(uint8_t *codes, uint8_t *scale) const
    {
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < 32; i++) {
            const unsigned u = gg_a8_mag(get(i));
            m = m > u ? m : u;
        }
        const unsigned byte = gg_a8_byte(m);
        const float s = gg_a8_unscale(byte);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            gg_u32x4 o;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int e = 16 * i + 4 * j;
                o[j] = gg_a8_enc4(gg_a8_ready(get(e), s), gg_a8_ready(get(e + 1), s), gg_a8_ready(get(e + 2), s), gg_a8_ready(get(e + 3), s));
            }
            *(gg_u32x4 *)(codes + 16 * i) = o;
        }
        *scale = (uint8_t)byte;
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

// W of a contraction step (64 channels) in LDS, in operand order: [tile of 32 columns][s of 4][piece][lane], 16 bytes each; the
// lanes 32.. start one slot later so that the eight k-groups of a column land on different banks when they are written.
// Tile nt holds the columns NT * j + nt: a lane's NT results of a row are then neighbours in memory.
constexpr int FRAG = 66 * 16;

template <class T, bool TRANS, int NT, int THREADS> struct Wstage {
    static constexpr int P = Ty<T>::P;
    static constexpr int ITEMS_ALL = TRANS ? 8 * NT * 16 : 8 * NT * 32;
    static constexpr int ITEMS = (ITEMS_ALL + THREADS - 1) / THREADS;
    static constexpr int BYTES = NT * 4 * P * FRAG;
    // not TRANS: 8 consecutive k of a column; TRANS: 8 consecutive k (rows of w) of two neighbouring columns
    static constexpr int WORDS = TRANS ? (sizeof(T) == 4 ? 16 : 8) : (sizeof(T) == 4 ? 8 : 4);
    unsigned r[ITEMS][WORDS];

    __device__ __forceinline__ void load(const Mm &p, int n0, int k0)
    {
        const T *w = (const T *)p.w;
#pragma unroll
        for (int i = 0; i < ITEMS; i++) {
            const int e = (int)threadIdx.x + i * THREADS;
#pragma unroll
            for (int j = 0; j < WORDS; j++) r[i][j] = 0u;
            if (e >= ITEMS_ALL) continue;
            if constexpr (!TRANS) {
                const int k = k0 + 8 * (e & 7), n = n0 + (e >> 3);
                if (n >= p.N) continue;
                const T *q = w + (size_t)n * p.K + k;
                if (k + 8 <= p.K) {
#pragma unroll
                    for (int j = 0; j < WORDS / 4; j++) {
                        gg_u32x4 u;
                        if constexpr (sizeof(T) == 4) u = *(const gg_u32x4_a4 *)(q + 4 * j);
                        else u = *(const gg_u32x4_a2 *)q;
#pragma unroll
                        for (int t = 0; t < 4; t++) r[i][4 * j + t] = u[t];
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        if (k + j >= p.K) continue;
                        if constexpr (sizeof(T) == 4) r[i][j] = ((const unsigned *)q)[j];
                        else r[i][j / 2] |= (unsigned)((const unsigned short *)q)[j] << (16 * (j & 1));
                    }
                }
            } else {
                const int n = n0 + 2 * (e % (NT * 16)), k = k0 + 8 * (e / (NT * 16));
                if (n >= p.N) continue;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    if (k + j >= p.K) continue;
                    const T *q = w + (size_t)(k + j) * p.N + n;
                    if constexpr (sizeof(T) == 4) {
                        r[i][2 * j] = ((const unsigned *)q)[0];
                        if (n + 1 < p.N) r[i][2 * j + 1] = ((const unsigned *)q)[1];
                    } else {
                        r[i][j] = ((const unsigned short *)q)[0];
                        if (n + 1 < p.N) r[i][j] |= (unsigned)((const unsigned short *)q)[1] << 16;
                    }
                }
            }
        }
    }

    static __device__ __forceinline__ void put(char *lds, int nl, int k8, const gg_u32x4 (&f)[P])
    {
        const int nt = nl % NT, j = nl / NT, h = k8 >> 2, s = k8 & 3;
#pragma unroll
        for (int q = 0; q < P; q++) *(gg_u32x4 *)(lds + ((nt * 4 + s) * P + q) * FRAG + (h * 33 + j) * 16) = f[q];
    }

    __device__ __forceinline__ void store(char *lds) const
    {
#pragma unroll
        for (int i = 0; i < ITEMS; i++) {
            const int e = (int)threadIdx.x + i * THREADS;
            if (e >= ITEMS_ALL) continue;
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
                put(lds, e >> 3, e & 7, f);
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
                            f[0][j] = c == 0 ? (r[i][2 * j] & 0xffffu) | (r[i][2 * j + 1] << 16) : (r[i][2 * j] >> 16) | (r[i][2 * j + 1] & 0xffff0000u);
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

// ---- many rows: a wave owns MR x 32 rows and 32 NT columns, its rows straight from memory into registers (each row is read by
// one wave only), W through LDS, the next step of both in flight while this one is multiplied -------------------------------
template <class T, bool TRANS, bool SAVE, int NT, int WAVES, int MR>
__global__ __launch_bounds__(WAVES * 64) void gg_k_lin8(Mm p)
{
    constexpr int P = Ty<T>::P, THREADS = WAVES * 64;
    typedef Wstage<T, TRANS, NT, THREADS> W;
    extern __shared__ __attribute__((aligned(16))) char lds8[];
    unsigned brow, bcol;
    if (!place(p, brow, bcol)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, j = lane & 31;
    const int n0 = (int)bcol * 32 * NT;
    const long long m0 = (long long)brow * (WAVES * MR * 32) + wave * (MR * 32);
    const int Cp = gg_a8_cp(p.K);
    const int steps = (p.K + 63) / 64;
    const T *rows[MR];
    bool live[MR];
#pragma unroll
    for (int m = 0; m < MR; m++) {
        const long long r = m0 + m * 32 + j;
        live[m] = r < p.R;
        rows[m] = (const T *)p.a + (size_t)(live[m] ? r : p.R - 1) * p.lda;
    }
    F16 acc[MR][NT];
#pragma unroll
    for (int m = 0; m < MR; m++)
#pragma unroll
        for (int t = 0; t < NT; t++) acc[m][t] = zero16();

    W ws;
    Block<T> a[MR];
    ws.load(p, n0, 0);
#pragma unroll
    for (int m = 0; m < MR; m++) a[m].load(rows[m], 32 * h, p.K);
    ws.store(lds8);
    __syncthreads();
    for (int st = 0; st < steps; st++) {
        const char *cur = lds8 + (st & 1) * W::BYTES;
        Block<T> nx[MR];
        const bool more = st + 1 < steps;
        if (more) {
            ws.load(p, n0, 64 * (st + 1));
#pragma unroll
            for (int m = 0; m < MR; m++) nx[m].load(rows[m], 64 * (st + 1) + 32 * h, p.K);
        }
        if (SAVE && bcol == 0) {
            const int blk = 2 * st + h;
#pragma unroll
            for (int m = 0; m < MR; m++) {
                const long long r = m0 + m * 32 + j;
                if (live[m] && blk * 32 < p.K) a[m].save(p.codes + (size_t)r * Cp + blk * 32, p.scales + (size_t)r * (Cp / 32) + blk);
            }
        }
#pragma unroll
        for (int s = 0; s < 4; s++) {
            gg_u32x4 fa[MR][P];
#pragma unroll
            for (int m = 0; m < MR; m++) a[m].frag(s, fa[m]);
#pragma unroll
            for (int t = 0; t < NT; t++) {
                gg_u32x4 fb[P];
#pragma unroll
                for (int q = 0; q < P; q++) fb[q] = *(const gg_u32x4 *)(cur + ((t * 4 + s) * P + q) * FRAG + (h * 33 + j) * 16);
#pragma unroll
                for (int m = 0; m < MR; m++) acc[m][t] = mul<T>(fa[m], fb, acc[m][t]);
            }
        }
        if (more) {
            ws.store(lds8 + ((st + 1) & 1) * W::BYTES);
#pragma unroll
            for (int m = 0; m < MR; m++) a[m] = nx[m];
        }
        __syncthreads();
    }
    const int n = n0 + NT * j;
    float b[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) b[t] = n + t < p.N ? gg_ld_param(p.bias, GGRowT<T>::id, n + t, 0.f) : 0.f;
#pragma unroll
    for (int m = 0; m < MR; m++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const long long row = m0 + m * 32 + ggm_row(r, lane);
            if (row >= p.R) continue;
            float v[NT];
#pragma unroll
            for (int t = 0; t < NT; t++) v[t] = acc[m][t][r] + b[t];
            put_row<T, NT>((T *)p.y, row, n, p.N, v);
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
    const int Cp = gg_a8_cp(p.K), steps = (p.K + 63) / 64;
    const T *row = (const T *)p.a + (size_t)(r < p.R ? r : p.R - 1) * p.lda;
    const T *w = (const T *)p.w;
    F16 acc = zero16();
    for (int st = wave; st < steps; st += SW) {
        const int k0 = 64 * st + 32 * h;
        Block<T> a, b;
        a.load(row, k0, p.K);
        if constexpr (!TRANS) {
            b.load(w + (size_t)(n < p.N ? n : p.N - 1) * p.K, k0, p.K);
        } else {
            const int nn = n < p.N ? n : p.N - 1;
#pragma unroll
            for (int i = 0; i < Block<T>::NW; i++) b.w[i] = gg_u32x4{0u, 0u, 0u, 0u};
#pragma unroll
            for (int i = 0; i < 32; i++) {
                if (k0 + i >= p.K) continue;
                const T *q = w + (size_t)(k0 + i) * p.N + nn;
                if constexpr (sizeof(T) == 4) b.w[i / 4][i % 4] = *(const unsigned *)q;
                else b.w[i / 8][(i % 8) / 2] |= (unsigned)*(const unsigned short *)q << (16 * (i & 1));
            }
        }
        if (SAVE && bcol == 0) {
            const int blk = 2 * st + h;
            if (r < p.R && blk * 32 < p.K) a.save(p.codes + (size_t)r * Cp + blk * 32, p.scales + (size_t)r * (Cp / 32) + blk);
        }
#pragma unroll
        for (int s = 0; s < 4; s++) {
            gg_u32x4 fa[P], fb[P];
            a.frag(s, fa);
            b.frag(s, fb);
            acc = mul<T>(fa, fb, acc);
        }
    }
#pragma unroll
    for (int i = 0; i < 16; i++) part[wave][i][lane] = acc[i];
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
    const uint8_t *codes, *scales; // NULL: no dw, only db (tk = 1)
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
    __device__ __forceinline__ void load(const Wg &p, long long r0, int n, int k, bool rows)
    {
        const int nb = p.Cp / 32;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const long long r = r0 + i;
            const bool in = rows && r < p.R;
            const T *q = (const T *)p.dy + (size_t)(in ? r : 0) * p.ldy + n;
#pragma unroll
            for (int t = 0; t < DW; t++) d[i][t] = 0u;
            c[i] = 0u;
            s[i] = GG_A8_MIN_BYTE;
            if (in && n + 4 <= p.N) {
                if constexpr (sizeof(T) == 4) {
                    const gg_u32x4 u = *(const gg_u32x4_a4 *)q;
#pragma unroll
                    for (int t = 0; t < 4; t++) d[i][t] = u[t];
                } else {
                    const gg_u32x2 u = *(const gg_u32x2_a2 *)q;
                    d[i][0] = u[0]; d[i][1] = u[1];
                }
            } else if (in && n < p.N) {
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    if (n + t >= p.N) continue;
                    if constexpr (sizeof(T) == 4) d[i][t] = ((const unsigned *)q)[t];
                    else d[i][t / 2] |= (unsigned)((const unsigned short *)q)[t] << (16 * (t & 1));
                }
            }
            if (in && p.codes && k < p.Cp) {
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
                const unsigned u = d[2 * q][t / 2], v = d[2 * q + 1][t / 2];
                f[0][q] = (t & 1) ? (u >> 16) | (v & 0xffff0000u) : (u & 0xffffu) | (v << 16);
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
                else f[t][0][q] = (__float_as_uint(u[t] * su) >> 16) | (__float_as_uint(v[t] * sv) & 0xffff0000u);
            }
        }
    }
};

template <class T>
__global__ __launch_bounds__(GW * 64, 1) void gg_k_lin8_wgrad(Wg p)
{
    constexpr int P = Ty<T>::P;
    extern __shared__ __attribute__((aligned(16))) float ldsf[];    // [GW][4][16][64]
    // (the tiles of one split read the same rows: same XCD, as in place())
    const unsigned tiles = p.tn * p.tk, id = blockIdx.x, xcd = id & 7, slot = id >> 3;
    const unsigned tile = slot % tiles, split = (slot / tiles) * 8 + xcd;
    if (split >= p.splits) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, j = lane & 31;
    const int n0 = (int)(tile / p.tk) * GT, k0 = (int)(tile % p.tk) * GT, n = n0 + 4 * j, k = k0 + 4 * j;
    const bool first = tile % p.tk == 0;
    const long long strips = (p.R + 15) / 16, stride = (long long)p.splits * GW;
    F16 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int t = 0; t < 4; t++) acc[i][t] = zero16();
    float dbs[4] = {0.f, 0.f, 0.f, 0.f};
    long long g = (long long)split * GW + wave;
    Strip<T> cur, nxt;
    cur.load(p, g * 16 + 8 * h, n, k, g < strips);
    for (; g < strips; g += stride) {
        const long long gn = g + stride;
        nxt.load(p, gn * 16 + 8 * h, n, k, gn < strips);
        gg_u32x4 fx[4][1];
        cur.frag_x(fx);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            gg_u32x4 fd[P];
            cur.frag_dy(i, fd);
#pragma unroll
            for (int t = 0; t < 4; t++) acc[i][t] = mul<T>(fd, fx[t], acc[i][t]);
        }
        if (first) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float s = cur.dyv(0, i);
#pragma unroll
                for (int q = 1; q < 8; q++) s += cur.dyv(q, i);
                dbs[i] += s;
            }
        }
        cur = nxt;
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
template <class T, bool TRANS, bool SAVE, int NT, int WAVES, int MR> int launch_many(Mm &p, hipStream_t st)
{
    constexpr int LDS = 2 * Wstage<T, TRANS, NT, WAVES * 64>::BYTES;
    static GGDevOnce done;
    if (!done) {
        if (hipFuncSetAttribute((const void *)gg_k_lin8<T, TRANS, SAVE, NT, WAVES, MR>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS) != hipSuccess)
            return GRIDGCN_ELAUNCH;
        done = true;
    }
    const long long rows = (long long)WAVES * MR * 32;
    p.nrow = (unsigned)((p.R + rows - 1) / rows);
    p.ncol = (unsigned)((p.N + 32 * NT - 1) / (32 * NT));
    gg_k_lin8<T, TRANS, SAVE, NT, WAVES, MR><<<place_grid(p.nrow, p.ncol), WAVES * 64, LDS, st>>>(p);
    return 0;
}

template <class T, bool TRANS, bool SAVE> int launch_mm(Mm &p, hipStream_t st)
{
    constexpr int WAVES = sizeof(T) == 4 ? 8 : 4, MR = sizeof(T) == 4 ? 1 : 2;
    const long long blocks = (p.R + WAVES * MR * 32 - 1) / (WAVES * MR * 32) * ((p.N + 127) / 128);
    // fewer workgroups than half the CUs: smaller ones, their waves on the contraction
    if (blocks < 128) {
        p.nrow = (unsigned)((p.R + 31) / 32);
        p.ncol = (unsigned)((p.N + 31) / 32);
        gg_k_lin8_few<T, TRANS, SAVE><<<place_grid(p.nrow, p.ncol), SW * 64, 0, st>>>(p);
        return 0;
    }
    return launch_many<T, TRANS, SAVE, 4, WAVES, MR>(p, st);
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
    if (!x || !W || !y || !type_ok(dtype) || !sizes_ok(R, K, N) || ldx < K || !codes != !scales || ((uintptr_t)codes & 15))
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
    if (!dy || !type_ok(dtype) || !sizes_ok(R, K, N) || ldy < N || (dx && !W) || (dW && (!codes || !scales)) ||
        ((uintptr_t)codes & 15))
        return GRIDGCN_EINVAL;
    Wg g = {};
    g.dy = dy; g.dw = dW; g.db = dbias; g.R = R; g.ldy = ldy; g.N = N; g.K = K; g.Cp = gg_a8_cp(K);
    if (dW) { g.codes = codes; g.scales = scales; }
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
