// gridgcn_lin8.hip -- the linear layer that keeps its input in 8 bits (gridgcn_act8.h) between forward and backward.
//
//   forward   y [R, N] = x [R, K] W^T + b, and in the same pass over x its 8-bit form
//   backward  dx [R, K] = dy W;   dW [N, K] = dy^T x^, x^ the values of the 8-bit form;   db = sum of dy's rows
//
// Rows are many (one per point or edge), K and N a few hundred: with 16-bit rows all three products wait for memory, with
// 32-bit rows they would wait for the fp32 matrix instruction (1/16 of the bf16 rate).  So a 32-bit operand enters as a sum of
// three bf16 numbers, x = hi + mid + lo, to nearest each: 8 + 8 + 8 bits, all of float32's 24 for any finite x up to 3.39e38,
// whatever stands beside it in its row.  A product is the six partial products that are above float32's own rounding (what is
// dropped, mid lo + lo mid + lo lo, is below 2^-24 of it) -- three in dW, as a value of the 8-bit form is exact in bf16 as it is.
// (Two fp16 numbers and three partial products under one power of two per row and column: 272 us for the y below, and what lies 2^-33
// under the largest value of its row was gone, against a weight of zero too.)
//
// Average (least) of ten calls, us.  655360 rows, 256 -> 128, fp32: y and codes 352 (288; 1.18 GB: 3.4 TB/s, six products: 732 TFLOP/s), dx
// 357 (295; 1.0 GB), dW 180 (139; 0.5 GB, three products: 716 TFLOP/s), W laid out 5 - 11, dW's partial sums 5: matrix pipe busy 43 - 48 %
// of the cycles, vector 26 - 41.
// 262144 rows, 256 -> 512, bf16: y and codes 178 (166; 0.47 GB, 386 TFLOP/s), dx 133 (123), dW 106 (96; 648 TFLOP/s): matrix 18, 26, 36 %,
// vector 23, 15, 33 %; what is left of y and dx are waits (a step of K ends at a barrier and at all of its loads).
// Few rows: 32, 512 -> 256, fp32: y 9 (7), dx 5 (5), dW 12 (11).
#include "../../include/gridgcn.h"
#include "gridgcn_act8.h"
#include "gridgcn_mma.h"
#include "gridgcn_once.h"
#include <initializer_list>
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
template <class M, int TN, int PA, int PB>
__device__ __forceinline__ void mul(const gg_u32x4 (&a)[PA], const gg_u32x4 (&b)[TN][PB], F16 (&c)[TN])
{
    auto one = [&](int i, int j) {
#pragma unroll
        for (int t = 0; t < TN; t++) c[t] = M::mfma(a[i], b[t][j], c[t]);
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
            if (k0 + i * VW < K) {
                const GGCol<T> col(k0 + i * VW, K);
                c.load(row, col, K);
                c.align(col);
            }
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
    // Scale byte of the 8-bit form: 16-bit rows, the lane holds a block of 32; 32-bit rows, the two halves hold one together (every
    // lane of the wave calls).  clean: as gg_a8_block_byte
    __device__ __forceinline__ unsigned byte(bool &clean) const
    {
        if constexpr (CH == 32) {
            // 16-bit rows: the largest of the bit patterns, two at a time
            typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
            u16x2 m2 = {0, 0};
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const unsigned u = w[i][j] & 0x7fff7fffu;
                    m2 = __builtin_elementwise_max(m2, __builtin_bit_cast(u16x2, u));
                }
            const unsigned m = m2[0] > m2[1] ? m2[0] : m2[1];
            constexpr bool BF = std::is_same<T, gg_bf16>::value;
            clean = !__any(m >= (BF ? 0x7f80u : 0x7c00u));
            if (clean) return gg_a8_byte(BF ? m << 16 : __float_as_uint(gg_f16of(m, 0)));
        }
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
        clean = !__any(m >= 0x7f800000u);
        if (!clean) m = top(true);
        return gg_a8_byte(m);
    }
    // four values of 16 bits / scale as codes
    static __device__ __forceinline__ unsigned enc(unsigned lo, unsigned hi, float scale)
    {
        typedef short s16x2 __attribute__((ext_vector_type(2)));
        s16x2 r = {0, 0};
        if constexpr (std::is_same<T, gg_f16>::value) {
            r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(gg_f16x2, lo), scale, false);
            r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(gg_f16x2, hi), scale, true);
        } else {
            r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(gg_bf16x2, lo), scale, false);
            r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(gg_bf16x2, hi), scale, true);
        }
        return __builtin_bit_cast(unsigned, r);
    }
    // codes of channels 16 i .. 16 i + 15 of the lane's share
    __device__ __forceinline__ gg_u32x4 codes(int i, unsigned byte, bool clean) const
    {
        gg_u32x4 o;
        if constexpr (CH == 32) {
            if (clean) {                          // two values of 16 bits to two codes in one instruction
                const float scale = gg_a8_scale(byte);
#pragma unroll
                for (int j = 0; j < 4; j++) o[j] = enc(w[2 * i + j / 2][2 * (j & 1)], w[2 * i + j / 2][2 * (j & 1) + 1], scale);
                return o;
            }
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float v[4];
            unsigned w[1];
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = get(16 * i + 4 * j + e);
            gg_a8_encode<4>(v, byte, clean, w);
            o[j] = w[0];
        }
        return o;
    }
};

struct Mm {
    const void *a;             // [R][K] rows, stride lda
    const void *w;             // few rows: TRANS ? [K][N] : [N][K], contiguous
    const char *wp;            // many rows: W in operand order (gg_k_lin8_pack)
    const void *bias;
    void *y;                   // [R][N] contiguous
    uint8_t *codes, *scales;
    long long R, lda;
    int K, N;
    unsigned ncol;             // column blocks
    unsigned nrow;             // row blocks
    bool past;                 // many rows: y around the caches
    bool spread;               // place()
};

// Workgroup -> (row block, column block): workgroups of consecutive numbers go to different XCDs; the column blocks of one row
// block read the same rows, so they get numbers that are 8 apart and share an L2.  With fewer than 64 row blocks, not a multiple
// of 8, that would leave XCDs short of work (one row block: seven of eight idle): then one after the other.
__device__ __forceinline__ bool place(const Mm &p, unsigned &row, unsigned &col)
{
    const unsigned id = blockIdx.x, xcd = id & 7, slot = id >> 3;
    if (p.spread) {
        col = id % p.ncol;
        row = id / p.ncol;
    } else {
        col = slot % p.ncol;
        row = (slot / p.ncol) * 8 + xcd;
    }
    return row < p.nrow;
}
unsigned place_grid(Mm &p)
{
    p.spread = p.nrow < 64 && p.nrow % 8 != 0;
    return (p.spread ? p.nrow : (p.nrow + 7) / 8 * 8) * p.ncol;
}

// ---- W in operand order, for many rows: [column block][step][tile of 32 columns][s][piece][lane], 16 bytes each; zeros behind K and N.
// Tile nt of a column block holds its columns NT * j + nt: a lane's NT results of a row are then neighbours in memory.
// 32-bit: its three pieces.  A workgroup = 32 columns. -----------------------------------------------------------------
constexpr int NT = 4, PT = 512;
template <class T> constexpr int STEP = NT * SS<T> * Ty<T>::P * 1024;          // bytes of a step: 24 KB (32-bit), 16 KB
struct Pk {
    const void *w;
    char *wp;
    int K, N, steps;
};
// 8 consecutive k of column n, zeros outside W (loaded from inside and dropped: eight loads in flight instead of eight branches)
template <class T, bool TRANS> __device__ __forceinline__ void ld8(const T *w, int n, int k, int K, int N, gg_u32x4 (&u)[sizeof(T) / 2])
{
    unsigned v[8];
    const int nn = n < N ? n : N - 1;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const int kk = k + e < K ? k + e : K - 1;
        const T *q = w + (TRANS ? (size_t)kk * N + nn : (size_t)nn * K + kk);
        if constexpr (sizeof(T) == 4) v[e] = *(const unsigned *)q;
        else v[e] = *(const unsigned short *)q;
    }
#pragma unroll
    for (int e = 0; e < 8; e++) {
        if (n >= N || k + e >= K) v[e] = 0u;
        if constexpr (sizeof(T) == 4) u[e / 4][e % 4] = v[e];
        else if (e & 1) u[0][e / 2] = v[e - 1] | (v[e] << 16);
    }
}
template <class T, bool TRANS> __global__ __launch_bounds__(PT) void gg_k_lin8_pack(Pk p)
{
    constexpr int S = SS<T>, P = Ty<T>::P, L = PT / 32;            // L lanes share a column
    const int c = TRANS ? (int)threadIdx.x & 31 : (int)threadIdx.x / L, kl = TRANS ? (int)threadIdx.x >> 5 : (int)threadIdx.x % L;
    const int n = blockIdx.x * 32 + c, groups = p.steps * (KS<T> / 8);
    const int nl = n % (32 * NT), nt = nl % NT, j = nl / NT;
    char *base = p.wp + (size_t)(n / (32 * NT)) * p.steps * STEP<T>;
    for (int g = kl; g < groups; g += L) {
        const int st = g / (KS<T> / 8), gi = g % (KS<T> / 8), h = gi / S, s = gi % S;
        gg_u32x4 u[sizeof(T) / 2], f[P];
        ld8<T, TRANS>((const T *)p.w, n, 8 * g, p.K, p.N, u);
        if constexpr (P == 3) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                unsigned hi, mid, lo;
                split2(__uint_as_float(u[e / 2][2 * (e & 1)]), __uint_as_float(u[e / 2][2 * (e & 1) + 1]), hi, mid, lo);
                f[0][e] = hi; f[1][e] = mid; f[2][e] = lo;
            }
        } else {
            f[0] = u[0];
        }
#pragma unroll
        for (int q = 0; q < P; q++)
            *(gg_u32x4 *)(base + (size_t)st * STEP<T> + ((nt * S + s) * P + q) * 1024 + (h * 32 + j) * 16) = f[q];
    }
}

// y of one row for M neighbouring columns
template <class T, int M> __device__ __forceinline__ void put_row(T *y, long long row, int n, int N, const float (&v)[M], bool past = false)
{
    T *q = y + (size_t)row * N + n;
    if (M == 4 && n + 4 <= N) {
        if constexpr (sizeof(T) == 4) {
            gg_st(q, gg_u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])}, past);
        } else if constexpr (std::is_same<T, gg_bf16>::value) {
            gg_st(q, gg_u32x2{gg_cvt_bf16(v[0], v[1]), gg_cvt_bf16(v[2], v[3])}, past);
        } else {
            gg_st(q, gg_u32x2{gg_cvt_f16(v[0], v[1]), gg_cvt_f16(v[2], v[3])}, past);
        }
    } else {
#pragma unroll
        for (int t = 0; t < M; t++)
            if (n + t < N) GGRowT<T>::put(q + t, v[t]);
    }
}

// ---- many rows: a wave owns 32 rows and 32 NT columns, its rows straight from memory into registers (each row is read by one wave
// only), W through LDS (copied there without passing registers), the next step of both in flight while this one is multiplied;
// three workgroups per CU, so that one's barriers and stores are another's matrix instructions.
// The 8-bit form is held back until 128 bytes of a row are complete: stored as they come, 16 bytes of a line per step, lines left the
// L2 half written and the kernel moved a third more bytes.  The column blocks of one row block take turns at it. ----------------
constexpr int MW = 4;             // waves
template <class T, bool SAVE>
__global__ __launch_bounds__(MW * 64, 3) void gg_k_lin8(Mm p)
{
    constexpr int P = Ty<T>::P, S = SS<T>, PC = Block<T>::CH / 16, GROUP = 128 / KS<T>;      // GROUP steps make 128 codes of a row
    __shared__ __attribute__((aligned(16))) char lds[2][STEP<T>];
    unsigned brow, bcol;
    if (!place(p, brow, bcol)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), h = lane >> 5, j = lane & 31;
    const long long m0 = (long long)brow * (MW * 32) + wave * 32, r = m0 + j;
    const bool live = r < p.R;
    const int Cp = gg_a8_cp(p.K), steps = (p.K + KS<T> - 1) / KS<T>, full = p.K / KS<T>, kh = KS<T> / 2 * h;
    const T *row = (const T *)p.a + (size_t)(live ? r : p.R - 1) * p.lda;
    const char *wp = p.wp + (size_t)bcol * steps * STEP<T> + threadIdx.x * 16;
    F16 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) acc[t] = zero16();
    gg_u32x4 held[4];             // codes of the group so far, the last ones behind
    unsigned heldb = 0;           // ... scale bytes likewise

    auto fetch_w = [&](int st) {
#pragma unroll
        for (int i = 0; i < STEP<T> / (MW * 64 * 16); i++)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(wp + (size_t)st * STEP<T> + i * (MW * 64 * 16)),
                                             (__attribute__((address_space(3))) void *)(&lds[st & 1][i * (MW * 64 * 16) + wave * 1024]), 16, 0, 0);
    };
    auto arrived = [&]() {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    };
    auto step = [&](Block<T> &b, int st) {
        const bool mine = SAVE && (unsigned)(st / GROUP) % p.ncol == bcol;
        if (mine) {
            bool clean;
            const unsigned byte = b.byte(clean);
#pragma unroll
            for (int i = 0; i < 4 - PC; i++) held[i] = held[i + PC];
#pragma unroll
            for (int i = 0; i < PC; i++) held[4 - PC + i] = b.codes(i, byte, clean);
            if constexpr (PC == 1) {
                heldb = (heldb >> 8) | (byte << 24);
            } else {
                const unsigned o = (unsigned)__shfl_xor((int)byte, 32);
                heldb = (heldb >> 16) | ((h ? o | (byte << 8) : byte | (o << 8)) << 16);
            }
            const int in = st % GROUP;                            // place of the step in its group
            if ((in == GROUP - 1 || st == steps - 1) && live) {
                const int k0 = (st - in) * KS<T>;
                uint8_t *q = p.codes + (size_t)r * Cp;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int e = i - (4 - (in + 1) * PC);            // piece of the group
                    const int k = k0 + (PC == 1 ? 32 * e + 16 * h : 64 * (e / 2) + 32 * h + 16 * (e & 1));
                    if (e >= 0 && k < Cp) *(gg_u32x4 *)(q + k) = held[i];
                }
                if (h == 0) {
                    const int have = (in + 1) * PC, left = (Cp - k0) / 32, n = have < left ? have : left;
                    const unsigned w = heldb >> (8 * (4 - have));
                    uint8_t *sq = p.scales + (size_t)r * (Cp / 32) + k0 / 32;
                    if (n == 4) *(gg_u32_a1 *)sq = w;
                    else
                        for (int i = 0; i < n; i++) sq[i] = (uint8_t)(w >> (8 * i));
                }
            }
        }
        const char *cur = lds[st & 1];
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
                    for (int q = 0; q < P; q++) fb[u][q] = *(const gg_u32x4 *)(cur + (((t + u) * S + s) * P + q) * 1024 + lane * 16);
                F16(&two)[2] = *(F16(*)[2])&acc[t];
                mul<Ty<T>>(fa, fb, two);
            }
        }
    };
    Block<T> a, nx;
    fetch_w(0);
    if (full) a.load_full(row + kh);
    arrived();
    for (int st = 0; st < full; st++) {
        if (st + 1 < steps) fetch_w(st + 1);
        if (st + 1 < full) nx.load_full(row + (st + 1) * KS<T> + kh);
        __builtin_amdgcn_sched_barrier(0);              // (loads first)
        step(a, st);
        a = nx;
        arrived();
    }
    if (full < steps) {
        a.load(row, full * KS<T> + kh, p.K);
        step(a, full);
    }
    const int n = ((int)bcol * 32 + j) * NT;
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
        put_row<T, NT>((T *)p.y, o, n, p.N, v, p.past);
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
unsigned v[Block<T>::CH];
#pragma unroll
            for (int i = 0; i < Block<T>::CH; i++) {
                const T *q = w + (size_t)(k0 + i < p.K ? k0 + i : p.K - 1) * p.N + nn;
                if constexpr (sizeof(T) == 4) v[i] = *(const unsigned *)q;
                else v[i] = *(const unsigned short *)q;
            }
#pragma unroll
            for (int i = 0; i < Block<T>::CH; i++) {
                if (k0 + i >= p.K) v[i] = 0u;
                if constexpr (sizeof(T) == 4) b.w[i / 4][i % 4] = v[i];
                else if (i & 1) b.w[i / 8][(i % 8) / 2] = v[i - 1] | (v[i] << 16);
            }
        }
        if (SAVE && bcol == 0) {
            bool clean;
            const unsigned byte = a.byte(clean);
            if (r < p.R && k0 < Cp) {
#pragma unroll
                for (int i = 0; i < Block<T>::CH / 16; i++) *(gg_u32x4 *)(p.codes + (size_t)r * Cp + k0 + 16 * i) = a.codes(i, byte, clean);
                if (k0 % 32 == 0) p.scales[(size_t)r * (Cp / 32) + k0 / 32] = (uint8_t)byte;
            }
        }
#pragma unroll
        for (int s = 0; s < SS<T>; s++) {
            gg_u32x4 fa[P], fb[1][P];
            a.frag(s, fa);
            b.frag(s, fb[0]);
            mul<Ty<T>>(fa, fb, acc);
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
// strips of 16 rows; the waves of a workgroup add up in LDS, the workgroups of a tile through memory in one order.
// What counts here is the number of vector instructions: on a SIMD they take turns with the matrix instructions (5 cycles each
// beside 32 per matrix instruction, measured on both layouts; two waves of 64 x 128 unpack the codes twice and were slower).
constexpr int GT = 128;           // results of a tile per side
constexpr int GW = 4;             // waves
struct Wg {
    const void *dy;               // [R][N], stride ldy
    const uint8_t *codes, *scales; // without dw (tk = 1): any four readable bytes, Cp = 0
    void *dw, *db;                // [N][K], [N]
    float *part;                  // splits > 1: [split][tile][128][128]
    double *dbpart;               // ... [split][tiles_n * 128]
    long long R, ldy;
    int N, K, Cp;
    unsigned tn, tk, splits, share;
};

template <class T> struct Strip {
    static constexpr int DW = sizeof(T) == 4 ? 4 : 2;
    unsigned d[8][DW];                // four columns of dy
    unsigned c[8], s[8];              // four codes; the scale bytes of the tile's four blocks (one word: a loop-carried byte is widened
                                      // at the loop's end, which waits for its load)
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
            s[i] = *(const gg_u32_a1 *)(scales + (size_t)i * (p.Cp / 32) + os);
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
            const T *q = (const T *)p.dy + (size_t)(in ? r : 0) * p.ldy;
#pragma unroll
            for (int t = 0; t < 4; t++) {
                unsigned v;
                const T *e = q + (n + t < p.N ? n + t : 0);
                if constexpr (sizeof(T) == 4) v = *(const unsigned *)e;
                else v = *(const unsigned short *)e;
                if (!in || n + t >= p.N) v = 0u;
                if constexpr (sizeof(T) == 4) d[i][t] = v;
                else d[i][t / 2] = t & 1 ? d[i][t / 2] | (v << 16) : v;
            }
            c[i] = 0u;
            s[i] = 0u;
            if (in && k < p.Cp) {
                c[i] = *(const unsigned *)(p.codes + (size_t)r * p.Cp + k);
                s[i] = (unsigned)p.scales[(size_t)r * nb + k / 32] << (8 * (k / 32 % 4));
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
    // two codes of a row with their scale, as two 16-bit numbers (exact)
    static __device__ __forceinline__ unsigned two(unsigned c, float scale, bool high)
    {
        if constexpr (std::is_same<T, gg_f16>::value) {
            if (high) return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)c, scale, true));
            return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)c, scale, false));
        } else {
            if (high) return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)c, scale, true));
            return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)c, scale, false));
        }
    }
    // bits of 2^E: the lane's byte turned to the exponent's place
    static __device__ __forceinline__ unsigned scale_bits(unsigned w, unsigned turn)
    {
        return (unsigned)__builtin_amdgcn_alignbit(w, w, turn) & 0x7f800000u;
    }
    // fp16 rows: a magnitude of 63488 or more has the 8-bit value 65536 (E = 8), which fp16 does not hold.  Blocks of such a scale enter
    // as two halves of x^ (exact: no value of theirs is below 2^-1 but 0).  big: a scale of the strip may be one (the bits of all together)
    static constexpr unsigned BIG = 135u << 23;
    __device__ __forceinline__ bool big(unsigned turn) const
    {
        unsigned o = s[0];
#pragma unroll
        for (int i = 1; i < 8; i++) o |= s[i];
        return scale_bits(o, turn) >= BIG;
    }
    // the four columns of x^ as operands; `halve`: of BIG blocks the half.  REST: their other half alone
    template <bool REST> __device__ __forceinline__ void frag_x(gg_u32x4 (&f)[4][1], unsigned turn, bool halve) const
    {
        unsigned sc[8], cc[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            sc[i] = scale_bits(s[i], turn);
            cc[i] = REST && sc[i] < BIG ? 0u : c[i];
        }
        if (halve) {
#pragma unroll
            for (int i = 0; i < 8; i++) sc[i] -= sc[i] >= BIG ? 1u << 23 : 0u;
        }
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const float su = __uint_as_float(sc[2 * q]), sv = __uint_as_float(sc[2 * q + 1]);
#pragma unroll
            for (int t = 0; t < 4; t += 2) {
                const unsigned u = two(cc[2 * q], su, t != 0), v = two(cc[2 * q + 1], sv, t != 0);
                f[t][0][q] = gg_pair16(u, v, 0);
                f[t + 1][0][q] = gg_pair16(u, v, 1);
            }
        }
    }
};

template <class T>
__global__ __launch_bounds__(GW * 64, 1) void gg_k_lin8_wgrad(Wg p)
{
    constexpr int P = Ty<T>::P;
    constexpr int D = 3;                                            // strips in registers, one of them in use
    extern __shared__ __attribute__((aligned(16))) float ldsf[];    // [GW][4][16][64]
    // (the tiles of one split read the same rows: one XCD, or `share` of them)
    const unsigned tiles = p.tn * p.tk, per = (tiles + p.share - 1) / p.share, id = blockIdx.x, slot = id >> 3;
    const unsigned unit = (slot / per) * 8 + (id & 7), split = unit / p.share, tile = (unit % p.share) * per + slot % per;
    if (split >= p.splits || tile >= tiles) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), h = lane >> 5, j = lane & 31;
    const int n0 = (int)(tile / p.tk) * GT, k0 = (int)(tile % p.tk) * GT, n = n0 + 4 * j, k = k0 + 4 * j;
    const bool first = tile % p.tk == 0 && p.db;
    const long long strips = (p.R + 15) / 16, stride = (long long)p.splits * GW;
    // Strips that are loaded unchecked.  What a lane reads behind the last column belongs to results that nobody stores (such lanes
    // read the columns from 0 on, and at most three values of dy and three scale bytes behind a row's end: the rows of these strips
    // have four more behind them).
    const long long whole = p.R > 4 ? (p.R - 4) / 16 : 0;
    const unsigned od = (unsigned)((8 * h * p.ldy + (n < p.N ? n : 0)) * (long long)sizeof(T));
    const int kc = k < p.Cp ? k : 0;
    const unsigned oc = (unsigned)(8 * h * p.Cp + kc), os = (unsigned)(8 * h * (p.Cp / 32) + (p.Cp ? k0 / 32 : 0));
    const unsigned turn = (8 * (k / 32 % 4) + 9) & 31;
    F16 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int t = 0; t < 4; t++) acc[i][t] = zero16();
    double dbs[4] = {0.0, 0.0, 0.0, 0.0};                          // (a lane's column over thousands of strips: 64 bits)
    Strip<T> q[D];
    // (never skipped -- past the end a strip is loaded again: behind a load that may or may not have been issued the compiler waits
    //  for everything in flight)
    auto fetch = [&](long long g, Strip<T> &s) {
        const size_t e = (size_t)(g < whole ? g : whole - 1);
        s.load_full(p, (const char *)p.dy + e * 16 * p.ldy * sizeof(T), (const char *)p.codes + e * 16 * p.Cp,
                    (const char *)p.scales + e * 16 * (p.Cp / 32), od, oc, os);
    };
    auto add = [&](const Strip<T> &s, const gg_u32x4 (&fx)[4][1]) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            gg_u32x4 fd[P];
            s.frag_dy(i, fd);
            mul<Ty<T>>(fd, fx, acc[i]);
        }
    };
    bool halved = false;
    auto use = [&](const Strip<T> &s) {
        gg_u32x4 fx[4][1];
        bool halve = false;
        if constexpr (std::is_same<T, gg_f16>::value) {
            halve = __any(s.big(turn));
            halved |= halve;
        }
        s.template frag_x<false>(fx, turn, halve);
        add(s, fx);
        if (first) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float v = s.dyv(0, i);
#pragma unroll
                for (int e = 1; e < 8; e++) v += s.dyv(e, i);
                dbs[i] += (double)v;
            }
        }
    };
    long long g = (long long)split * GW + wave;
    if (g < whole) {
#pragma unroll
        for (int d = 0; d < D - 1; d++) fetch(g + d * stride, q[d]);
        for (; g + (D - 1) * stride < whole; g += D * stride) {
#pragma unroll
            for (int d = 0; d < D; d++) {
                fetch(g + (d + D - 1) * stride, q[(d + D - 1) % D]);
                __builtin_amdgcn_sched_barrier(0);      // (the scheduler put the loads behind the matrix instructions: no overlap at all)
                use(q[d]);
            }
        }
#pragma unroll
        for (int d = 0; d < D - 1; d++) {
            if (g >= whole) continue;
            use(q[d]);
            g += stride;
        }
    }
    for (; g < strips; g += stride) {                             // (the last one or two strips of all)
        Strip<T> s;
        s.load_tail(p, g * 16 + 8 * h, n, k);
        use(s);
    }
    if (halved) {             // (fp16: the strips with BIG blocks once more; 262144 rows, 256 -> 512: 128 us, one in 1000 rows BIG 225)
        for (g = (long long)split * GW + wave; g < strips; g += stride) {
            unsigned top = 0;                                     // (the scales alone: such strips are few)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const long long r = g * 16 + 8 * h + i;
                const unsigned e = r < p.R && k < p.Cp ? p.scales[(size_t)r * (p.Cp / 32) + k / 32] : 0u;
                top = top > e ? top : e;
            }
            if (!__any(top >= Strip<T>::BIG >> 23)) continue;
            Strip<T> s;
            s.load_tail(p, g * 16 + 8 * h, n, k);
            gg_u32x4 fx[4][1];
            s.template frag_x<true>(fx, turn, true);
            add(s, fx);
        }
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
        for (int e = 0; e < 16 / GW; e++) {
            const int r = wave * (16 / GW) + e;
            float v[4];
#pragma unroll
            for (int t = 0; t < 4; t++) {
                v[t] = ldsf[(t * 16 + r) * 64 + lane];
#pragma unroll
                for (int o = 1; o < GW; o++) v[t] += ldsf[((o * 4 + t) * 16 + r) * 64 + lane];
            }
            const int nl = 4 * ggm_row(r, lane) + i;
            if (pt) *(float4 *)(pt + (size_t)nl * GT + 4 * j) = make_float4(v[0], v[1], v[2], v[3]);
            else if (p.dw && n0 + nl < p.N) put_row<T, 4>((T *)p.dw, n0 + nl, k, p.K, v);
        }
    }
    if (!first) return;
    __syncthreads();
    double *ldsd = (double *)ldsf;
#pragma unroll
    for (int i = 0; i < 4; i++) ldsd[(wave * 4 + i) * 64 + lane] = dbs[i];
    __syncthreads();
    if ((int)threadIdx.x < GT) {
        const int jj = threadIdx.x / 4, i = threadIdx.x % 4;
        double v = 0.0;
#pragma unroll
        for (int o = 0; o < GW; o++) v += ldsd[(o * 4 + i) * 64 + jj] + ldsd[(o * 4 + i) * 64 + jj + 32];
        const int nn = n0 + (int)threadIdx.x;
        if (p.part) p.dbpart[(size_t)split * p.tn * GT + nn] = v;
        else if (nn < p.N) GGRowT<T>::put((T *)p.db + nn, (float)v);
    }
}

// sums of the splits: a workgroup = 32 groups of 4 results (db: 32 results, in 64 bits) x 8 lanes over the splits
template <class T>
__global__ __launch_bounds__(256) void gg_k_lin8_wsum(Wg p, unsigned nw)
{
    __shared__ float4 red[8][32];
    const unsigned tiles = p.tn * p.tk;
    const int e = threadIdx.x & 31, l = threadIdx.x >> 5;
    if (blockIdx.x >= nw) {
        __shared__ double redd[8][32];
        const size_t nn = (size_t)(blockIdx.x - nw) * 32 + e;
        double v = 0.0;
#pragma unroll 8
        for (unsigned q = l; q < p.splits; q += 8) v += p.dbpart[q * (size_t)p.tn * GT + nn];
        redd[l][e] = v;
        __syncthreads();
        if (l || nn >= (size_t)p.N) return;
#pragma unroll
        for (int q = 1; q < 8; q++) v += redd[q][e];
        GGRowT<T>::put((T *)p.db + nn, (float)v);
        return;
    }
    const size_t at = ((size_t)blockIdx.x * 32 + e) * 4;
    const size_t stride = (size_t)tiles * GT * GT;
    const float *src = p.part + at;
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
    const unsigned tile = (unsigned)(at / (GT * GT));
    const int rem = (int)(at % (GT * GT)), n = (int)(tile / p.tk) * GT + rem / GT, k = (int)(tile % p.tk) * GT + rem % GT;
    if (n < p.N) put_row<T, 4>((T *)p.dw, n, k, p.K, v);
}

// ---- host side ------------------------------------------------------------------------------------------------------
// Many rows: more than one block of 128, and larger workgroups that fill at least half the CUs; below that smaller ones, their waves on
// the contraction.  Measured (fp32 / bf16 forward, us; few | many):  8192 x 256 -> 128 (64 workgroups) 15 | 28 / 10 | 15;
// 16384 (128) 27 | 30 / 16 | 15;  32768 50 | 32 / 30 | 17;  128 x 256 -> 16384 (one row block: W is laid out for it alone)
// 23 | 37 / 15 | 19;  256 x 512 -> 8192 40 | 48 / 22 | 23.
bool many(long long R, int N) { return R > MW * 32 && (R + MW * 32 - 1) / (MW * 32) * ((N + 32 * NT - 1) / (32 * NT)) >= 128; }
size_t pack_bytes(long long R, int K, int N, int dtype)
{
    if (!many(R, N)) return 0;
    const bool f32 = dtype == GRIDGCN_F32;
    const int ks = f32 ? KS<float> : KS<gg_bf16>;
    const size_t ncol = (N + 32 * NT - 1) / (32 * NT), steps = (K + ks - 1) / ks;
    return ncol * steps * (f32 ? STEP<float> : STEP<gg_bf16>);
}

template <class T, bool TRANS, bool SAVE> void launch_mm(Mm &p, void *ws, hipStream_t st)
{
    if (!many(p.R, p.N)) {
        p.nrow = (unsigned)((p.R + 31) / 32);
        p.ncol = (unsigned)((p.N + 31) / 32);
        gg_k_lin8_few<T, TRANS, SAVE><<<place_grid(p), SW * 64, 0, st>>>(p);
        return;
    }
    p.nrow = (unsigned)((p.R + MW * 32 - 1) / (MW * 32));
    p.ncol = (unsigned)((p.N + 32 * NT - 1) / (32 * NT));
    Pk k = {};
    k.w = p.w; k.wp = (char *)ws; k.K = p.K; k.N = p.N;
    k.steps = (p.K + KS<T> - 1) / KS<T>;
    gg_k_lin8_pack<T, TRANS><<<p.ncol * NT, PT, 0, st>>>(k);
    p.wp = k.wp;
    p.past = gg_past_caches(p.R, p.N, GGRowT<T>::id);
    gg_k_lin8<T, SAVE><<<place_grid(p), MW * 64, 0, st>>>(p);
}

// Splits of the rows for dW: a multiple of 8 (an XCD each), or 1, 2, 4 of which 8, 4, 2 XCDs share the tiles.  A CU holds one workgroup,
// an XCD 32: the fewest splits with the least time in (generations) x (strips of a wave + 6 for summing up), at least four strips
// and at most two generations.  Measured, float32 dW: rows 32768, K = N = 1024 (64 tiles): 4 splits on four XCDs 363 us,
// 8 splits 207;   rows 262144, K = 256, N = 128 (2 tiles): 64 splits 97, 128 splits 66, 256 splits 73.
unsigned splits_of(long long R, unsigned tiles)
{
    const long long most = (R + 16 * GW * 4 - 1) / (16 * GW * 4), strips = R / (16 * GW);
    unsigned best = 1;
    long long least = -1;
    for (unsigned s = 1; s <= 256 && s <= most; s = s < 8 ? s * 2 : s + 8) {
        const long long load = s < 8 ? ((long long)tiles * s + 7) / 8 : (long long)(s / 8) * tiles, gens = (load + 31) / 32;
        const long long time = gens * (strips / s + 6);
        if (gens > 2 && s > 1) break;
        if (least < 0 || time < least) { least = time; best = s; }
    }
    return best;
}

size_t wgrad_bytes(long long R, unsigned tn, unsigned tk)
{
    const unsigned s = splits_of(R, tn * tk);
    return s > 1 ? (size_t)s * ((size_t)tn * tk * GT * GT * sizeof(float) + (size_t)tn * GT * sizeof(double)) : 0;
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
    p.share = p.splits < 8 ? 8 / p.splits : 1;
    const unsigned units = (p.splits * p.share + 7) / 8 * 8;
    gg_k_lin8_wgrad<T><<<units * ((tiles + p.share - 1) / p.share), GW * 64, LDS, st>>>(p);
    if (p.splits > 1) {
        const unsigned nw = p.dw ? tiles * (GT * GT / 128) : 0, nd = p.db ? p.tn * (GT / 32) : 0;
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

int gridgcn_linear_act8_workspace_bytes(long long R, int K, int N, int dtype, int backward, size_t *bytes)
{
    if (!bytes || !sizes_ok(R, K, N) || !type_ok(dtype)) return GRIDGCN_EINVAL;
    if (!backward) {
        *bytes = pack_bytes(R, K, N, dtype);
        return GRIDGCN_OK;
    }
    // (dx, then dW or db alone: one after the other in the same memory)
    const unsigned tn = (N + GT - 1) / GT;
    size_t n = pack_bytes(R, N, K, dtype);
    for (size_t o : {wgrad_bytes(R, tn, (K + GT - 1) / GT), wgrad_bytes(R, tn, 1)}) n = n > o ? n : o;
    *bytes = n;
    return GRIDGCN_OK;
}

int gridgcn_linear_act8_fwd(const void *x, int dtype, long long R, int K, long long ldx, const void *W, const void *bias,
                            int N, void *y, uint8_t *codes, uint8_t *scales, void *ws, size_t ws_bytes, void *stream)
{
    if (!x || !W || !y || !type_ok(dtype) || !sizes_ok(R, K, N) || ldx < K || ldx > GRIDGCN_MAX_LD || !codes != !scales ||
        ((uintptr_t)codes & 15))
        return GRIDGCN_EINVAL;
    const size_t need = pack_bytes(R, K, N, dtype);
    if (need && (!ws || ws_bytes < need || ((uintptr_t)ws & 15))) return GRIDGCN_EWORKSPACE;
    Mm p = {};
    p.a = x; p.w = W; p.bias = bias; p.y = y; p.codes = codes; p.scales = scales; p.R = R; p.lda = ldx; p.K = K; p.N = N;
    const hipStream_t st = (hipStream_t)stream;
    const int rc = with_type(dtype, [&](auto *t) {
        typedef typename std::remove_pointer<decltype(t)>::type T;
        if (codes) launch_mm<T, false, true>(p, ws, st);
        else launch_mm<T, false, false>(p, ws, st);
        return 0;
    });
    if (rc) return rc;
    return hipGetLastError() == hipSuccess ? GRIDGCN_OK : GRIDGCN_ELAUNCH;
}

int gridgcn_linear_act8_bwd(const void *dy, int dtype, long long R, int N, long long ldy, const void *W, int K,
                            const uint8_t *codes, const uint8_t *scales, void *dx, void *dW, void *dbias, void *ws,
                            size_t ws_bytes, void *stream)
{
    if (!dy || !type_ok(dtype) || !sizes_ok(R, K, N) || ldy < N || ldy > GRIDGCN_MAX_LD || (dx && !W) ||
        (dW && (!codes || !scales)) || ((uintptr_t)codes & 15))
        return GRIDGCN_EINVAL;
    Wg g = {};
    g.dy = dy; g.dw = dW; g.db = dbias; g.R = R; g.ldy = ldy; g.N = N; g.K = K;
    g.Cp = dW ? gg_a8_cp(K) : 0;
    g.codes = dW ? codes : (const uint8_t *)dy;
    g.scales = dW ? scales : (const uint8_t *)dy;
    g.tn = (N + GT - 1) / GT;
    g.tk = dW ? (K + GT - 1) / GT : 1;
    g.splits = splits_of(R, g.tn * g.tk);
    size_t need = dx ? pack_bytes(R, N, K, dtype) : 0;
    if (dW || dbias) need = need > wgrad_bytes(R, g.tn, g.tk) ? need : wgrad_bytes(R, g.tn, g.tk);
    if (need && (!ws || ws_bytes < need || ((uintptr_t)ws & 15))) return GRIDGCN_EWORKSPACE;
    if (g.splits > 1) {
        g.part = (float *)ws;
        g.dbpart = (double *)(g.part + (size_t)g.splits * g.tn * g.tk * GT * GT);
    }
    const hipStream_t st = (hipStream_t)stream;
    const int rc = with_type(dtype, [&](auto *t) {
        typedef typename std::remove_pointer<decltype(t)>::type T;
        if (dx) {
            Mm p = {};
            p.a = dy; p.w = W; p.y = dx; p.R = R; p.lda = ldy; p.K = N; p.N = K;
            launch_mm<T, true, false>(p, ws, st);
        }
        return dW || dbias ? launch_wgrad<T>(g, st) : 0;
    });
    if (rc) return rc;
    return hipGetLastError() == hipSuccess ? GRIDGCN_OK : GRIDGCN_ELAUNCH;
}

}  // extern "C"
