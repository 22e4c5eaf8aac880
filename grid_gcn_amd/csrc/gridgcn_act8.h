// gridgcn_act8.h -- rows of 32-, 16- and 8-bit activations: vector access, and the 8-bit form of a row that the
// training layers keep between forward and backward.
//
// The 8-bit form: every 32 consecutive channels of a row share one power of two 2^E, the smallest with
// max |x| <= 448 * 2^E (448: the largest e4m3 number), E >= -117; a channel is the e4m3 number nearest to x * 2^-E.
//   * a power of two: scaling and unscaling are exact, the one rounding is the e4m3 conversion (half a step: 2^-4 of the
//     value, or 2^-10 * 2^E where the value is below 2^-6 * 2^E);
//   * a value has 4 significant bits and (E >= -117) is never a subnormal float32: it is EXACT in bf16, and in fp16 when x
//     was fp16 (x is a multiple of 2^-24, and so is its rounding to 4 bits) -- so it enters a bf16 / fp16 matrix instruction
//     without a second rounding.  One exception: an fp16 magnitude of 63488 or more rounds to 65536, infinite as an fp16;
//   * infinities and NaN become NaN and do not take part in the maximum; a magnitude above 3.29e38 rounds to 2^128, which
//     is infinite as a float32.
// Layout: codes [rows][Cp], Cp = C rounded up to 32 (the padding holds zeros: rows start on 32 bytes whatever C is),
// scales [rows][Cp / 32] with byte E + 127.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#define GG_T_F32 0
#define GG_T_BF16 1
#define GG_T_F16 2

typedef __bf16 gg_bf16;
typedef _Float16 gg_f16;
typedef unsigned gg_u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned gg_u32x2 __attribute__((ext_vector_type(2)));
// the same as memory operands that are only as aligned as an element of a row is (a row may start anywhere; the
// hardware's vector loads take that)
typedef gg_u32x4 gg_u32x4_a4 __attribute__((aligned(4)));
typedef gg_u32x4 gg_u32x4_a2 __attribute__((aligned(2)));
typedef gg_u32x2 gg_u32x2_a2 __attribute__((aligned(2)));
typedef unsigned gg_u32_a1 __attribute__((aligned(1)));
typedef unsigned gg_u32_a2 __attribute__((aligned(2)));

__device__ __forceinline__ float gg_lo16f(unsigned u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float gg_hi16f(unsigned u) { return __uint_as_float(u & 0xffff0000u); }
// two floats -> two bf16 / fp16 of one register, to nearest even (the compiler's conversion: v_cvt_pk_*)
typedef float gg_pair __attribute__((ext_vector_type(2)));
typedef gg_bf16 gg_bf16x2 __attribute__((ext_vector_type(2)));
typedef gg_f16 gg_f16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ unsigned gg_cvt_bf16(float a, float b)
{
    const gg_pair v = {a, b};
    return __builtin_bit_cast(unsigned, __builtin_convertvector(v, gg_bf16x2));
}
__device__ __forceinline__ unsigned gg_cvt_f16(float a, float b)
{
    const gg_pair v = {a, b};
    return __builtin_bit_cast(unsigned, __builtin_convertvector(v, gg_f16x2));
}
// (by value: __builtin_bit_cast of an ELEMENT of a vector takes element 0)
__device__ __forceinline__ float gg_f16of(unsigned u, int i) { return (float)__builtin_bit_cast(gg_f16x2, u)[i]; }

// Results that no cache can hold are stored around them (`past`): what an ordinary store leaves dirty is written back while the
// next pass reads.  Forward and backward of a group normalisation, and a pass over its output, fp32 rows of 128:
//   336 MB   518 -> 473 us, forward + scaling it 314 -> 308, + sum of it 286 -> 274;    268 MB   413 -> 376, 256 -> 248, 240 -> 222
//   134 MB   203 -> 187,                         128 -> 123,             106 -> 114;     67 MB   104 -> 105,  61 ->  64,  61 ->  68
// so the border is where the reader of the result would find little of it in the 256 MB of the last cache anyway.
static inline bool gg_past_caches(long long rows, long long C, int dtype)
{
    return rows * C >= (192ll << 20) / (dtype == GG_T_F32 ? 4 : 2);
}
// one store of a 16- or 8-byte vector that is aligned to an element of T
#define GG_STORE(TYPE)                                                                                              \
    if (past) {                                                                                                     \
        asm volatile("");              /* keep the two stores apart: merged, they are an ordinary one */            \
        __builtin_nontemporal_store(v, (TYPE *)p);                                                                  \
        asm volatile("");                                                                                           \
    } else {                                                                                                        \
        *(TYPE *)p = v;                                                                                             \
    }
template <class T> __device__ __forceinline__ void gg_st(T *p, gg_u32x4 v, bool past)
{
    if constexpr (sizeof(T) == 4) { GG_STORE(gg_u32x4_a4) }
    else { GG_STORE(gg_u32x4_a2) }
}
template <class T> __device__ __forceinline__ void gg_st(T *p, gg_u32x2 v, bool past) { GG_STORE(gg_u32x2_a2) }
#undef GG_STORE

// ---- rows of T, 16 bytes at a time: V channels ----------------------------------------------------------------------
template <class T> struct GGRowT;
template <> struct GGRowT<float> {
    static constexpr int V = 4, id = GG_T_F32;
    static __device__ __forceinline__ void st(float *p, const float (&v)[4], bool past)
    {
        gg_u32x4 u;
#pragma unroll
        for (int i = 0; i < 4; i++) u[i] = __float_as_uint(v[i]);
        gg_st(p, u, past);
    }
    static __device__ __forceinline__ float get(const float *p) { return *p; }
    static __device__ __forceinline__ void put(float *p, float v) { *p = v; }
};
template <> struct GGRowT<gg_bf16> {
    static constexpr int V = 8, id = GG_T_BF16;
    static __device__ __forceinline__ void st(gg_bf16 *p, const float (&v)[8], bool past)
    {
        gg_u32x4 u;
#pragma unroll
        for (int i = 0; i < 4; i++) u[i] = gg_cvt_bf16(v[2 * i], v[2 * i + 1]);
        gg_st(p, u, past);
    }
    static __device__ __forceinline__ float get(const gg_bf16 *p) { return __uint_as_float((unsigned)*(const unsigned short *)p << 16); }
    static __device__ __forceinline__ void put(gg_bf16 *p, float v) { *(unsigned short *)p = (unsigned short)gg_cvt_bf16(v, 0.f); }
};
template <> struct GGRowT<gg_f16> {
    static constexpr int V = 8, id = GG_T_F16;
    static __device__ __forceinline__ void st(gg_f16 *p, const float (&v)[8], bool past)
    {
        gg_u32x4 u;
#pragma unroll
        for (int i = 0; i < 4; i++) u[i] = gg_cvt_f16(v[2 * i], v[2 * i + 1]);
        gg_st(p, u, past);
    }
    static __device__ __forceinline__ float get(const gg_f16 *p) { return (float)*p; }
    static __device__ __forceinline__ void put(gg_f16 *p, float v) { *(unsigned short *)p = (unsigned short)gg_cvt_f16(v, 0.f); }
};

// V channels of a row from channel c on; what lies past C is left alone
template <class T> __device__ __forceinline__ void gg_st_chunk(T *row, int c, int C, const float (&v)[GGRowT<T>::V], bool past)
{
    constexpr int V = GGRowT<T>::V;
    if (c + V <= C) {
        GGRowT<T>::st(row + c, v, past);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (c + i < C) GGRowT<T>::put(row + c + i, v[i]);
    }
}

// A thread's column: the V channels from c on.  It loads the V channels from `at` on, which end with the row at the latest, and
// drops the first `drop` of them afterwards: the last chunk of a row costs no branch around its loads (a batch of loads with
// branches between them goes out one by one).
template <class T> struct GGCol {
    int at, drop;
    bool narrow;                              // rows shorter than a chunk: by element
    __device__ __forceinline__ GGCol(int c, int C)
    {
        constexpr int V = GGRowT<T>::V;
        narrow = C < V;
        at = narrow || c + V <= C ? c : C - V;
        drop = c - at < V ? c - at : V;
    }
};

// a chunk as it stands in memory: 4 registers until it is used
template <class T> struct GGChunk {
    gg_u32x4 w;
    __device__ __forceinline__ void load(const T *row, const GGCol<T> &k, int C)
    {
        constexpr int V = GGRowT<T>::V;
        if (!k.narrow) {
            if constexpr (V == 4) w = *(const gg_u32x4_a4 *)(row + k.at);
            else w = *(const gg_u32x4_a2 *)(row + k.at);
        } else {
            w = gg_u32x4{0u, 0u, 0u, 0u};
#pragma unroll
            for (int i = 0; i < V - 1; i++) {
                if (k.at + i >= C) continue;
                if constexpr (V == 4) w[i] = ((const unsigned *)row)[k.at + i];
                else w[i / 2] |= (unsigned)((const unsigned short *)row)[k.at + i] << (16 * (i & 1));
            }
        }
    }
    // what `load` read, from the column's first channel on; zeros past the row's end
    __device__ __forceinline__ void align(const GGCol<T> &k)
    {
        constexpr int V = GGRowT<T>::V;
        if (!k.drop) return;
        int n = k.drop;
        if constexpr (V == 8) {
            if (n & 1) {
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] = (w[i] >> 16) | (i < 3 ? w[(i + 1) & 3] << 16 : 0u);
            }
            n >>= 1;
        }
        if (n & 1) w = gg_u32x4{w[1], w[2], w[3], 0u};
        if (n & 2) w = gg_u32x4{w[2], w[3], 0u, 0u};
        if (n & 4) w = gg_u32x4{0u, 0u, 0u, 0u};
    }
    __device__ __forceinline__ void zero() { w = gg_u32x4{0u, 0u, 0u, 0u}; }
    __device__ __forceinline__ void get(float (&v)[GGRowT<T>::V]) const
    {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (GGRowT<T>::id == GG_T_F32) v[i] = __uint_as_float(w[i]);
            else if constexpr (GGRowT<T>::id == GG_T_BF16) { v[2 * i] = gg_lo16f(w[i]); v[2 * i + 1] = gg_hi16f(w[i]); }
            else { v[2 * i] = gg_f16of(w[i], 0); v[2 * i + 1] = gg_f16of(w[i], 1); }
        }
    }
};

// a parameter vector of either type; none: the given value
__device__ __forceinline__ float gg_ld_param(const void *p, int ptype, int i, float none)
{
    if (!p) return none;
    if (ptype == GG_T_F32) return ((const float *)p)[i];
    if (ptype == GG_T_BF16) return GGRowT<gg_bf16>::get((const gg_bf16 *)p + i);
    return GGRowT<gg_f16>::get((const gg_f16 *)p + i);
}
__device__ __forceinline__ void gg_st_param(void *p, int ptype, size_t i, float v)
{
    if (ptype == GG_T_F32) ((float *)p)[i] = v;
    else if (ptype == GG_T_BF16) GGRowT<gg_bf16>::put((gg_bf16 *)p + i, v);
    else GGRowT<gg_f16>::put((gg_f16 *)p + i, v);
}

// ---- the 8-bit form -------------------------------------------------------------------------------------------------
#define GG_A8_BLOCK 32
#define GG_A8_MIN_BYTE 10          // E = -117
static inline __host__ __device__ int gg_a8_cp(int C) { return (C + GG_A8_BLOCK - 1) & ~(GG_A8_BLOCK - 1); }

// magnitude of x for the maximum of a block: its bits without the sign, 0 where x is not finite
__device__ __forceinline__ unsigned gg_a8_mag(float x)
{
    const unsigned u = __float_as_uint(x) & 0x7fffffffu;
    return u < 0x7f800000u ? u : 0u;
}
// scale byte of a block from the bits of its largest magnitude 1.m * 2^(e - 127): 448 = 1.75 * 2^8
__device__ __forceinline__ unsigned gg_a8_byte(unsigned amax)
{
    const int b = (int)(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
    return (unsigned)(b > GG_A8_MIN_BYTE ? b : GG_A8_MIN_BYTE);
}
__device__ __forceinline__ float gg_a8_scale(unsigned byte) { return __uint_as_float(byte << 23); }          // 2^E
__device__ __forceinline__ float gg_a8_unscale(unsigned byte) { return __uint_as_float((254u - byte) << 23); } // 2^-E
// x * 2^-E, NaN where x is not finite (an infinity would saturate or not by a mode of the converter)
__device__ __forceinline__ float gg_a8_ready(float x, float unscale)
{
    return (__float_as_uint(x) & 0x7fffffffu) < 0x7f800000u ? x * unscale : __uint_as_float(0x7fc00000u);
}
__device__ __forceinline__ unsigned gg_a8_enc4(float a, float b, float c, float d)
{
    int w = 0;
    w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, w, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    return (unsigned)w;
}
// (without the scale)
__device__ __forceinline__ void gg_a8_dec4(unsigned w, float &a, float &b, float &c, float &d)
{
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    a = lo[0]; b = lo[1]; c = hi[0]; d = hi[1];
}

// V channels of one block, the other 32 / V - 1 lanes of the block beside this one: its scale byte.  Every lane of the wave
// takes part (lanes without data pass zeros).  clean: no value of the WAVE is infinite or NaN, which saves the tests on each
// (the largest bit pattern tells); where one is, all lanes look again at the finite ones only.
template <int V> __device__ __forceinline__ unsigned gg_a8_block_max(unsigned m)
{
#pragma unroll
    for (int d = 1; d < GG_A8_BLOCK / V; d *= 2) {
        const unsigned o = (unsigned)__shfl_xor((int)m, d);
        m = m > o ? m : o;
    }
    return m;
}
template <int V> __device__ __forceinline__ unsigned gg_a8_block_byte(const float (&v)[V], bool &clean)
{
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < V; i++) {
        const unsigned u = __float_as_uint(v[i]) & 0x7fffffffu;
        m = m > u ? m : u;
    }
    m = gg_a8_block_max<V>(m);
    clean = !__any(m >= 0x7f800000u);
    if (!clean) {
        m = 0;
#pragma unroll
        for (int i = 0; i < V; i++) {
            const unsigned u = gg_a8_mag(v[i]);
            m = m > u ? m : u;
        }
        m = gg_a8_block_max<V>(m);
    }
    return gg_a8_byte(m);
}
template <int V> __device__ __forceinline__ void gg_a8_encode(const float (&v)[V], unsigned byte, bool clean, unsigned (&w)[V / 4])
{
    const float s = gg_a8_unscale(byte);
    if (clean) {
#pragma unroll
        for (int i = 0; i < V / 4; i++) w[i] = gg_a8_enc4(v[4 * i] * s, v[4 * i + 1] * s, v[4 * i + 2] * s, v[4 * i + 3] * s);
    } else {
#pragma unroll
        for (int i = 0; i < V / 4; i++)
            w[i] = gg_a8_enc4(gg_a8_ready(v[4 * i], s), gg_a8_ready(v[4 * i + 1], s), gg_a8_ready(v[4 * i + 2], s), gg_a8_ready(v[4 * i + 3], s));
    }
}
template <int V> __device__ __forceinline__ void gg_a8_st_codes(uint8_t *p, const unsigned (&w)[V / 4])
{
    if constexpr (V == 4) *(unsigned *)p = w[0];
    else *(gg_u32x2 *)p = gg_u32x2{w[0], w[1]};
}
// V channels of a block as they stand in memory
template <int V> struct GGCodes {
    unsigned w[V / 4], byte;
    __device__ __forceinline__ void load(const uint8_t *codes, const uint8_t *scale)
    {
        if constexpr (V == 4) w[0] = *(const unsigned *)codes;
        else { const gg_u32x2 u = *(const gg_u32x2 *)codes; w[0] = u[0]; w[1] = u[1]; }
        byte = *scale;
    }
    __device__ __forceinline__ void zero()
    {
#pragma unroll
        for (int i = 0; i < V / 4; i++) w[i] = 0u;
        byte = GG_A8_MIN_BYTE;
    }
    __device__ __forceinline__ void get(float (&v)[V]) const
    {
        const float s = gg_a8_scale(byte);
#pragma unroll
        for (int i = 0; i < V / 4; i++) {
            float a, b, c, d;
            gg_a8_dec4(w[i], a, b, c, d);
            v[4 * i] = a * s; v[4 * i + 1] = b * s; v[4 * i + 2] = c * s; v[4 * i + 3] = d * s;
        }
    }
};
template <int V> __device__ __forceinline__ void gg_a8_ld(const uint8_t *codes, const uint8_t *scale, float (&v)[V])
{
    GGCodes<V> c;
    c.load(codes, scale);
    c.get(v);
}
