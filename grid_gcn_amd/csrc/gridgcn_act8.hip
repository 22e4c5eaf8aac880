// gridgcn_act8.hip -- rows to and from the 8-bit form of gridgcn_act8.h.  Bound by memory: T + 1.03 bytes per value.
// A thread keeps ONE column chunk of 16 bytes and walks rows: no division in the loop, whole lines per wave; the 8 (fp32)
// or 4 (16-bit) neighbouring lanes of a 32-channel block find its maximum with cross-lane moves.
// 655360 rows of fp32: C = 128 pack 80 us (5.3 TB/s), unpack 62 (6.8); C = 131 (rows that start anywhere, codes of 160) 86 (5.2), 111 (4.1).
#include "../../include/gridgcn.h"
#include "gridgcn_act8.h"

namespace {
constexpr int THREADS = 256;
constexpr int UNROLL = 4;           // rows in flight per thread: loads of a batch are issued before the first is used

// threads of a workgroup laid over (row, chunk): tpr chunks of one row, rpb rows (the threads past rpb * tpr idle)
struct Lay { int nq, tpr, rpb; };
Lay lay_of(int nq)
{
    Lay l;
    l.nq = nq;
    l.tpr = nq < THREADS ? nq : THREADS;
    l.rpb = THREADS / l.tpr;
    return l;
}

template <class T>
__global__ __launch_bounds__(THREADS) void gg_k_act8_pack(const T *__restrict__ x, long long R, int C, long long ldx, Lay l,
                                                          uint8_t *__restrict__ codes, uint8_t *__restrict__ scales)
{
    constexpr int V = GGRowT<T>::V;
    const int Cp = gg_a8_cp(C), nb = Cp / GG_A8_BLOCK;
    const int tr = threadIdx.x / l.tpr, q = blockIdx.y * l.tpr + threadIdx.x % l.tpr, c = q * V;
    const bool on = tr < l.rpb && q < l.nq;     // (a chunk behind C: zeros)
    const GGCol<T> col(on ? c : 0, C);
    const long long step = (long long)gridDim.x * l.rpb * UNROLL;
    for (long long r0 = (long long)blockIdx.x * l.rpb * UNROLL; r0 < R; r0 += step) {
        GGChunk<T> in[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            const long long r = r0 + (long long)u * l.rpb + tr;
            in[u].load(x + (r < R ? r : R - 1) * ldx, col, C);          // (rows past the end: encoded, not stored)
        }
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            const long long r = r0 + (long long)u * l.rpb + tr;
            float v[V];
            in[u].align(col);
            in[u].get(v);
            bool clean;
            const unsigned byte = gg_a8_block_byte<V>(v, clean);
            unsigned w[V / 4];
            gg_a8_encode<V>(v, byte, clean, w);
            if (on && r < R) {
                gg_a8_st_codes<V>(codes + r * Cp + c, w);
                if (c % GG_A8_BLOCK == 0) scales[r * nb + c / GG_A8_BLOCK] = (uint8_t)byte;
            }
        }
    }
}

template <class T>
__global__ __launch_bounds__(THREADS) void gg_k_act8_unpack(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales,
                                                            long long R, int C, Lay l, T *__restrict__ x, long long ldx, bool past)
{
    constexpr int V = GGRowT<T>::V;
    const int Cp = gg_a8_cp(C), nb = Cp / GG_A8_BLOCK;
    const int tr = threadIdx.x / l.tpr, q = blockIdx.y * l.tpr + threadIdx.x % l.tpr, c = q * V;
    if (tr >= l.rpb || q >= l.nq) return;
    const long long step = (long long)gridDim.x * l.rpb * UNROLL;
    for (long long r0 = (long long)blockIdx.x * l.rpb * UNROLL + tr; r0 < R; r0 += step) {
        float v[UNROLL][V];
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            const long long r = r0 + (long long)u * l.rpb;
            const long long rr = r < R ? r : R - 1;
            gg_a8_ld<V>(codes + rr * Cp + c, scales + rr * nb + c / GG_A8_BLOCK, v[u]);
        }
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            const long long r = r0 + (long long)u * l.rpb;
            if (r < R) gg_st_chunk(x + r * ldx, c, C, v[u], past);
        }
    }
}

dim3 grid_of(long long R, const Lay &l)
{
    const long long rows = (long long)l.rpb * UNROLL;
    long long g = (R + rows - 1) / rows;
    const long long most = 256 * 16;       // (16 workgroups per CU: eight resident, and a tail that evens out)
    if (g > most) g = most;
    return dim3((unsigned)g, (unsigned)((l.nq + l.tpr - 1) / l.tpr));
}

template <class T> void pack(const void *x, long long R, int C, long long ldx, uint8_t *codes, uint8_t *scales, hipStream_t st)
{
    const Lay l = lay_of(gg_a8_cp(C) / GGRowT<T>::V);
    gg_k_act8_pack<T><<<grid_of(R, l), THREADS, 0, st>>>((const T *)x, R, C, ldx, l, codes, scales);
}
template <class T> void unpack(const uint8_t *codes, const uint8_t *scales, long long R, int C, void *x, long long ldx, hipStream_t st)
{
    const Lay l = lay_of((C + GGRowT<T>::V - 1) / GGRowT<T>::V);
    gg_k_act8_unpack<T><<<grid_of(R, l), THREADS, 0, st>>>(codes, scales, R, C, l, (T *)x, ldx,
                                                                 gg_past_caches(R, C, GGRowT<T>::id));
}
}  // namespace

extern "C" {

int gridgcn_act8_pack(const void *x, int dtype, long long R, int C, long long ldx, uint8_t *codes, uint8_t *scales, void *stream)
{
    if (!x || !codes || !scales || R < 1 || C < 1 || C > GRIDGCN_ACT8_MAX_C || ldx < C || ldx > GRIDGCN_MAX_LD || ((uintptr_t)codes & 15)) return GRIDGCN_EINVAL;
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == GRIDGCN_F32) pack<float>(x, R, C, ldx, codes, scales, st);
    else if (dtype == GRIDGCN_BF16) pack<gg_bf16>(x, R, C, ldx, codes, scales, st);
    else if (dtype == GRIDGCN_F16) pack<gg_f16>(x, R, C, ldx, codes, scales, st);
    else return GRIDGCN_EINVAL;
    return hipGetLastError() == hipSuccess ? GRIDGCN_OK : GRIDGCN_ELAUNCH;
}

int gridgcn_act8_unpack(const uint8_t *codes, const uint8_t *scales, long long R, int C, int dtype, void *x, long long ldx, void *stream)
{
    if (!x || !codes || !scales || R < 1 || C < 1 || C > GRIDGCN_ACT8_MAX_C || ldx < C || ldx > GRIDGCN_MAX_LD || ((uintptr_t)codes & 15)) return GRIDGCN_EINVAL;
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == GRIDGCN_F32) unpack<float>(codes, scales, R, C, x, ldx, st);
    else if (dtype == GRIDGCN_BF16) unpack<gg_bf16>(codes, scales, R, C, x, ldx, st);
    else if (dtype == GRIDGCN_F16) unpack<gg_f16>(codes, scales, R, C, x, ldx, st);
    else return GRIDGCN_EINVAL;
    return hipGetLastError() == hipSuccess ? GRIDGCN_OK : GRIDGCN_ELAUNCH;
}

}  // extern "C"
