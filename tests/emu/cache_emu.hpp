// TEST INFRASTRUCTURE: what the kernels of the 4-bit cache use beyond amdgcn_emu.hpp, as plain C++.
#pragma once

#include "hip/hip_runtime.h"

#include <math.h>

// ---- the matrix instruction of 16 x 16 x 32: lane l holds, of A and of B, row or column l % 16, terms 8 (l / 16) .. + 7, and gets rows
// 4 (l / 16) .. + 3 of column l % 16.  Numbers below the normal range count at their value, as in the matrix unit.
struct emu_operands {
    float a[2][64][8], b[2][64][8];   // (two sets: a lane may be at its next product before the last one has read this one's)
};
extern thread_local emu_operands emu_products;
typedef float emu_f32x4 __attribute__((ext_vector_type(4)));
inline emu_f32x4 emu_mfma_16x16x32(unsigned site, const float *a, const float *b, emu_f32x4 c)
{
    const unsigned p = emu_cur->parity++ & 1u;
    memcpy(emu_products.a[p][emu_lane], a, sizeof(float) * 8);
    memcpy(emu_products.b[p][emu_lane], b, sizeof(float) * 8);
    emu_meet(site, (int)p);
    const int n = emu_lane & 15, g = emu_lane >> 4;
    for (int r = 0; r < 4; ++r) {
        float sum = c[r];
        for (int k = 0; k < 32; ++k) sum += emu_products.a[p][(4 * g + r) + 16 * (k >> 3)][k & 7] * emu_products.b[p][n + 16 * (k >> 3)][k & 7];
        c[r] = sum;
    }
    return c;
}
inline float emu_widen(_Float16 v) { return (float)v; }
inline float emu_widen(__bf16 v)
{
    uint16_t bits;
    memcpy(&bits, &v, 2);
    const uint32_t wide = (uint32_t)bits << 16;
    float f;
    memcpy(&f, &wide, 4);
    return f;
}
template <typename V>
inline emu_f32x4 emu_mfma_of(unsigned site, V a, V b, emu_f32x4 c, int, int, int)
{
    float x[8], y[8];
    for (int i = 0; i < 8; ++i) x[i] = emu_widen(a[i]), y[i] = emu_widen(b[i]);
    return emu_mfma_16x16x32(site, x, y, c);
}
#define __builtin_amdgcn_mfma_f32_16x16x32_f16(...) emu_mfma_of(__LINE__, __VA_ARGS__)
#define __builtin_amdgcn_mfma_f32_16x16x32_bf16(...) emu_mfma_of(__LINE__, __VA_ARGS__)

// to nearest, ties to even; a NaN stays one
inline uint32_t emu_f32_to_bf16(float x)
{
    uint32_t u;
    memcpy(&u, &x, 4);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (u >> 16) | 0x40u;
    return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
}
template <typename T>
inline T emu_shfl(unsigned site, T v, int src)
{
    uint64_t bits = 0;
    memcpy(&bits, &v, sizeof(T));
    const uint64_t got = emu_exchange(site, bits, src & 63);
    T out;
    memcpy(&out, &got, sizeof(T));
    return out;
}
#define __shfl(v, src, width) emu_shfl(__LINE__, v, src)
#define __builtin_amdgcn_exp2f(x) exp2f(x)
#define __builtin_amdgcn_logf(x) log2f(x)
#define __builtin_amdgcn_sched_barrier(x) ((void)0)
#define __builtin_amdgcn_rcpf(x) (1.0f / (x))
#define __builtin_amdgcn_fractf(x) ((x) - floorf(x))
inline uint32_t atomicAdd(uint32_t *p, uint32_t v) { return __atomic_fetch_add(p, v, __ATOMIC_SEQ_CST); }
