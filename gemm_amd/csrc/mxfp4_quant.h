/*
 * mxfp4_quant.h - eight floats per lane to e2m1 codes and a power of two per block of 32 (mxfp4_pack.hip has the rule), for the kernels
 * that make operands and for the one that quantises its own activations.
 */
#ifndef QLIN_MXFP4_QUANT_H
#define QLIN_MXFP4_QUANT_H

#include "mxfp4.h"

namespace qlin {
namespace mxfp4 {

struct Bf16 { uint16_t bits; };

template <class T> struct alignas(16) Eight { T v[8]; };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(Bf16 v) { return __uint_as_float((uint32_t)v.bits << 16); }

/* elements p[0..7], those at `left` and behind as zeros; VEC: p is on 16 bytes and `left` a multiple of 8 */
template <class T, bool VEC> __device__ __forceinline__ void load8(const T *p, int left, float (&x)[8]) {
    if constexpr (VEC) {
        Eight<T> e = {};
        if (left > 0) e = *reinterpret_cast<const Eight<T> *>(p);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = to_f32(e.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            x[i] = 0.0f;
            if (i < left) x[i] = to_f32(p[i]);
        }
    }
}

template <int CTRL> __device__ __forceinline__ uint32_t quad_perm(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true);
}
constexpr int kXor1 = 0xB1, kXor2 = 0x4E; /* lane q of four takes lane q ^ 1, q ^ 2 */

/* four codes in 16 bits to a byte each */
__device__ __forceinline__ uint32_t spread(uint32_t v) {
    v = (v | v << 8) & 0x00FF00FFu;
    return (v | v << 4) & 0x0F0F0F0Fu;
}

/* the four lanes of a block, 8 elements each in order: its exponent (in all four) and this lane's dword of its 16 code bytes, whose
 * place is dword_of(q) */
struct Packed { uint32_t exponent, codes; };
__device__ __forceinline__ int dword_of(int q) { return (q & 1) * 2 + (q >> 1); }
__device__ __forceinline__ Packed pack8(const float (&x)[8], int q) {
    uint32_t m = 0, negative = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t b = __float_as_uint(x[i]);
        m = max(m, b & 0x7FFFFFFFu);
        negative |= (b >> 31) << (4 * i + 3);
    }
    m = max(m, quad_perm<kXor1>(m));
    m = max(m, quad_perm<kXor2>(m));
    const bool not_finite = m >= 0x7F800000u;
    const uint32_t e = not_finite ? 255u : (uint32_t)max((int)(m >> 23) - 2, 0);
    const float power = __uint_as_float(e == 0 ? 0x00400000u : e << 23);
    uint32_t own = 0;
    own = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(own, x[0], x[1], power, 0);
    own = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(own, x[2], x[3], power, 1);
    own = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(own, x[4], x[5], power, 2);
    own = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(own, x[6], x[7], power, 3);
    if (not_finite) own = negative | 0x77777777u;
    /* byte j = element j | element j + 16: lanes 0 and 2 (1 and 3) make bytes 0..7 (8..15) together, the lower one the first four */
    const uint32_t other = quad_perm<kXor2>(own);
    const uint32_t low = q < 2 ? own : other >> 16, high = q < 2 ? other : own >> 16;
    return {e, spread(low & 0xFFFFu) | spread(high & 0xFFFFu) << 4};
}

/* rows that can be read in 16-byte loads */
template <class T> bool reads_wide(const void *X, int n_cols, int ldx) {
    return (reinterpret_cast<uintptr_t>(X) & 15) == 0 && n_cols % 8 == 0 && (size_t)ldx * sizeof(T) % 16 == 0;
}

}  // namespace mxfp4
}  // namespace qlin
#endif
