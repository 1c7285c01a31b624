// The 8-bit paged cache: an element is an e4m3 value (1 sign, 4 exponent, 3 fraction bits; largest 448;
// 0x7f and 0xff are NaN, there are no infinities) that stands for itself times the 32-bit scale of its
// page and KV head.
#pragma once

#include "common.cuh"

namespace dvb {

// Two e4m3 values, the low 16 bits of x, as f16 (exact: f16 holds every e4m3 value).
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t x) {
    uint32_t r;
    asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %1;\n cvt.rn.f16x2.e4m3x2 %0, l;\n}\n" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ uint32_t e4m3x2_hi_to_f16x2(uint32_t x) {
    uint32_t r;
    asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %1;\n cvt.rn.f16x2.e4m3x2 %0, h;\n}\n" : "=r"(r) : "r"(x));
    return r;
}
// Two f32 values rounded to e4m3 (to nearest even, NaN stays NaN; |x| <= 448 or NaN), lo in the low byte.
__device__ __forceinline__ uint32_t f32x2_to_e4m3x2(float lo, float hi) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
// Bit 7 of every byte of x that is an e4m3 NaN.
__device__ __forceinline__ uint32_t e4m3_nan(uint32_t x) { return ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// Bytes of x whose bit 7 is set in `flags` replaced by zeros.
__device__ __forceinline__ uint32_t clear_bytes(uint32_t x, uint32_t flags) {
    const uint32_t m = flags >> 7;  // 1 in each flagged byte
    return x & ~(m * 255u);
}

// Elements [e0, e0 + 8) of a row, and of a row rotated by its angles: element e < R / 2 pairs with e + R / 2,
// products and sum rounded separately, the result rounded to T (the other elements as they are).  FULL: the
// angle of element e is entry e of cos and sin (keys, as the paged append rotates them), else e mod R / 2
// (queries: the first half of the row).  vec: the rotary halves are whole groups of 8, cos / sin rows 16-byte
// aligned.
template <class T> __device__ __forceinline__ void load8(const T* x, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(x)), b = __ldg(reinterpret_cast<const float4*>(x) + 1);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        const uint4 a = __ldg(reinterpret_cast<const uint4*>(x));
        const T* y = reinterpret_cast<const T*>(&a);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = Elem<T>::to_f(y[i]);
    }
}
template <class T, bool FULL>
__device__ __forceinline__ void rotated8(const T* x, const float* cr, const float* sr, int e0, int R, bool vec, float (&v)[8]) {
    load8(x + e0, v);
    if (e0 >= R) return;
    const int h = R >> 1;
    if (vec) {
        const bool lo = e0 < h;
        float y[8], c[8], s[8];
        const int j = FULL || lo ? e0 : e0 - h;
        load8(x + (lo ? e0 + h : e0 - h), y);
        load8(cr + j, c);
        load8(sr + j, s);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = Elem<T>::to_f(Elem<T>::from_f(__fadd_rn(__fmul_rn(v[i], c[i]), __fmul_rn(lo ? -y[i] : y[i], s[i]))));
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int e = e0 + i;
        if (e >= R) break;
        const int j = FULL || e < h ? e : e - h;
        const float y = e < h ? -Elem<T>::to_f(x[e + h]) : Elem<T>::to_f(x[e - h]);
        v[i] = Elem<T>::to_f(Elem<T>::from_f(__fadd_rn(__fmul_rn(v[i], __ldg(cr + j)), __fmul_rn(y, __ldg(sr + j)))));
    }
}

}  // namespace dvb
