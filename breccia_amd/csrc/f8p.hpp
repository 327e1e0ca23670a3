// The e4m3 layout (BKV_LAYOUT_F8P): how a page lies in memory, and the arithmetic of its codes.
//
// A unit is one (page, kv head) of K or of V: 16 cells x 256 values, a byte each, 4096 bytes.  Its values share one scale, a
// power of two 2^e.  A power of two loses nothing against any other scale -- codes are floating point, their relative step
// is the same wherever the page's largest value falls within the last binade -- and makes exact what a cache does with its
// rows later: a value coded again under another scale is the same number unless it falls among the subnormal codes.
//
// A K page is n_kv units and then one 128-byte line with the exponents of K and V, int32 [kv head][2]; a V page is n_kv units.
//
// Both units keep their cells in blocks of four, 1024 bytes each (what a selection list picks is one run of memory), and
// inside a block the bytes stand as the matrix cores take them, so that the attention kernels load operands straight from
// memory, 16 bytes a lane and 256 bytes in one piece an instruction:
//   K  byte 64 s + 16 (cell % 4) + 4 u + k     for element 128 (s / 8) + 32 u + 4 (s % 8) + k,  s < 16, u and k < 4
//   V  byte 4 d + cell % 4                     for element d
// K: the lane that has 16 bytes of row c and piece s has two 8-element shares of a contraction over the head dim (q is put in the
// same order).  V: a dword is one column of four cells, a lane's 16 bytes four columns: its share of P.V.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace bkv {

constexpr int kF8Hd = 256, kF8Page = 16, kF8Waves = 4;
constexpr int kF8Unit = kF8Hd * kF8Page;  // bytes
constexpr int kF8Line = 128;              // of a K page, behind its units
constexpr int kF8ExpLo = -32, kF8ExpHi = 31;
constexpr float kF8Top = 448.0f;
constexpr float kF8Finite = 0x1.fffffep+127f;

typedef unsigned f8_u4 __attribute__((ext_vector_type(4)));
typedef float f8_f2 __attribute__((ext_vector_type(2)));
typedef int f8_i2 __attribute__((ext_vector_type(2)));

__host__ __device__ inline size_t f8p_k_page_bytes(int n_kv) { return (size_t)n_kv * kF8Unit + kF8Line; }
__host__ __device__ inline size_t f8p_v_page_bytes(int n_kv) { return (size_t)n_kv * kF8Unit; }

// the smallest e of the range with amax <= 448 * 2^e (amax >= 0 and finite); the largest where none is
__device__ __forceinline__ int f8p_exponent(float amax) {
    const uint32_t b = __float_as_uint(amax);
    const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(max(e, kF8ExpLo), kF8ExpHi);
}
// An exponent as it is read: whatever the line holds, one of the range.  (Pools are zeroed at creation: a scale of 1.)
__device__ __forceinline__ int f8p_exponent_read(int e) { return min(max(e, kF8ExpLo), kF8ExpHi); }
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

__device__ __forceinline__ float amax_finite(float a, float x) {
    const float m = fabsf(x);
    return fmaxf(a, m <= kF8Finite ? m : 0.0f);
}

// Four values as codes, `inv` the reciprocal of the scale: rounded once (the product with a power of two is exact, or so small
// that its code is 0), beyond the range the largest code, NaN for what is not finite.
__device__ __forceinline__ unsigned f8p_codes4(const float (&x)[4], float inv) {
#pragma clang fp contract(off)
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = fabsf(x[i]) <= kF8Finite ? fminf(fmaxf(x[i] * inv, -kF8Top), kF8Top) : __builtin_nanf("");
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
}
__device__ __forceinline__ void f8p_values4(unsigned w, float scale, float (&x)[4]) {
    const f8_f2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    x[0] = a[0] * scale, x[1] = a[1] * scale, x[2] = b[0] * scale, x[3] = b[1] * scale;
}

}  // namespace bkv
