// What the attention kernels over e4m3 pages (f8p.hpp) share: a wave that walks pages two at a time with tiles of 16 query rows.
//
//   S^T[cell][row] = K[cell][:] . Q[row][:]      v_mfma_f32_16x16x32_f16, A = K (codes as f16, exact), B = q
//   z              = S^T * 2^(e_K) + e_V          base-2 logits plus the exponent of the page's V
//   w              = exp2(z - M)                  M: a running maximum of z, moved when it is passed by more than kF8Slack
//   O^T[d][row]   += V^T[d][cell] . w[cell][row]  A = V (codes as f16, exact), 32 cells of two pages a product
//   l             += w * 2^(-e_V)
//
// So the scale of K is a factor of the page's scores and that of V rides on the weights: the largest terms have weights near 1
// whatever the magnitude of their values, pages of different scales meet in one product, and out = O / l with both relative to
// M.  Exponents lie in -32 .. 31, which keeps the terms of l below 2^(kF8Slack + 32 + log2 of the cells) and its largest one
// above 2^-70.
//
// q and the weights enter as the sum of two f16 numbers (two products each): 22 bits and more.  q's row is brought to a largest
// value of 2^13 .. 2^14 first, by a power of two that rejoins the scale of K: neither part leaves what f16 can hold, whatever the
// queries' size.  The sums are f32, in the matrix cores.
//
// A lane (c = lane % 16, g = lane / 16) holds of a tile row c, and cells 4 g .. 4 g + 3 of either page: weights come out of the
// softmax in the order the second product takes them in.
#pragma once

#include <hip/hip_runtime.h>

#include "f8p.hpp"
#include "lane_groups.hpp"

namespace bkv {

typedef _Float16 f8_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 f8_h2 __attribute__((ext_vector_type(2)));
typedef float f8_f4 __attribute__((ext_vector_type(4)));

constexpr float kF8Slack = 6.0f;

__device__ __forceinline__ f8_f4 f8_mfma(f8_h8 a, f8_h8 b, f8_f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// 4 + 4 codes as f16 numbers; the conversion is exact (e4m3's subnormals are f16 normals), NaN stays NaN
__device__ __forceinline__ f8_h8 f8_to_f16(unsigned a, unsigned b) {
    const f8_h2 p = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)a, 1.0f, false), q = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)a, 1.0f, true);
    const f8_h2 r = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)b, 1.0f, false), s = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)b, 1.0f, true);
    return f8_h8{p[0], p[1], q[0], q[1], r[0], r[1], s[0], s[1]};
}

// One row of q (already known to be readable) as the B operand of eight 32-deep products, in the order of K's pieces; rows of
// other lane groups c hold other rows.  Returns the power of two its values were multiplied by, as an exponent.
__device__ __forceinline__ int f8_split_q(const float* row, bool live, float scale_log2e, int g, f8_h8 (&hi)[8], f8_h8 (&lo)[8]) {
    f8_f4 raw[8][2];
#pragma unroll
    for (int f = 0; f < 8; ++f) {
        const int s = 4 * (f >> 1) + g;
        const float* const at = row + 128 * (s >> 3) + 4 * (s & 7) + 64 * (f & 1);
        raw[f][0] = *reinterpret_cast<const f8_f4*>(at);
        raw[f][1] = *reinterpret_cast<const f8_f4*>(at + 32);
    }
    float top = 0.0f;
#pragma unroll
    for (int f = 0; f < 8; ++f)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float x = raw[f][j >> 2][j & 3] * scale_log2e;
            x = live ? x : 0.0f;
            asm("" : "+v"(x));  // an f32 number: not fused into what follows
            raw[f][j >> 2][j & 3] = x;
            top = fmaxf(top, fabsf(x));
        }
    top = max_over_lane_groups(top);
    const int up = min(max(13 - ((int)(__float_as_uint(top) >> 23) - 127), -126), 126);
    const float by = exp2_int(up);
#pragma unroll
    for (int f = 0; f < 8; ++f)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float x = raw[f][j >> 2][j & 3] * by;
            hi[f][j] = (_Float16)x;
            lo[f][j] = (_Float16)(x - (float)hi[f][j]);
        }
    return up;
}

// The factor of a page's scores: 2^(e_K - up), kept among the normal numbers (beyond them the logits are far past f32's
// range, or all but zero, either way).
__device__ __forceinline__ float f8_score_factor(int ek, int up) {
    return __uint_as_float((uint32_t)min(max(ek - up + 127, 1), 254) << 23);
}

// 0xff in byte i where cell `first + i` is at most `last`
__device__ __forceinline__ unsigned f8_live_bytes(int first, int last) {
    const int n = min(max(last - first + 1, 0), 4);
    return n == 4 ? 0xffffffffu : (1u << (8 * n)) - 1u;
}

template <int TILES>
struct F8Walk {
    f8_h8 qhi[TILES][8], qlo[TILES][8];
    f8_f4 o[TILES][4][4];  // [m][j][r]: element 64 m + 16 g + 4 r + j of row c
    float m[TILES];        // M, the same in the row's four lanes
    float l[TILES];        // the lane's share
    int up[TILES];

    __device__ __forceinline__ void begin() {
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            m[t] = -INFINITY;
            l[t] = 0.0f;
#pragma unroll
            for (int a = 0; a < 4; ++a)
#pragma unroll
                for (int b = 0; b < 4; ++b) o[t][a][b] = f8_f4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    // z of a pair of pages; k: 16 bytes of piece 4 i + g of row c.  ek, ev: of the page (or the lane's cells) of either half
    __device__ __forceinline__ void scores(const f8_u4 (&k)[2][4], const int (&ek)[2], const int (&ev)[2], float (&z)[TILES][2][4]) const {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            f8_f4 s[TILES], sl[TILES];
#pragma unroll
            for (int t = 0; t < TILES; ++t) s[t] = sl[t] = f8_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const f8_h8 a = h ? f8_to_f16(k[p][i].z, k[p][i].w) : f8_to_f16(k[p][i].x, k[p][i].y);
#pragma unroll
                    for (int t = 0; t < TILES; ++t) {
                        s[t] = f8_mfma(a, qhi[t][2 * i + h], s[t]);
                        sl[t] = f8_mfma(a, qlo[t][2 * i + h], sl[t]);
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                const float by = f8_score_factor(ek[p], up[t]);
#pragma unroll
                for (int r = 0; r < 4; ++r) z[t][p][r] = __builtin_fmaf(s[t][r] + sl[t][r], by, (float)ev[p]);
            }
        }
    }
    // weights of a pair, as the second product takes them; M, l and O follow
    __device__ __forceinline__ void softmax(const float (&z)[TILES][2][4], const int (&ev)[2], f8_h8 (&ph)[TILES], f8_h8 (&pl)[TILES]) {
        bool any = false;
        float was[TILES], at[TILES];
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            float pm = fmaxf(fmaxf(fmaxf(z[t][0][0], z[t][0][1]), fmaxf(z[t][0][2], z[t][0][3])),
                             fmaxf(fmaxf(z[t][1][0], z[t][1][1]), fmaxf(z[t][1][2], z[t][1][3])));
            pm = max_over_lane_groups(pm);
            was[t] = m[t];
            const bool moved = pm > m[t] + kF8Slack;
            m[t] = moved ? pm : m[t];
            any = any || moved;
            at[t] = m[t] == -INFINITY ? 0.0f : m[t];  // nothing attended yet
        }
        if (__builtin_amdgcn_ballot_w64(any) != 0) {
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                const float keep = __builtin_amdgcn_exp2f(was[t] - at[t]);
                l[t] *= keep;
#pragma unroll
                for (int a = 0; a < 4; ++a)
#pragma unroll
                    for (int b = 0; b < 4; ++b) o[t][a][b] *= keep;
            }
        }
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                float sum = 0.0f;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float w = __builtin_amdgcn_exp2f(z[t][p][r] - at[t]);
                    sum += w;
                    const _Float16 hi = (_Float16)w;
                    ph[t][4 * p + r] = hi;
                    pl[t][4 * p + r] = (_Float16)(w - (float)hi);
                }
                l[t] = __builtin_fmaf(sum, exp2_int(-ev[p]), l[t]);
            }
        }
    }
    // v: 16 bytes of columns 64 m + 4 c .. of cells 4 g .. of either page
    __device__ __forceinline__ void add_values(const f8_u4 (&v)[2][4], const f8_h8 (&ph)[TILES], const f8_h8 (&pl)[TILES]) {
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f8_h8 x = f8_to_f16(v[0][a][j], v[1][a][j]);
#pragma unroll
                for (int t = 0; t < TILES; ++t) o[t][a][j] = f8_mfma(x, ph[t], o[t][a][j]);
#pragma unroll
                for (int t = 0; t < TILES; ++t) o[t][a][j] = f8_mfma(x, pl[t], o[t][a][j]);
            }
    }
};

}  // namespace bkv
