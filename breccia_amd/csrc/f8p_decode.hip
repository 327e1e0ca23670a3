// Paged decode attention over e4m3 pages (f8p.hpp, f8p_attn.hpp) on gfx950: the split-K kernel; cut of a batch, merge and launch
// are those of the other layouts (decode_attn.hip).
//
// A work-group of four waves has one (entry, kv head, page range); a wave has every fourth page of it, and takes them two at a
// time with all heads of the kv head as its tile of 16.  512 bytes a cell and kv head have to come from memory, against 32 matrix
// products a page, a fifth of the time the bytes take: the kernel is bound by its stream.  Pages lie in memory as the products
// take them, so they go straight to registers, 16 KiB a wave in flight, the next pair asked for as soon as the last use of this
// one's is behind.
#include <type_traits>

#include "decode_attn_common.hpp"
#include "f8p_attn.hpp"

namespace bkv {

namespace {

constexpr int kFoldRow = kHd + 4;  // floats of a head's row on its way through LDS: rows 16 bytes apart in the banks
struct FoldLds {
    float o[kWaves][16][kFoldRow];
    float m[kWaves][16], l[kWaves][16];
};

typedef const __attribute__((address_space(1))) uint8_t* gptr;

// SEL: the cells of a list of 4-cell blocks instead of all; a wave's unit is then a group of four listed blocks, which stand for
// the four blocks of a page.
template <bool SEL, bool DESC>
__global__ __launch_bounds__(kBlock, 2) void decode_attn_f8p_kernel(const AttnArgsOf<DESC> P) {
    __shared__ __attribute__((aligned(16))) FoldLds L;
    int e, rem, pos, row, pps;
    const int unit = blockIdx.x;
    if (!unit_of_work_group<false, DESC>(P, unit, e, rem, pos, row, pps)) return;
    const int range = small_div(rem, P.inv_kv16), kvh = rem - range * P.n_kv;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int32_t* const table = P.tables + (size_t)row * (size_t)P.max_pages_per_seq;
    const size_t k_page = f8p_k_page_bytes(P.n_kv), v_page = f8p_v_page_bytes(P.n_kv);
    const uint8_t* const kpool = P.kpool + (size_t)kvh * kF8Unit;
    const uint8_t* const vpool = P.vpool + (size_t)kvh * kF8Unit;
    const uint8_t* const lines = P.kpool + (size_t)P.n_kv * kF8Unit + 8 * (size_t)kvh;

    // this wave's units: pages (groups of listed blocks) first + wave + 4 i, i < mine
    int listed = 0;
    if constexpr (SEL) listed = (int)min(P.counts[e], (uint32_t)P.max_ids);
    const int total = SEL ? (listed + 3) >> 2 : pos / kPage + 1;
    const int first = range * pps + wave;
    const int mine = max((min((range + 1) * pps, total) - first + kWaves - 1) / kWaves, 0);

    // Pages of units, 64 at a time: lane i has the page of unit i (SEL: the id of block i % 4 of unit i / 4, and its page).
    // Past the end the last one again: everything asked for is in the pool.
    constexpr int kAhead = SEL ? 16 : 64;  // units
    int ids = 0, blocks = 0;
    const auto fetch_ids = [&](int from) {
        if constexpr (SEL) {
            const int i = (first + kWaves * (from + (lane >> 2))) * 4 + (lane & 3);
            const uint32_t id = i < listed ? P.ids[(size_t)e * (size_t)P.id_stride + (size_t)i] : 0xffffffffu;
            blocks = (int)id;
            ids = table[min(id, (uint32_t)pos >> 2) >> 2];
        } else {
            ids = table[first + kWaves * min(from + lane, mine - 1)];
        }
    };

    f8_u4 k[2][4], v[2][4];
    f8_i2 ex[2];
    int vb[2] = {0, 0};  // SEL: the block of cells 4 g ..
    const auto k_at = [&](int u) -> gptr {
        if constexpr (SEL) {
            const int from = 4 * (u & (kAhead - 1)) + (c >> 2);
            const int id = __shfl(blocks, from, 64), page = __shfl(ids, from, 64);
            return (gptr)(kpool + (size_t)(unsigned)page * k_page + (size_t)((min((uint32_t)id, (uint32_t)pos >> 2) & 3) * 1024 + g * 64 + (c & 3) * 16));
        } else {
            const int page = __builtin_amdgcn_readlane(ids, u & (kAhead - 1));
            return (gptr)(kpool + (size_t)(unsigned)page * k_page) + ((c >> 2) * 1024 + g * 64 + (c & 3) * 16);
        }
    };
    const auto load_k = [&](int u) {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const gptr at = k_at(min(u + p, mine - 1));
#pragma unroll
            for (int i = 0; i < 4; ++i) k[p][i] = *(const __attribute__((address_space(1))) f8_u4*)(at + 256 * i);
        }
    };
    const auto load_v = [&](int u) {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const int uu = min(u + p, mine - 1);
            if constexpr (SEL) {
                const int from = 4 * (uu & (kAhead - 1)) + g;
                const int id = __shfl(blocks, from, 64), page = __shfl(ids, from, 64);
                vb[p] = id;
                const gptr at = (gptr)(vpool + (size_t)(unsigned)page * v_page + (size_t)((min((uint32_t)id, (uint32_t)pos >> 2) & 3) * 1024 + c * 16));
#pragma unroll
                for (int i = 0; i < 4; ++i) v[p][i] = *(const __attribute__((address_space(1))) f8_u4*)(at + 256 * i);
                ex[p] = *(const __attribute__((address_space(1))) f8_i2*)(gptr)(lines + (size_t)(unsigned)page * k_page);
            } else {
                const int page = __builtin_amdgcn_readlane(ids, uu & (kAhead - 1));
                const gptr at = (gptr)(vpool + (size_t)(unsigned)page * v_page) + (g * 1024 + c * 16);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[p][i] = *(const __attribute__((address_space(1))) f8_u4*)(at + 256 * i);
                ex[p] = *(const __attribute__((address_space(1))) f8_i2*)(gptr)(lines + (size_t)(unsigned)page * k_page);
            }
        }
    };

    F8Walk<1> W;
    W.begin();
    if (mine > 0) {
        fetch_ids(0);
        load_k(0);
        load_v(0);
        const bool head_live = c < P.group;
        W.up[0] = f8_split_q(P.q + ((size_t)e * P.n_q + (size_t)kvh * P.group + (size_t)(head_live ? c : 0)) * kHd, head_live, P.scale_log2e, g,
                             W.qhi[0], W.qlo[0]);
        for (int u = 0; u < mine; u += 2) {
            const bool more = u + 2 < mine;
            int ek[2], ev[2];
#pragma unroll
            for (int p = 0; p < 2; ++p) ek[p] = f8p_exponent_read(ex[p].x), ev[p] = f8p_exponent_read(ex[p].y);
            float z[1][2][4];
            unsigned live_v[2] = {0xffffffffu, 0xffffffffu};
            W.scores(k, ek, ev, z);
            if (more) {
                if (((u + 2) & (kAhead - 1)) == 0) fetch_ids(u + 2);
                load_k(u + 2);
            }
            if constexpr (SEL) {
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    live_v[p] = 0;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const bool live = u + p < mine && block_cell_live((uint32_t)vb[p], r, pos);
                        z[0][p][r] = live ? z[0][p][r] : -INFINITY;
                        live_v[p] |= live ? 0xffu << (8 * r) : 0u;
                    }
                }
            } else if (!more) {
                // cells past the position, and the page asked for twice
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const int at = u + p < mine ? (first + kWaves * (u + p)) * kPage + 4 * g : pos + 1;
                    live_v[p] = f8_live_bytes(at, pos);
#pragma unroll
                    for (int r = 0; r < 4; ++r) z[0][p][r] = at + r <= pos ? z[0][p][r] : -INFINITY;
                }
            }
            f8_h8 ph[1], pl[1];
            W.softmax(z, ev, ph, pl);
            if (SEL || !more) {
                // values that no weight belongs to may be anything (a weight of 0 would not keep NaN away)
#pragma unroll
                for (int p = 0; p < 2; ++p)
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[p][i] &= live_v[p];
            }
            W.add_values(v, ph, pl);
            if (more) load_v(u + 2);
        }
    }

    // ---- the four waves' results folded; wave w sums columns 64 w .. 64 w + 63 and writes them ----
    W.l[0] = sum_over_lane_groups(W.l[0]);
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            *reinterpret_cast<f8_f4*>(&L.o[wave][c][64 * a + 16 * g + 4 * r]) =
                f8_f4{W.o[0][a][0][r], W.o[0][a][1][r], W.o[0][a][2][r], W.o[0][a][3][r]};
    if (g == 0) L.m[wave][c] = W.m[0], L.l[wave][c] = W.l[0];
    __syncthreads();
    const int col = 64 * wave + 4 * c;
    for (int h = g; h < P.group; h += 4) {
        float mx = L.m[0][h];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) mx = fmaxf(mx, L.m[w][h]);
        const float ref = mx == -INFINITY ? 0.0f : mx;
        f8_f4 sum = f8_f4{0.0f, 0.0f, 0.0f, 0.0f};
        float l = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(L.m[w][h] - ref);
            sum += *reinterpret_cast<const f8_f4*>(&L.o[w][h][col]) * f;
            l = __builtin_fmaf(L.l[w][h], f, l);
        }
        // a denominator that is no number, for the merge: it takes outputs without one for those of an empty list
        if (!(l < INFINITY)) {
            sum = f8_f4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
            mx = 0.0f;
            l = 1.0f;
        }
        const size_t at = (size_t)unit * P.group + h;
        *reinterpret_cast<f8_f4*>(P.part_o + at * kHd + col) = sum;
        if (wave == 0 && c == 0) *reinterpret_cast<float2*>(P.part_ml + at * 2) = make_float2(mx, l);
    }
}

}  // namespace

hipError_t launch_decode_attn_f8p(const AttnKernelParams& kp, const AttnBatch& b, bool sel, int32_t total, hipStream_t stream, hipEvent_t start,
                                  hipEvent_t stop) {
    const auto launch = [&](auto kernel, const auto& args) {
        if (start) hipExtLaunchKernelGGL(kernel, dim3((unsigned)total), dim3(kBlock), 0, stream, start, stop, 0, args);
        else hipLaunchKernelGGL(kernel, dim3((unsigned)total), dim3(kBlock), 0, stream, args);
    };
    if (kp.bd) {
        launch(decode_attn_f8p_kernel<false, true>, kp);
    } else {
        AttnKernelArgs<AttnBatch> args;
        static_cast<AttnKernelParams&>(args) = kp;
        args.b = b;
        if (sel) launch(decode_attn_f8p_kernel<true, false>, args);
        else launch(decode_attn_f8p_kernel<false, false>, args);
    }
    return hipGetLastError();
}

}  // namespace bkv
