// Paged causal attention for chunks of many query tokens over e4m3 pages (f8p.hpp, f8p_attn.hpp) on gfx950; blocks of rows, the cut
// of long walks, order and merge are those of the other layouts (prefill_plan.hpp, prefill_attn.hip).
//
// A work-group of four waves has 64 or 128 query rows ((token, head) pairs of one kv head), a wave one tile of 16 of them or two.
// The waves share nothing: pages lie in memory as the products take them, so each wave loads its operands straight into
// registers, 16 KiB a pair of pages, from the cache of the compute unit or the die where its neighbours' loads have left them,
// and there is no barrier in the walk.
#include <type_traits>

#include "f8p_attn.hpp"
#include "gate.hpp"
#include "prefill_common.hpp"

namespace bkv {

namespace {

constexpr int kHd = kF8Hd, kPage = kF8Page;
typedef const __attribute__((address_space(1))) uint8_t* gptr;
typedef __attribute__((address_space(1))) f8_f4* out_f4;
typedef const __attribute__((address_space(1))) f8_f4* in_f4;

// 1.0 for every byte that is a NaN code, as f16 operand; 0 elsewhere
__device__ __forceinline__ f8_h8 f8_nan_marks(unsigned a, unsigned b) {
    f8_h8 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[i] = ((a >> (8 * i)) & 0x7fu) == 0x7fu ? (_Float16)1.0f : (_Float16)0.0f;
        x[i + 4] = ((b >> (8 * i)) & 0x7fu) == 0x7fu ? (_Float16)1.0f : (_Float16)0.0f;
    }
    return x;
}
// a NaN code among four: bit 7 of its byte
__device__ __forceinline__ unsigned f8_nan_bytes(unsigned w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
// the four codes with NaN ones replaced by zeros
__device__ __forceinline__ unsigned f8_without_nan(unsigned w) {
    const unsigned n = f8_nan_bytes(w);
    return w & ~((n >> 7) * 0xffu);
}

// Which (entry, kv head, block of query rows) this work-group has; false where it has none.  idx: which of the unit's blocks,
// in dispatch order; cut: the block's walk is cut at all, range: which range of its pages.  (The kernel of the other layouts finds
// it the same way, in its body: as a function there it trips this compiler's register allocation.)
template <bool SPLIT, int kRowsPerWg>
__device__ __forceinline__ bool chunk_unit(const std::conditional_t<SPLIT, PrefillSplitParams, PrefillKernelParams>& P, int& e, int& kvh, int& idx,
                                           int& range, bool& cut) {
    if constexpr (SPLIT) {
        while (e + 1 < P.b.n && (int)blockIdx.x >= P.s.wg_base[e + 1]) ++e;
        int rem = (int)blockIdx.x - P.s.wg_base[e];
        // uncut blocks first: the longest of them are longer than a range
        const int blocks = (P.b.n_tok[e] * P.group + kRowsPerWg - 1) / kRowsPerWg;
        const int uncut = (blocks - P.s.n_cut[e]) * P.n_kv;
        cut = rem >= uncut;
        if (cut) {
            rem -= uncut;
            range = rem % P.s.splits[e];
            rem /= P.s.splits[e];
        }
        idx = divided_by(rem, P.n_kv, P.n_kv_inverse, kvh) + (cut ? 0 : P.s.n_cut[e]);
    } else if (P.by_xcd) {
        const int units = P.b.n * P.n_kv;
        const int x = (int)blockIdx.x % kXcds;
        int j = (int)blockIdx.x / kXcds;
        int u;
        if (units >= kXcds) {
            u = x;
            for (;;) {
                if (u >= units) return false;  // this die's share of the grid is shorter than the longest
                const int nb = (P.b.n_tok[divided_by(u, P.n_kv, P.n_kv_inverse)] * P.group + kRowsPerWg - 1) / kRowsPerWg;
                if (j < nb) break;
                j -= nb;
                u += kXcds;
            }
            idx = j;
        } else {
            u = x % units;
            const int dies = (kXcds - u + units - 1) / units;  // dies x with x % units == u
            idx = j * dies + x / units;
        }
        e = divided_by(u, P.n_kv, P.n_kv_inverse, kvh);
    } else {
        while (e + 1 < P.b.n && (int)blockIdx.x >= P.b.wg_base[e + 1]) ++e;
        const int rem = (int)blockIdx.x - P.b.wg_base[e];
        idx = divided_by(rem, P.n_kv, P.n_kv_inverse, kvh);
    }
    return true;
}

template <int TILES, bool SPLIT>
__global__ __launch_bounds__(256, TILES == 2 ? 1 : 2) void chunk_attn_f8p_kernel(const std::conditional_t<SPLIT, PrefillSplitParams, PrefillKernelParams> P) {
    constexpr int kRowsPerWg = 4 * TILES * kPrefillRowsPerWave;
    now(P.b, P.n_kv, P.by_xcd);
    if constexpr (SPLIT) now(P.s);
    int e = 0, kvh, idx, range = 0;
    bool cut = false;
    if (!chunk_unit<SPLIT, kRowsPerWg>(P, e, kvh, idx, range, cut)) return;
    const int n_rows = P.b.n_tok[e] * P.group;  // query rows of this kv head
    const int n_blocks = (n_rows + kRowsPerWg - 1) / kRowsPerWg;
    if (idx >= n_blocks) return;
    // later rows attend more cells: the heaviest blocks are dispatched first
    const int rb = n_blocks - 1 - idx;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int row0 = rb * kRowsPerWg + wave * TILES * kPrefillRowsPerWave;
    if (row0 >= n_rows) return;
    const int pos0 = P.b.pos0[e];

    // pages of the walk, or of this range of it
    int end_pg = (pos0 + divided_by(min(row0 + TILES * kPrefillRowsPerWave, n_rows) - 1, P.group, P.group_inverse)) / kPage + 1;
    int first_pg = 0;
    if constexpr (SPLIT) {
        if (cut) {
            const int wg_last_row = min(rb * kRowsPerWg + kRowsPerWg, n_rows) - 1;
            const int wg_pages = (pos0 + divided_by(wg_last_row, P.group, P.group_inverse)) / kPage + 1;
            int each;
            const int ranges = split_ranges(wg_pages, P.s.pps, P.s.splits[e], each);
            if (range >= ranges) return;  // the entry's longest block has more
            first_pg = range * each;
            end_pg = min(end_pg, first_pg + each);
        }
    }
    int tok[TILES], head[TILES], last_cell[TILES];
    bool row_live[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        const int row = row0 + t * kPrefillRowsPerWave + c;
        row_live[t] = row < n_rows;
        int h;
        tok[t] = divided_by(row_live[t] ? row : row0, P.group, P.group_inverse, h);
        head[t] = kvh * P.group + h;
        last_cell[t] = pos0 + tok[t];
    }
    // the last cell that every row of the wave attends: pages wholly at or below it need no mask
    const int all_live = pos0 + divided_by(row0, P.group, P.group_inverse);

    const int32_t* const table = P.tables + (size_t)P.b.row[e] * (size_t)P.max_pages_per_seq;
    const size_t k_page = f8p_k_page_bytes(P.n_kv), v_page = f8p_v_page_bytes(P.n_kv);
    const uint8_t* const kpool = P.kpool + (size_t)kvh * kF8Unit;
    const uint8_t* const vpool = P.vpool + (size_t)kvh * kF8Unit;
    const uint8_t* const lines = P.kpool + (size_t)P.n_kv * kF8Unit + 8 * (size_t)kvh;
    const int mine = end_pg - first_pg;  // pages; none of a range behind the wave's rows

    F8Walk<TILES> W;
    W.begin();
    if (mine > 0) {
        int ids = 0;  // lane i: page i of the 64 from here on; past the end the last again
        const auto fetch_ids = [&](int from) { ids = table[first_pg + min(from + lane, mine - 1)]; };
        f8_u4 k[2][4], v[2][4];
        f8_i2 ex[2];
        const int k_lane = (c >> 2) * 1024 + g * 64 + (c & 3) * 16, v_lane = g * 1024 + c * 16;
        const auto load_k = [&](int u) {
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const gptr at = (gptr)(kpool + (size_t)(unsigned)__builtin_amdgcn_readlane(ids, min(u + p, mine - 1) & 63) * k_page) + k_lane;
#pragma unroll
                for (int i = 0; i < 4; ++i) k[p][i] = *(const __attribute__((address_space(1))) f8_u4*)(at + 256 * i);
            }
        };
        const auto load_v = [&](int u) {
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const size_t page = (size_t)(unsigned)__builtin_amdgcn_readlane(ids, min(u + p, mine - 1) & 63);
                const gptr at = (gptr)(vpool + page * v_page) + v_lane;
#pragma unroll
                for (int i = 0; i < 4; ++i) v[p][i] = *(const __attribute__((address_space(1))) f8_u4*)(at + 256 * i);
                ex[p] = *(const __attribute__((address_space(1))) f8_i2*)(gptr)(lines + page * k_page);
            }
        };
        fetch_ids(0);
        load_k(0);
        load_v(0);
#pragma unroll
        for (int t = 0; t < TILES; ++t)
            W.up[t] = f8_split_q(P.q + ((size_t)(P.b.src0[e] + tok[t]) * P.n_q + head[t]) * kHd, row_live[t], P.scale_log2e, g, W.qhi[t], W.qlo[t]);
        for (int u = 0; u < mine; u += 2) {
            const bool more = u + 2 < mine;
            int ek[2], ev[2];
#pragma unroll
            for (int p = 0; p < 2; ++p) ek[p] = f8p_exponent_read(ex[p].x), ev[p] = f8p_exponent_read(ex[p].y);
            float z[TILES][2][4];
            W.scores(k, ek, ev, z);
            if (more) {
                if (((u + 2) & 63) == 0) fetch_ids(u + 2);
                load_k(u + 2);
            }
            const int cell0 = (first_pg + u) * kPage;
            const bool masked = cell0 + 2 * kPage - 1 > all_live || u + 1 >= mine;
            if (masked) {
#pragma unroll
                for (int t = 0; t < TILES; ++t)
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        const int at = u + p < mine ? cell0 + p * kPage + 4 * g : 0x7fffff00;
#pragma unroll
                        for (int r = 0; r < 4; ++r) z[t][p][r] = at + r <= last_cell[t] ? z[t][p][r] : -INFINITY;
                    }
            }
            f8_h8 ph[TILES], pl[TILES];
            W.softmax(z, ev, ph, pl);
            if (masked) {
                // A weight of 0 would not keep NaN away from rows that must not see it.  NaN codes are taken out of such a
                // pair, and rows that do see one get their NaN by itself: where a column's marks meet a live cell.
                unsigned any = 0;
#pragma unroll
                for (int p = 0; p < 2; ++p)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) any |= f8_nan_bytes(v[p][i][j]);
                if (__builtin_amdgcn_ballot_w64(any != 0) != 0) {
#pragma unroll
                    for (int t = 0; t < TILES; ++t) {
                        f8_h8 live;
#pragma unroll
                        for (int p = 0; p < 2; ++p) {
                            const int at = u + p < mine ? cell0 + p * kPage + 4 * g : 0x7fffff00;
#pragma unroll
                            for (int r = 0; r < 4; ++r) live[4 * p + r] = at + r <= last_cell[t] ? (_Float16)1.0f : (_Float16)0.0f;
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const f8_f4 seen = f8_mfma(f8_nan_marks(v[0][i][j], v[1][i][j]), live, f8_f4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
                                for (int r = 0; r < 4; ++r) W.o[t][i][j][r] = seen[r] > 0.0f ? __builtin_nanf("") : W.o[t][i][j][r];
                            }
                    }
#pragma unroll
                    for (int p = 0; p < 2; ++p)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int j = 0; j < 4; ++j) v[p][i][j] = f8_without_nan(v[p][i][j]);
                }
            }
            W.add_values(v, ph, pl);
            if (more) load_v(u + 2);
        }
    }

    // ---- normalise, gate, store ----
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        const float l = sum_over_lane_groups(W.l[t]);
        if (!row_live[t]) continue;
        if constexpr (SPLIT) {
            if (cut) {
                const size_t slot = (size_t)P.s.slot_base[e] + (size_t)(idx * P.n_kv + kvh) * P.s.splits[e] + range;
                const size_t at = slot * kRowsPerWg + (size_t)((wave * TILES + t) * kPrefillRowsPerWave + c);
                float* const po = P.part_o + at * kHd + 16 * g;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        *reinterpret_cast<f8_f4*>(po + 64 * i + 4 * r) = f8_f4{W.o[t][i][0][r], W.o[t][i][1][r], W.o[t][i][2][r], W.o[t][i][3][r]};
                if (g == 0) *reinterpret_cast<float2*>(P.part_ml + at * 2) = make_float2(W.m[t], l);
                continue;
            }
        }
        const float inv = l > 0.0f ? 1.0f / l : l == l ? 0.0f : l;
        const size_t row = (size_t)(P.b.src0[e] + tok[t]);
        float* const op = P.out + (row * P.n_q + head[t]) * kHd + 16 * g;
        const float* const gp = P.gate ? P.gate + (int64_t)row * P.gate_tok_stride + (int64_t)head[t] * P.gate_head_stride + 16 * g : nullptr;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f8_f4 y[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) y[r] = f8_f4{W.o[t][i][0][r], W.o[t][i][1][r], W.o[t][i][2][r], W.o[t][i][3][r]} * inv;
            if (gp) {
                f8_f4 z[4];
                if (P.gate_in_fours) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) z[r] = *(in_f4)(gptr)(gp + 64 * i + 4 * r);
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int j = 0; j < 4; ++j) z[r][j] = gp[64 * i + 4 * r + j];
                }
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int j = 0; j < 4; ++j) y[r][j] *= sigmoid(z[r][j]);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) *reinterpret_cast<f8_f4*>(op + 64 * i + 4 * r) = y[r];
        }
    }
}

}  // namespace

hipError_t launch_chunk_attn_f8p(bkv_pool* p, const PrefillSplitParams& kp, int32_t rows_per_wg, bool split, uint32_t grid, hipStream_t stream) {
    const auto launch = [&](auto kernel, const auto& args) {
        launch_staged(p, BKV_STAGE_PREFILL_ATTN, kernel, dim3(grid), dim3(256), 0, stream, args);
    };
    const PrefillKernelParams& whole = kp;
    const bool two = rows_per_wg == 8 * kPrefillRowsPerWave;
    if (!split) {
        if (two) launch(chunk_attn_f8p_kernel<2, false>, whole);
        else launch(chunk_attn_f8p_kernel<1, false>, whole);
        return hipGetLastError();
    }
    if (two) launch(chunk_attn_f8p_kernel<2, true>, kp);
    else launch(chunk_attn_f8p_kernel<1, true>, kp);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    return launch_prefill_merge(p, kp, rows_per_wg, stream);
}

}  // namespace bkv
