// Paged causal attention for chunks of many query tokens over e4m3 pages (f8p.hpp, f8p_attn.hpp) on gfx950; blocks of rows, the cut
// of long walks, order and merge are those of the other layouts (prefill_plan.hpp, prefill_attn.hip).
//
// A work-group of four waves has 64 or 128 query rows ((token, head) pairs of one kv head), a wave one tile of 16 of them or two.
// The waves share nothing in the walk: pages lie in memory as the products take them, so each wave loads its operands straight into
// registers, 16 KiB a pair of pages, from the cache of the compute unit where its neighbours' loads have left seven of ten lines,
// and there is no barrier.
//
// What bounds it: power first (1.85 to 2.1 GHz under it), then issue.  q and the weights are two f16 numbers each, so twice the
// useful products are issued; a library product reaches 1245 TFLOP/s on this card, and four chunks of 1024 tokens behind 1536 take
// 221 us, as long as their products would there.  A prompt of 4096 at 12 heads a kv head takes 370 of 331: the start and the end
// of its 768 work-groups are a tenth of their time (an order of dispatch that evens out when they end brought 1 %).  16x16x32
// products and two tiles because 32x32x16 ones cost more power (from registers alone 1403 TFLOP/s against 1647); pages shared
// through LDS took 250 us where this took 242.
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

// Which (entry, kv head, block of query rows) this work-group has, if any.  idx: which of the unit's blocks, in dispatch order; cut:
// the block's walk is cut at all, range: which range of its pages.  (The kernel of the other layouts finds it the same way, in its
// body: as a function there it trips this compiler's register allocation.)
struct ChunkUnit {
    bool any;
    int e, kvh, idx, range;
    bool cut;
};
template <bool SPLIT, int kRowsPerWg>
__device__ __forceinline__ ChunkUnit chunk_unit(const std::conditional_t<SPLIT, PrefillSplitParams, PrefillKernelParams>& P) {
    int e = 0, kvh = 0, idx = 0, range = 0;
    bool cut = false;
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
                if (u >= units) return ChunkUnit{};  // this die's share of the grid is shorter than the longest
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
    return ChunkUnit{true, e, kvh, idx, range, cut};
}

__device__ __forceinline__ int wave_value(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ unsigned lds_at(const float* p) { return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) float*)p; }
// a maximum whose operands are known not to be signalling NaNs; fmaxf would quiet each of them first
__device__ __forceinline__ float max3(float a, float b, float c) {
    float x;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(x) : "v"(a), "v"(b), "v"(c));
    return x;
}

// Two tiles: x * by of an accumulator that stays in the upper half of the register file.  (Written out in C++, the copies to the lower half are
// made ahead of the branch around it, for every pair.)  `products_done` stands between the last product that wrote x and the first of
// these, `settle` between the last of these and the next product: the compiler does not see which registers asm reads and writes
// when it works out those waits.
__device__ __forceinline__ void scale_accumulator(float& x, float by) {
    float t;
    asm volatile("v_accvgpr_read_b32 %1, %0\n\tv_mul_f32 %1, %1, %2\n\tv_accvgpr_write_b32 %0, %1" : "+a"(x), "=&v"(t) : "v"(by));
}
__device__ __forceinline__ void products_done() { asm volatile("s_nop 15\n\ts_nop 15"); }
__device__ __forceinline__ void settle() { asm volatile("s_nop 4"); }

// The waves' rows of q on their way in and of the output on their way out, 16 bytes apart in the banks.  A lane holds pieces of one
// row; a load or store straight from there touches 16 rows 64 bytes at a time, which the path to memory takes line by line.
constexpr int kStagedRow = kHd + 4;
template <int TILES>
struct ChunkLds {
    float row[4][16 * TILES][kStagedRow];
};

// Lane (c, g) has of tile t row 16 t + c, and cells 4 g .. 4 g + 3 of either page of a pair: scores z[t][4 page + cell % 4].
template <int TILES, bool SPLIT>
__global__ __launch_bounds__(256, TILES == 2 ? 1 : 2) void chunk_attn_f8p_kernel(const std::conditional_t<SPLIT, PrefillSplitParams, PrefillKernelParams> P) {
    constexpr int kRowsPerWave = 16 * TILES, kRowsPerWg = 4 * kRowsPerWave;
    __shared__ __attribute__((aligned(16))) ChunkLds<TILES> L;
    now(P.b, P.n_kv, P.by_xcd);
    if constexpr (SPLIT) now(P.s);
    const ChunkUnit unit_of = chunk_unit<SPLIT, kRowsPerWg>(P);
    if (!unit_of.any) return;
    // (the same for every lane, which the compiler has lost sight of in the search)
    const int e = wave_value(unit_of.e), kvh = wave_value(unit_of.kvh), idx = wave_value(unit_of.idx), range = wave_value(unit_of.range);
    const bool cut = unit_of.cut;
    const int n_rows = P.b.n_tok[e] * P.group;  // query rows of this kv head
    const int n_blocks = (n_rows + kRowsPerWg - 1) / kRowsPerWg;
    if (idx >= n_blocks) return;
    // later rows attend more cells: the heaviest blocks are dispatched first
    const int rb = n_blocks - 1 - idx;
    const int wave = wave_value(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int row0 = rb * kRowsPerWg + wave * kRowsPerWave;
    if (row0 >= n_rows) return;
    const int live_rows = min(n_rows - row0, kRowsPerWave);
    const int pos0 = P.b.pos0[e];

    // pages of the walk, or of this range of it
    int end_pg = (pos0 + divided_by(row0 + live_rows - 1, P.group, P.group_inverse)) / kPage + 1;
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
    first_pg = wave_value(first_pg);
    const int mine = wave_value(end_pg) - first_pg;  // pages; none of a range behind the wave's rows
    // Lane x: (token, head) of the wave's row x % kRowsPerWave; past the chunk's end the first row's again, whose results are not
    // stored.
    const int my_row = lane & (kRowsPerWave - 1);
    int my_head;
    const int my_tok = divided_by(my_row < live_rows ? row0 + my_row : row0, P.group, P.group_inverse, my_head);
    my_head += kvh * P.group;
    int last_cell[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) last_cell[t] = pos0 + __shfl(my_tok, 16 * t + c, 64);
    // the last cell that every row of the wave attends: pages wholly at or below it need no mask
    const int all_live = wave_value(pos0 + divided_by(row0, P.group, P.group_inverse));
    const uint64_t out_row = (uint64_t)(P.b.src0[e] + my_tok);
    const uint64_t row_at = (out_row * (uint64_t)P.n_q + (uint64_t)my_head) * (kHd * 4);  // of q and of the output, in bytes

    const int32_t* const table = P.tables + (size_t)P.b.row[e] * (size_t)P.max_pages_per_seq;
    const size_t k_page = f8p_k_page_bytes(P.n_kv), v_page = f8p_v_page_bytes(P.n_kv);
    const uint8_t* const kpool = P.kpool + (size_t)kvh * kF8Unit;
    const uint8_t* const vpool = P.vpool + (size_t)kvh * kF8Unit;
    const uint8_t* const lines = P.kpool + (size_t)P.n_kv * kF8Unit + 8 * (size_t)kvh;

    float minus_one = -1.0f;
    asm("" : "+v"(minus_one));
    f8_f4 o[TILES][4][4];  // [m][j][r]: element 64 m + 16 g + 4 r + j of the row
    float at[TILES];       // M, once anything is attended
    float limit[TILES];    // what a pair's maximum has to pass for M to move, relative to it
    float l_run[TILES];
    unsigned poison[TILES][2];  // elements that are NaN whatever the products say: bit 16 (m % 2) + 4 j + r of word m / 2
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        at[t] = l_run[t] = 0.0f;
        limit[t] = -INFINITY;
        poison[t][0] = poison[t][1] = 0;
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[t][m][j] = f8_f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    float* const rows = &L.row[wave][0][0];

    if (mine > 0) {
        // ---- q's rows into LDS, an instruction each ----
        {
            const uint64_t q_at = (uint64_t)(uintptr_t)P.q + row_at;
#pragma unroll
            for (int r = 0; r < kRowsPerWave; ++r) load_to_lds(lds_at(rows + r * kStagedRow), (gptr)lane_value(q_at, r), 16 * lane);
        }
        // The wave's pages, through the scalar path: pair u's are asked for three steps ahead.  Past the end the last again.
        typedef const __attribute__((address_space(4))) int32_t* id_ptr;
        typedef const __attribute__((address_space(4))) f8_i2* line_ptr;
        const id_ptr my_table = (id_ptr)(uintptr_t)(table + first_pg);
        struct Pair {
            size_t p[2];
        };
        const auto page_id = [&](int u) { return (size_t)(unsigned)my_table[min(u, mine - 1)]; };
        const auto pair_ids = [&](int u) { return Pair{{page_id(u), page_id(u + 1)}}; };
        const auto exps = [&](const Pair& x, int p) { return *(line_ptr)(uintptr_t)(lines + x.p[p] * k_page); };
        const int k_lane = (c >> 2) * 1024 + g * 64 + (c & 3) * 16, v_lane = g * 1024 + c * 16;
        const auto k_base = [&](const Pair& x, int p) -> gptr { return (gptr)(kpool + x.p[p] * k_page) + k_lane; };
        const auto v_base = [&](const Pair& x, int p) -> gptr { return (gptr)(vpool + x.p[p] * v_page) + v_lane; };
        f8_u4 k[2][4], v[2][4];
        const auto load_k = [&](gptr base, int p, int i) { k[p][i] = *(const __attribute__((address_space(1))) f8_u4*)(base + 256 * i); };
        const auto load_v = [&](gptr base, int p, int m) { v[p][m] = *(const __attribute__((address_space(1))) f8_u4*)(base + 256 * m); };
        Pair ids_0 = pair_ids(0), ids_1 = pair_ids(2), ids_2 = pair_ids(4);  // this pair, the next, the one after
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const gptr base = k_base(ids_0, p);
#pragma unroll
            for (int i = 0; i < 4; ++i) load_k(base, p, i);
        }
        // With two tiles, a wave alone on its SIMD, V is asked for a step ahead.  With one the registers of a step's K become those
        // of its V and back: the other wave's products cover what is left of the way (and 180 bytes a lane no longer spill).
        constexpr bool kVAhead = TILES == 2;
        if constexpr (kVAhead) {
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const gptr base = v_base(ids_0, p);
#pragma unroll
                for (int m = 0; m < 4; ++m) load_v(base, p, m);
            }
        }
        f8_i2 ex[2] = {exps(ids_0, 0), exps(ids_0, 1)};

        // ---- q as high and low parts: fragment f = 2 i + half of piece 4 i + g ----
        wait_for_loads();
        wave_lds_fence();
        f8_h8 qhi[TILES][8], qlo[TILES][8];
        float down[TILES];  // what brings scores to base-2 logits
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const float* const qrow = rows + (16 * t + c) * kStagedRow;
            f8_f4 raw[8][2];
            float top = 0.0f;
#pragma unroll
            for (int f = 0; f < 8; ++f) {
                const int s = 4 * (f >> 1) + g;
                const float* const from = qrow + 128 * (s >> 3) + 4 * (s & 7) + 64 * (f & 1);
                raw[f][0] = *reinterpret_cast<const f8_f4*>(from);
                raw[f][1] = *reinterpret_cast<const f8_f4*>(from + 32);
#pragma unroll
                for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(raw[f][j >> 2][j & 3]));
            }
            top = max_over_lane_groups(top);
            const int up = min(max(13 - ((int)(__float_as_uint(top) >> 23) - 127), -126), 126);
            const float by = f8_lift_q(up, P.scale_log2e);
            down[t] = exp2_int(-up) * P.scale_log2e;
#pragma unroll
            for (int f = 0; f < 8; ++f)
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const float a = raw[f][j >> 2][j & 3] * by, b = raw[f][j >> 2][(j & 3) + 1] * by;
                    const f8_h2 hi = to_f16(a, b);
                    const f8_h2 lo = to_f16(remainder_of(a, hi[0], minus_one), remainder_of(b, hi[1], minus_one));
                    qhi[t][f][j] = hi[0], qhi[t][f][j + 1] = hi[1];
                    qlo[t][f][j] = lo[0], qlo[t][f][j + 1] = lo[1];
                }
        }

        f8_f4 s[TILES][2];
        const auto multiply_k = [&](int f) {  // 16 of them: fragment f % 8 of page f / 8
            const int p = f >> 3, i = (f >> 1) & 3;
            const f8_h8 a = (f & 1) ? f8_to_f16(k[p][i].z, k[p][i].w) : f8_to_f16(k[p][i].x, k[p][i].y);
#pragma unroll
            for (int t = 0; t < TILES; ++t) s[t][p] = f8_mfma(a, qhi[t][f & 7], (f & 7) ? s[t][p] : f8_f4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
            for (int t = 0; t < TILES; ++t) s[t][p] = f8_mfma(a, qlo[t][f & 7], s[t][p]);
        };
        // The pair's logits in base 2, plus the exponents of its values, relative to `at`.
        float z[TILES][8], unit[2], by[TILES][2], plus[TILES][2], pm[TILES];
        const auto factors = [&]() {
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const int ek = f8p_exponent_read(ex[p].x), ev = f8p_exponent_read(ex[p].y);
                unit[p] = exp2_int(-ev);
#pragma unroll
                for (int t = 0; t < TILES; ++t) {
                    // (kept finite: beyond f32's range the logits are far past it, or zero, either way)
                    by[t][p] = fminf(fmaxf(down[t] * exp2_int(ek), -kF8Finite), kF8Finite);
                    plus[t][p] = (float)ev - at[t];
                }
            }
        };
        const auto logits_part = [&](int part) {  // 12 of them
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                if (part < 8) {
                    z[t][part] = __builtin_fmaf(s[t][part >> 2][part & 3], by[t][part >> 2], plus[t][part >> 2]);
                    stay(z[t][part]);
                }
                if (part == 8) pm[t] = max3(z[t][0], z[t][1], z[t][2]);
                if (part == 9) pm[t] = max3(pm[t], z[t][3], z[t][4]);
                if (part == 10) pm[t] = max3(pm[t], z[t][5], z[t][6]);
                if (part == 11) pm[t] = max3(pm[t], z[t][7], z[t][7]);
            }
        };
        const auto has_dead = [&](int u) { return (first_pg + u + 2) * kPage - 1 > all_live || u + 1 >= mine; };
        // the first of the lane's cells of page p of pair u; past the end one that nobody attends
        const auto cell_of = [&](int u, int p) { return u + p < mine ? (first_pg + u + p) * kPage + 4 * g : 0x7fffff00; };
        // dead cells out of pair u, and M moved where the pair passes it by more than kF8Lift + kF8Slack
        const auto move_reference = [&](int u) {
            if (has_dead(u)) {
#pragma unroll
                for (int t = 0; t < TILES; ++t) {
                    pm[t] = -INFINITY;
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        z[t][r] = cell_of(u, r >> 2) + (r & 3) <= last_cell[t] ? z[t][r] : -INFINITY;
                        pm[t] = fmaxf(pm[t], z[t][r]);
                    }
                }
            }
            bool any = false;
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                pm[t] = max_over_lane_groups(pm[t]);
                any = any || pm[t] > limit[t];
            }
            if (__builtin_amdgcn_ballot_w64(any) != 0) {
                if constexpr (TILES == 2) products_done();
#pragma unroll
                for (int t = 0; t < TILES; ++t) {
                    // (nothing attended yet: nothing to keep, whatever the exponential of it would be)
                    const bool moved = pm[t] > limit[t];
                    const float up = moved ? f8_reference(pm[t]) : 0.0f, keep = limit[t] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(-up);
                    limit[t] = moved ? kF8Lift + kF8Slack : limit[t];
                    at[t] += up;
                    l_run[t] *= keep;
#pragma unroll
                    for (int r = 0; r < 8; ++r) z[t][r] -= up;
#pragma unroll
                    for (int m = 0; m < 4; ++m)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                if constexpr (TILES == 2) {
                                    float x = o[t][m][j][r];
                                    scale_accumulator(x, keep);
                                    o[t][m][j][r] = x;
                                } else {
                                    o[t][m][j][r] *= keep;
                                }
                            }
                }
                if constexpr (TILES == 2) settle();
            }
        };

#pragma unroll
        for (int f = 0; f < 16; ++f) multiply_k(f);
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const gptr next = k_base(ids_1, p);
#pragma unroll
            for (int i = 0; i < 4; ++i) load_k(next, p, i);
        }
        factors();
#pragma unroll
        for (int part = 0; part < 12; ++part) logits_part(part);
        move_reference(0);
        ex[0] = exps(ids_1, 0), ex[1] = exps(ids_1, 1);

        // A step: the next pair's scores with this one's weights between them, then this one's values with the next one's logits
        // between them.
        for (int u = 0; u < mine; u += 2) {
            if constexpr (TILES == 2) {
                // half of q in the upper half of the register file, beside the accumulators: only matrix products read it
#pragma unroll
                for (int t = 0; t < TILES; ++t)
#pragma unroll
                    for (int f = 0; f < 8; ++f) {
                        f8_u4 x = __builtin_bit_cast(f8_u4, qlo[t][f]);
                        asm("" : "+a"(x));
                        qlo[t][f] = __builtin_bit_cast(f8_h8, x);
                    }
            }
            const Pair ids_next = pair_ids(u + 6);
            const f8_i2 ex_next[2] = {exps(ids_2, 0), exps(ids_2, 1)};
            float sum[TILES][2];
            f8_h8 ph[TILES], pl[TILES];
#pragma unroll
            for (int t = 0; t < TILES; ++t) sum[t][0] = sum[t][1] = 0.0f;
            const auto weights_part = [&](int part) {
                if (part < 8) {
#pragma unroll
                    for (int t = 0; t < TILES; ++t) {
                        z[t][part] = __builtin_amdgcn_exp2f(z[t][part]);
                        stay(z[t][part]);
                    }
                }
                if (part >= 4 && part < 4 + 4 * TILES) {
                    const int t = (part - 4) >> 2, r = 2 * ((part - 4) & 3);
                    sum[t][r >> 2] += z[t][r];
                    sum[t][r >> 2] += z[t][r + 1];
                    f8_h2 hi = to_f16(z[t][r], z[t][r + 1]);
                    f8_h2 lo = to_f16(remainder_of(z[t][r], hi[0], minus_one), remainder_of(z[t][r + 1], hi[1], minus_one));
                    stay(hi), stay(lo);
                    ph[t][r] = hi[0], ph[t][r + 1] = hi[1];
                    pl[t][r] = lo[0], pl[t][r + 1] = lo[1];
                }
            };
            {
                const gptr next[2] = {kVAhead ? k_base(ids_2, 0) : v_base(ids_0, 0), kVAhead ? k_base(ids_2, 1) : v_base(ids_0, 1)};
#pragma unroll
                for (int f = 0; f < 16; ++f) {
                    multiply_k(f);
                    weights_part(f);
                    if (kVAhead && (f & 1)) load_k(next[f >> 3], f >> 3, (f >> 1) & 3);
                    if (!kVAhead && (f & 1)) load_v(next[(f >> 1) & 1], (f >> 1) & 1, f >> 2);
                }
            }
#pragma unroll
            for (int t = 0; t < TILES; ++t) l_run[t] = __builtin_fmaf(sum[t][0], unit[0], __builtin_fmaf(sum[t][1], unit[1], l_run[t]));
            if (has_dead(u)) {
                // A weight of 0 would not keep NaN away from rows that must not see it.  NaN codes are taken out of such a
                // pair, and noted for the rows that do see one: where a column's marks meet a live cell.
                unsigned any = 0;
#pragma unroll
                for (int p = 0; p < 2; ++p)
#pragma unroll
                    for (int m = 0; m < 4; ++m)
#pragma unroll
                        for (int j = 0; j < 4; ++j) any |= f8_nan_bytes(v[p][m][j]);
                if (__builtin_amdgcn_ballot_w64(any != 0) != 0) {
                    f8_h8 live[TILES];
#pragma unroll
                    for (int t = 0; t < TILES; ++t)
#pragma unroll
                        for (int r = 0; r < 8; ++r) live[t][r] = cell_of(u, r >> 2) + (r & 3) <= last_cell[t] ? (_Float16)1.0f : (_Float16)0.0f;
#pragma unroll
                    for (int m = 0; m < 4; ++m)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const f8_h8 marks = f8_nan_marks(v[0][m][j], v[1][m][j]);
#pragma unroll
                            for (int t = 0; t < TILES; ++t) {
                                const f8_f4 seen = f8_mfma(marks, live[t], f8_f4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
                                for (int r = 0; r < 4; ++r) poison[t][m >> 1] |= seen[r] > 0.0f ? 1u << (16 * (m & 1) + 4 * j + r) : 0u;
                            }
#pragma unroll
                            for (int p = 0; p < 2; ++p) v[p][m][j] = f8_without_nan(v[p][m][j]);
                            __builtin_amdgcn_sched_barrier(0);
                        }
                }
            }
            factors();
            const gptr after[2] = {kVAhead ? v_base(ids_1, 0) : k_base(ids_2, 0), kVAhead ? v_base(ids_1, 1) : k_base(ids_2, 1)};
#pragma unroll
            for (int m = 0; m < 4; ++m) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f8_h8 x = f8_to_f16(v[0][m][j], v[1][m][j]);
#pragma unroll
                    for (int t = 0; t < TILES; ++t) o[t][m][j] = f8_mfma(x, ph[t], o[t][m][j]);
#pragma unroll
                    for (int t = 0; t < TILES; ++t) o[t][m][j] = f8_mfma(x, pl[t], o[t][m][j]);
                    logits_part(4 * m + j);
                }
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    if constexpr (kVAhead) load_v(after[p], p, m);
                    else load_k(after[p], p, m);
                }
            }
            move_reference(u + 2);
            ids_0 = ids_1, ids_1 = ids_2, ids_2 = ids_next;
            ex[0] = ex_next[0], ex[1] = ex_next[1];
        }
    }

    // ---- normalise, gate, store ----
    // The gate's values of every row are asked for ahead of the rows' way through LDS, into the registers that q had: in batches of
    // eight rows behind it they were a chain of trips to memory.
    const bool gated = P.gate && !(SPLIT && cut);
    const uint64_t gate_at = (uint64_t)(uintptr_t)P.gate + (uint64_t)((int64_t)out_row * P.gate_tok_stride + (int64_t)my_head * P.gate_head_stride) * 4;
    f8_f4 gate[kRowsPerWave];
    if (gated) {
        if (P.gate_in_fours) {
#pragma unroll
            for (int r = 0; r < kRowsPerWave; ++r) gate[r] = *((in_f4)lane_value(gate_at, r) + lane);
        } else {
            typedef const __attribute__((address_space(1))) float* in_float;
#pragma unroll
            for (int r = 0; r < kRowsPerWave; ++r)
#pragma unroll
                for (int j = 0; j < 4; ++j) gate[r][j] = ((in_float)lane_value(gate_at, r))[4 * lane + j];
        }
    }
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        if (__builtin_amdgcn_ballot_w64((poison[t][0] | poison[t][1]) != 0) != 0) {
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[t][m][j][r] = poison[t][m >> 1] >> (16 * (m & 1) + 4 * j + r) & 1u ? __builtin_nanf("") : o[t][m][j][r];
        }
        const float l = sum_over_lane_groups(l_run[t]);
        if constexpr (SPLIT) {
            if (cut) {
                const size_t slot = (size_t)P.s.slot_base[e] + (size_t)(idx * P.n_kv + kvh) * P.s.splits[e] + range;
                const int r = 16 * t + c;
                float* const ml = P.part_ml + (slot * kRowsPerWg + (size_t)(wave * kRowsPerWave + r)) * 2;
                if (g == 0 && r < live_rows) *reinterpret_cast<float2*>(ml) = make_float2(limit[t] == -INFINITY ? -INFINITY : at[t], l);
            }
        }
        const float inv = SPLIT && cut ? 1.0f : l > 0.0f ? 1.0f / l : l == l ? 0.0f : l;
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                *reinterpret_cast<f8_f4*>(rows + (16 * t + c) * kStagedRow + 64 * m + 16 * g + 4 * r) =
                    f8_f4{o[t][m][0][r], o[t][m][1][r], o[t][m][2][r], o[t][m][3][r]} * inv;
    }
    wave_lds_fence();
    // from here on lane x has elements 4 x .. 4 x + 3 of every row
    const auto staged = [&](int r) { return *reinterpret_cast<const f8_f4*>(rows + r * kStagedRow + 4 * lane); };
    if constexpr (SPLIT) {
        if (cut) {
            const size_t slot = (size_t)P.s.slot_base[e] + (size_t)(idx * P.n_kv + kvh) * P.s.splits[e] + range;
            float* const po = P.part_o + (slot * kRowsPerWg + (size_t)(wave * kRowsPerWave)) * kHd + 4 * lane;
#pragma unroll 8
            for (int r = 0; r < kRowsPerWave; ++r)
                if (r < live_rows) *reinterpret_cast<f8_f4*>(po + r * kHd) = staged(r);
            return;
        }
    }
    const uint64_t out_at = (uint64_t)(uintptr_t)P.out + row_at;
#pragma unroll
    for (int r = 0; r < kRowsPerWave; ++r) {
        f8_f4 y = staged(r);
        if (gated) {
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] *= sigmoid(gate[r][j]);
        }
        if (r < live_rows) *((out_f4)lane_value(out_at, r) + lane) = y;
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
    // (a call is cut while it leaves half of the compute units idle, and takes two tiles from two work-groups a unit on: not both)
    if (two) launch(chunk_attn_f8p_kernel<2, true>, kp);
    else launch(chunk_attn_f8p_kernel<1, true>, kp);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    return launch_prefill_merge(p, kp, rows_per_wg, stream);
}

}  // namespace bkv
