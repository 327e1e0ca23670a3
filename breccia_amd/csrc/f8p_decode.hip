// Paged decode attention over e4m3 pages (f8p.hpp, f8p_attn.hpp) on gfx950: the split-K kernel; cut of a batch, merge and launch
// are those of the other layouts (decode_attn.hip).
//
// A work-group of four waves has one (entry, kv head, page range); a wave has every fourth page of it, and takes them two at a
// time with all heads of the kv head as its tile of 16.  512 bytes a cell and kv head have to come from memory, against 32 matrix
// products a page, a fifth of the time the bytes take: the kernel is bound by its stream.  Pages lie in memory as the products
// take them, so they go straight to registers, 16 KiB a wave in flight, the next pair asked for as soon as the last use of this
// one's is behind.  Sixteen contexts of 8k to 128k, 1.41 GB: 222 us, 6.4 TB/s of the 6.8 that a plain read reaches; short ones are
// 9 us of start, fold and merge.
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
typedef const __attribute__((address_space(1))) f8_u4* gptr_u4;
typedef const __attribute__((address_space(1))) f8_i2* gptr_i2;

// 0xff in byte i where cell `first + i` is at most `last`
__device__ __forceinline__ unsigned live_bytes(int first, int last) {
    const int n = min(max(last - first + 1, 0), 4);
    return n == 4 ? 0xffffffffu : (1u << (8 * n)) - 1u;
}

// A wave's walk: lane (c, g) has head c, and cells 4 g .. 4 g + 3 of either page of a pair.
struct Walk {
    f8_h8 qhi[8], qlo[8];  // fragment 2 i + half of piece 4 i + g
    float down;            // what brings scores to base-2 logits
    f8_f4 o[4][4];         // [m][j][r]: element 64 m + 16 g + 4 r + j
    float m = -INFINITY;   // M, the same in the head's four lanes
    float l = 0.0f;        // the lane's share

    __device__ __forceinline__ void split_q(const f8_f4 (&raw)[8][2], float scale_log2e) {
        float top = 0.0f;
#pragma unroll
        for (int f = 0; f < 8; ++f)
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(raw[f][j >> 2][j & 3]));
        top = max_over_lane_groups(top);
        const int up = min(max(13 - ((int)(__float_as_uint(top) >> 23) - 127), -126), 126);
        const float by = f8_lift_q(up, scale_log2e);
        down = exp2_int(-up) * scale_log2e;
#pragma unroll
        for (int f = 0; f < 8; ++f)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float x = raw[f][j >> 2][j & 3] * by;
                qhi[f][j] = (_Float16)x;
                qlo[f][j] = (_Float16)(x - (float)qhi[f][j]);
            }
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int b = 0; b < 4; ++b) o[a][b] = f8_f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // z of a pair of pages; k: 16 bytes of piece 4 i + g of row c.  ek, ev: of the page (or the lane's cells) of either half
    __device__ __forceinline__ void scores(const f8_u4 (&k)[2][4], const int (&ek)[2], const int (&ev)[2], float (&z)[2][4]) const {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            f8_f4 hi = f8_f4{0.0f, 0.0f, 0.0f, 0.0f}, lo = hi;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const f8_h8 a = h ? f8_to_f16(k[p][i].z, k[p][i].w) : f8_to_f16(k[p][i].x, k[p][i].y);
                    hi = f8_mfma(a, qhi[2 * i + h], hi);
                    lo = f8_mfma(a, qlo[2 * i + h], lo);
                }
            }
            // (kept finite: beyond f32's range the logits are far past it, or zero, either way)
            const float by = fminf(fmaxf(down * exp2_int(ek[p]), -kF8Finite), kF8Finite);
#pragma unroll
            for (int r = 0; r < 4; ++r) z[p][r] = __builtin_fmaf(hi[r] + lo[r], by, (float)ev[p]);
        }
    }
    // weights of a pair, as the second product takes them; M, l and O follow
    __device__ __forceinline__ void softmax(const float (&z)[2][4], const int (&ev)[2], f8_h8& ph, f8_h8& pl) {
        float pm = fmaxf(fmaxf(fmaxf(z[0][0], z[0][1]), fmaxf(z[0][2], z[0][3])), fmaxf(fmaxf(z[1][0], z[1][1]), fmaxf(z[1][2], z[1][3])));
        pm = max_over_lane_groups(pm);
        const float was = m;
        const bool moved = pm - m > kF8Lift + kF8Slack;  // (of sums with M the rounding could hide that)
        m = moved ? f8_reference(pm) : m;
        const float at = m == -INFINITY ? 0.0f : m;  // nothing attended yet
        if (__builtin_amdgcn_ballot_w64(moved) != 0) {
            const float keep = __builtin_amdgcn_exp2f(was - at);
            l *= keep;
#pragma unroll
            for (int a = 0; a < 4; ++a)
#pragma unroll
                for (int b = 0; b < 4; ++b) o[a][b] *= keep;
        }
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            float sum = 0.0f;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float w = __builtin_amdgcn_exp2f(z[p][r] - at);
                sum += w;
                const _Float16 hi = (_Float16)w;
                ph[4 * p + r] = hi;
                pl[4 * p + r] = (_Float16)(w - (float)hi);
            }
            l = __builtin_fmaf(sum, exp2_int(-ev[p]), l);
        }
    }
    // v: 16 bytes of columns 64 m + 4 c .. of cells 4 g .. of either page
    __device__ __forceinline__ void add_values(const f8_u4 (&v)[2][4], f8_h8 ph, f8_h8 pl) {
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f8_h8 x = f8_to_f16(v[0][a][j], v[1][a][j]);
                o[a][j] = f8_mfma(x, ph, o[a][j]);
                o[a][j] = f8_mfma(x, pl, o[a][j]);
            }
    }
};

// SEL: the cells of a list of 4-cell blocks instead of all; a wave's unit is then a group of four listed blocks, which stand for
// the four blocks of a page.
// ONCE: the pages go past the caches.  What a call of many pages leaves there is gone before anyone comes back to it, and its way
// in costs: sixteen contexts of 8k to 128k 250 -> 222 us (5.6 -> 6.3 TB/s), eight of 1k to 32k 33.4 -> 30.0.  Eight of 6000,
// which stay in the 256 MB behind the dies' caches between two calls, 15.8 -> 18.0.
template <bool SEL, bool ONCE, typename Args>
__global__ __launch_bounds__(kBlock, 2) void decode_attn_f8p_kernel(const Args P) {
    constexpr bool DESC = std::is_same<Args, AttnKernelParams>::value;
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
    const int first = range * pps + wave;  // this wave's units: pages (groups of listed blocks) first + wave + 4 i, i < mine

    // Pages of units, 64 at a time: lane i has the page of unit i (SEL: the id of block i % 4 of unit i / 4, and its page).
    // Past the end the last one again: everything asked for is in the pool.
    constexpr int kAhead = SEL ? 16 : 64;  // units
    int ids = 0, blocks = 0, listed = 0;
    if constexpr (SEL) listed = (int)min(P.counts[e], (uint32_t)P.max_ids);
    const int total = SEL ? (listed + 3) >> 2 : pos / kPage + 1;
    const int mine = __builtin_amdgcn_readfirstlane(max((min((range + 1) * pps, total) - first + kWaves - 1) / kWaves, 0));
    const auto fetch_ids = [&](int from) {
        if constexpr (SEL) {
            // (a list need not be there past its length)
            const int i = (first + kWaves * (from + (lane >> 2))) * 4 + (lane & 3);
            const uint32_t id = i < listed ? P.ids[(size_t)e * (size_t)P.id_stride + (size_t)i] : 0xffffffffu;
            blocks = (int)id;
            ids = table[min(id, (uint32_t)pos >> 2) >> 2];
        } else {
            ids = table[first + kWaves * min(from + lane, mine - 1)];
        }
    };
    if (mine > 0) fetch_ids(0);

    // q is asked for behind the first pages, which take longer (32 contexts of 2048: 19.2 us against 19.8 in front of them); SEL
    // asks before, while it still follows its list to the pages (eight lists of 513 blocks: 14.8 us against 15.5).
    f8_f4 raw[8][2];
    const auto fetch_q = [&] {
        // (a lane without a head has the first one's row: its column of the products is its own, and nothing of it is stored)
        const float* const qrow = P.q + ((size_t)e * P.n_q + (size_t)kvh * P.group + (size_t)(c < P.group ? c : 0)) * kHd;
#pragma unroll
        for (int f = 0; f < 8; ++f) {
            const int s = 4 * (f >> 1) + g;
            const float* const at = qrow + 128 * (s >> 3) + 4 * (s & 7) + 64 * (f & 1);
            raw[f][0] = *reinterpret_cast<const f8_f4*>(at);
            raw[f][1] = *reinterpret_cast<const f8_f4*>(at + 32);
        }
    };
    if constexpr (SEL) fetch_q();

    f8_u4 k[2][4], v[2][4];
    f8_i2 ex[2];
    int vb[2] = {0, 0};  // SEL: the block of cells 4 g ..
    const auto load = [](gptr at) {
        if constexpr (ONCE) return __builtin_nontemporal_load((gptr_u4)at);
        else return *(gptr_u4)at;
    };
    const auto block_at = [&](uint32_t id) { return (size_t)((min(id, (uint32_t)pos >> 2) & 3) * 1024); };
    // (the exponents ahead of K: the scores wait for K alone, not for the V asked for since)
    const auto load_k = [&](int u) {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const int w = min(u + p, mine - 1) & (kAhead - 1);
            gptr at;
            if constexpr (SEL) {
                ex[p] = *(gptr_i2)(gptr)(lines + (size_t)(unsigned)__shfl(ids, 4 * w + g, 64) * k_page);
                const int from = 4 * w + (c >> 2);
                const size_t page = (size_t)(unsigned)__shfl(ids, from, 64);
                at = (gptr)(kpool + page * k_page + block_at((uint32_t)__shfl(blocks, from, 64))) + (g * 64 + (c & 3) * 16);
            } else {
                const size_t page = (size_t)(unsigned)__builtin_amdgcn_readlane(ids, w);
                ex[p] = *(gptr_i2)(gptr)(lines + page * k_page);
                at = (gptr)(kpool + page * k_page) + ((c >> 2) * 1024 + g * 64 + (c & 3) * 16);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) k[p][i] = load(at + 256 * i);
        }
    };
    const auto load_v = [&](int u) {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const int w = min(u + p, mine - 1) & (kAhead - 1);
            gptr at;
            if constexpr (SEL) {
                const int from = 4 * w + g;
                vb[p] = __shfl(blocks, from, 64);
                at = (gptr)(vpool + (size_t)(unsigned)__shfl(ids, from, 64) * v_page + block_at((uint32_t)vb[p])) + c * 16;
            } else {
                at = (gptr)(vpool + (size_t)(unsigned)__builtin_amdgcn_readlane(ids, w) * v_page) + (g * 1024 + c * 16);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) v[p][i] = load(at + 256 * i);
        }
    };

    Walk W;
    if (mine > 0) {
        load_k(0);
        load_v(0);
    }
    if constexpr (!SEL) fetch_q();
    W.split_q(raw, P.scale_log2e);
    // Two forms of a step, the last one asks for nothing: of one with branches around its loads the compiler cannot tell what is in
    // flight behind them, and waits for V with K (eight contexts of 1k to 32k 31.2 us instead of 30.0).
    const auto step = [&](int u, auto asks) __attribute__((always_inline)) {
        constexpr bool more = decltype(asks)::value;
        int ek[2], ev[2];
#pragma unroll
        for (int p = 0; p < 2; ++p) ek[p] = f8p_exponent_read(ex[p].x), ev[p] = f8p_exponent_read(ex[p].y);
        float z[2][4];
        unsigned live_v[2] = {0xffffffffu, 0xffffffffu};
        W.scores(k, ek, ev, z);
        if constexpr (more) {
            if (((u + 2) & (kAhead - 1)) == 0) {
                fetch_ids(u + 2);
                asm volatile("" : "+v"(ids));  // waited for here: behind the branch every trip would wait for the V it has in flight
            }
            load_k(u + 2);
        }
        if constexpr (SEL) {
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                live_v[p] = 0;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool live = u + p < mine && block_cell_live((uint32_t)vb[p], r, pos);
                    z[p][r] = live ? z[p][r] : -INFINITY;
                    live_v[p] |= live ? 0xffu << (8 * r) : 0u;
                }
            }
        } else if constexpr (!more) {
            // cells past the position, and the page asked for twice
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const int at = u + p < mine ? (first + kWaves * (u + p)) * kPage + 4 * g : pos + 1;
                live_v[p] = live_bytes(at, pos);
#pragma unroll
                for (int r = 0; r < 4; ++r) z[p][r] = at + r <= pos ? z[p][r] : -INFINITY;
            }
        }
        f8_h8 ph, pl;
        W.softmax(z, ev, ph, pl);
        if constexpr (SEL || !more) {
            // values that no weight belongs to may be anything (a weight of 0 would not keep NaN away)
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
                for (int i = 0; i < 4; ++i) v[p][i] &= live_v[p];
        }
        W.add_values(v, ph, pl);
        if constexpr (more) load_v(u + 2);
    };
    int last = 0;
    for (; last + 2 < mine; last += 2) step(last, std::true_type{});
    if (mine > 0) step(last, std::false_type{});

    // ---- the four waves' results folded; wave w sums columns 64 w .. 64 w + 63 and writes them ----
    W.l = sum_over_lane_groups(W.l);
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            *reinterpret_cast<f8_f4*>(&L.o[wave][c][64 * a + 16 * g + 4 * r]) = f8_f4{W.o[a][0][r], W.o[a][1][r], W.o[a][2][r], W.o[a][3][r]};
    if (g == 0) L.m[wave][c] = W.m, L.l[wave][c] = W.l;
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

// Bytes from which on pages go past the caches (ONCE): what the calls of one token walk, of all layers of the pool, before they come
// back to the first page.  (Eight contexts of 12000, 94 MiB: 22.3 us kept, 22.6 past; of 14000, 109 MiB: 26.3 kept, 25.2 past.)
constexpr int64_t kOnceFrom = 96ll << 20;

}  // namespace

hipError_t launch_decode_attn_f8p(const AttnKernelParams& kp, const AttnBatch& b, int32_t n_layers, bool sel, int32_t total, hipStream_t stream,
                                  hipEvent_t start, hipEvent_t stop) {
    const auto launch = [&](auto kernel, const auto& args) {
        if (start) hipExtLaunchKernelGGL(kernel, dim3((unsigned)total), dim3(kBlock), 0, stream, start, stop, 0, args);
        else hipLaunchKernelGGL(kernel, dim3((unsigned)total), dim3(kBlock), 0, stream, args);
    };
    int64_t cells = 0;
    for (int i = 0; i < b.n; ++i) cells += b.pos[i] + 1;
    const bool once = cells * kp.n_kv * 2 * kF8Hd * n_layers >= kOnceFrom;
    if (kp.bd) {
        // (the device's positions are a plan's; b has those that it began with)
        if (once) launch(decode_attn_f8p_kernel<false, true, AttnKernelParams>, kp);
        else launch(decode_attn_f8p_kernel<false, false, AttnKernelParams>, kp);
        return hipGetLastError();
    }
    const auto with = [&](auto& args) {
        using Args = std::decay_t<decltype(args)>;
        static_cast<AttnKernelParams&>(args) = kp;
        if (sel) launch(decode_attn_f8p_kernel<true, false, Args>, args);
        else if (once) launch(decode_attn_f8p_kernel<false, true, Args>, args);
        else launch(decode_attn_f8p_kernel<false, false, Args>, args);
    };
    if (b.n <= kFewEntries) {
        AttnKernelArgs<AttnBatchFew> args{};
        args.b.n = b.n;
        for (int i = 0; i < b.n; ++i) args.b.row[i] = b.row[i], args.b.pos[i] = b.pos[i], args.b.wg_base[i] = b.wg_base[i], args.b.pps[i] = b.pps[i];
        with(args);
    } else {
        AttnKernelArgs<AttnBatch> args;
        args.b = b;
        with(args);
    }
    return hipGetLastError();
}

}  // namespace bkv
