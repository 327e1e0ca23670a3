// Rows into and out of pools in the e4m3 layout (f8p.hpp), for gfx950.
//
// Written rows join a page under one scale with the rows below them that it holds already.  So a work-group has a whole unit,
// K or V of a (page, kv head): it holds all 16 rows in registers, 16 values a thread, agrees on the largest magnitude, and
// writes all codes.  Rows behind the last one written are cleared: of what others left in a page nothing counts that lies behind a
// written row.  (K and V in one work-group: five ragged chunks of 2073 rows at n_kv = 4 9.5 us, apart 8.7.)
//
// Everything here moves bytes.  Small calls take what a launch and two dependent trips to memory take, 3.5 us; reading back
// 131072 cells as binary16, 402 MB, takes 67 us, 6.0 TB/s, what a copy reaches here.  131072 rows in take 108 us from f32 rows (672 MB, 6.2
// TB/s) into pages that the caches behind the dies hold, 136 into pages scattered over 2.3 GB; from binary16 rows (404 MB) 113 to
// 119: K is read 64 bytes of a row at a time.  131072 cells out of the other layouts as f32 / f16: f16 182 / 144 us, q8_0 V 139 / 107,
// int8 95 / 87.
#include <algorithm>
#include <type_traits>

#include "bkv_internal.hpp"
#include "f8p.hpp"
#include "quant_decode.hpp"
#include "quant_encode.hpp"

namespace bkv {

namespace {

constexpr int kBlock = 64 * kF8Waves;
typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));

struct F8MoveGeom {
    int32_t n_kv, max_pages_per_seq;
};

// Four consecutive source values; binary16 under the cache's load rule (exponent field 0 reads as zero).
__device__ __forceinline__ void load4(const float* p, float (&x)[4]) {
    const v4u a = __builtin_nontemporal_load(reinterpret_cast<const v4u*>(p));
    x[0] = __uint_as_float(a.x), x[1] = __uint_as_float(a.y), x[2] = __uint_as_float(a.z), x[3] = __uint_as_float(a.w);
}
__device__ __forceinline__ void load4(const uint16_t* p, float (&x)[4]) {
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    const h4 h = __builtin_bit_cast(h4, __builtin_nontemporal_load(reinterpret_cast<const v2u*>(p)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float v = (float)h[i];
        x[i] = fabsf(v) < 0x1p-14f ? __builtin_copysignf(0.0f, v) : v;
    }
}

__device__ __forceinline__ float wave_max_of(float a) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) a = fmaxf(a, __shfl_xor(a, off, 64));
    return a;
}

// What thread (wave w, lane l) has of a unit.
//   K  rows 8 (w / 2) + l / 8, piece s = 8 (w % 2) + l % 8: elements k_col + 32 u + 0..3, u < 4, 16 bytes at k_at.
//      Eight lanes read 128 bytes of a row at a time and write 128 bytes of codes.
//   V  rows 4 w + 0..3, elements 4 l .. 4 l + 3, 16 bytes at v_at.
struct F8Share {
    int k_row, k_col, k_at;
    int v_row, v_col, v_at;
    __device__ __forceinline__ explicit F8Share(int tid) {
        const int w = tid >> 6, l = tid & 63;
        k_row = 8 * (w >> 1) + (l >> 3);
        k_col = 128 * (w & 1) + 4 * (l & 7);
        k_at = (k_row >> 2) * 1024 + (8 * (w & 1) + (l & 7)) * 64 + (k_row & 3) * 16;
        v_row = 4 * w;
        v_col = 4 * l;
        v_at = w * 1024 + l * 16;
    }
};

// One half (K or V) of a unit that lies in registers, x[u]: K's elements k_col + 32 u .., V's row v_row + u, coded and stored.
// Rows below `kept` are in the page and come from `old` (loaded by the caller) under their old scale, rows from `end` on are
// cleared.
struct F8Old {
    v4u w;
    int e;
};
// First the page's rows as they are to be, and the wave's largest magnitude to red[wave]; behind a barrier, the codes.
template <bool V>
__device__ __forceinline__ void settle_rows(const F8Share& at, float (&x)[4][4], int kept, int end, const F8Old& old, float* red, int tid) {
    const auto row = [&](int u) { return V ? at.v_row + u : at.k_row; };
    if (kept > 0) {
        const float scale = exp2_int(old.e);
        unsigned in[4] = {old.w.x, old.w.y, old.w.z, old.w.w}, rows[4];
        if constexpr (V) transpose4x4_bytes(in, rows);
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (row(u) < kept) f8p_values4(V ? rows[u] : in[u], scale, x[u]);
    }
    float top = 0.0f;
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (row(u) >= end) x[u][i] = 0.0f;
            top = amax_finite(top, x[u][i]);
        }
    top = wave_max_of(top);
    if ((tid & 63) == 0) red[tid >> 6] = top;
}
template <bool V>
__device__ __forceinline__ void store_codes(const F8Share& at, const float (&x)[4][4], const float* red, uint8_t* unit, int32_t* exponent, int tid) {
    const int e = f8p_exponent(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    const float by = exp2_int(-e);
    unsigned codes[4], out[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) out[u] = codes[u] = f8p_codes4(x[u], by);
    if constexpr (V) transpose4x4_bytes(codes, out);
    *reinterpret_cast<v4u*>(unit + (V ? at.v_at : at.k_at)) = v4u{out[0], out[1], out[2], out[3]};
    if (tid == 0) *exponent = e;
}

struct F8Target {
    uint8_t *kunit, *vunit;
    int32_t* line;
};
__device__ __forceinline__ F8Target target_of(const F8MoveGeom& g, uint8_t* kpool, uint8_t* vpool, const int32_t* tables, int row, int page, int kvh) {
    const int32_t phys = tables[(size_t)row * (size_t)g.max_pages_per_seq + (size_t)page];
    F8Target t;
    uint8_t* const kp = kpool + (size_t)phys * f8p_k_page_bytes(g.n_kv);
    t.kunit = kp + (size_t)kvh * kF8Unit;
    t.vunit = vpool + (size_t)phys * f8p_v_page_bytes(g.n_kv) + (size_t)kvh * kF8Unit;
    t.line = reinterpret_cast<int32_t*>(kp + (size_t)g.n_kv * kF8Unit) + 2 * kvh;
    return t;
}
template <bool V>
__device__ __forceinline__ F8Old old_of(const F8Target& t, const F8Share& at) {
    return F8Old{*reinterpret_cast<const v4u*>(V ? t.vunit + at.v_at : t.kunit + at.k_at), f8p_exponent_read(t.line[V])};
}

// Which entry's page a work-group has.  By the grid: a row of it for each entry, as long as the longest (AppendBatchOf); or, where
// that leaves many work-groups with nothing, by a search of the entries, the grid as long as the batch has pages (F8Batch).
// find: `at`, which page of the launch, becomes which page of the entry; false where there is none.
struct F8Rows {
    int row, pos0, n_tok, src0;
};
__host__ __device__ inline int pages_touched(int pos0, int n_tok) { return n_tok > 0 ? (pos0 + (n_tok - 1)) / kF8Page - pos0 / kF8Page + 1 : 0; }
template <int N>
__device__ __forceinline__ bool find(const AppendBatchOf<N>& b, int& at, F8Rows& r) {
    const int e = blockIdx.y;
    r = F8Rows{b.row[e], b.pos0[e], b.n_tok[e], b.src0[e]};
    return at < pages_touched(r.pos0, r.n_tok);
}
// base[i]: pages of the entries before i; behind the last one INT32_MAX
template <int N>
struct F8Batch : AppendBatchOf<N> {
    int32_t base[N];
};
template <int N>
__device__ __forceinline__ bool find(const F8Batch<N>& b, int& at, F8Rows& r) {
    int e = -1;
#pragma unroll
    for (int i = 0; i < N; ++i) e += at >= b.base[i] ? 1 : 0;
    at -= b.base[e];
    r = F8Rows{b.row[e], b.pos0[e], b.n_tok[e], b.src0[e]};
    return true;
}
// a step plan's: one token of every entry of the descriptor
struct F8DescBatch {
    const AttnBatch* bd;
};
__device__ __forceinline__ bool find(const F8DescBatch& b, int& at, F8Rows& r) {
    const int e = blockIdx.y;
    r = F8Rows{b.bd->row[e], b.bd->pos[e], 1, e};
    return true;
}

// Which of a launch's work a work-group has, of which there is one for (page, kv head, K or V): both halves of a (page, kv head)
// side by side, in turns so that the dies, which have every eighth work-group, get as much of K as of V.
struct F8Work {
    int page, kvh;  // page: of the launch
    bool v;
};
__device__ __forceinline__ F8Work work_of(int x, int n_kv) {
    F8Work w;
    w.v = ((x ^ (x >> 3)) & 1) != 0;
    w.page = (x >> 1) / n_kv;
    w.kvh = (x >> 1) - w.page * n_kv;
    return w;
}

// The rows of a work-group's page: where they come from, which of them the call writes.
struct F8Span {
    int page, kept, end;
};
__device__ __forceinline__ F8Span span_of(const F8Rows& r, int at_page) {
    F8Span s;
    s.page = r.pos0 / kF8Page + at_page;
    s.kept = max(r.pos0 - s.page * kF8Page, 0);
    s.end = min(r.pos0 + r.n_tok - s.page * kF8Page, kF8Page);
    return s;
}
// (rows outside of the call's are clamped to it and dropped: no branch around a load)
__device__ __forceinline__ size_t source_of(const F8Rows& r, const F8Span& s, int n_kv, int kvh, int row, int col) {
    const int tok = min(max(s.page * kF8Page + row - r.pos0, 0), r.n_tok - 1);
    return (((size_t)r.src0 + (size_t)tok) * (size_t)n_kv + (size_t)kvh) * kF8Hd + (size_t)col;
}

template <bool V, typename SrcT>
__device__ __forceinline__ void append_unit(const F8Rows& r, const F8Span& s, int n_kv, int kvh, const F8Target& t, const SrcT* __restrict__ src,
                                            float* red) {
    const int tid = threadIdx.x;
    const F8Share at(tid);
    float x[4][4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
        load4(src + (V ? source_of(r, s, n_kv, kvh, at.v_row + u, at.v_col) : source_of(r, s, n_kv, kvh, at.k_row, at.k_col + 32 * u)), x[u]);
    F8Old old{};
    if (s.kept > 0) old = old_of<V>(t, at);
    settle_rows<V>(at, x, s.kept, s.end, old, red, tid);
    __syncthreads();
    store_codes<V>(at, x, red, V ? t.vunit : t.kunit, t.line + V, tid);
}
template <typename SrcT, typename Batch>
__global__ __launch_bounds__(kBlock) void append_f8p_kernel(Batch b, F8MoveGeom g, uint8_t* __restrict__ kpool, uint8_t* __restrict__ vpool,
                                                            const int32_t* __restrict__ tables, const SrcT* __restrict__ ks,
                                                            const SrcT* __restrict__ vs) {
    __shared__ float red[kF8Waves];
    F8Work w = work_of(blockIdx.x, g.n_kv);
    F8Rows r;
    if (!find(b, w.page, r)) return;
    const F8Span s = span_of(r, w.page);
    const F8Target t = target_of(g, kpool, vpool, tables, r.row, s.page, w.kvh);
    if (w.v) append_unit<true>(r, s, g.n_kv, w.kvh, t, vs, red);
    else append_unit<false>(r, s, g.n_kv, w.kvh, t, ks, red);
}

// The same with K through RMSNorm and the rotary first; arithmetic as in append_kprep_kernel (kv_move.hip).  A work-group has both
// halves of a (page, kv head): V arrives, is coded and stored while one wave adds up K's squares, one after the other as the sum
// is defined.  Eight work-groups a compute unit, as many as LDS and threads let be there, hide what they can of that chain
// (registers are kept to that: 86 of them and five work-groups cost two prompts of 8191 tokens 3 us).  Those, 84 MB, take 21.7 us;
// without the sums, the products and the rotary, 17 us.
struct F8Prep {
    const float* gamma;
    const float* table;
    const int32_t* positions;
    float eps;
    int32_t n_rot, max_pos;
};
constexpr int kPrepStride = kF8Hd + 4;
template <typename Batch>
__global__ __launch_bounds__(kBlock, 8) void append_kprep_f8p_kernel(Batch b, F8MoveGeom g, F8Prep kp, uint8_t* __restrict__ kpool,
                                                                     uint8_t* __restrict__ vpool, const int32_t* __restrict__ tables,
                                                                     const float* __restrict__ ks, const float* __restrict__ vs) {
#pragma clang fp contract(off)
    __shared__ float red_v[kF8Waves], red_k[kF8Waves];
    __shared__ __attribute__((aligned(16))) float rows_s[kF8Page * kPrepStride];
    __shared__ double inv_s[kF8Page];
    int at_page = (int)blockIdx.x / g.n_kv;
    const int kvh = (int)blockIdx.x - at_page * g.n_kv;
    F8Rows r;
    if (!find(b, at_page, r)) return;
    const F8Span s = span_of(r, at_page);
    const int tid = threadIdx.x;
    const F8Share at(tid);
    const F8Target t = target_of(g, kpool, vpool, tables, r.row, s.page, kvh);
    float v[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float x[4];
        load4(ks + source_of(r, s, g.n_kv, kvh, at.v_row + i, at.v_col), x);
        *reinterpret_cast<float4*>(rows_s + (at.v_row + i) * kPrepStride + at.v_col) = make_float4(x[0], x[1], x[2], x[3]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) load4(vs + source_of(r, s, g.n_kv, kvh, at.v_row + i, at.v_col), v[i]);
    const float gamma = kp.gamma[tid];
    F8Old old{};
    if (s.kept > 0) old = old_of<true>(t, at);
    __syncthreads();
    // (one wave of the four, another in the next work-group: a compute unit's would all wait for one SIMD: 0.7 us of the prompts')
    const int sum_row = (tid ^ (int)(blockIdx.x << 6)) & (kBlock - 1);
    if (sum_row < kF8Page) {
        double ss = 0.0;  // in element order; a product of two floats is exact, fused it is the same sum
#pragma unroll 4
        for (int i = 0; i < kF8Hd; i += 4) {
            const float4 x = *reinterpret_cast<const float4*>(rows_s + sum_row * kPrepStride + i);
            ss = __builtin_fma((double)x.x, (double)x.x, ss);
            ss = __builtin_fma((double)x.y, (double)x.y, ss);
            ss = __builtin_fma((double)x.z, (double)x.z, ss);
            ss = __builtin_fma((double)x.w, (double)x.w, ss);
        }
        inv_s[sum_row] = 1.0 / sqrt(ss / (double)kF8Hd + (double)kp.eps);
    }
    settle_rows<true>(at, v, s.kept, s.end, old, red_v, tid);
    __syncthreads();
    store_codes<true>(at, v, red_v, t.vunit, t.line + 1, tid);
#pragma unroll 4
    for (int row = 0; row < kF8Page; ++row) {
        float* d = rows_s + row * kPrepStride + tid;
        *d = (float)((double)*d * inv_s[row] * (double)gamma);
    }
    __syncthreads();
    // the rotary: pairs tid / 16 + 16 i of row tid % 16 (clamped to the call's cells: positions need not cover others)
    const int half = kp.n_rot / 2, rot_row = tid & (kF8Page - 1);
    const int cell = min(max(s.page * kF8Page + rot_row, r.pos0), r.pos0 + r.n_tok - 1);
    const int pos = min(max(kp.positions ? kp.positions[cell] : cell, 0), kp.max_pos - 1);
    const float2* const factors = reinterpret_cast<const float2*>(kp.table) + (size_t)pos * half;
    float* const d = rows_s + rot_row * kPrepStride;
    for (int j = tid / kF8Page; j < half; j += kBlock / kF8Page) {
        const float2 cs = factors[j];
        const double x = (double)d[j], y = (double)d[j + half], c = (double)cs.x, si = (double)cs.y;
        const double xc = x * c, ys = y * si, xs = x * si, yc = y * c;
        d[j] = (float)(xc - ys);
        d[j + half] = (float)(xs + yc);
    }
    __syncthreads();
    float k[4][4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const float4 x = *reinterpret_cast<const float4*>(rows_s + at.k_row * kPrepStride + at.k_col + 32 * u);
        k[u][0] = x.x, k[u][1] = x.y, k[u][2] = x.z, k[u][3] = x.w;
    }
    if (s.kept > 0) old = old_of<false>(t, at);
    settle_rows<false>(at, k, s.kept, s.end, old, red_k, tid);
    __syncthreads();
    store_codes<false>(at, k, red_k, t.kunit, t.line, tid);
}

// ---- rows read back -----------------------------------------------------------------------------------
// The values of cells cell0[i] .. of sequence i as rows [sum n_tok][n_kv][hd], f32 or binary16 (rounded to nearest).
// The batch's pos0 = first cell, n_tok = cells, src0 = first row of the output.
__device__ __forceinline__ void put4(float* p, const float (&x)[4]) {
    __builtin_nontemporal_store(v4u{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])}, reinterpret_cast<v4u*>(p));
}
__device__ __forceinline__ void put4(uint16_t* p, const float (&x)[4]) {
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    const h4 h = {(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
    __builtin_nontemporal_store(__builtin_bit_cast(v2u, h), reinterpret_cast<v2u*>(p));
}

__device__ __forceinline__ void put8(uint16_t* p, const float (&x)[8]) {
    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
    h8 h;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = (_Float16)x[i];
    __builtin_nontemporal_store(__builtin_bit_cast(v4u, h), reinterpret_cast<v4u*>(p));
}
// the neighbour's (lane ^ 1) value
__device__ __forceinline__ unsigned of_neighbour(unsigned x) { return (unsigned)__builtin_amdgcn_mov_dpp((int)x, 0xb1, 0xf, 0xf, true); }

// e4m3 pools: a work-group per (page, kv head), shares as on the way in.
template <typename DstT, typename Batch>
__global__ __launch_bounds__(kBlock) void read_rows_f8p_kernel(Batch b, F8MoveGeom g, const uint8_t* __restrict__ kpool,
                                                               const uint8_t* __restrict__ vpool, const int32_t* __restrict__ tables,
                                                               DstT* __restrict__ ko, DstT* __restrict__ vo) {
    int at_page = (int)blockIdx.x / g.n_kv;
    const int kvh = (int)blockIdx.x - at_page * g.n_kv;
    F8Rows r;
    if (!find(b, at_page, r)) return;
    const int page = r.pos0 / kF8Page + at_page;
    const F8Share at(threadIdx.x);
    const F8Target t = target_of(g, const_cast<uint8_t*>(kpool), const_cast<uint8_t*>(vpool), tables, r.row, page, kvh);
    const F8Old k = old_of<false>(t, at), v = old_of<true>(t, at);
    const auto live = [&](int row) { return page * kF8Page + row >= r.pos0 && page * kF8Page + row < r.pos0 + r.n_tok; };
    const auto dst = [&](int row, int col) -> size_t {
        return (((size_t)r.src0 + (size_t)(page * kF8Page + row - r.pos0)) * (size_t)g.n_kv + (size_t)kvh) * kF8Hd + (size_t)col;
    };
    const float ks = exp2_int(k.e), vs = exp2_int(v.e);
    unsigned cols[4] = {v.w.x, v.w.y, v.w.z, v.w.w}, rows[4];
    transpose4x4_bytes(cols, rows);
    if constexpr (std::is_same<DstT, uint16_t>::value) {
        // Two lanes have neighbouring fours: the even one takes both fours of the even dwords, the odd one of the odd dwords, and
        // stores are 16 bytes a lane, whole 128-byte lines an instruction.
        const bool odd = threadIdx.x & 1;
        const auto store = [&](unsigned even_w, unsigned odd_w, float scale, DstT* to) {
            const unsigned mine = odd ? odd_w : even_w, theirs = of_neighbour(odd ? even_w : odd_w);
            float lo[4], hi[4];
            f8p_values4(odd ? theirs : mine, scale, lo);
            f8p_values4(odd ? mine : theirs, scale, hi);
            const float y[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            if (to) put8(to, y);
        };
#pragma unroll
        for (int i = 0; i < 2; ++i)
            store(k.w[2 * i], k.w[2 * i + 1], ks, live(at.k_row) ? ko + dst(at.k_row, at.k_col - 4 * odd + 32 * (2 * i + odd)) : nullptr);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            store(rows[2 * i], rows[2 * i + 1], vs, live(at.v_row + 2 * i + odd) ? vo + dst(at.v_row + 2 * i + odd, at.v_col - 4 * odd) : nullptr);
    } else {
        if (live(at.k_row)) {
            const size_t k0 = dst(at.k_row, at.k_col);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                float y[4];
                f8p_values4(k.w[u], ks, y);
                put4(ko + k0 + 32 * u, y);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float y[4];
            f8p_values4(rows[i], vs, y);
            if (live(at.v_row + i)) put4(vo + dst(at.v_row + i, at.v_col), y);
        }
    }
}

// The other layouts: a thread has four consecutive elements of a (cell, kv head) row of K and of V.
template <int LAYOUT, typename DstT, typename Batch>
__global__ __launch_bounds__(kBlock) void read_rows_kernel(Batch b, F8MoveGeom g, int hd, const uint8_t* __restrict__ kpool,
                                                           const uint8_t* __restrict__ vpool, const int32_t* __restrict__ tables,
                                                           DstT* __restrict__ ko, DstT* __restrict__ vo, unsigned rows) {
    const unsigned per_cell = (unsigned)(g.n_kv * (hd / 4));
    const unsigned idx = blockIdx.x * (unsigned)kBlock + threadIdx.x;  // (below 2^32: checked on the host)
    const unsigned i = idx / per_cell, rest = idx - i * per_cell;
    if (i >= rows) return;
    const unsigned kvh = rest / (unsigned)(hd / 4), d = 4 * (rest - kvh * (unsigned)(hd / 4));
    // the entry of the work-group's first row, and from there on
    int e = -1;
#pragma unroll
    for (int k = 0; k < (int)(sizeof(b.src0) / sizeof(b.src0[0])); ++k)
        e += k < b.n && blockIdx.x * (unsigned)kBlock / per_cell >= (unsigned)b.src0[k] ? 1 : 0;
    while (e + 1 < b.n && i >= (unsigned)b.src0[e + 1]) ++e;
    const unsigned cell = (unsigned)b.pos0[e] + i - (unsigned)b.src0[e];
    const int32_t phys = tables[(size_t)b.row[e] * (size_t)g.max_pages_per_seq + cell / kF8Page];
    const size_t row = ((size_t)phys * g.n_kv + kvh) * kF8Page + cell % kF8Page;
    const auto halves = [&](const uint8_t* pool, float (&x)[4]) {
        const v2u w = *reinterpret_cast<const v2u*>(pool + (row * (size_t)hd + d) * 2);
        x[0] = f16_load(w.x & 0xffffu), x[1] = f16_load(w.x >> 16), x[2] = f16_load(w.y & 0xffffu), x[3] = f16_load(w.y >> 16);
    };
    const auto codes = [](unsigned w, float scale, float (&x)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = (float)(int8_t)(w >> (8 * j)) * scale;
    };
    const auto i8h = [&](const uint8_t* pool, float (&x)[4]) {
        const uint8_t* const p = pool + row * ((size_t)hd + (size_t)(hd / 32) * 2);
        codes(*reinterpret_cast<const unsigned*>(p + d), f16_load(*reinterpret_cast<const uint16_t*>(p + hd + (d / 32) * 2)), x);
    };
    float k[4], v[4];
    if constexpr (LAYOUT == BKV_LAYOUT_I8H) {
        i8h(kpool, k);
        i8h(vpool, v);
    } else {
        halves(kpool, k);
        if constexpr (LAYOUT == BKV_LAYOUT_F16) {
            halves(vpool, v);
        } else {
            const unsigned* const w = reinterpret_cast<const unsigned*>(vpool) + (row * (size_t)(hd / 32) + d / 32) * 9u;
            codes(w[1 + (d % 32) / 4], __uint_as_float(w[0]), v);
        }
    }
    const size_t to = ((size_t)i * (size_t)g.n_kv + kvh) * (size_t)hd + d;
    put4(ko + to, k);
    put4(vo + to, v);
}

F8MoveGeom f8_geom(const bkv_pool* p) { return F8MoveGeom{p->g.n_kv, p->desc.max_pages_per_seq}; }

// f of the batch in the argument struct that suits it, and of the launch's grid, `each` work-groups a page: the smaller structs
// where they fit (kFewEntries), a search of the entries where the other way leaves more than kIdle work-groups with nothing.
// Those cost what starting them costs, the search a trip to the arguments, 0.7 us: one prompt of 8192 and 63 tokens beside it, 128k
// of them idle, 71 us by the grid and 21 by the search; 64 chunks of 64, none, 12.0 and 13.6; five ragged chunks, 1552, 12.6 and 12.8.
constexpr int64_t kIdle = 2048;
template <typename Batch>
void fill_batch(Batch& out, const AppendBatch& b) {
    out.n = b.n;
    for (int i = 0; i < b.n; ++i) {
        out.row[i] = b.row[i];
        out.pos0[i] = b.pos0[i];
        out.n_tok[i] = b.n_tok[i];
        out.src0[i] = b.src0[i];
    }
}
template <int N, typename F>
void with_entries(const AppendBatch& b, int each, F f) {
    int64_t pages = 0, most = 0;
    for (int i = 0; i < b.n; ++i) {
        const int n = pages_touched(b.pos0[i], b.n_tok[i]);
        pages += n;
        most = std::max<int64_t>(most, n);
    }
    if ((most * b.n - pages) * each <= kIdle) {
        AppendBatchOf<N> out{};
        fill_batch(out, b);
        return f(out, dim3((unsigned)(most * each), (unsigned)b.n));
    }
    F8Batch<N> out{};
    fill_batch(out, b);
    int32_t base = 0;
    for (int i = 0; i < N; ++i) {
        out.base[i] = i < b.n ? base : INT32_MAX;
        if (i < b.n) base += pages_touched(b.pos0[i], b.n_tok[i]);
    }
    f(out, dim3((unsigned)(pages * each)));
}
template <typename F>
void with_batch(const AppendBatch& b, int each, F f) {
    if (b.n > kFewEntries) with_entries<BKV_MAX_BATCH>(b, each, f);
    else with_entries<kFewEntries>(b, each, f);
}

}  // namespace

hipError_t launch_append_f8p(bkv_pool* p, int32_t layer, const AppendBatch& b, const void* k, const void* v, bool src_is_f16,
                             hipStream_t stream) {
    with_batch(b, 2 * p->g.n_kv, [&](const auto& batch, dim3 grid) {
        using Batch = std::decay_t<decltype(batch)>;
        const auto launch = [&](auto kernel, auto ks, auto vs) {
            launch_staged(p, BKV_STAGE_APPEND, kernel, grid, dim3(kBlock), 0, stream, batch, f8_geom(p), p->k_layer[(size_t)layer],
                          p->v_layer[(size_t)layer], (const int32_t*)p->table_dev, ks, vs);
        };
        if (src_is_f16) launch(append_f8p_kernel<uint16_t, Batch>, (const uint16_t*)k, (const uint16_t*)v);
        else launch(append_f8p_kernel<float, Batch>, (const float*)k, (const float*)v);
    });
    return hipGetLastError();
}

hipError_t launch_append_f8p_desc(bkv_pool* p, int32_t layer, const AttnBatch* desc, int32_t n, const float* k, const float* v,
                                  hipStream_t stream) {
    hipLaunchKernelGGL((append_f8p_kernel<float, F8DescBatch>), dim3((unsigned)p->g.n_kv * 2, (unsigned)n), dim3(kBlock), 0, stream,
                       F8DescBatch{desc}, f8_geom(p), p->k_layer[(size_t)layer], p->v_layer[(size_t)layer], (const int32_t*)p->table_dev, k, v);
    return hipGetLastError();
}

hipError_t launch_append_kprep_f8p(bkv_pool* p, int32_t layer, const AppendBatch& b, const float* k, const float* v, const float* gamma,
                                   float eps, const float* table, int32_t n_rot, int32_t max_pos, const int32_t* positions,
                                   hipStream_t stream) {
    with_batch(b, p->g.n_kv, [&](const auto& batch, dim3 grid) {
        launch_staged(p, BKV_STAGE_APPEND_KPREP, append_kprep_f8p_kernel<std::decay_t<decltype(batch)>>, grid, dim3(kBlock), 0, stream, batch,
                      f8_geom(p), F8Prep{gamma, table, positions, eps, n_rot, max_pos}, p->k_layer[(size_t)layer], p->v_layer[(size_t)layer],
                      (const int32_t*)p->table_dev, k, v);
    });
    return hipGetLastError();
}

hipError_t launch_read_rows(bkv_pool* p, int32_t layer, const AppendBatch& b, int64_t rows, void* k, void* v, bool to_f16,
                            hipStream_t stream) {
    const uint8_t* const kpool = p->k_layer[(size_t)layer];
    const uint8_t* const vpool = p->v_layer[(size_t)layer];
    const int32_t* const tables = p->table_dev;
    const auto with_outputs = [&](auto ko, auto vo) {
        using DstT = std::remove_pointer_t<decltype(ko)>;
        if (p->g.layout == BKV_LAYOUT_F8P)
            return with_batch(b, p->g.n_kv, [&](const auto& batch, dim3 grid) {
                launch_staged(p, BKV_STAGE_READ_ROWS, read_rows_f8p_kernel<DstT, std::decay_t<decltype(batch)>>, grid, dim3(kBlock), 0, stream, batch,
                              f8_geom(p), kpool, vpool, tables, ko, vo);
            });
        const int64_t threads = rows * p->g.n_kv * (p->g.hd / 4);
        const dim3 grid((unsigned)((threads + kBlock - 1) / kBlock));
        const auto by_layout = [&](const auto& batch) {
            using Batch = std::decay_t<decltype(batch)>;
            const auto launch = [&](auto kernel) {
                launch_staged(p, BKV_STAGE_READ_ROWS, kernel, grid, dim3(kBlock), 0, stream, batch, f8_geom(p), p->g.hd, kpool, vpool, tables, ko, vo,
                              (unsigned)rows);
            };
            if (p->g.layout == BKV_LAYOUT_F16) launch(read_rows_kernel<BKV_LAYOUT_F16, DstT, Batch>);
            else if (p->g.layout == BKV_LAYOUT_Q8V) launch(read_rows_kernel<BKV_LAYOUT_Q8V, DstT, Batch>);
            else launch(read_rows_kernel<BKV_LAYOUT_I8H, DstT, Batch>);
        };
        if (b.n > kFewEntries) return by_layout(b);
        AppendBatchOf<kFewEntries> few{};
        fill_batch(few, b);
        by_layout(few);
    };
    if (to_f16) with_outputs((uint16_t*)k, (uint16_t*)v);
    else with_outputs((float*)k, (float*)v);
    return hipGetLastError();
}

}  // namespace bkv
