// Rows into and out of pools in the e4m3 layout (f8p.hpp), for gfx950.
//
// Written rows join a page under one scale with the rows below them that it holds already.  So a work-group has a whole
// (page, kv head), K and V: it holds all 16 rows of both in registers, 16 + 16 values a thread, agrees on the two largest
// magnitudes, and writes all codes of the page.  Rows behind the last one written are cleared: what a page holds follows from
// the rows written into it, whoever had it before.
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
__device__ __forceinline__ void transpose4x4(const unsigned (&w)[4], unsigned (&t)[4]) { transpose4x4_bytes(w, t); }

// The values of a page that lie in registers, coded and stored.  k[u]: elements k_col + 32 u ..; v[i]: row v_row + i.
// Rows below `kept` are in the page and come from old_k / old_v (loaded by the caller, under their old scales), rows from `end`
// on are cleared.
struct F8Old {
    v4u k, v;
    int ek, ev;
};
__device__ __forceinline__ void store_page(const F8Share& at, float (&k)[4][4], float (&v)[4][4], int kept, int end, const F8Old& old, float* red,
                                           uint8_t* kunit, uint8_t* vunit, int32_t* line, int tid) {
    float ka = 0.0f, va = 0.0f;
    if (kept > 0) {
        const float ks = exp2_int(old.ek), vs = exp2_int(old.ev);
        if (at.k_row < kept) {
#pragma unroll
            for (int u = 0; u < 4; ++u) f8p_values4(old.k[u], ks, k[u]);
        }
        unsigned cols[4] = {old.v.x, old.v.y, old.v.z, old.v.w}, rows[4];
        transpose4x4(cols, rows);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (at.v_row + i < kept) f8p_values4(rows[i], vs, v[i]);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (at.k_row >= end) k[u][i] = 0.0f;
            if (at.v_row + u >= end) v[u][i] = 0.0f;
            ka = amax_finite(ka, k[u][i]);
            va = amax_finite(va, v[u][i]);
        }
    ka = wave_max_of(ka);
    va = wave_max_of(va);
    if ((tid & 63) == 0) red[(tid >> 6) * 2] = ka, red[(tid >> 6) * 2 + 1] = va;
    __syncthreads();
    const int ek = f8p_exponent(fmaxf(fmaxf(red[0], red[2]), fmaxf(red[4], red[6])));
    const int ev = f8p_exponent(fmaxf(fmaxf(red[1], red[3]), fmaxf(red[5], red[7])));
    const float ki = exp2_int(-ek), vi = exp2_int(-ev);
    v4u ko;
#pragma unroll
    for (int u = 0; u < 4; ++u) ko[u] = f8p_codes4(k[u], ki);
    unsigned rows[4], cols[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) rows[i] = f8p_codes4(v[i], vi);
    transpose4x4(rows, cols);
    *reinterpret_cast<v4u*>(kunit + at.k_at) = ko;
    *reinterpret_cast<v4u*>(vunit + at.v_at) = v4u{cols[0], cols[1], cols[2], cols[3]};
    if (tid == 0) line[0] = ek, line[1] = ev;
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
__device__ __forceinline__ F8Old old_of(const F8Target& t, const F8Share& at) {
    F8Old o;
    o.k = *reinterpret_cast<const v4u*>(t.kunit + at.k_at);
    o.v = *reinterpret_cast<const v4u*>(t.vunit + at.v_at);
    o.ek = f8p_exponent_read(t.line[0]);
    o.ev = f8p_exponent_read(t.line[1]);
    return o;
}

// One work-group per (page of an entry, kv head): grid (pages of the longest entry x kv heads, entries).
// Batch: of the call, or (a step plan's) one token of every entry of the descriptor.
struct F8Rows {
    int row, pos0, n_tok, src0;
};
template <typename Batch>
__device__ __forceinline__ F8Rows rows_of(const Batch& b, int s) {
    return F8Rows{b.row[s], b.pos0[s], b.n_tok[s], b.src0[s]};
}
struct F8DescBatch {
    const AttnBatch* bd;
};
__device__ __forceinline__ F8Rows rows_of(const F8DescBatch& b, int s) { return F8Rows{b.bd->row[s], b.bd->pos[s], 1, s}; }

template <typename SrcT, typename Batch>
__global__ __launch_bounds__(kBlock) void append_f8p_kernel(Batch b, F8MoveGeom g, uint8_t* __restrict__ kpool, uint8_t* __restrict__ vpool,
                                                            const int32_t* __restrict__ tables, const SrcT* __restrict__ ks,
                                                            const SrcT* __restrict__ vs) {
    __shared__ float red[2 * kF8Waves];
    const F8Rows r = rows_of(b, blockIdx.y);
    const int first_page = r.pos0 / kF8Page;
    const int at_page = (int)blockIdx.x / g.n_kv, kvh = (int)blockIdx.x - at_page * g.n_kv;
    const int page = first_page + at_page;
    if (r.n_tok == 0 || page > (r.pos0 + r.n_tok - 1) / kF8Page) return;
    const int tid = threadIdx.x;
    const F8Share at(tid);
    const F8Target t = target_of(g, kpool, vpool, tables, r.row, page, kvh);
    const int kept = max(r.pos0 - page * kF8Page, 0), end = min(r.pos0 + r.n_tok - page * kF8Page, kF8Page);
    // rows outside of the call's are clamped to it and dropped: no branch around a load
    const auto src = [&](int row, int col) -> size_t {
        const int tok = min(max(page * kF8Page + row - r.pos0, 0), r.n_tok - 1);
        return (((size_t)r.src0 + (size_t)tok) * (size_t)g.n_kv + (size_t)kvh) * kF8Hd + (size_t)col;
    };
    float k[4][4], v[4][4];
    const size_t k0 = src(at.k_row, at.k_col);
#pragma unroll
    for (int u = 0; u < 4; ++u) load4(ks + k0 + 32 * u, k[u]);
#pragma unroll
    for (int i = 0; i < 4; ++i) load4(vs + src(at.v_row + i, at.v_col), v[i]);
    F8Old old{};
    if (kept > 0) old = old_of(t, at);
    store_page(at, k, v, kept, end, old, red, t.kunit, t.vunit, t.line, tid);
}

// The same with K through RMSNorm and the rotary first; stages and arithmetic as in append_kprep_kernel (kv_move.hip), which this
// layout shares but for the unit of work, a (page, kv head).
struct F8Prep {
    const float* gamma;
    const float* table;
    const int32_t* positions;
    float eps;
    int32_t n_rot, max_pos;
};
constexpr int kPrepStride = kF8Hd + 4;
__global__ __launch_bounds__(kBlock) void append_kprep_f8p_kernel(AppendBatch b, F8MoveGeom g, F8Prep kp, uint8_t* __restrict__ kpool,
                                                                  uint8_t* __restrict__ vpool, const int32_t* __restrict__ tables,
                                                                  const float* __restrict__ ks, const float* __restrict__ vs) {
#pragma clang fp contract(off)
    __shared__ float red[2 * kF8Waves];
    __shared__ __attribute__((aligned(16))) float rows_s[kF8Page * kPrepStride];
    __shared__ double inv_s[kF8Page];
    __shared__ int pos_s[kF8Page];
    const F8Rows r = rows_of(b, blockIdx.y);
    const int first_page = r.pos0 / kF8Page;
    const int at_page = (int)blockIdx.x / g.n_kv, kvh = (int)blockIdx.x - at_page * g.n_kv;
    const int page = first_page + at_page;
    if (r.n_tok == 0 || page > (r.pos0 + r.n_tok - 1) / kF8Page) return;
    const int tid = threadIdx.x;
    const F8Share at(tid);
    const F8Target t = target_of(g, kpool, vpool, tables, r.row, page, kvh);
    const int kept = max(r.pos0 - page * kF8Page, 0), end = min(r.pos0 + r.n_tok - page * kF8Page, kF8Page);
    const auto src = [&](int row, int col) -> size_t {
        const int tok = min(max(page * kF8Page + row - r.pos0, 0), r.n_tok - 1);
        return (((size_t)r.src0 + (size_t)tok) * (size_t)g.n_kv + (size_t)kvh) * kF8Hd + (size_t)col;
    };
    float v[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float x[4];
        load4(ks + src(at.v_row + i, at.v_col), x);
#pragma unroll
        for (int j = 0; j < 4; ++j) rows_s[(at.v_row + i) * kPrepStride + at.v_col + j] = x[j];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) load4(vs + src(at.v_row + i, at.v_col), v[i]);
    const float gamma = kp.gamma[tid];
    F8Old old{};
    if (kept > 0) old = old_of(t, at);
    if (tid >= 64 && tid < 64 + kF8Page) {
        // (clamped to the call's cells: positions need not cover others)
        const int cell = min(max(page * kF8Page + tid - 64, r.pos0), r.pos0 + r.n_tok - 1);
        const int64_t pos = kp.positions ? (int64_t)kp.positions[cell] : (int64_t)cell;
        pos_s[tid - 64] = (int)(pos < 0 ? 0 : (pos > kp.max_pos - 1 ? kp.max_pos - 1 : pos));
    }
    __syncthreads();
    if (tid < kF8Page) {
        double ss = 0.0;  // in element order
#pragma unroll 8
        for (int i = 0; i < kF8Hd; i += 4) {
            const float4 x = *reinterpret_cast<const float4*>(rows_s + tid * kPrepStride + i);
            ss += (double)x.x * (double)x.x;
            ss += (double)x.y * (double)x.y;
            ss += (double)x.z * (double)x.z;
            ss += (double)x.w * (double)x.w;
        }
        inv_s[tid] = 1.0 / sqrt(ss / (double)kF8Hd + (double)kp.eps);
    }
    __syncthreads();
#pragma unroll
    for (int row = 0; row < kF8Page; ++row) {
        float* d = rows_s + row * kPrepStride + tid;
        *d = (float)((double)*d * inv_s[row] * (double)gamma);
    }
    __syncthreads();
    const int half = kp.n_rot / 2;
    for (int idx = tid; idx < kF8Page * half; idx += kBlock) {
        const int row = idx & (kF8Page - 1), j = idx / kF8Page;
        const float2 cs = reinterpret_cast<const float2*>(kp.table)[(size_t)pos_s[row] * half + j];
        float* d = rows_s + row * kPrepStride;
        const double x = (double)d[j], y = (double)d[j + half], c = (double)cs.x, s = (double)cs.y;
        const double xc = x * c, ys = y * s, xs = x * s, yc = y * c;
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
    store_page(at, k, v, kept, end, old, red, t.kunit, t.vunit, t.line, tid);
}

// ---- rows read back -----------------------------------------------------------------------------------
// The values of cells cell0[i] .. of sequence i as rows [sum n_tok][n_kv][hd], f32 or binary16 (rounded to nearest).
// AppendBatch: pos0 = first cell, n_tok = cells, src0 = first row of the output.
__device__ __forceinline__ void put4(float* p, const float (&x)[4]) {
    __builtin_nontemporal_store(v4u{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])}, reinterpret_cast<v4u*>(p));
}
__device__ __forceinline__ void put4(uint16_t* p, const float (&x)[4]) {
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    const h4 h = {(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
    __builtin_nontemporal_store(__builtin_bit_cast(v2u, h), reinterpret_cast<v2u*>(p));
}

// e4m3 pools: a work-group per (page, kv head), shares as on the way in.
template <typename DstT, typename Batch>
__global__ __launch_bounds__(kBlock) void read_rows_f8p_kernel(Batch b, F8MoveGeom g, const uint8_t* __restrict__ kpool,
                                                               const uint8_t* __restrict__ vpool, const int32_t* __restrict__ tables,
                                                               DstT* __restrict__ ko, DstT* __restrict__ vo) {
    const F8Rows r = rows_of(b, blockIdx.y);
    const int first_page = r.pos0 / kF8Page;
    const int at_page = (int)blockIdx.x / g.n_kv, kvh = (int)blockIdx.x - at_page * g.n_kv;
    const int page = first_page + at_page;
    if (r.n_tok == 0 || page > (r.pos0 + r.n_tok - 1) / kF8Page) return;
    const F8Share at(threadIdx.x);
    const F8Target t = target_of(g, const_cast<uint8_t*>(kpool), const_cast<uint8_t*>(vpool), tables, r.row, page, kvh);
    const F8Old x = old_of(t, at);
    const auto live = [&](int row) { return page * kF8Page + row >= r.pos0 && page * kF8Page + row < r.pos0 + r.n_tok; };
    const auto dst = [&](int row, int col) -> size_t {
        return (((size_t)r.src0 + (size_t)(page * kF8Page + row - r.pos0)) * (size_t)g.n_kv + (size_t)kvh) * kF8Hd + (size_t)col;
    };
    const float ks = exp2_int(x.ek), vs = exp2_int(x.ev);
    if (live(at.k_row)) {
        const size_t k0 = dst(at.k_row, at.k_col);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            float y[4];
            f8p_values4(x.k[u], ks, y);
            put4(ko + k0 + 32 * u, y);
        }
    }
    unsigned cols[4] = {x.v.x, x.v.y, x.v.z, x.v.w}, rows[4];
    transpose4x4(cols, rows);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float y[4];
        f8p_values4(rows[i], vs, y);
        if (live(at.v_row + i)) put4(vo + dst(at.v_row + i, at.v_col), y);
    }
}

// The other layouts: a thread has four consecutive elements of a (cell, kv head) row of K and of V.
template <int LAYOUT, typename DstT, typename Batch>
__global__ __launch_bounds__(kBlock) void read_rows_kernel(Batch b, F8MoveGeom g, int hd, const uint8_t* __restrict__ kpool,
                                                           const uint8_t* __restrict__ vpool, const int32_t* __restrict__ tables,
                                                           DstT* __restrict__ ko, DstT* __restrict__ vo) {
    const F8Rows r = rows_of(b, blockIdx.y);
    const unsigned per_cell = (unsigned)(g.n_kv * (hd / 4));
    const int64_t idx = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (idx >= (int64_t)r.n_tok * per_cell) return;
    const unsigned i = (unsigned)(idx / per_cell), rest = (unsigned)(idx - (int64_t)i * per_cell);
    const unsigned kvh = rest / (unsigned)(hd / 4), d = 4 * (rest - kvh * (unsigned)(hd / 4));
    const unsigned cell = (unsigned)r.pos0 + i;
    const int32_t phys = tables[(size_t)r.row * (size_t)g.max_pages_per_seq + cell / kF8Page];
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
    const size_t to = (((size_t)r.src0 + i) * (size_t)g.n_kv + kvh) * (size_t)hd + d;
    put4(ko + to, k);
    put4(vo + to, v);
}

F8MoveGeom f8_geom(const bkv_pool* p) { return F8MoveGeom{p->g.n_kv, p->desc.max_pages_per_seq}; }

// pages the longest of the batch's entries touches
unsigned pages_of(const AppendBatch& b) {
    int most = 0;
    for (int i = 0; i < b.n; ++i)
        if (b.n_tok[i] > 0) most = std::max(most, (b.pos0[i] + b.n_tok[i] - 1) / kF8Page - b.pos0[i] / kF8Page + 1);
    return (unsigned)most;
}

// f of the batch, in the smaller argument struct where it fits (kFewEntries)
template <typename F>
void with_batch(const AppendBatch& b, F f) {
    if (b.n > kFewEntries) return f(b);
    AppendBatchOf<kFewEntries> few{};
    few.n = b.n;
    for (int i = 0; i < b.n; ++i) {
        few.row[i] = b.row[i];
        few.pos0[i] = b.pos0[i];
        few.n_tok[i] = b.n_tok[i];
        few.src0[i] = b.src0[i];
    }
    f(few);
}

}  // namespace

hipError_t launch_append_f8p(bkv_pool* p, int32_t layer, const AppendBatch& b, const void* k, const void* v, bool src_is_f16,
                             hipStream_t stream) {
    const dim3 grid(pages_of(b) * (unsigned)p->g.n_kv, (unsigned)b.n);
    with_batch(b, [&](const auto& batch) {
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
    hipLaunchKernelGGL((append_f8p_kernel<float, F8DescBatch>), dim3((unsigned)p->g.n_kv, (unsigned)n), dim3(kBlock), 0, stream,
                       F8DescBatch{desc}, f8_geom(p), p->k_layer[(size_t)layer], p->v_layer[(size_t)layer], (const int32_t*)p->table_dev, k, v);
    return hipGetLastError();
}

hipError_t launch_append_kprep_f8p(bkv_pool* p, int32_t layer, const AppendBatch& b, const float* k, const float* v, const float* gamma,
                                   float eps, const float* table, int32_t n_rot, int32_t max_pos, const int32_t* positions,
                                   hipStream_t stream) {
    const dim3 grid(pages_of(b) * (unsigned)p->g.n_kv, (unsigned)b.n);
    launch_staged(p, BKV_STAGE_APPEND_KPREP, append_kprep_f8p_kernel, grid, dim3(kBlock), 0, stream, b, f8_geom(p),
                  F8Prep{gamma, table, positions, eps, n_rot, max_pos}, p->k_layer[(size_t)layer], p->v_layer[(size_t)layer],
                  (const int32_t*)p->table_dev, k, v);
    return hipGetLastError();
}

hipError_t launch_read_rows(bkv_pool* p, int32_t layer, const AppendBatch& b, int32_t max_cells, void* k, void* v, bool to_f16,
                            hipStream_t stream) {
    const uint8_t* const kpool = p->k_layer[(size_t)layer];
    const uint8_t* const vpool = p->v_layer[(size_t)layer];
    const int32_t* const tables = p->table_dev;
    with_batch(b, [&](const auto& batch) {
        using Batch = std::decay_t<decltype(batch)>;
        const auto to = [&](auto* ko, auto* vo) {
            using DstT = std::remove_pointer_t<decltype(ko)>;
            if (p->g.layout == BKV_LAYOUT_F8P) {
                launch_staged(p, BKV_STAGE_READ_ROWS, read_rows_f8p_kernel<DstT, Batch>, dim3(pages_of(b) * (unsigned)p->g.n_kv, (unsigned)b.n),
                              dim3(kBlock), 0, stream, batch, f8_geom(p), kpool, vpool, tables, ko, vo);
                return;
            }
            const int64_t threads = (int64_t)max_cells * p->g.n_kv * (p->g.hd / 4);
            const dim3 grid((unsigned)((threads + kBlock - 1) / kBlock), (unsigned)b.n);
            const auto launch = [&](auto kernel) {
                launch_staged(p, BKV_STAGE_READ_ROWS, kernel, grid, dim3(kBlock), 0, stream, batch, f8_geom(p), p->g.hd, kpool, vpool, tables, ko, vo);
            };
            if (p->g.layout == BKV_LAYOUT_F16) launch(read_rows_kernel<BKV_LAYOUT_F16, DstT, Batch>);
            else if (p->g.layout == BKV_LAYOUT_Q8V) launch(read_rows_kernel<BKV_LAYOUT_Q8V, DstT, Batch>);
            else launch(read_rows_kernel<BKV_LAYOUT_I8H, DstT, Batch>);
        };
        if (to_f16) to((uint16_t*)k, (uint16_t*)v);
        else to((float*)k, (float*)v);
    });
    return hipGetLastError();
}

}  // namespace bkv
