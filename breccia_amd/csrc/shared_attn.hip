// Decode attention of a batch whose entries share pages (a prompt's samples, questions to one document, branches of a search), for
// gfx950.  For query row r = (entry, head), whose group shares cells 0 .. S - 1 and whose entry has cells S .. pos of its own,
//   (m, l, O)_f = max, sum and value sum of exp2(x - m) over the shared cells, x = scale log2(e) q . k
//   (m, l, O)_o = the same over the entry's own
//   out = (O_f 2^(m_f - M) + O_o 2^(m_o - M)) / (l_f 2^(m_f - M) + l_o 2^(m_o - M)),  M = max(m_f, m_o)
// The shared cells are a matrix product: every entry's rows meet the same K and V, so the chunk kernels walk them once for all (their
// form without a causal mask, cut into ranges, shared_plan.hpp).  The own cells are streams: walks of a few rows in the same launch, or
// where there are many of them the decode kernels.  All leave partial results, whole rows of f32; the kernel below puts a row's together.
// 32 entries of 8192 shared cells, 2 kv heads of 8, f16: 19 us of walks and 7 of the merge, 26 where each entry for itself reads 268 MB
// in 55; 64 of 65519 and up to 2000 of their own, 12 heads:
// 208 + 28 + 11, 690 each for itself.
#include <type_traits>

#include "decode_attn_common.hpp"
#include "gate.hpp"
#include "lane_groups.hpp"

namespace bkv {

namespace {

// Rows of partial results: where the first range's of the entry's head 0 lies, rows between kv heads and between ranges.
struct SharedMergeParams {
    const float *front_o, *front_ml;  // of the shared pages
    const float *own_o, *own_ml;      // of the entry's own
    const float* gate;
    float* out;
    int64_t gate_seq_stride, gate_head_stride;
    int32_t n_q, group, rows_shift;  // blocks of 1 << rows_shift rows
    int32_t n_kv;
    uint32_t inv_group16;
    int32_t own_stride;              // rows between the ranges of an entry's own pages
};
template <int N>
struct SharedMergeArgs : SharedMergeParams {
    int32_t own_splits[N], own_row[N], own_kv[N];     // own_kv: rows between kv heads
    int32_t front_splits[N];                          // ranges of the group's walk; 0: it has none
    int32_t front_slot[N], front_blocks[N], first[N]; // its first slot, its blocks of rows, its first entry
};

constexpr int kMergeWaves = 4;
constexpr int kMergeCols = 64;                 // columns of a work-group
constexpr int kMergeGroups = kMergeWaves * 4;  // 16 lanes, 4 columns each, take partial results i, i + kMergeGroups, ...

// exp2(x - ref), and 0 where nothing has been attended yet (both -inf)
__device__ __forceinline__ float weight_of(float x, float ref) { return __builtin_amdgcn_exp2f(x - (ref == -INFINITY ? 0.0f : ref)); }

// A work-group per (entry, q head, quarter of the columns), as in decode_attn_merge_kernel (decode_attn.hip).  A row has up to
// kMaxSharedRanges partial results of shared pages and, of its own, up to as many from walks or what the decode kernels cut a long part
// into; most have a few.  A quarter of a wave's lanes takes every 16th.  512 rows of 35 partial results 7 us, 18 MB that lie in the
// caches: two trips to memory (maxima and sums, rows), a launch and two barriers.
template <int N>
__global__ __launch_bounds__(64 * kMergeWaves) void shared_merge_kernel(const SharedMergeArgs<N> P) {
    __shared__ __attribute__((aligned(16))) float red[kMergeWaves][kMergeCols];
    __shared__ __attribute__((aligned(16))) float red_m[kMergeWaves], red_l[kMergeWaves];
    const int e = blockIdx.y;
    const int h = blockIdx.x / (kHd / kMergeCols);
    const int col = blockIdx.x % (kHd / kMergeCols) * kMergeCols;
    const int own_splits = P.own_splits[e], own_first = P.own_row[e], own_kv = P.own_kv[e], front_splits = P.front_splits[e];
    const int front_slot = P.front_slot[e], front_blocks = P.front_blocks[e], first = P.first[e];
    asm volatile("" ::"s"(own_splits), "s"(own_first), "s"(own_kv), "s"(front_splits), "s"(front_slot), "s"(front_blocks), "s"(first),
                 "s"(P.front_o), "s"(P.front_ml), "s"(P.own_o), "s"(P.own_ml), "s"(P.gate), "s"(P.out), "s"(P.gate_seq_stride),
                 "s"(P.gate_head_stride), "s"(P.n_kv), "s"(P.n_q), "s"(P.group), "s"(P.rows_shift), "s"(P.inv_group16), "s"(P.own_stride));
    const int kvh = small_div(h, P.inv_group16);
    const int hl = h - kvh * P.group;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    float gt = 0.0f;
    if (P.gate && wave == 0) gt = P.gate[(size_t)e * P.gate_seq_stride + (size_t)h * P.gate_head_stride + col + lane];
    const uint32_t own_row = (uint32_t)(own_first + kvh * own_kv + hl), own_stride = (uint32_t)P.own_stride;
    // the group's rows, block by block; a group of no more than 16 has slots of 16
    const int row = (e - first) * P.group + hl, rb = row >> P.rows_shift;
    const uint32_t front_stride = front_blocks < 0 ? 16u : 1u << P.rows_shift;
    const int blocks = front_blocks < 0 ? 1 : front_blocks;
    const uint32_t front_row = 16u * (uint32_t)front_slot + (uint32_t)((blocks - 1 - rb) * P.n_kv + kvh) * (uint32_t)front_splits * front_stride +
                               (uint32_t)(row & ((1 << P.rows_shift) - 1));
    const int total = front_splits + own_splits;
    const int at = threadIdx.x >> 4, lane_at = col + 4 * (lane & 15);
    f4 o = f4{0.0f, 0.0f, 0.0f, 0.0f};
    float m_run = -INFINITY, l_run = 0.0f;
    // everything of a round is requested before the first use, without branches: past the end the last one again, which counts as
    // zeros
    const auto round = [&](auto n, int s0) {
        constexpr int kIn = decltype(n)::value;
        float m[kIn], l[kIn];
        f4 v[kIn];
#pragma unroll
        for (int u = 0; u < kIn; ++u) {
            const int s = min(s0 + u * kMergeGroups, total - 1);
            const bool front = s < front_splits;
            // (a workspace has 2^15 rows: 32 bits hold any offset in floats)
            const uint32_t r = front ? front_row + (uint32_t)s * front_stride : own_row + (uint32_t)(s - front_splits) * own_stride;
            const float2 ml = *reinterpret_cast<const float2*>((front ? P.front_ml : P.own_ml) + r * 2u);
            m[u] = ml.x, l[u] = ml.y;
            v[u] = *reinterpret_cast<const f4*>((front ? P.front_o : P.own_o) + (r * (uint32_t)kHd + (uint32_t)lane_at));
        }
        __builtin_amdgcn_sched_barrier(0);
        float mx = m_run;
#pragma unroll
        for (int u = 0; u < kIn; ++u) {
            const bool mine = s0 + u * kMergeGroups < total;
            m[u] = mine ? m[u] : -INFINITY;
            l[u] = mine ? l[u] : 0.0f;
            v[u] = mine ? v[u] : f4{0.0f, 0.0f, 0.0f, 0.0f};
            mx = fmaxf(mx, m[u]);
        }
        const float keep = weight_of(m_run, mx);
        o *= keep;
        l_run *= keep;
        m_run = mx;
#pragma unroll
        for (int u = 0; u < kIn; ++u) {
            const float f = weight_of(m[u], mx);
            o += v[u] * f;
            l_run = fmaf(f, l[u], l_run);
        }
    };
    if (total <= kMergeGroups) round(std::integral_constant<int, 1>(), at);
    else if (total <= 2 * kMergeGroups) round(std::integral_constant<int, 2>(), at);
    else if (total <= 3 * kMergeGroups) round(std::integral_constant<int, 3>(), at);
    else if (total <= 4 * kMergeGroups) round(std::integral_constant<int, 4>(), at);
    else
        for (int s0 = 0; s0 < total; s0 += 5 * kMergeGroups) round(std::integral_constant<int, 5>(), s0 + at);
    // the four 16-lane groups of a wave, then the waves
    const float m_wave = max_over_lane_groups(m_run);
    const float f = weight_of(m_run, m_wave);
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = sum_over_lane_groups(o[k] * f);
    const float l_wave = sum_over_lane_groups(l_run * f);
    if (lane < 16) *reinterpret_cast<f4*>(&red[wave][4 * lane]) = o;
    if (lane == 0) {
        red_m[wave] = m_wave;
        red_l[wave] = l_wave;
    }
    __syncthreads();
    if (wave != 0) return;
    const f4 m = *reinterpret_cast<const f4*>(red_m), l = *reinterpret_cast<const f4*>(red_l);
    const float mx = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
    float r = 0.0f, lt = 0.0f;
#pragma unroll
    for (int w = 0; w < kMergeWaves; ++w) {
        const float fw = weight_of(m[w], mx);
        r = fmaf(red[w][lane], fw, r);
        lt = fmaf(l[w], fw, lt);
    }
    r = lt > 0.0f ? r / lt : lt == lt ? 0.0f : lt;  // (a sum that is no number stays one)
    if (P.gate) r *= sigmoid(gt);
    P.out[((size_t)e * P.n_q + h) * kHd + col + lane] = r;
}

template <int N>
void launch_merge(bkv_pool* p, const SharedMergeParams& mp, const SharedPlan& plan, int32_t n, const AttnBatch* own, hipStream_t stream) {
    SharedMergeArgs<N> args{};
    static_cast<SharedMergeParams&>(args) = mp;
    for (int i = 0; i < n; ++i) {
        if (own) {
            args.own_splits[i] = own->splits[i];
            args.own_row[i] = own->wg_base[i] * mp.group;
            args.own_kv[i] = mp.group;
        } else {
            const int w = plan.own_of[i];
            args.own_splits[i] = plan.ranges[w];
            args.own_row[i] = 16 * plan.slot_base[w];
            args.own_kv[i] = 16 * plan.ranges[w];
        }
        const int g = plan.group_of[i];
        if (g < 0) continue;
        const int rows = plan.entries[g] * mp.group;
        args.front_splits[i] = plan.ranges[g];
        args.front_slot[i] = plan.slot_base[g];
        args.front_blocks[i] = rows <= 16 ? -1 : (rows + plan.rows_per_wg - 1) / plan.rows_per_wg;
        args.first[i] = plan.first[g];
    }
    launch_staged(p, BKV_STAGE_ATTN_MERGE, shared_merge_kernel<N>, dim3((unsigned)mp.n_q * (kHd / kMergeCols), (unsigned)n),
                  dim3(64 * kMergeWaves), 0, stream, args);
}

}  // namespace

hipError_t launch_shared_attn(bkv_pool* p, int32_t layer, const SharedPlan& plan, int32_t n, const AttnBatch* own, const AttnArgs& a,
                              const ChunkWorkspace& ws, hipStream_t stream) {
    hipError_t err = launch_shared_walk(p, layer, plan, a, ws, stream);
    if (err != hipSuccess) return err;
    if (own) {
        err = launch_decode_ranges(p, layer, *own, a, stream);
        if (err != hipSuccess) return err;
    }
    SharedMergeParams mp{};
    mp.front_o = ws.o, mp.front_ml = ws.ml;
    mp.own_o = own ? p->part_o : ws.o, mp.own_ml = own ? p->part_ml : ws.ml;
    mp.gate = a.gate;
    mp.out = a.out;
    mp.gate_seq_stride = a.gate_seq_stride, mp.gate_head_stride = a.gate_head_stride;
    mp.n_kv = p->g.n_kv, mp.n_q = a.n_q_head, mp.group = a.n_q_head / p->g.n_kv;
    mp.rows_shift = __builtin_ctz((unsigned)plan.rows_per_wg);
    mp.inv_group16 = small_divisor_inverse(mp.group);
    mp.own_stride = own ? mp.n_kv * mp.group : 16;
    if (n <= kFewEntries) launch_merge<kFewEntries>(p, mp, plan, n, own, stream);
    else launch_merge<kMaxBatch>(p, mp, plan, n, own, stream);
    return hipGetLastError();
}

}  // namespace bkv
