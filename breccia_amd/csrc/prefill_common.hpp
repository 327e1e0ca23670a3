// What the chunk attention kernels share: their arguments, and how they take them in.
#pragma once

#include <type_traits>

#include "bkv_internal.hpp"

namespace bkv {

struct PrefillKernelParams {
    PrefillBatch b;
    const uint8_t* kpool;
    const uint8_t* vpool;
    const int32_t* tables;
    const float* q;     // [sum n_tok][n_q][256]
    const float* gate;  // optional
    float* out;         // [sum n_tok][n_q][256]
    int64_t gate_tok_stride, gate_head_stride;
    int32_t max_pages_per_seq, n_kv, n_q, group;
    float scale_log2e;
    uint32_t group_inverse, n_kv_inverse;  // floor((2^32 - 1) / n), for divided_by
    int32_t gate_in_fours;                 // four gate values can be read at once
    int32_t by_xcd;  // work-groups are dealt to the chip's 8 dies so that each die sees few (entry, kv head) units
};

// A cut call: a work-group walks one range of its block's pages and leaves a partial result,
// prefill_merge_kernel puts the ranges of a row together.
struct PrefillSplitParams : PrefillKernelParams {
    PrefillSplit s;
    float* part_o;   // [slot][row of the block][256], relative to the range's own softmax reference
    float* part_ml;  // [slot][row of the block][reference, denominator]
};

// x / n and the rest, for x >= 0: the inverse is below 2^32 / n by 1 at most, so the product's quotient is right or one
// too small.  (A division by a number that only the launch knows is some 40 instructions.)
__device__ __forceinline__ int divided_by(int x, int n, uint32_t inverse, int& rest) {
    int q = (int)__umulhi((uint32_t)x, inverse);
    rest = x - q * n;
    if (rest >= n) ++q, rest -= n;
    return q;
}
__device__ __forceinline__ int divided_by(int x, int n, uint32_t inverse) {
    int rest;
    return divided_by(x, n, inverse, rest);
}

// The arguments' cache lines, asked for at once as a kernel begins: left to where each field is used, they are a chain of
// trips to memory (41 tokens behind 517 cells through 12 layers: 234 us, 218 with this and `held`).
template <typename S>
__device__ __forceinline__ void now(const PrefillBatch& b, int n_kv, const S& at_end) {
    asm volatile("" : : "s"(b.row[0]), "s"(b.pos0[0]), "s"(b.n_tok[0]), "s"(b.src0[0]), "s"(b.wg_base[0]), "s"(n_kv), "s"(at_end));
}
__device__ __forceinline__ void now(const PrefillSplit& s) {
    asm volatile("" : : "s"(s.pps), "s"(s.splits[0]), "s"(s.wg_base[0]), "s"(s.unit_base[0]), "s"(s.slot_base[0]));
}
// keeps an argument in registers from here on instead of asking for it again
template <typename T>
__device__ __forceinline__ T held(T x) {
    asm volatile("" : "+s"(x));
    return x;
}
// A pointer that came through `held` is not known to be to global memory any more: used as it is, each access is a flat one,
// which LDS counts too and which are waited for together.
template <typename T>
__device__ __forceinline__ __attribute__((address_space(1))) T* in_global(T* p) {
    return (__attribute__((address_space(1))) T*)p;
}

// what lane i has in x
__device__ __forceinline__ uint64_t lane_value(uint64_t x, int i) {
    const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)x, i);
    const unsigned hi = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)(x >> 32), i);
    return (uint64_t)hi << 32 | lo;
}

// two f32 numbers as f16, rounded to nearest
typedef _Float16 f16_pair __attribute__((ext_vector_type(2)));
__device__ __forceinline__ f16_pair to_f16(float a, float b) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    return __builtin_convertvector(f2{a, b}, f16_pair);
}
// x - (the f16 number hi): one v_fma_mix_f32 takes the f16 operand as it is (minus_one: -1.0f that the compiler
// cannot see through, a plain subtraction would be preceded by a conversion)
__device__ __forceinline__ float remainder_of(float x, _Float16 hi, float minus_one) {
    return __builtin_fmaf((float)hi, minus_one, x);
}
// keeps a value where it is computed: between matrix products, not behind the branch that its use stands behind
template <typename T>
__device__ __forceinline__ void stay(T& x) {
    asm volatile("" : "+v"(x));
}

typedef const __attribute__((address_space(1))) uint8_t* page_ptr;  // said to be global memory: its address goes through integers
// 16 bytes a lane straight into LDS: lane l's go to byte lds + 16 l.  Nothing but the vector-memory count says when they
// have landed; each wave waits for its own ahead of the barrier that publishes them.
__device__ __forceinline__ void load_to_lds(unsigned lds, page_ptr base, unsigned lane_off) {
    // (the base came from a VALU instruction, which a vector-memory one must not follow closely: the copy is a scalar
    // instruction, and the wait state that m0 wants)
    uint64_t at;
    // (m0 is reserved: the compiler keeps nothing there of its own accord, and warns that it would not; what it must not do is
    // let a value that it puts there for an instruction of its own live across this)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
    asm volatile("s_mov_b32 m0, %1\n\ts_mov_b64 %0, %3\n\tglobal_load_lds_dwordx4 %2, %0"
                 : "=&s"(at)
                 : "s"(lds), "v"(lane_off), "s"(base)
                 : "m0", "memory");
#pragma clang diagnostic pop
}
__device__ __forceinline__ void wait_for_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// The ranges of a cut call's rows put together (prefill_attn.hip).
hipError_t launch_prefill_merge(bkv_pool* p, const PrefillSplitParams& kp, int32_t rows_per_wg, hipStream_t stream);
// The chunk attention kernel of the e4m3 layout (f8p_chunk.hip), over `grid` work-groups of rows_per_wg rows; split: cut walks, which
// leave partial results.
hipError_t launch_chunk_attn_f8p(bkv_pool* p, const PrefillSplitParams& kp, int32_t rows_per_wg, bool split, uint32_t grid, hipStream_t stream);

}  // namespace bkv
