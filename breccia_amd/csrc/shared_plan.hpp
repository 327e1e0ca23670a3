// Attention of a decode batch whose entries share pages: what is walked once for all entries of a group, and how the walks are cut.
// No HIP types: host-only tests run the same functions.
//
// A walk takes query rows over pages, each row over all of them, and leaves partial results (prefill_attn.hip, f8p_chunk_kernel.hpp):
// the rows of a group -- (entry, head) pairs of one kv head -- over the pages that the group shares, in blocks of 64 or 128 as a
// chunk's rows, and the rows of an entry over its own pages, 16 of a block.  Where the own pages are much of the work they are left to the
// decode kernels, whose stream is faster.  One kernel puts a row's partial results together (shared_attn.hip).
#pragma once

#include <algorithm>
#include <cstdint>

#include "prefill_plan.hpp"

namespace bkv {

constexpr int kMaxWalks = kMaxBatch + kMaxBatch / 2;  // a group that shares has two entries at least
constexpr int kFewWalks = 24;
constexpr int kMaxSharedRanges = 256;  // of a block
// Pairs of pages that a range of a walk of `pairs` has at least: 128 ranges, and more of them only of six pairs or more.  One block's walk
// at 128 / up to 256 ranges (us of a call): 54000 cells, e4m3 27.4 / 23.2; 34000 23.0 / 22.9; 21000, f16 20.1 / 22.9 (ranges of three).
constexpr int64_t least_pairs(int64_t pairs) {
    const int64_t even = (pairs + 127) / 128, most = (pairs + kMaxSharedRanges - 1) / kMaxSharedRanges;
    return std::max(std::min<int64_t>(even, 6), most);
}

struct SharedPlan {
    int32_t rows_per_wg;
    // the walks, those of groups first: where the table begins in the arena, last cell, entries, first entry, ranges of a block,
    // first work-group, first slot of 16 rows of partial results
    int32_t n, groups, wgs;
    int32_t table[kMaxWalks], pos[kMaxWalks], entries[kMaxWalks], first[kMaxWalks], ranges[kMaxWalks], wg_base[kMaxWalks], slot_base[kMaxWalks];
    // of the batch's entries: the walk of its group or -1, pages that it does not read for itself, and the walk of its own pages
    int32_t group_of[kMaxBatch], front[kMaxBatch], own_of[kMaxBatch];
    bool own_walks;  // the entries' own pages are among the walks
};

struct SharedPlanLimits {
    int32_t layout;  // bkv_layout: 0 f16, 1 q8_0 V, 2 int8, 3 e4m3
    int32_t n_kv;
    int32_t group;  // q heads of a kv head
    int32_t n_cu;
    int64_t rows;   // query rows the workspace holds partial results for
    int64_t table_row;  // entries of a table
};

inline int32_t shared_blocks(const SharedPlanLimits& lim, int32_t entries, int32_t rows) { return (entries * lim.group + rows - 1) / rows; }

// What is decided here, and what it was measured against (us of a call, 2 kv heads of 8 heads; "each": bkv_decode_attn, every entry reading
// all of its pages, most of them out of the caches):
// - Whether to share.  A call of walks begins and ends 3.5 us later than one of decode kernels (pages of 8 bits: 5.5) and has ranges of three
//   pairs at least; a pair of pages takes a block of 64 rows 0.8 us, a quantised pool's block of 128 2.2, an entry's own rows 1.1 and 2.0.
//   Entries that need not read a page save it at 9 TB/s (10.5); what the group then reads once, and what entries have of their own, would
//   have been read anyway.  Of 1500 batches drawn (f16) that shared with 2.5, 1.0 and 10.5, 89 were slower than each for itself by 139 us in all;
//   with these a third of that is left, and 20 us of gains are lost; e4m3, 500 batches: 155 us, 52 and 64.
//       f16, each / shared: 4 of 2048 cells 10.2 / 12.5, 2 of 8192 13.4 / 15.9, 16 of 1024 12.8 / 13.6 (these stay apart); 8 of 4096
//       17.0 / 14.9, 4 of 32768 50 / 23, 64 of 4096 52 / 26, 32 of 8192 55 / 26, 64 of 16384 160 / 49
//       e4m3: 2 of 32768 19.3 / 21.4, 16 of 4096 and 4000 of their own 24 / 33 (apart); 8 of 4096 14.6 / 14.9; 4 of 32768 22.6 / 21.9,
//       64 of 4096 32.9 / 26.3, 64 of 16384 86 / 50
//       int8: 8 of 4096 15.9 / 19, 64 of 512 18.9 / 28.6, 16 of 8192 and 1000 of their own 32 / 41 (apart); 8 of 32768 60 / 35, 64 of 4096
//       52 / 38, 64 of 16384 161 / 72
//       q8_0 V goes by int8's constants: 2 of 8192 15.3 / 16.3, 16 of 1024 15.7 / 23.4, 64 of 512 21.8 / 28.0, 32 of 2048 24.7 / 27.7, 16 of
//       4096 25.0 / 27.0 (apart); 4 of 32768 44.5 / 27.2, 64 of 4096 58.5 / 40.9, 64 of 16384 180 / 66; its K need not be decoded, so a pair
//       costs less and there are calls apart that sharing would help: 8 of 8192 25.1 / 23.4, 4 of 16384 24.7 / 21.4, 2 of 32768 28.0 / 25.7
//   What it comes to: of 4902 drawn batches that share, 104 are more than 1 us slower than each for itself, 322 us of the 448 ms that they take
//   apart (175 shared).  f16 49 of 3337, at worst 66 / 83; int8 5 of 606, 31 / 34; e4m3 50 of 959: dozens of own parts of a
//   hundred cells behind 1400 shared ones, whose walks it takes to cost what f16's do, 31 / 45.  q8_0 V 33 of 2475, 86 / 99.
//   Where the own pages are read apart the call is two launches behind, 13 us, and on e4m3 pools, whose pages are small, 20: 32 of 8192
//   and 4000 of their own, f16 89 / 60, int8 71 / 67, e4m3 47 / 52 (with 13).
// - Blocks of 64 rows, and of 128 (quantised pools: always) where the walks are long: such a block takes 1.57 us a pair, two of 64 1.9.
//   64 / 128: f16, 64 of 16384 49 / 56, of 32768 80 / 81, of 49152 113 / 107; four groups of 16 of 32768 100 / 91; e4m3 51 / 54, 86 / 77,
//   122 / 102, 90 / 80.
// - Own pages by walks, in the same launch, or by the decode kernels: 5 us a call for the start of another kernel; but a walk of 16 rows
//   uses a quarter of a work-group.  By walks / apart: f16, 32 of 8192 and 4000 of their own 61 / 70, 64 of 4096 and 100 of their own
//   28 / 35, 8 of 8192 with 8 others of 30000 beside them 114 / 98; e4m3 56 / 52, 30 / 35, 110 / 63; int8 90 / 65, 38 / 44, 134 / 74; q8_0 V
//   87 / 73, 41 / 42, 16 of 16384 and 4000 of their own 62 / 58.  A wave
//   of 512 registers leaves no room for another work-group: blocks of 128 rows leave the own pages apart, on quantised pools unless all is
//   short.
// - As many ranges as compute units: a second work-group a unit brings little (the products bound it: 64 rows a pair 0.94 us alone, 0.88
//   beside another) and its partial results cost; 32 of 8192 with 128 / 256 / 512 ranges 27 / 28 / 37 us, 64 of 16384 74 / 50 / 59.  Where
//   walks are short, or their waves leave no room beside them, a unit for each work-group of own pages, up to a quarter: 16 of 16384 with
//   192 / 256 24.1 / 25.7, 64 of 4096 26.9 / 28.1, four groups of 16 of 4096 26.6 / 27.5.
// - Own walks in ranges of half the length, since a wave alone takes longer for a pair: 16 of 65519 and up to 2000 of their own at 12
//   heads 81 -> 69, 64 of 4096 29 -> 26; e4m3 30 -> 26.
//
// entries[g], pages[g]: of group g, whose entries stand behind those of the groups before.  row, pos: block-table row and position of
// each entry.  False where no group's walk pays, or the workspace does not hold the rows' partial results.
inline bool plan_shared(const SharedPlanLimits& lim, int32_t n_groups, const int32_t* entries, const int32_t* pages, const int32_t* row,
                        const int32_t* pos, SharedPlan& plan) {
    const bool quantised = lim.layout == 1 || lim.layout == 2, f16 = lim.layout == 0;
    const int32_t n_cu = lim.n_cu > 0 ? lim.n_cu : 256;
    // bytes of a page that one kv head reads
    const double page_bytes = kPrefillPage * (f16 ? 1024.0 : lim.layout == 1 ? 800.0 : lim.layout == 2 ? 544.0 : 512.0);
    const int32_t least_rows = (quantised ? 8 : 4) * kPrefillRowsPerWave;
    const double pair_us = quantised ? 2.2 : 0.8;  // of a block of least_rows
    const double each_rate = f16 ? 9e6 : 10.5e6, once_rate = f16 ? 10e6 : 6e6;  // bytes a us
    // Which groups: those whose walk, as a share of the chip's time, costs less than what their entries no longer read (out of the
    // caches, most of it) ...
    double gain = 0.0, once = 0.0;
    int64_t work = 0, range = 3;
    const auto units_of = [&](int32_t g, int32_t rows) { return (int64_t)shared_blocks(lim, entries[g], rows) * lim.n_kv; };
    const auto saved_us = [&](int32_t g) { return (entries[g] - 1.0) * pages[g] * lim.n_kv * page_bytes / each_rate; };
    const auto read_us = [&](int32_t g) { return (double)pages[g] * lim.n_kv * page_bytes / once_rate; };
    const auto pays = [&](int32_t g) {
        if (entries[g] < 2 || pages[g] < 1) return false;
        return saved_us(g) > pair_us * (double)(units_of(g, least_rows) * ((pages[g] + 1) / 2)) / n_cu - read_us(g);
    };
    int32_t at = 0;
    plan.n = 0;
    for (int32_t g = 0; g < n_groups; ++g) {
        const bool walks = pays(g);
        for (int32_t i = at; i < at + entries[g]; ++i) {
            plan.group_of[i] = walks ? plan.n : -1;
            plan.front[i] = walks ? pages[g] : 0;
        }
        if (walks) {
            plan.table[plan.n] = (int32_t)(row[at] * lim.table_row);
            plan.pos[plan.n] = pages[g] * kPrefillPage - 1;
            plan.entries[plan.n] = entries[g];
            plan.first[plan.n++] = at;
            work += units_of(g, least_rows) * ((pages[g] + 1) / 2);
            range = std::max(range, least_pairs((pages[g] + 1) / 2));
            gain += saved_us(g);
            once += read_us(g);
        }
        at += entries[g];
    }
    plan.groups = plan.n;
    // ... and the call as a whole.
    if (plan.n == 0) return false;
    const auto pairs_of = [&](int32_t i) { return (plan.pos[i] / kPrefillPage + 2) / 2; };
    int64_t own_work = 0;
    for (int32_t i = 0; i < at; ++i) own_work += lim.n_kv * ((pos[i] / kPrefillPage - plan.front[i] + 2) / 2);
    const bool two = !quantised && work > (f16 ? 56 : 44) * (int64_t)n_cu;
    plan.rows_per_wg = quantised || two ? 8 * kPrefillRowsPerWave : 4 * kPrefillRowsPerWave;
    plan.own_walks = quantised ? own_work <= 4 * (int64_t)n_cu && work <= 10 * (int64_t)n_cu : !two && own_work <= (f16 ? 40 : 24) * (int64_t)n_cu;
    const double own_us = std::max((quantised ? 2.0 : 1.1) * (double)own_work / n_cu - (double)own_work * 2.0 * page_bytes / each_rate, 0.0);
    const double cost = (!plan.own_walks ? (lim.layout == 3 ? 20.0 : 13.0) : (f16 ? 3.5 : 5.5) + own_us) +
                        std::max(pair_us * std::max((double)range, (double)work / n_cu) - once, 0.0);
    if (gain <= cost) return false;
    if (plan.own_walks)
        for (int32_t i = 0; i < at; ++i) {
            plan.own_of[i] = plan.n;
            plan.table[plan.n] = (int32_t)(row[i] * lim.table_row) + plan.front[i];
            plan.pos[plan.n] = pos[i] - plan.front[i] * kPrefillPage;
            plan.entries[plan.n] = 1;
            plan.first[plan.n++] = i;
        }
    // Ranges of walks from .. to - 1, `least` page pairs or more each, so that they are no more than fit work-groups (one a unit if that
    // is more) and their partial results find room.  With many blocks there may be more of them once ranges have `most` pairs: one long
    // walk among short ones would have a range or two otherwise (62 entries, one with 33603 cells of its own: 480 us / 47).
    // -> pairs of a range, or -1.  The longer the ranges, the fewer: the shortest that will do are found in steps twice as long each and
    // then between the last two, a dozen looks at all walks at most (pair by pair up to thousands: of 200000 random batches the slowest took
    // 1200 us of the host, now 17).
    int64_t wgs = 0, slots = 0;
    const auto cut = [&](int32_t from, int32_t to, int64_t fit, int64_t least, int64_t most, int64_t room) {
        int64_t total = 0, units = 0, longest = 1;
        for (int32_t i = from; i < to; ++i) {
            const int64_t nb = (int64_t)shared_blocks(lim, plan.entries[i], plan.rows_per_wg) * lim.n_kv;
            total += nb * pairs_of(i);
            units += nb;
            longest = std::max<int64_t>(longest, pairs_of(i));
        }
        const int64_t wgs0 = wgs, slots0 = slots;
        bool holds = false;
        const auto does = [&](int64_t each) {
            wgs = wgs0, slots = slots0;
            for (int32_t i = from; i < to; ++i) {
                int32_t even;
                plan.ranges[i] = split_ranges(plan.pos[i] / kPrefillPage + 1, 2, (int32_t)((pairs_of(i) + each - 1) / each), even);
                plan.wg_base[i] = (int32_t)wgs;
                plan.slot_base[i] = (int32_t)slots;
                const int64_t mine = (int64_t)shared_blocks(lim, plan.entries[i], plan.rows_per_wg) * lim.n_kv * plan.ranges[i];
                wgs += mine;
                slots += mine * (plan.entries[i] * lim.group <= 16 ? 1 : plan.rows_per_wg / 16);
            }
            holds = slots <= room;
            return holds && wgs - wgs0 <= std::max(fit, units) + (each >= most && 4 * units > fit ? std::min(fit, units) : 0);
        };
        int64_t each = std::max<int64_t>({least, (total + fit - 1) / fit, least_pairs(longest)}), short_of = each - 1;
        for (int64_t step = 1; !does(each); step *= 2) {
            if (each >= longest) {  // one range each
                if (!holds) return (int64_t)-1;
                break;
            }
            short_of = each;
            each = std::min(each + step, longest);
        }
        int64_t looked_at = each;
        while (each - short_of > 1) {
            looked_at = short_of + (each - short_of) / 2;
            (does(looked_at) ? each : short_of) = looked_at;
        }
        if (looked_at != each) (void)does(each);
        return each;
    };
    const int64_t own_slots = (int64_t)lim.n_kv * (plan.n - plan.groups);
    const int64_t beside = plan.own_walks && (quantised || work <= 10 * (int64_t)n_cu) ? std::min<int64_t>(own_slots, n_cu / 4) : 0;
    const int64_t each = cut(0, plan.groups, n_cu - beside, 3, 24, lim.rows / 16 - own_slots);
    if (each < 0 || (plan.own_walks && cut(plan.groups, plan.n, n_cu, std::max<int64_t>(3, each / 2), each + 12, lim.rows / 16) < 0)) return false;
    plan.wgs = (int32_t)wgs;
    return true;
}

}  // namespace bkv
