// How often plan_shared (csrc/shared_plan.hpp) works out how a walk is cut: it is asked on every layer's call, and a batch may have walks of
// thousands of pages.
#include <cstdio>
#include <cstdlib>
#include <random>

#include "../../breccia_amd/csrc/prefill_plan.hpp"

static long g_cuts;
namespace bkv {
inline int counted_split_ranges(int pages, int pps, int max_splits, int& each) { return ++g_cuts, split_ranges(pages, pps, max_splits, each); }
}  // namespace bkv
#define split_ranges counted_split_ranges
#include "../../breccia_amd/csrc/shared_plan.hpp"

using namespace bkv;

int main(int argc, char** argv) {
    (void)argc;
    std::mt19937 rng((unsigned)std::atoi(argv[1]));
    const int trials = std::atoi(argv[2]);
    const auto pick = [&](int lo, int hi) { return (int)(lo + rng() % (unsigned)(hi - lo + 1)); };
    const auto log_pick = [&](int hi) { return pick(0, pick(0, 3) ? hi : hi / 64 + 1); };
    int planned = 0;
    double worst = 0.0;
    for (int trial = 0; trial < trials; ++trial) {
        const SharedPlanLimits lim{pick(0, 3), pick(0, 1) ? 2 : pick(1, 16), pick(1, 16), 256, pick(0, 9) ? 32768 : pick(64, 40000), 8192};
        int32_t entries[kMaxBatch], pages[kMaxBatch], row[kMaxBatch], pos[kMaxBatch];
        int n = 0, groups = 0;
        const int want = pick(1, kMaxBatch);
        while (n < want) {
            const int e = pick(1, pick(0, 1) ? want - n : 1);
            entries[groups] = e;
            pages[groups] = log_pick(4096);
            for (int i = 0; i < e; ++i) row[n] = pick(0, 99), pos[n++] = pages[groups] * 16 + log_pick(pick(0, 9) ? 4000 : 60000);
            ++groups;
        }
        SharedPlan plan;
        g_cuts = 0;
        if (!plan_shared(lim, groups, entries, pages, row, pos, plan)) continue;
        ++planned;
        worst = std::max(worst, (double)g_cuts / plan.n);
    }
    // walks of up to 7846 pages, 3923 pairs: twelve steps out, eleven back, the last one again
    std::printf("%d planned, at most %.1f cuts a walk\n", planned, worst);
    return planned > trials / 10 && worst <= 26 ? 0 : 1;
}
