// What a compaction's list of table changes costs goes by the call and not by how many sequences a pool may have: memory that it asks for, and
// the list itself against one made entry by entry.
#include <cstdio>
#include <cstdlib>
#include <map>
#include <new>
#include <random>
#include <string>
#include <vector>

#include "../../breccia_amd/csrc/allocator.hpp"

static size_t g_asked;
void* operator new(size_t n) {
    g_asked += n;
    if (void* p = std::malloc(n)) return p;
    throw std::bad_alloc();
}
void operator delete(void* p) noexcept { std::free(p); }
void operator delete(void* p, size_t) noexcept { std::free(p); }

using namespace bkv;

#define REQUIRE(x)                                                                \
    do {                                                                          \
        if (!(x)) {                                                               \
            std::printf("trial %d: %s fails (line %d)\n", trial, #x, __LINE__);   \
            return 1;                                                             \
        }                                                                         \
    } while (0)

int main() {
    constexpr int32_t kSeqs = 1 << 18, kRow = 40;
    PageAllocator a(4000, 16, kSeqs, kRow);
    std::mt19937 rng(3);
    std::string err;
    const auto pick = [&](int lo, int hi) { return (int)(lo + rng() % (unsigned)(hi - lo + 1)); };
    std::vector<int32_t> live;
    for (int i = 0; i < 60; ++i) {
        int32_t s, n_cow, trial = -1;
        REQUIRE(a.seq_create(&s, err) == AllocErr::Ok && a.seq_reserve(s, pick(1, kRow * 16), nullptr, 0, &n_cow, err) == AllocErr::Ok);
        live.push_back(s);
    }
    for (int trial = 0; trial < 300; ++trial) {
        // changes of this and that sequence are pending
        if (pick(0, 3) == 0) a.pending_settled();
        for (int k = pick(0, 3); k-- > 0;) {
            PagePair cow[2];
            int32_t n_cow, child;
            const int32_t s = live[(size_t)pick(0, (int)live.size() - 1)];
            if (pick(0, 1)) (void)a.seq_reserve(s, std::min<int64_t>(a.seq_len(s) + pick(1, 60), kRow * 16), cow, 2, &n_cow, err);
            else if (a.seq_fork(s, pick(0, (int)a.seq_len(s)), &child, err) == AllocErr::Ok && a.seq_free(child, err) != AllocErr::Ok) return 1;
        }
        std::vector<int32_t> seqs;
        std::vector<int64_t> first, end;
        const int n = pick(1, 8);
        for (int i = 0; i < n; ++i) {
            const int32_t s = live[(size_t)(trial * 8 + i) % live.size()];
            seqs.push_back(s);
            first.push_back(pick(0, (int)a.seq_len(s)));
            end.push_back(pick((int)first.back(), (int)a.seq_len(s)));
        }
        std::vector<int32_t> fresh, words;
        REQUIRE(a.compact_begin(n, seqs.data(), first.data(), end.data(), fresh, err) == AllocErr::Ok);
        std::map<uint32_t, int32_t> want;
        for (const TableUpdate& u : a.pending_updates()) want[u.offset] = u.value;
        const size_t before = g_asked;
        a.compact_updates(n, seqs.data(), first.data(), end.data(), fresh, words);
        REQUIRE(g_asked - before <= 64 + sizeof(int32_t) * 2 * (want.size() + (size_t)n * kRow) + 64 * (size_t)n);
        a.compact_commit(n, seqs.data(), first.data(), end.data(), fresh);
        for (const TableUpdate& u : a.pending_updates()) want[u.offset] = u.value;
        std::map<uint32_t, int32_t> got;
        REQUIRE(words.size() % 2 == 0);
        for (size_t i = 0; i < words.size(); i += 2) REQUIRE(got.emplace((uint32_t)words[i], words[i + 1]).second);
        REQUIRE(got.size() <= want.size());
        // (an entry that the compaction leaves as it was need not be in both)
        for (const auto& w : want) REQUIRE(got.count(w.first) && got[w.first] == w.second);
        REQUIRE(got.size() == want.size());
        if (trial % 50 == 0) REQUIRE(a.check(err));
    }
    std::puts("ok");
    return 0;
}
