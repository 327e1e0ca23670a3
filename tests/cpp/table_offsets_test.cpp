// Changes of block tables behind the 2^31st entry of their arena: where the allocator says they are.
#include <cstdio>
#include <string>

#include "../../breccia_amd/csrc/allocator.hpp"

using namespace bkv;

#define REQUIRE(x)                                              \
    do {                                                        \
        if (!(x)) {                                             \
            std::printf("%s fails (line %d)\n", #x, __LINE__);  \
            return 1;                                           \
        }                                                       \
    } while (0)

int main() {
    constexpr int32_t kRow = 1 << 21, kSeqs = 1025;
    PageAllocator a(64, 16, kSeqs, kRow);
    std::string err;
    int32_t last = -1, n_cow;
    for (int32_t i = 0; i < kSeqs; ++i) REQUIRE(a.seq_create(&last, err) == AllocErr::Ok);
    REQUIRE(last == kSeqs - 1);
    for (int round = 0; round < 2; ++round) {
        REQUIRE(a.seq_reserve(last, 40 + 32 * round, nullptr, 0, &n_cow, err) == AllocErr::Ok);
        const auto& changes = a.pending_updates();
        REQUIRE(changes.size() == (round ? 2u : 3u));
        for (size_t i = 0; i < changes.size(); ++i) {
            const size_t col = i + (round ? 3 : 0);
            REQUIRE((size_t)changes[i].offset == (size_t)last * kRow + col && changes[i].value == a.seq_table(last)[col]);
        }
        a.pending_settled();
        REQUIRE(!a.pending());
    }
    REQUIRE(a.seq_free(last, err) == AllocErr::Ok);
    REQUIRE(a.pending_updates().size() == 5 && a.pending_updates()[4].value == -1);
    a.pending_settled();
    std::puts("ok");
    return 0;
}
