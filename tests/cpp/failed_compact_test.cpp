// A compaction that fails has enqueued no kernel of its own that is still to run, and leaves sequence, tables and free pages as they were;
// one whose kernels are out has happened.  Run on the host: the HIP calls that the library makes are the ones below (an
// executable's come before a library's), which launch nothing and fail, or are not done yet, when they are told to.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>

#include "breccia_kv.h"

// The launches of a compaction, and of the tables' changes (in work-groups of 128 threads, and of others); those of the former that nothing
// has waited for.
static int g_compactions, g_others, g_running;
// Which record of an event fails (0: none), from which question on the answer is "not yet", which launch fails; a launch's error, or one that
// somebody else left.
static int g_records, g_fail_record, g_queries, g_late_query, g_fail_launch;
static hipError_t g_left = hipSuccess;

static hipError_t launched(dim3 block) {
    if (block.x != 128) return ++g_others, hipSuccess;
    if (++g_compactions == g_fail_launch) return g_left = hipErrorInvalidConfiguration;
    return ++g_running, hipSuccess;
}
static dim3 g_grid, g_block;
extern "C" {
hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t, hipStream_t) { return g_grid = g, g_block = b, hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3* g, dim3* b, size_t* s, hipStream_t* st) {
    *g = g_grid, *b = g_block, *s = 0, *st = nullptr;
    return hipSuccess;
}
hipError_t hipDeviceSynchronize() { return g_running = 0, hipSuccess; }
static char g_event;
hipError_t hipEventCreate(hipEvent_t* e) { return *e = (hipEvent_t)&g_event, hipSuccess; }
hipError_t hipEventCreateWithFlags(hipEvent_t* e, unsigned) { return *e = (hipEvent_t)&g_event, hipSuccess; }
hipError_t hipEventDestroy(hipEvent_t) { return hipSuccess; }
hipError_t hipEventElapsedTime(float* ms, hipEvent_t, hipEvent_t) { return *ms = 0.0f, hipSuccess; }
hipError_t hipEventQuery(hipEvent_t) { return ++g_queries >= g_late_query && g_late_query ? hipErrorNotReady : hipSuccess; }
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return ++g_records == g_fail_record ? g_left = hipErrorInvalidHandle : hipSuccess; }
hipError_t hipExtLaunchKernel(const void*, dim3, dim3 b, void**, size_t, hipStream_t, hipEvent_t, hipEvent_t, int) { return launched(b); }
hipError_t hipLaunchKernel(const void*, dim3, dim3 b, void**, size_t, hipStream_t) { return launched(b); }
hipError_t hipMalloc(void** p, size_t n) { return *p = aligned_alloc(256, (n + 255) & ~(size_t)255), *p ? hipSuccess : hipErrorOutOfMemory; }
hipError_t hipFree(void* p) { return free(p), hipSuccess; }
hipError_t hipHostMalloc(void** p, size_t n, unsigned) { return hipMalloc(p, n); }
hipError_t hipHostFree(void* p) { return hipFree(p); }
hipError_t hipGetDevice(int* d) { return *d = 0, hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetDeviceCount(int* n) { return *n = 1, hipSuccess; }
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600* p, int) {
    memset(p, 0, sizeof(*p));
    p->multiProcessorCount = 256;
    return hipSuccess;
}
const char* hipGetErrorString(hipError_t) { return "as told"; }
hipError_t hipGetLastError() {
    const hipError_t e = g_left;
    return g_left = hipSuccess, e;
}
static char g_symbol[1 << 26];
hipError_t hipGetSymbolAddress(void** p, const void*) { return *p = g_symbol, hipSuccess; }
hipError_t hipMemcpy(void*, const void*, size_t, hipMemcpyKind) { return hipSuccess; }
hipError_t hipMemcpyAsync(void*, const void*, size_t, hipMemcpyKind, hipStream_t) { return hipSuccess; }
hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) { return *s = (hipStream_t)&g_event, hipSuccess; }
hipError_t hipStreamDestroy(hipStream_t) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* s) { return *s = hipStreamCaptureStatusNone, hipSuccess; }
hipError_t hipStreamQuery(hipStream_t) { return hipSuccess; }
hipError_t hipStreamWaitEvent(hipStream_t, hipEvent_t, unsigned) { return hipSuccess; }
hipError_t hipThreadExchangeStreamCaptureMode(hipStreamCaptureMode*) { return hipSuccess; }
}

static const char* g_what;
static int g_at;
#define EXPECT(x)                                                                                                                            \
    do {                                                                                                                                     \
        if (!(x)) {                                                                                                                          \
            printf("%s %d: %s fails (line %d); %d launches, %s\n", g_what, g_at, #x, __LINE__, g_compactions, bkv_last_error());             \
            exit(1);                                                                                                                         \
        }                                                                                                                                    \
    } while (0)

struct State {
    int64_t len;
    int32_t free;
    std::vector<int32_t> table;
    bool operator==(const State& o) const { return len == o.len && free == o.free && table == o.table; }
};
static State state(bkv_pool* p, int32_t seq) {
    State s{bkv_seq_len(p, seq), 0, std::vector<int32_t>((size_t)bkv_seq_n_pages(p, seq))};
    const int32_t* const table = bkv_seq_block_table(p, seq);
    std::copy(table, table + s.table.size(), s.table.begin());
    s.free = bkv_pool_free_pages(p);
    return s;
}

// A sequence of `cells` is compacted to `keep` of them, again and again until the ring has gone round, then once with something that goes
// wrong, then once more.  -> whether that call failed
template <typename Wrong>
static bool once(int64_t cells, int32_t keep, const char* what, int at, Wrong wrong) {
    g_what = what, g_at = at;
    bkv_pool_desc d{};
    d.n_layers = 1, d.page_cells = 16, d.n_kv_head = 1, d.head_dim = 32, d.max_seqs = 2, d.layout = BKV_LAYOUT_F16;
    d.max_pages_per_seq = (int32_t)(cells / 16 + 1), d.n_pages = 2 * d.max_pages_per_seq + 2;
    bkv_pool* p = nullptr;
    EXPECT(bkv_pool_create(&d, &p) == BKV_OK);
    int32_t seq, other, n_cow;
    EXPECT(bkv_seq_create(p, &seq) == BKV_OK && bkv_seq_reserve(p, seq, cells, nullptr, 0, &n_cow) == BKV_OK);
    EXPECT(bkv_seq_create(p, &other) == BKV_OK && bkv_seq_reserve(p, other, 5, nullptr, 0, &n_cow) == BKV_OK);
    alignas(16) static uint32_t list[4];
    char streams[2];
    const auto compact = [&](int64_t n, void* stream) {
        const int64_t first = 0;
        const int32_t n_keep = (int32_t)n;
        return bkv_seq_compact(p, 1, &seq, &first, &n_keep, list, 0, 0, stream);
    };
    for (int64_t i = 0, slots = 0; slots < 40; ++i, slots += 1 + cells / 16 / 16384) EXPECT(compact(cells, streams) == BKV_OK);
    const State was = state(p, seq);
    g_compactions = g_others = g_running = g_records = g_queries = 0;
    wrong();
    const bkv_status st = compact(keep, streams);
    g_fail_record = g_late_query = g_fail_launch = 0, g_left = hipSuccess;
    const State now = state(p, seq);
    if (st != BKV_OK) {
        EXPECT(now == was);
        EXPECT(g_running == 0);  // none that would write tables, or pages that are free again
    } else {
        EXPECT(now.len == keep && (int64_t)now.table.size() == (keep + 15) / 16);
        EXPECT(now.free == was.free + (int32_t)(was.table.size() - now.table.size()));
        EXPECT(keep == 0 || g_compactions >= 1);
    }
    EXPECT(bkv_pool_check(p) == BKV_OK);
    EXPECT(compact(1 <= now.len, streams + 1) == BKV_OK && bkv_pool_check(p) == BKV_OK);
    EXPECT(bkv_pool_destroy(p) == BKV_OK);
    return st != BKV_OK;
}

int main() {
    EXPECT(bkv_wait_options(1, 1) == BKV_OK);
    // pages in one slot with the tables' changes; more than one slot holds; more than all of them
    const struct {
        int64_t cells;
        int at_most;
    } sizes[] = {{1000, 6}, {20 * 16384 + 7, 12}, {(int64_t)34 * 16384 * 16, 0}};
    for (const auto& s : sizes) {
        const int32_t keeps[] = {(int32_t)(s.cells - 3), 700, 0};
        for (const int32_t keep : keeps) {
            int late = 0, launch = 0;
            for (int i = 1; i <= s.at_most; ++i) {
                EXPECT(!once(s.cells, keep, "record", i, [&] { g_fail_record = i; }));
                late += once(s.cells, keep, "not yet from question", i, [&] { g_late_query = i; });
                launch += once(s.cells, keep, "launch", i, [&] { g_fail_launch = i; });
            }
            if (s.at_most && keep) EXPECT(late > 0 && launch > 0);
            EXPECT(!once(s.cells, keep, "an error that was there", 0, [] { g_left = hipErrorOutOfMemory; }));
            if (keep == 0) EXPECT(!once(s.cells, keep, "not yet", 1, [] { g_late_query = 1; }));
        }
    }
    // between its launches, once the ring has gone round
    const int64_t most = sizes[2].cells;
    EXPECT(once(most, (int32_t)most, "not yet from question", 34, [] { g_late_query = 34; }));
    EXPECT(once(most, (int32_t)most, "launch", 33, [] { g_fail_launch = 33; }));
    puts("ok");
    return 0;
}
