// A decode step whose ordering behind another stream fails reports that and enqueues nothing: no row is in the cache of a
// call that failed.  Run on the host: the HIP calls that the library makes are the ones below (an executable's come before a
// library's), which launch nothing, count launches and fail the wait that they are told to.
#include <hip/hip_runtime.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "breccia_kv.h"

static int g_launches, g_waits, g_fail_wait;

extern "C" {
hipError_t __hipPushCallConfiguration(dim3, dim3, size_t, hipStream_t) { return hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3* g, dim3* b, size_t* s, hipStream_t* st) {
    *g = *b = dim3(1), *s = 0, *st = nullptr;
    return hipSuccess;
}
hipError_t hipDeviceSynchronize() { return hipSuccess; }
static char g_event;
hipError_t hipEventCreate(hipEvent_t* e) { return *e = (hipEvent_t)&g_event, hipSuccess; }
hipError_t hipEventCreateWithFlags(hipEvent_t* e, unsigned) { return *e = (hipEvent_t)&g_event, hipSuccess; }
hipError_t hipEventDestroy(hipEvent_t) { return hipSuccess; }
hipError_t hipEventElapsedTime(float* ms, hipEvent_t, hipEvent_t) { return *ms = 0.0f, hipSuccess; }
hipError_t hipEventQuery(hipEvent_t) { return hipSuccess; }
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }
hipError_t hipExtLaunchKernel(const void*, dim3, dim3, void**, size_t, hipStream_t, hipEvent_t, hipEvent_t, int) { return ++g_launches, hipSuccess; }
hipError_t hipLaunchKernel(const void*, dim3, dim3, void**, size_t, hipStream_t) { return ++g_launches, hipSuccess; }
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
hipError_t hipGetLastError() { return hipSuccess; }
static char g_symbol[1 << 26];
hipError_t hipGetSymbolAddress(void** p, const void*) { return *p = g_symbol, hipSuccess; }
hipError_t hipMemcpy(void*, const void*, size_t, hipMemcpyKind) { return hipSuccess; }
hipError_t hipMemcpyAsync(void*, const void*, size_t, hipMemcpyKind, hipStream_t) { return hipSuccess; }
hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) { return *s = (hipStream_t)&g_event, hipSuccess; }
hipError_t hipStreamDestroy(hipStream_t) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* s) { return *s = hipStreamCaptureStatusNone, hipSuccess; }
hipError_t hipStreamQuery(hipStream_t) { return hipSuccess; }
hipError_t hipStreamWaitEvent(hipStream_t, hipEvent_t, unsigned) { return ++g_waits == g_fail_wait ? hipErrorInvalidValue : hipSuccess; }
hipError_t hipThreadExchangeStreamCaptureMode(hipStreamCaptureMode*) { return hipSuccess; }
}

#define EXPECT(x)                                                                                             \
    do {                                                                                                      \
        if (!(x)) {                                                                                           \
            printf("layout %d, plan %d, wait %d: %s (%s)\n", layout, plan, fail, #x, bkv_last_error());       \
            return 1;                                                                                         \
        }                                                                                                     \
    } while (0)

int main() {
    alignas(16) static float rows[4096];
    char streams[2];
    for (int layout = BKV_LAYOUT_F16; layout <= BKV_LAYOUT_F8P; ++layout)
        for (int plan = 0; plan < 2; ++plan) {
            int failed = 0, fail = 0;
            for (fail = 1; fail < 10; ++fail) {
                bkv_pool_desc d{};
                d.n_layers = 1, d.n_pages = 8, d.page_cells = 16, d.n_kv_head = 2, d.head_dim = 256, d.max_seqs = 1, d.max_pages_per_seq = 8;
                d.layout = (decltype(d.layout))layout;
                bkv_pool* p = nullptr;
                g_fail_wait = 0;
                EXPECT(bkv_pool_create(&d, &p) == BKV_OK);
                int32_t seq, n_cow;
                int64_t pos = 0;
                EXPECT(bkv_seq_create(p, &seq) == BKV_OK);
                EXPECT(bkv_seq_reserve(p, seq, 10, nullptr, 0, &n_cow) == BKV_OK);
                bkv_step_plan* pl = nullptr;
                if (plan) EXPECT(bkv_step_plan_create(p, 1, &seq, &pos, 4, 16, streams, &pl) == BKV_OK);
                const auto step = [&](void* stream) {
                    return plan ? bkv_step_plan_decode(pl, 0, rows, rows, rows, nullptr, 0, 0, 0.0625f, rows, stream)
                                : bkv_decode_step(p, 0, 1, &seq, &pos, rows, rows, 16, rows, nullptr, 0, 0, 0.0625f, rows, stream);
                };
                EXPECT(step(streams) == BKV_OK);
                g_launches = g_waits = 0, g_fail_wait = fail;
                const bkv_status st = step(streams + 1);
                g_fail_wait = 0;
                if (st != BKV_OK) {
                    ++failed;
                    EXPECT(st == BKV_ERR_HIP && g_launches == 0);
                } else {
                    EXPECT(g_launches >= 2 && g_waits < fail);
                }
                if (pl) EXPECT(bkv_step_plan_destroy(pl) == BKV_OK);
                EXPECT(bkv_pool_destroy(p) == BKV_OK);
            }
            EXPECT(failed > 0);
        }
    puts("ok");
    return 0;
}
