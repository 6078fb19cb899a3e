// scratch_threads.cpp -- calls of several host threads on one stream, against mocks of the HIP calls that
// tiny-llm_amd/csrc/scratch.cpp makes (compiled with g++, no GPU and no HIP runtime). A call that holds its stream's
// scratch (ScratchCall) keeps its buffers, contents and addresses, until it lets go.
#include <atomic>
#include <chrono>
#include <cstdio>
#include <cstdlib>
#include <mutex>
#include <set>
#include <thread>

#include "tq_common.h"

namespace {

std::mutex g_mu;
std::set<void *> g_live;

void check(bool ok, const char *what) {
    if (!ok) {
        std::printf("FAIL %s\n", what);
        std::exit(1);
    }
    std::printf("ok %s\n", what);
}
bool live(void *p) {
    std::lock_guard<std::mutex> lock(g_mu);
    return g_live.count(p) != 0;
}
hipStream_t stream(int i) { return reinterpret_cast<hipStream_t>(static_cast<uintptr_t>(0x1000 * i)); }

}  // namespace

extern "C" {
hipError_t hipGetDevice(int *d) {
    *d = 0;
    return hipSuccess;
}
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus *st) {
    *st = hipStreamCaptureStatusNone;
    return hipSuccess;
}
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipMalloc(void **p, size_t n) {
    *p = std::malloc(n);
    std::lock_guard<std::mutex> lock(g_mu);
    g_live.insert(*p);
    return hipSuccess;
}
hipError_t hipMemsetAsync(void *, int, size_t, hipStream_t) { return hipSuccess; }
hipError_t hipFree(void *p) {
    std::lock_guard<std::mutex> lock(g_mu);
    g_live.erase(p);  // (kept allocated: no later buffer can have its address)
    return hipSuccess;
}
}

using namespace tqhip;

int main() {
    std::atomic<bool> grown{false}, other{false};
    std::thread same, elsewhere;
    {
        ScratchCall call(stream(1));
        void *p = nullptr, *again = nullptr;
        unsigned long long *slots = nullptr;
        check(call.workspace(1000, &p) == kOk && live(p), "a call gets a buffer");
        check(scratch_split_slots(stream(1), 100, &slots) == kOk && slots, "and a second one under its own hold");
        same = std::thread([&] {
            ScratchCall call2(stream(1));
            void *q = nullptr;
            check(call2.workspace(8 << 20, &q) == kOk && q != p, "a larger one of the same stream, afterwards");
            grown = true;
        });
        elsewhere = std::thread([&] {
            ScratchCall call2(stream(2));
            void *q = nullptr;
            check(call2.workspace(1000, &q) == kOk && q != p, "another stream does not wait");
            other = true;
        });
        for (int i = 0; i < 2000 && !other; ++i) std::this_thread::sleep_for(std::chrono::milliseconds(5));
        check(other, "another stream went ahead");
        std::this_thread::sleep_for(std::chrono::milliseconds(200));
        check(!grown && live(p), "the buffer stays while the call goes on");
        check(call.workspace(1000, &again) == kOk && again == p, "at its address");
    }
    same.join();
    elsewhere.join();
    check(grown, "the waiting call went on");
    std::printf("all ok\n");
    return 0;
}
