// What the tcgen05 kernels of gemm_sm100.cu and lora.cu share: tile constants, the bounded wait and its status codes.
#pragma once

#include <stdint.h>

#include "ptx.cuh"

namespace pg {
namespace {

constexpr uint32_t kBM = 128;           // rows of A per CTA
constexpr uint32_t kBK = 64;            // k elements per stage = one 128-byte swizzle row
constexpr uint32_t kUmmaK = 16;         // k elements per tcgen05.mma (16-bit inputs)
constexpr uint32_t kThreads = 192;
#ifdef PG_TEST_SHORT_WAIT
// Test build (libPeakGemm_device_waittest.so, never shipped as the product): waits give up after 2 ms.
constexpr uint64_t kWaitTimeoutNs = 2000000ull;
#else
constexpr uint64_t kWaitTimeoutNs = 2000000000ull;                // 2 s
#endif

// Codes written to the device status word (role that gave up).
enum : int {
    kStProducerEmpty = 1,
    kStMmaFull = 2,
    kStMmaAccEmpty = 3,
    kStEpiAccFull = 4,
    kStEpiTailFlag = 5,
};

struct WaitCtx {
    volatile uint32_t *abort_flag;  // shared memory
    int *status;                    // global memory
};

// Bounded mbarrier wait.  Returns false if the wait was abandoned.  The clock is
// only consulted every 1024 failed probes (each probe already suspends the thread
// for a hardware-defined interval), so the common short wait costs nothing extra.
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, const WaitCtx &ctx, int code) {
    if (ptx::mbar_try_wait(bar, parity)) return true;
    uint64_t t0 = 0;
    uint32_t spins = 0;
    while (true) {
        if (ptx::mbar_try_wait(bar, parity)) return true;
        if ((++spins & 1023u) == 0) {
            if (*ctx.abort_flag) return false;
            const uint64_t now = ptx::globaltimer_ns();
            if (t0 == 0) t0 = now;
            else if (now - t0 > kWaitTimeoutNs) {
                *ctx.abort_flag = 1;
                if (ctx.status) atomicCAS(ctx.status, 0, code);
                return false;
            }
        }
    }
}

}  // namespace
}  // namespace pg
