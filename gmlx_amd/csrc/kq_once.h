// What the host does once on each device.
#pragma once
#include <atomic>
#include <cstdint>

// Limits of a kernel (its dynamic LDS) hold on the device that they are set on:
// f, on the device that is current, at the first call there and after failures;
// says whether it has succeeded.  Two threads may both run it, which is harmless.
class OncePerDevice {
    std::atomic<uint64_t> done_{0};

  public:
    template <class F>
    bool operator()(int device, F &&f) {
        if (device < 0) return false;
        const uint64_t bit = device < 64 ? (uint64_t)1 << device : 0;
        if (done_.load(std::memory_order_acquire) & bit) return true;
        if (!f()) return false;
        done_.fetch_or(bit, std::memory_order_release);
        return true;
    }
};
