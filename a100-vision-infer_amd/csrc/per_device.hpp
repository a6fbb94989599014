// An action that is due once on every device of a process (kernel attributes
// belong to a device's copy of a kernel).  No HIP here: the CPU tests compile it.
#pragma once
#include <stdint.h>

#include <atomic>

namespace fp8lin {

class OncePerDevice {
public:
    // act() the first time on this device, and again while it fails: what it
    // returned, 0 for done.  Two threads that come first together both act.
    template <class F>
    int operator()(int device, F&& act) {
        const uint64_t bit = device >= 0 && device < 64 ? (uint64_t)1 << device : 0;
        if (done_.load(std::memory_order_acquire) & bit) return 0;
        const int e = act();
        if (e == 0) done_.fetch_or(bit, std::memory_order_release);
        return e;
    }

private:
    std::atomic<uint64_t> done_{0};
};

}  // namespace fp8lin
