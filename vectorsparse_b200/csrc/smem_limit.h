// How much dynamic shared memory a kernel has been allowed, per device.  Nothing of CUDA here, so that it can be tested alone.
#pragma once
#include <atomic>
#include <mutex>

namespace vs {

class SmemLimit {   // of one kernel
public:
    static constexpr int kDevices = 64;

    // Calls set() (0: it went well) unless `bytes` are allowed already.  The lock is held around the call and the note of it: of two host threads with unlike sizes neither
    // takes back what the other was allowed, so the limit only grows.
    template <typename Set> int raise(int device, int bytes, Set set) {
        if (known_[device].load(std::memory_order_acquire) >= bytes) return 0;
        std::lock_guard<std::mutex> lock(mutex_);
        if (known_[device].load(std::memory_order_relaxed) >= bytes) return 0;
        const int rc = set();
        if (rc == 0) known_[device].store(bytes, std::memory_order_release);
        return rc;
    }

private:
    std::atomic<int> known_[kDevices] = {};
    std::mutex mutex_;
};

}  // namespace vs
