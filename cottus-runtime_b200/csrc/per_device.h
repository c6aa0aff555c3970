// Facts about a device, looked up at its first use.
#pragma once

#include <atomic>
#include <mutex>

namespace cb200 {

// One T per device, filled in by the first call of get() whose `find` succeeds.
// A failure is returned and not kept: the next call looks again.
template <typename T, typename Err, int kMaxDevices = 64>
class PerDevice {
public:
    // find(T&) -> Err, Err{} for success; `out_of_range` for a device past the table.
    template <typename Find>
    Err get(int device, T& out, Err out_of_range, Find find) {
        if (device < 0 || device >= kMaxDevices) return out_of_range;
        if (!known_[device].load(std::memory_order_acquire)) {
            std::lock_guard<std::mutex> lock(mutex_);
            if (!known_[device].load(std::memory_order_relaxed)) {
                T found{};
                const Err e = find(found);
                if (e != Err{}) return e;
                value_[device] = found;
                known_[device].store(true, std::memory_order_release);
            }
        }
        out = value_[device];
        return Err{};
    }

private:
    std::mutex mutex_;
    T value_[kMaxDevices] = {};
    std::atomic<bool> known_[kMaxDevices] = {};
};

}  // namespace cb200
