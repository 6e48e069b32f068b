// What the library has found out, or set up, once for a device.  Host threads may ask for it at the same time: both then find it out,
// to the same end, and a value that is seen is whole and was set after what it stands for was done.
#pragma once

#include <atomic>

namespace catccos {

template <typename T, int kDevices>
class PerDevice {
public:
    // the device's value; T() where there is none yet, or no place for the device
    T get(int device) const { return device >= 0 && device < kDevices ? values_[device].load(std::memory_order_acquire) : T(); }
    void set(int device, T value)
    {
        if (device >= 0 && device < kDevices) {
            values_[device].store(value, std::memory_order_release);
        }
    }

private:
    std::atomic<T> values_[kDevices] = {};
};

}  // namespace catccos
