// What a process sets or asks once for each of its devices, such as the shared memory that a kernel may take and how many of its clusters are
// resident together.  What failed is not remembered, and tried again at the next call.
#pragma once

#include <atomic>

constexpr int kMostDevices = 64;      // devices beyond these are asked every time

struct OncePerDevice {
    std::atomic<bool> done[kMostDevices] = {};
    // go() returns 0 when it has succeeded; returns what it returned, or 0 where it has succeeded before.
    template <typename Go>
    int operator()(int device, Go go) {
        const bool known = device >= 0 && device < kMostDevices;
        if (known && done[device].load(std::memory_order_acquire)) return 0;
        const int status = go();
        if (known && status == 0) done[device].store(true, std::memory_order_release);
        return status;
    }
};

struct NumberPerDevice {
    std::atomic<int> held[kMostDevices] = {};      // one more than the number; 0: not known yet
    // go() returns the number, or one below zero when it has failed: 0 for this call.
    template <typename Go>
    int operator()(int device, Go go) {
        const bool known = device >= 0 && device < kMostDevices;
        const int before = known ? held[device].load(std::memory_order_acquire) : 0;
        if (before > 0) return before - 1;
        const int number = go();
        if (number < 0) return 0;
        if (known) held[device].store(number + 1, std::memory_order_release);
        return number;
    }
};
