// Something that the runtime is to be asked once for each kernel on each device.
#pragma once
#include <mutex>
#include <set>
#include <utility>

struct AskedOnce {
    std::mutex lock;                       // launchers are called from several threads, each on the device that is its own
    std::set<std::pair<int, const void*>> done;

    // `ask` for this kernel on this device, unless it has answered 0 before; gives its answer back.  Held while it asks: whoever finds
    // the pair here, finds it asked for.
    template <typename Ask> int once(const void* kern, int dev, Ask ask) {
        std::lock_guard<std::mutex> held(lock);
        const std::pair<int, const void*> key(dev, kern);
        if (done.count(key)) return 0;
        const int status = ask();
        if (status == 0) done.insert(key);
        return status;
    }
};
