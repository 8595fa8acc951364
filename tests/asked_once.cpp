// Threads on devices of their own ask for the same kernels at once.  Whatever the table then takes for granted on a device must have been
// asked for on that device, and what it was asked for must have been done when `once` returns.  Exit code 0: so it is.
#include "asked_once.h"
#include <atomic>
#include <cstdio>
#include <thread>
#include <vector>

constexpr int KERNELS = 90, DEVICES = 4, ROUNDS = 400;
static char kernels[KERNELS];                            // (their addresses stand for kernels)

int main() {
    for (int round = 0; round < ROUNDS; ++round) {
        AskedOnce table;
        std::atomic<int> done[KERNELS][DEVICES] = {}, ready{0}, wrong{0};
        auto run = [&](int dev, int turn) {
            ++ready;
            while (ready < 2 * DEVICES) {}
            for (int i = 0; i < KERNELS; ++i) {
                const int k = (i + turn * 7) % KERNELS;
                const int st = table.once(&kernels[k], dev, [&] { ++done[k][dev]; return 0; });
                if (st || !done[k][dev]) ++wrong;        // the launch that follows would fail
            }
        };
        std::vector<std::thread> threads;
        for (int t = 0; t < 2 * DEVICES; ++t) threads.emplace_back(run, t % DEVICES, t / DEVICES);
        for (auto& t : threads) t.join();
        if (wrong) { std::printf("round %d: %d calls without their kernel\n", round, (int)wrong); return 1; }
        // known from here on; an answer other than 0 is given back, and asked for again
        int asked = 0;
        for (int k = 0; k < KERNELS; ++k)
            for (int d = 0; d < DEVICES; ++d) table.once(&kernels[k], d, [&] { ++asked; return 0; });
        char other;
        for (int i = 0; i < 2; ++i)
            if (table.once(&other, 0, [&] { ++asked; return 7; }) != 7) return 2;
        if (asked != 2) { std::printf("asked %d times again\n", asked - 2); return 3; }
    }
    return 0;
}
