// Values of a device (per_device.hpp) that several threads find out at once: compiled with the race detector.
#include <cstdio>
#include <thread>
#include <vector>

#include "../../catccos_b200/csrc/per_device.hpp"

int main()
{
    static catccos::PerDevice<int, 4> found;
    static int done[4][8];  // what a value stands for, done before it is set
    bool good = found.get(0) == 0 && found.get(-1) == 0 && found.get(4) == 0;
    found.set(4, 7);
    found.set(-1, 7);
    std::vector<std::thread> threads;
    std::atomic<int> wrong{0};
    for (int t = 0; t < 8; ++t) {
        threads.emplace_back([t, &wrong] {
            for (int n = 0; n < 1000; ++n) {
                const int device = (n + t) % 4, seen = found.get(device);
                if (seen == 0) {
                    done[device][t] = 1;
                    found.set(device, t + 1);
                } else if (done[device][seen - 1] != 1) {
                    wrong++;
                }
            }
        });
    }
    for (std::thread& t : threads) {
        t.join();
    }
    good = good && wrong == 0;
    for (int d = 0; d < 4; ++d) {
        good = good && found.get(d) >= 1 && found.get(d) <= 8;
    }
    printf(good ? "per device ok\n" : "per device wrong\n");
    return good ? 0 : 1;
}
