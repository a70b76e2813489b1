// The library's count of launches, raised by threads side by side: none may be lost.
#include <cstdio>
#include <thread>
#include <vector>

#include "../llama2.rs_b200/csrc/kernels.cuh"

decltype(l2::g_launches) l2::g_launches{};

int main() {
    constexpr int THREADS = 4, EACH = 1000000;
    std::vector<std::thread> all;
    for (int i = 0; i < THREADS; i++)
        all.emplace_back([] {
            for (int n = 0; n < EACH; n++) {
                l2::g_launches++;
                asm volatile("" ::: "memory");
            }
        });
    for (auto& t : all) t.join();
    const bool ok = l2::g_launches.all == 1ull * THREADS * EACH && l2::LaunchCount::mine == 0;
    std::printf("%s\n", ok ? "ok" : "launches lost");
    return !ok;
}
