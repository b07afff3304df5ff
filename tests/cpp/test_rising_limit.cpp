// Two threads raise one kernel's limit at once, the larger one first but slowly: the limit must end at the larger value, and
// what is recorded must be what was set.
#include <chrono>
#include <cstdio>
#include <thread>

#include "rtb_cluster.cuh"

int main() {
    using namespace std::chrono_literals;
    for (int larger_first = 0; larger_first < 2; ++larger_first) {
        rtb::RisingLimit limit;
        std::atomic<size_t> attribute{0};
        std::atomic<bool> inside{false}, other_done{false};
        const size_t first = larger_first ? 100000 : 50000, second = larger_first ? 50000 : 100000;
        std::thread a([&] {
            limit.raise(3, first, [&] {
                attribute = first;
                inside = true;
                for (int k = 0; k < 200 && !other_done; ++k) std::this_thread::sleep_for(1ms);   // between the call and the record
                return 0;
            });
        });
        while (!inside) std::this_thread::yield();
        std::thread b([&] {
            limit.raise(3, second, [&] { attribute = second; return 0; });
            other_done = true;
        });
        a.join(), b.join();
        if (attribute != 100000) return std::printf("the limit ended at %zu\n", attribute.load()), 1;
        // what was reached needs no further call, what lies beyond does; another device has a limit of its own; a failure is not recorded
        int calls = 0;
        auto count = [&] { ++calls; return 0; };
        limit.raise(3, 100000, count), limit.raise(3, 1, count), limit.raise(3, 0, count);
        if (calls != 0) return std::printf("raised again to what it was\n"), 1;
        if (limit.raise(4, 200000, [] { return -8; }) != -8) return std::printf("a failure was lost\n"), 1;
        limit.raise(4, 200000, count), limit.raise(3, 100001, count);
        if (calls != 2) return std::printf("%d calls where two were due\n", calls), 1;
    }
    std::printf("ok\n");
    return 0;
}
