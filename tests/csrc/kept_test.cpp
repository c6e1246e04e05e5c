// Host test of kept.h: prints what `kept` returned and how often it had asked, in order.
#include <cstdio>
#include <thread>
#include <vector>

#include "../../fluke_b200/csrc/kept.h"

int main() {
    std::atomic<int> slot{0}, shared{0}, wrong{0};
    int asked = 0;
    const int answers[] = {0, -1, 7, 9};
    for (int call = 0; call < 5; ++call) {
        const int got = fluke_sm100::kept(slot, [&] { return answers[asked++]; });
        std::printf("%d/%d ", got, asked);
    }
    std::vector<std::thread> threads;
    for (int t = 0; t < 8; ++t)
        threads.emplace_back([&] {
            for (int i = 0; i < 10000; ++i) wrong += fluke_sm100::kept(shared, [] { return 74; }) != 74;
        });
    for (auto &t : threads) t.join();
    std::printf("%d\n", wrong.load());
}
