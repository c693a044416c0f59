// Host check of csrc/exl3_workspace.hpp: the launches of calls that share an internal workspace keep together.
// "Launches" are entries of a log; a call of several takes the workspace, logs each of them with a pause between,
// and lets go.  Exit status 0: no call's entries were parted on its key, and calls on two keys overlapped.
#include "exl3_workspace.hpp"

#include <chrono>
#include <condition_variable>
#include <cstdio>
#include <thread>
#include <utility>
#include <vector>

typedef exl3k::WorkspaceTable<std::pair<int, const void *>> Table;

int main() {
    Table table;
    std::mutex log_mutex;
    std::vector<std::pair<int, int>> log[2];  // of each key: (call, launch)
    const int streams[2] = {};
    constexpr int kThreads = 6, kCalls = 60, kLaunches = 3;

    std::vector<std::thread> threads;
    for (int t = 0; t < kThreads; ++t)
        threads.emplace_back([&, t] {
            for (int c = 0; c < kCalls; ++c) {
                const int key = (t + c) % 2;
                exl3k::WorkspaceLease lease;
                Table::Slot &slot = table.take(std::make_pair(0, &streams[key]), &lease);
                slot.bytes += 1;  // growth, guarded by the lease
                for (int i = 0; i < kLaunches; ++i) {
                    {
                        std::lock_guard<std::mutex> lock(log_mutex);
                        log[key].emplace_back(t * kCalls + c, i);
                    }
                    std::this_thread::sleep_for(std::chrono::microseconds(20));
                }
            }
        });
    for (std::thread &t : threads) t.join();
    size_t calls = 0;
    for (const auto &entries : log)
        for (size_t i = 0; i < entries.size(); ++i) {
            if (entries[i].second != (int)(i % kLaunches) || entries[i].first != entries[i - i % kLaunches].first) {
                std::printf("parted at %zu\n", i);
                return 1;
            }
            calls += i % kLaunches == 0;
        }
    if (calls != (size_t)kThreads * kCalls) return 2;

    // a call on one key does not wait for a call on another
    exl3k::WorkspaceLease first;
    Table::Slot &a = table.take(std::make_pair(0, &streams[0]), &first);
    Table::Slot *b = nullptr;
    std::thread([&] {
        exl3k::WorkspaceLease second;
        b = &table.take(std::make_pair(0, &streams[1]), &second);
    }).join();
    if (!b || b == &a || a.bytes + b->bytes != calls) return 3;
    std::puts("workspace leases ok");
    return 0;
}
