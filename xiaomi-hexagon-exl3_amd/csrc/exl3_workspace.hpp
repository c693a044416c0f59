// exl3_workspace.hpp -- who may enqueue on an internal workspace (host only, no HIP in it).
//
// A call of several launches (a walk in parts and its join, a split GEMM and its sum, packing and a
// product) hands data from one to the next in its workspace.  The launches of two threads on one stream run in
// the order in which they were enqueued, so between a call's launches no other call may enqueue one: a call
// holds its stream's workspace from the moment it gets it until its last launch is enqueued.  A workspace that
// the caller passes is the caller's to order.
#pragma once

#include <stddef.h>

#include <map>
#include <mutex>

namespace exl3k {

// held by a call until it returns; empty for a workspace of the caller's
typedef std::unique_lock<std::mutex> WorkspaceLease;

// One workspace per key (device and stream), never removed: references to a slot stay good.
template <typename Key>
class WorkspaceTable {
  public:
    struct Slot {
        std::mutex busy;  // guards the rest, and the order of launches on the workspace
        void *ptr = nullptr;
        size_t bytes = 0;
    };
    // waits until no other call holds it; calls on other keys go on
    Slot &take(const Key &key, WorkspaceLease *lease) {
        Slot *slot;
        {
            std::lock_guard<std::mutex> lock(mutex_);
            slot = &slots_[key];
        }
        *lease = WorkspaceLease(slot->busy);
        return *slot;
    }

  private:
    std::mutex mutex_;
    std::map<Key, Slot> slots_;
};

}  // namespace exl3k
