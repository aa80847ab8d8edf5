// What is set once on each device: per-kernel attributes (more than 64 KB of dynamic LDS).  hipFuncSetAttribute applies to the current device, so a process that drives a second GPU
// sets them there, too.  Host only; behind hip_runtime.h.
#pragma once
#include <atomic>
#include <mutex>
#include <utility>

namespace lcc {

//   static DeviceOnce once;
//   if (auto turn = once.first()) ...set...;
// The first caller on a device sets, with the lock held; the device counts as done at the end of its `if`.  Callers that come meanwhile wait there: whoever passes may launch.
class DeviceOnce {
  std::atomic<unsigned long long> done_{0};
  std::mutex mu_;

 public:
  class Turn {
    std::unique_lock<std::mutex> lock_;
    std::atomic<unsigned long long>* done_ = nullptr;
    unsigned long long bit_ = 0;

   public:
    Turn() = default;
    Turn(std::unique_lock<std::mutex> lock, std::atomic<unsigned long long>& done, unsigned long long bit) : lock_(std::move(lock)), done_(&done), bit_(bit) {}
    Turn(Turn&&) = delete;
    ~Turn() { if (done_ != nullptr) done_->fetch_or(bit_, std::memory_order_release); }      // ahead of lock_'s release
    explicit operator bool() const { return done_ != nullptr; }
  };
  Turn first() {
    int d = 0;
    (void)hipGetDevice(&d);
    const unsigned long long bit = 1ull << (d & 63);
    if (done_.load(std::memory_order_acquire) & bit) return Turn();
    std::unique_lock<std::mutex> lock(mu_);
    if (done_.load(std::memory_order_relaxed) & bit) return Turn();
    return Turn(std::move(lock), done_, bit);
  }
};

}  // namespace lcc
