// Records of waits that kernels gave up, one word a device. A kernel writes its
// code into its device's word; every host thread that uses the device then
// learns of it once, whichever thread looks first.
#pragma once

#include <atomic>
#include <cstdint>
#include <mutex>

namespace mx {

class WaitRecords {
 public:
  static constexpr int kDevices = 64;

  // `words` are kDevices ints that the kernels can write, zero at first. There is
  // one object a process (what a thread has seen is kept by thread).
  explicit WaitRecords(int* words) : words_(words) {}

  // The code of a record on the device that this thread has not taken, or 0. A
  // thread is not told of records that others had taken before its first call.
  int pending(int device) {
    Seen& seen = this_thread(device);
    if (word(device) == 0 && seen.count == count_[device].load(std::memory_order_acquire)) return 0;
    std::lock_guard<std::mutex> lock(mu_);
    collect(device);
    return seen.count == count_[device].load(std::memory_order_relaxed) ? 0 : code_[device];
  }

  // The same, and it counts as taken by this thread (and by no other).
  int take(int device) {
    const int code = pending(device);
    if (code) {
      std::lock_guard<std::mutex> lock(mu_);
      this_thread(device).count = count_[device].load(std::memory_order_relaxed);
    }
    return code;
  }

 private:
  struct Seen {
    bool known = false;
    uint64_t count = 0;
  };
  Seen& this_thread(int device) {
    static thread_local Seen seen[kDevices];
    Seen& s = seen[device];
    if (!s.known) s.known = true, s.count = count_[device].load(std::memory_order_acquire);
    return s;
  }
  int word(int device) const { return __atomic_load_n(words_ + device, __ATOMIC_ACQUIRE); }
  void collect(int device) {
    const int code = __atomic_exchange_n(words_ + device, 0, __ATOMIC_ACQ_REL);
    if (!code) return;
    code_[device] = code;
    count_[device].fetch_add(1, std::memory_order_release);
  }

  int* words_;
  std::mutex mu_;
  std::atomic<uint64_t> count_[kDevices] = {};
  int code_[kDevices] = {};
};

}  // namespace mx
