// How much dynamic shared memory a kernel may be launched with: beyond 48 KB the runtime wants to be told, per kernel and
// device.  The limit is raised once, to the most that a launch can ever ask for, so that threads whose launches ask for
// different sizes cannot lower it for one another.
#pragma once

#include <atomic>
#include <cstddef>

namespace slora {

class SmemLimit {
 public:
  // `smem`: bytes of this launch; `most()`: bytes of the largest one; `set(bytes)`: raises the limit, false when it cannot.
  template <typename Most, typename Set>
  bool allow(int dev, size_t smem, const Most& most, const Set& set) {
    if (smem <= kGiven) return true;
    const bool known = dev >= 0 && dev < kDevices;
    if (known && raised_[dev].load(std::memory_order_acquire)) return true;
    if (!set(most())) return false;
    if (known) raised_[dev].store(true, std::memory_order_release);
    return true;
  }

 private:
  static constexpr int kDevices = 64;
  static constexpr size_t kGiven = 32 * 1024;  // what every kernel may take: 48 KB, up to 16 of them static
  std::atomic<bool> raised_[kDevices] = {};
};

}  // namespace slora
