// How much dynamic shared memory each kernel was allowed, per device (the standard library only, so that it is tested on the host).
#pragma once
#include <map>
#include <mutex>
#include <utility>

namespace q38 {

class SharedMemoryGrants {
 public:
  // Calls `raise` unless the kernel was allowed that much before.  An exception of it leaves what is remembered as it was.
  template <typename F> void ensure(const void* kernel, int device, int bytes, F&& raise) {
    const std::lock_guard<std::mutex> lock(mutex_);
    int& granted = granted_[{kernel, device}];
    if (bytes <= granted) return;
    raise();
    granted = bytes;
  }

 private:
  std::mutex mutex_;
  std::map<std::pair<const void*, int>, int> granted_;
};

}  // namespace q38
