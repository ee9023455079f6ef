// The dynamic shared memory that each kernel has been opted in to. Plain C++, so that a host
// program can go through it too.
#pragma once

#include <map>
#include <mutex>
#include <utility>

namespace fe {

// One entry for each (function, device), which only grows: the attribute is a maximum, so a
// launch that needs less than an earlier one leaves it alone, and a launch that needs more
// raises it. Check, set and record are one step under the lock; with a gap between them two
// threads could set 150 KB and then 120 KB of one kernel and record 150, after which every
// launch of 150 KB would fail.
class SmemOptin {
 public:
  // set(bytes): raises the attribute; 0 on success. Returns its result, or 0 without a call.
  template <typename Set>
  auto ensure(const void* func, int device, int bytes, Set set) -> decltype(set(bytes)) {
    std::lock_guard<std::mutex> lk(mu_);
    const auto it = bytes_.try_emplace(std::make_pair(func, device), 0).first;
    if (it->second >= bytes) return {};
    const auto e = set(bytes);
    if (e == decltype(e){}) it->second = bytes;
    return e;
  }

 private:
  std::mutex mu_;
  std::map<std::pair<const void*, int>, int> bytes_;
};

}  // namespace fe
