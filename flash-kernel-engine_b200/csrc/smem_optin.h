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
  // set(bytes): raises the attribute; 0 on success. Returns its result, 0 without a call, or
  // no_memory where there is none for a record (called from C entries: nothing is thrown).
  template <typename Set, typename Error>
  Error ensure(const void* func, int device, int bytes, Set set, Error no_memory) noexcept {
    std::lock_guard<std::mutex> lk(mu_);
    int* have = nullptr;
    try {
      have = &bytes_[std::make_pair(func, device)];
    } catch (...) {
      return no_memory;
    }
    if (*have >= bytes) return Error{};
    const Error e = set(bytes);
    if (e == Error{}) *have = bytes;
    return e;
  }

 private:
  std::mutex mu_;
  std::map<std::pair<const void*, int>, int> bytes_;
};

}  // namespace fe
