// Which streams end in a kernel of this library that writes block tables and lengths. Plain
// C++, so that a host program can go through it too.
//
// The paged decode reads block_tables and context_lens ahead of its griddepcontrol.wait, but
// only past that wait are the stores of the kernel before it sure to be seen, even where that
// kernel has left every SM. So a decode that follows a writer of them directly is launched
// without programmatic serialization. A kernel in between that waits for what is before it,
// and does not let its successor start early, ends this: the decode starts after it, and it
// ended after the writer.
#pragma once

#include <algorithm>
#include <atomic>
#include <mutex>
#include <utility>
#include <vector>

namespace fe {

class TableWriters {
 public:
  // A kernel that writes tables or lengths goes on the stream. These are called from C entries:
  // nothing is thrown, and where a stream cannot be recorded every stream counts as one that
  // ends in a writer from then on.
  void wrote(int device, const void* stream) noexcept {
    std::lock_guard<std::mutex> lk(mu_);
    if (find(device, stream) != last_.end()) return;
    try {
      last_.emplace_back(device, stream);
      count_ = static_cast<int>(last_.size());
    } catch (...) {
      all_ = true;
    }
  }
  // A kernel goes on the stream behind which the tables are sure to be seen. Returns whether
  // the stream ended in a writer.
  bool passed(int device, const void* stream) noexcept {
    if (all_) return true;
    if (count_ == 0) return false;
    std::lock_guard<std::mutex> lk(mu_);
    const auto it = find(device, stream);
    if (it == last_.end()) return false;
    *it = last_.back();
    last_.pop_back();
    count_ = static_cast<int>(last_.size());
    return true;
  }

 private:
  using Stream = std::pair<int, const void*>;
  std::vector<Stream>::iterator find(int device, const void* stream) {
    return std::find(last_.begin(), last_.end(), Stream(device, stream));
  }
  std::mutex mu_;
  std::atomic<int> count_{0};  // a call with no writer anywhere takes no lock
  std::atomic<bool> all_{false};
  std::vector<Stream> last_;
};

}  // namespace fe
