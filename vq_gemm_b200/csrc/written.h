// Which streams hold weights that this library has written and no product has followed yet (see note_weights_written in
// common.cuh).  Plain C++, no CUDA types.
#pragma once

#include <atomic>
#include <mutex>
#include <new>
#include <vector>

namespace vqg {

class WrittenMarks {
 public:
  // `stream` tells streams of one device apart, `capture` is the id of the capture that the stream is part of, 0 outside one: what
  // is captured runs later, so an eager mark is not met by a captured product, nor the other way round.
  struct Key {
    int device;
    const void* stream;
    unsigned long long capture;
    bool operator==(const Key& o) const { return device == o.device && stream == o.stream && capture == o.capture; }
  };

  // One entry per key, for as many as there are.  Where memory for it runs out every stream counts as marked from then on.
  void note(const Key& k) noexcept {
    std::lock_guard<std::mutex> lk(mu_);
    for (const Key& m : marks_)
      if (m == k) return;
    try {
      marks_.push_back(k);
    } catch (const std::bad_alloc&) {
      all_.store(true);
    }
    count_.store(marks_.size());
  }

  // Whether the stream may be marked, in any capture or none: take() need not be asked otherwise.
  bool maybe(int device, const void* stream) noexcept {
    if (all_.load(std::memory_order_relaxed)) return true;
    if (count_.load(std::memory_order_relaxed) == 0) return false;
    std::lock_guard<std::mutex> lk(mu_);
    for (const Key& m : marks_)
      if (m.device == device && m.stream == stream) return true;
    return false;
  }

  // Whether it is marked; the mark is then gone.
  bool take(const Key& k) noexcept {
    std::lock_guard<std::mutex> lk(mu_);
    for (Key& m : marks_)
      if (m == k) {
        m = marks_.back();
        marks_.pop_back();
        count_.store(marks_.size());
        return true;
      }
    return all_.load();
  }

 private:
  std::mutex mu_;
  std::vector<Key> marks_;
  std::atomic<size_t> count_{0};
  std::atomic<bool> all_{false};
};

}  // namespace vqg
