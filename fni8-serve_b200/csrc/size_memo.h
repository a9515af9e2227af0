// Answers that depend on sizes alone, asked for in every call: found once, then looked up.
#pragma once
#include <map>
#include <mutex>
#include <utility>

namespace fni8h {

// Grows with the keys seen, whatever their number: a list that fills up would make every size beyond it pay in every
// call. Any host thread may ask.
template <typename Key>
class SizeMemo {
 public:
  // The number of `key`, from find() where it is not known yet. A negative one (no answer) is not kept.
  template <typename Find>
  int get(const Key& key, Find&& find) {
    std::lock_guard<std::mutex> lock(mu_);
    const auto it = known_.find(key);
    if (it != known_.end()) return it->second;
    const int n = std::forward<Find>(find)();
    if (n >= 0) {
      try {
        known_.emplace(key, n);
      } catch (...) {  // no memory for it: found again next time (the callers are C entry points)
      }
    }
    return n;
  }

 private:
  std::mutex mu_;
  std::map<Key, int> known_;
};

}  // namespace fni8h
