// Whether the outputs of a call are memory of their own. Blocks write them in any
// order while others still read operands, so an output that lies in another one or in
// an operand would leave words that depend on that order. Host only.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include <algorithm>
#include <vector>

namespace cfhe {

// The polynomials that a call writes, each `bytes` long. Usually they are one tensor
// and the operands others: then a test is a comparison or two.
class Outputs {
 public:
  explicit Outputs(size_t bytes) : bytes_{bytes} {}
  template <typename T>
  void add(T *const *p, size_t n) {
    for (size_t i = 0; i < n; i++) at_.push_back(reinterpret_cast<uintptr_t>(p[i]));
  }
  // After the last add(): false if two of them overlap
  bool apart() {
    if (!std::is_sorted(at_.begin(), at_.end())) std::sort(at_.begin(), at_.end());
    for (size_t i = 1; i < at_.size(); i++)
      if (at_[i] - at_[i - 1] < bytes_) return false;
    return true;
  }
  // After apart(): whether `size` bytes at p overlap one of them
  bool meet(const void *p, size_t size) const {
    const uintptr_t lo = reinterpret_cast<uintptr_t>(p), hi = lo + size;
    if (at_.empty() || hi <= at_.front() || lo >= at_.back() + bytes_) return false;
    const auto next = std::upper_bound(at_.begin(), at_.end(), lo);
    return (next != at_.end() && *next < hi) || (next != at_.begin() && next[-1] + bytes_ > lo);
  }
  // The same for n polynomials; p[i] may be the very polynomial own[i], an output.
  // Null entries (an operand that is not there) meet nothing.
  template <typename T, typename U = T>
  bool meet(const T *const *p, size_t n, U *const *own = nullptr) const {
    for (size_t i = 0; i < n; i++)
      if (p[i] && !(own && p[i] == own[i]) && meet(p[i], bytes_)) return true;
    return false;
  }

 private:
  size_t bytes_;
  std::vector<uintptr_t> at_;
};

}  // namespace cfhe
