// Whether the outputs of a call are memory of their own. Blocks write them in any
// order while others still read operands, so an output that lies in another one or in
// an operand would leave words that depend on that order. Host only.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include <algorithm>
#include <initializer_list>
#include <vector>

namespace cfhe {

// The polynomials that a call writes, each `bytes` long. Usually they are one tensor
// and the operands others: then a test is a comparison or two, and the addresses are
// in order as they come (260 outputs and as many operands: 1.5 us of the host's time,
// sorted from scratch 4.2). Otherwise their ascending runs are merged.
class Outputs {
 public:
  explicit Outputs(size_t bytes) : bytes_{bytes} {}
  // n outputs of several polynomials each, parts[k][i] part k of output i
  template <typename T>
  void add(std::initializer_list<T *const *> parts, size_t n) {
    at_.reserve(at_.size() + parts.size() * n);
    for (size_t i = 0; i < n; i++)
      for (T *const *p : parts) at_.push_back(reinterpret_cast<uintptr_t>(p[i]));
  }
  // After the last add(): false if two of them overlap
  bool apart() {
    std::vector<size_t> runs = {0};  // where they begin
    for (size_t i = 1; i < at_.size(); i++)
      if (at_[i] < at_[i - 1]) runs.push_back(i);
    runs.push_back(at_.size());
    while (runs.size() > 2) {  // neighbours in pairs
      std::vector<size_t> longer = {0};
      for (size_t r = 0; r + 2 < runs.size(); r += 2) {
        std::inplace_merge(at_.begin() + runs[r], at_.begin() + runs[r + 1], at_.begin() + runs[r + 2]);
        longer.push_back(runs[r + 2]);
      }
      if (longer.back() != at_.size()) longer.push_back(at_.size());
      runs.swap(longer);
    }
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
