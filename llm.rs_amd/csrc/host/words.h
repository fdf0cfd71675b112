// words.h - small host arrays for a launch: in its own arguments where they fit,
// else in device memory filled by launches that carry them in theirs.  Either way
// the call returns without waiting and nothing of the caller's is read later.
#pragma once
#include <algorithm>
#include <vector>

#include "../kernel_args.h"
#include "internal.h"

namespace llmrs {

// Device memory from the caching allocator, given back at the end of the scope:
// reuse follows in stream order.
struct Scratch {
  void* p = nullptr;
  explicit Scratch(size_t bytes) : p(bytes ? ctx().alloc.alloc(bytes) : nullptr) {}
  Scratch(const Scratch&) = delete;
  Scratch& operator=(const Scratch&) = delete;
  ~Scratch() {
    if (p) ctx().alloc.release(p);
  }
};

// `n` words to device memory, in stream order.
inline void set_words(int* dst, const int* w, size_t n) {
  for (size_t i = 0; i < n; i += kPagedWords) {
    WordsArgs a;
    a.dst = dst + i;
    a.n = (int)std::min<size_t>(kPagedWords, n - i);
    std::copy(w + i, w + i + a.n, a.w);
    launch("paged_words", dim3(1), dim3(256), 0, ctx().stream, a);
  }
}

// Puts `w` into a launch's `inl` words or into device memory; the address for its
// `ext` (null: inl).  Lives until the launch is queued.
class LaunchWords {
 public:
  LaunchWords(const std::vector<int>& w, int* inl) : mem_(w.size() <= (size_t)kPagedWords ? 0 : 4 * w.size()) {
    if (mem_.p) set_words((int*)mem_.p, w.data(), w.size());
    else std::copy(w.begin(), w.end(), inl);
  }
  const int* ext() const { return (const int*)mem_.p; }

 private:
  Scratch mem_;
};

}  // namespace llmrs
