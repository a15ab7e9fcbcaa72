// Which of many tensors' bytes overlap (host code of tgx_clip.hip and tgx_adamw.hip).
#pragma once

#include <algorithm>
#include <cstdint>

namespace tgx {
namespace {

struct Range {
  uint64_t lo, hi;
  int64_t tensor;
  bool out;  // written
};

// whether bytes of a range that is written lie in another one; then the tensors of the two,
// the smaller first.  Sorts r.
bool overlap(Range* r, int64_t n, int64_t& one, int64_t& other) {
  std::sort(r, r + n, [](const Range& x, const Range& y) { return x.lo < y.lo; });
  const Range *any = nullptr, *out = nullptr;  // of those before, the one that reaches farthest
  for (int64_t i = 0; i < n; ++i) {
    const Range* before = r[i].out ? any : out;
    if (before != nullptr && before->hi > r[i].lo) {
      one = std::min(before->tensor, r[i].tensor);
      other = std::max(before->tensor, r[i].tensor);
      return true;
    }
    if (any == nullptr || r[i].hi > any->hi) any = &r[i];
    if (r[i].out && (out == nullptr || r[i].hi > out->hi)) out = &r[i];
  }
  return false;
}

}  // namespace
}  // namespace tgx
