// Argument checks shared by the row collectives.
#ifndef ROCSHMEM_MI355X_ROWS_COMMON_HPP
#define ROCSHMEM_MI355X_ROWS_COMMON_HPP

#include <string>

#include "cabi_common.hpp"

namespace rsm {

// What the MI355X's last-level cache holds.
constexpr size_t kInfinityCacheBytes = 256u << 20;

// The members of a team, as the kernels address them: a symmetric pointer of PE 0 moved by `first`
// bytes is the first member's copy, and every further `step` bytes the next member's.
struct Members {
  int size;
  int64_t first, step;
};

// The symmetric operands of one call: every one has to lie in a live allocation, and none that the
// call writes may share bytes with another, unless the two are one array on purpose.  (A call of few
// rows takes the GPU about as long as the host: no allocation and no text here but for a refusal.)
class Operands {
 public:
  explicit Operands(const char *call) : call_(call) {}

  static constexpr int kNone = -1;   // no operand

  // rows x cols elements of `size` bytes, `ld` elements from row to row.  It may be the same array as the
  // operand `may_be`, added before it, each row of which is read before it is written.  Returns the
  // operand's number.
  int matrix(const void *p, const char *name, size_t rows, size_t cols, size_t ld, size_t size, bool written, int may_be = kNone) {
    return add(p, name, rows && cols ? ((rows - 1) * ld + cols) * size : 0, size, written, may_be);
  }
  // `bytes` bytes that begin at a multiple of `align`; no operand where `p` is NULL.
  int add(const void *p, const char *name, size_t bytes, size_t align, bool written, int may_be = kNone) {
    if (!p) return kNone;
    spans_[count_] = {static_cast<const char *>(p), bytes, align, name, written, may_be};
    return count_++;
  }

  bool ok() const {
    const auto *rt = rocshmem::host::Runtime::get();
    for (int i = 0; i < count_; ++i) {
      const Span &s = spans_[i];
      const size_t offset = static_cast<size_t>(s.p - rt->arena());
      if (s.p >= rt->arena() && offset < rt->slice_stride()) {
        const size_t end = rt->allocation_end(offset);
        if (end != rocshmem::host::Pow2Allocator::kNoOffset && s.bytes <= end - offset && offset % s.align == 0) continue;
      }
      const std::string what = std::string(call_) + ": " + s.name;
      if (check_symmetric(s.p, what.c_str()) && check_extent(s.p, s.bytes, what.c_str())) fail(what + " is not aligned to " + std::to_string(s.align) + " bytes");
      return false;
    }
    return disjoint();
  }

  // No operand that is written shares bytes with another but the one that it may be: with that operand, not
  // with its array, which may serve as a further operand that is read in another order.
  bool disjoint() const {
    for (int i = 0; i < count_; ++i)
      for (int j = 0; j < i; ++j) {
        const Span &a = spans_[i], &b = spans_[j];
        if (!(a.written || b.written) || !(a.p < b.p + b.bytes && b.p < a.p + a.bytes)) continue;
        if (a.p == b.p && a.may_be == j) continue;
        fail(std::string(call_) + ": " + a.name + " and " + b.name + " overlap");
        return false;
      }
    return true;
  }

 private:
  struct Span {
    const char *p;
    size_t bytes, align;
    const char *name;
    bool written;
    int may_be;
  };
  static constexpr int kMost = 16;   // no call has more operands
  const char *call_;
  Span spans_[kMost];
  int count_ = 0;
};

// False, with the error set, when `team` is none; otherwise its members.
inline bool members_of(uint64_t team, const char *call, Members *out) {
  rocshmem::host::Runtime *rt = rocshmem::host::Runtime::get();
  if (!rt) {
    fail("rsm_init has not been called");
    return false;
  }
  const auto *rec = rt->team_record(reinterpret_cast<rocshmem::detail::Team *>(team));
  if (!rec) {
    fail(std::string(call) + ": invalid team");
    return false;
  }
  const auto &t = rec->image.wrt_world;
  const int64_t stride = static_cast<int64_t>(rt->slice_stride());
  *out = {t.size, t.pe_start * stride, t.stride * stride};
  return true;
}

}  // namespace rsm

#endif
