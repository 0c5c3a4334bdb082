// What the row collectives' check of operands takes for an overlap: addresses alone, no GPU.
// Prints one line per case that comes out wrong, and "ok" when there is none.
#include <cstdio>

#include "cabi/rows_common.hpp"

namespace {

int wrong = 0;
char arena[1 << 16];
char *const x = arena, *const y = arena + 4096, *const z = arena + 8192;

// A 4 x 8 matrix of floats at `p`; `same`: the array that it may be.
void put(rsm::Operands &o, const void *p, const char *name, bool written, const void *same = nullptr) {
  o.matrix(p, name, 4, 8, 8, 4, written, same);
}

void expect(const char *what, const rsm::Operands &o, bool disjoint) {
  if (o.disjoint() == disjoint) return;
  std::printf("%s: %s\n", what, disjoint ? "refused" : "let through");
  ++wrong;
}

}  // namespace

int main() {
  {
    rsm::Operands o("apart");
    put(o, x, "source", false);
    put(o, y, "residual", false);
    put(o, z, "residual_out", true, y);
    expect("arrays of their own", o, true);
  }
  {
    rsm::Operands o("in place");
    put(o, x, "source", false);
    put(o, y, "residual", false);
    put(o, y, "residual_out", true, y);
    put(o, x, "normed", true, x);
    expect("results in place of their operands", o, true);
  }
  {
    rsm::Operands o("shifted");
    put(o, x, "source", false);
    put(o, x + 16, "normed", true, x);
    expect("a result that begins inside its operand", o, false);
  }
  {
    rsm::Operands o("null");
    put(o, x, "source", false);
    put(o, y, "residual", false);
    put(o, x, "residual_out", true, y);
    put(o, nullptr, "normed", true, x);
    expect("another result over an operand that an absent one may replace", o, false);
  }
  {
    rsm::Operands o("null first");
    put(o, x, "grad_residual_out", false);
    put(o, x, "grad_source", true);
    put(o, nullptr, "grad_residual", true, x);
    expect("the same of a result without an operand of its own", o, false);
  }
  if (!wrong) std::printf("ok\n");
  return wrong != 0;
}
