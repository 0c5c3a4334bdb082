// What the row collectives' check of operands takes for an overlap: addresses alone, no GPU.
// Prints one line per case that comes out wrong, and "ok" when there is none.
#include <cstdio>

#include "cabi/rows_common.hpp"

namespace {

int wrong = 0;
char arena[1 << 16];
char *const x = arena, *const y = arena + 4096, *const z = arena + 8192;

// A 4 x 8 matrix of floats at `p`; `may_be`: the operand that it may share its array with.
int put(rsm::Operands &o, const void *p, const char *name, bool written, int may_be = rsm::Operands::kNone) {
  return o.matrix(p, name, 4, 8, 8, 4, written, may_be);
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
    const int residual = put(o, y, "residual", false);
    put(o, z, "residual_out", true, residual);
    expect("arrays of their own", o, true);
  }
  {
    rsm::Operands o("in place");
    const int source = put(o, x, "source", false), residual = put(o, y, "residual", false);
    put(o, y, "residual_out", true, residual);
    put(o, x, "normed", true, source);
    expect("results in place of their operands", o, true);
  }
  {
    rsm::Operands o("shifted");
    const int source = put(o, x, "source", false);
    put(o, x + 16, "normed", true, source);
    expect("a result that begins inside its operand", o, false);
  }
  {
    rsm::Operands o("null");
    const int source = put(o, x, "source", false), residual = put(o, y, "residual", false);
    put(o, x, "residual_out", true, residual);
    put(o, nullptr, "normed", true, source);
    expect("another result over an operand that an absent one may replace", o, false);
  }
  {
    rsm::Operands o("null first");
    const int grad_residual_out = put(o, x, "grad_residual_out", false);
    put(o, x, "grad_source", true);
    put(o, nullptr, "grad_residual", true, grad_residual_out);
    expect("the same of a result without an operand of its own", o, false);
  }
  {
    rsm::Operands o("chain");
    put(o, x, "source", false);
    const int residual = put(o, x, "residual", false);
    expect("one array read twice", o, true);
    put(o, x, "residual_out", true, residual);
    expect("a result in place of an operand whose array is read as another one too", o, false);
  }
  {
    rsm::Operands o("chain of the first");
    const int source = put(o, x, "source", false);
    put(o, x, "residual", false);
    put(o, x, "normed", true, source);
    expect("the same of the operand added first", o, false);
  }
  {
    rsm::Operands o("absent operand");
    const int grad_normed = put(o, nullptr, "grad_normed", false);
    put(o, x, "grad_source", true, grad_normed);
    put(o, x, "grad_residual_out", false);
    expect("a result whose own operand is absent", o, false);
  }
  if (!wrong) std::printf("ok\n");
  return wrong != 0;
}
