// Tensors [batch][token][head][dim] of the layer operators: addressing and
// the checks of arguments they share.
#pragma once

#include <cstdlib>

#include "../../include/cchip_operators.h"
#include "operators.hpp"

namespace cchip {
namespace op {

struct Heads {
  char *p;  // elements of the operator's type
  int64_t b, t, h;
};

// Whether two heads' elements of a tensor share a place, as far as one step
// along an axis, or one and some along another, shows it.
inline bool heads_overlap(int64_t batch, int64_t tokens, const cchip_heads &x, int heads, int dim) {
  const int64_t count[] = {batch, tokens, heads}, step[] = {std::llabs(x.batch), std::llabs(x.token), std::llabs(x.head)};
  for (int i = 0; i < 3; i++) {
    if (count[i] < 2) continue;
    if (step[i] < dim) return true;
    for (int j = 0; j < 3; j++) {
      if (i == j || count[j] < 2 || step[j] < dim || step[j] > step[i]) continue;
      const int64_t n = step[i] / step[j], over = step[i] % step[j];
      if ((over < dim && n < count[j]) || (step[j] - over < dim && n + 1 < count[j])) return true;
    }
  }
  return false;
}

// What a kernel takes of an operator's tensor. The distance of tokens is
// bounded so that a kernel may count the elements of some hundred of them in
// 32 bits.
inline Heads heads_of(const char *who, const char *name, int dtype, int64_t batch, int64_t tokens, int heads, int dim,
                      const cchip_heads &x, bool written) {
  if (batch * tokens == 0) return {static_cast<char *>(x.data), x.batch, x.token, x.head};
  if (!x.data) throw InvalidArgument(strf("%s: no %s", who, name));
  if (reinterpret_cast<uintptr_t>(x.data) % (dtype == CCHIP_F32 ? 4 : 2))
    throw InvalidArgument(strf("%s: %s is not aligned to its elements", who, name));
  if (x.token < 0 || x.token > (int64_t(1) << 23))
    throw InvalidArgument(strf("%s: tokens of %s are not 0 to 2^23 elements apart", who, name));
  if (written && heads_overlap(batch, tokens, x, heads, dim)) throw InvalidArgument(strf("%s: elements of %s overlap", who, name));
  return {static_cast<char *>(x.data), x.batch, x.token, x.head};
}

}  // namespace op
}  // namespace cchip
