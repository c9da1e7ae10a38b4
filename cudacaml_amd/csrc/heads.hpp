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

// A tensor's counts along its axes.
struct HeadCounts {
  int64_t n[3];  // batch, tokens, heads
};

// Whether elements of one tensor lie in another's. Of tensors with other
// distances along an axis that both go along, which may lie between one
// another, the first heads are looked at. Otherwise heads of the two are as far
// apart as the tensors and a whole number of steps along each axis. Where a
// step is longer than all that the shorter ones reach together, as it is
// unless a tensor reads elements twice, the whole number nearest to what is
// left is the one, or one beside it.
inline bool heads_meet(int dim, int size, const HeadCounts &nx, const Heads &x, const HeadCounts &ny, const Heads &y) {
  const int64_t sx[] = {x.b, x.t, x.h}, sy[] = {y.b, y.t, y.h};
  int64_t step[3], least[3], most[3];
  int axes = 0;
  __int128 low = 0, high = 0;
  for (int i = 0; i < 3; i++) {
    if (nx.n[i] < 1 || ny.n[i] < 1) return false;
    if (nx.n[i] > 1 && ny.n[i] > 1 && sx[i] != sy[i]) return meet(x.p, size_t(dim) * size, y.p, size_t(dim) * size);
    const int64_t s = nx.n[i] > 1 ? sx[i] : sy[i];
    if ((nx.n[i] < 2 && ny.n[i] < 2) || s == 0) continue;
    int at = axes++;
    for (; at > 0 && std::llabs(step[at - 1]) < std::llabs(s); at--) step[at] = step[at - 1], least[at] = least[at - 1], most[at] = most[at - 1];
    step[at] = s, least[at] = 1 - ny.n[i], most[at] = nx.n[i] - 1;
    low += __int128(s) * (s > 0 ? least[at] : most[at]);
    high += __int128(s) * (s > 0 ? most[at] : least[at]);
  }
  const __int128 apart = (reinterpret_cast<intptr_t>(y.p) - reinterpret_cast<intptr_t>(x.p)) / size;
  if (apart <= low - dim || apart >= high + dim) return false;
  const auto among = [&](const auto &self, int axis, __int128 left) -> bool {
    if (axis == axes) return left < dim && left > -dim;
    const __int128 near = left / step[axis];
    for (int i = -1; i <= 1; i++)
      if (near + i >= least[axis] && near + i <= most[axis] && self(self, axis + 1, left - (near + i) * step[axis])) return true;
    return false;
  };
  return among(among, 0, apart);
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
