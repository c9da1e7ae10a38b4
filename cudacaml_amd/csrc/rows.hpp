// Matrices of rows for the dropout, the norm block and the embedding:
// addressing, stores, dropout's parameters and the checks of arguments they
// share.
#pragma once

#include <cstdlib>

#include "../../include/cchip_operators.h"
#include "operators.hpp"

namespace cchip {
namespace op {

struct Rows {
  char *p;
  int64_t row;  // elements
};

template <typename T>
__device__ __forceinline__ T *row_at(const Rows &x, uint64_t row) {
  return reinterpret_cast<T *>(x.p) + int64_t(row) * x.row;
}

template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&x)[8], int n) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < 8; i++) r.x[i] = T(x[i]);
  if (n == 8) {
    const u32x4 *s = reinterpret_cast<const u32x4 *>(&r);
    u32x4_any *d = reinterpret_cast<u32x4_any *>(p);
#pragma unroll
    for (int i = 0; i < int(sizeof(T) * 8 / 16); i++) d[i] = s[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (i < n) p[i] = r.x[i];
  }
}

__device__ __forceinline__ uint64_t offset_of(const Drop &d) { return d.offset + (d.step ? *d.step : 0); }

// The kernel's form of a probability, seed and offset.
Drop drop_of(const char *who, double p, uint64_t seed, uint64_t offset, const uint64_t *step);

inline void check_rows_type(const char *who, int dtype) {
  if (dtype != CCHIP_F32 && dtype != CCHIP_BF16 && dtype != CCHIP_F16)
    throw InvalidArgument(strf("%s: dtype %d is not f32, bf16 or f16", who, dtype));
}

inline Rows rows_of(const char *who, const char *name, int dtype, int64_t rows, int64_t cols, const cchip_rows &x,
                    bool written, bool needed) {
  if (!x.data) {
    if (needed) throw InvalidArgument(strf("%s: no %s", who, name));
    return {nullptr, 0};
  }
  if (reinterpret_cast<uintptr_t>(x.data) % (dtype == CCHIP_F32 ? 4 : 2))
    throw InvalidArgument(strf("%s: %s is not aligned to its elements", who, name));
  if (written && rows > 1 && std::llabs(x.row) < cols) throw InvalidArgument(strf("%s: rows of %s overlap", who, name));
  return {static_cast<char *>(x.data), x.row};
}

// What a call reads and writes may lie in one place where each thread reads an
// element before it writes it: row for row. Any other overlap is refused, as
// far as the first rows show it.
inline void check_place(const char *who, int dtype, int64_t rows, int64_t cols, const char *out_name, const Rows &out,
                        const char *in_name, const Rows &in, bool in_place) {
  const size_t bytes = size_t(cols) * (dtype == CCHIP_F32 ? 4 : 2);
  if (!out.p || !in.p || !meet(out.p, bytes, in.p, bytes)) return;
  if (in_place && out.p == in.p && (rows == 1 || out.row == in.row)) return;
  throw InvalidArgument(strf("%s: %s is written over %s%s", who, out_name, in_name, in_place ? ", and not row for row" : ""));
}

template <typename F>
void with_rows_type(int dtype, F &&f) {
  if (dtype == CCHIP_F32) f(float());
  else if (dtype == CCHIP_F16) f(f16());
  else f(bf16());
}

}  // namespace op
}  // namespace cchip
