// Dropout whose mask is drawn from the counter-based generator each time it
// is needed and never stored.

#include "../../include/cchip_operators.h"
#include "operators.hpp"
#include "rows.hpp"

#include <cmath>

namespace cchip {
namespace op {
namespace {

struct DropoutArgs {
  Rows x, residual, out;
  uint64_t groups;   // rows times groups of 8 columns
  uint32_t per_row;  // groups a row
  int64_t cols;
  float scale;
  Drop drop;
};

// A thread a group of 8 columns. One call of the generator serves all 8, at
// 16 bits each: its ten rounds are 20 32-bit multiplications at a quarter of
// the vector rate, 2.5 for each value, and 32 bits each would make it the
// arithmetic and not the memory that bounds a 16-bit dropout.
template <typename T>
__global__ __launch_bounds__(256) void dropout(const DropoutArgs a) {
  const uint64_t i = uint64_t(blockIdx.x) * 256 + threadIdx.x;
  if (i >= a.groups) return;
  const uint64_t row = a.groups <= 0xFFFFFFFFu ? uint32_t(i) / a.per_row : i / a.per_row;
  const uint32_t group = uint32_t(i - row * a.per_row);
  const int64_t col = int64_t(group) * 8;
  const int n = a.cols - col > 8 ? 8 : int(a.cols - col);
  const Raw8<T> x = load8<T>(row_at<T>(a.x, row) + col, n);
  const bool add = a.residual.p != nullptr;
  Raw8<T> r = {};
  if (add) r = load8<T>(row_at<T>(a.residual, row) + col, n);
  const uint32_t bits = a.drop.bar ? keep_bits(a.drop, offset_of(a.drop), uint32_t(row), group) : 0xFFu;
  const float up = a.scale * a.drop.up;
  float out[8];
#pragma unroll
  for (int j = 0; j < 8; j++) out[j] = (bits >> j & 1 ? up * float(x.x[j]) : 0.0f) + (add ? float(r.x[j]) : 0.0f);
  store8<T>(row_at<T>(a.out, row) + col, out, n);
}

}  // namespace

Drop drop_of(const cchip_drop *d) {
  if (!d) return {0, 0, nullptr, 0, 1.0f};
  if (!(d->p >= 0.0 && d->p <= 1.0)) throw InvalidArgument(strf("dropout: p = %g is not in 0 .. 1", d->p));
  const uint32_t bar = uint32_t(std::nearbyint(d->p * 65536.0));
  return {d->seed, d->offset, d->step, bar, bar >= 65536 ? 0.0f : float(65536.0 / (65536 - bar))};
}

}  // namespace op
}  // namespace cchip

using namespace cchip;
using namespace cchip::op;

extern "C" int cchip_dropout(int dtype, int64_t rows, int64_t cols, const cchip_drop *drop, float scale, cchip_rows x,
                             cchip_rows residual, cchip_rows out, void *stream) {
  return guarded([&] {
    const char *who = "dropout";
    check_rows_type(who, dtype);
    if (!drop) throw InvalidArgument("dropout: no probability and seed");
    if (rows < 0 || cols < 0 || rows >= (int64_t(1) << 32) || cols >= (int64_t(1) << 35))
      throw InvalidArgument("dropout: rows are below 2^32 and columns below 2^35");
    if (!std::isfinite(scale)) throw InvalidArgument("dropout: scale is not finite");
    DropoutArgs a = {};
    a.drop = drop_of(drop);
    if (rows == 0 || cols == 0) return;
    a.x = rows_of(who, "x", dtype, rows, cols, x, false, true);
    a.residual = rows_of(who, "residual", dtype, rows, cols, residual, false, false);
    a.out = rows_of(who, "out", dtype, rows, cols, out, true, true);
    a.per_row = uint32_t((cols + 7) / 8);
    a.groups = uint64_t(rows) * a.per_row;
    if ((a.groups + 255) / 256 > uint64_t(INT32_MAX)) throw InvalidArgument("dropout: more elements than a launch can have");
    a.cols = cols;
    a.scale = scale;
    with_rows_type(dtype, [&](auto t) {
      typedef decltype(t) T;
      hipLaunchKernelGGL((dropout<T>), dim3(unsigned((a.groups + 255) / 256)), dim3(256), 0, (hipStream_t)stream, a);
    });
    check_launch("dropout");
  });
}
