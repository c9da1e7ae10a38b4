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
  uint64_t per_row;  // groups a row, up to 2^32
  int64_t cols;
  float scale;
  Drop drop;
};

// A thread a group of 8 columns. One call of the generator serves all 8, at
// 16 bits each: its ten rounds are 20 32-bit multiplications at a quarter of
// the vector rate, 2.5 for each value, and 32 bits each would make it the
// arithmetic and not the memory that bounds a 16-bit dropout. 16384 x 8192
// bf16 onto a residual and the gradient back, 1.34 GB, take 227 us: 5.9 TB/s,
// over a copy's 4.9 as the second finds some of its input in the cache.
template <typename T>
__global__ __launch_bounds__(256) void dropout(const DropoutArgs a) {
  const uint64_t i = uint64_t(block_index()) * 256 + threadIdx.x;
  if (i >= a.groups) return;
  const uint64_t row = a.groups <= 0xFFFFFFFFu ? uint32_t(i) / uint32_t(a.per_row) : i / a.per_row;
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

Drop drop_of(const char *who, double p, uint64_t seed, uint64_t offset, const uint64_t *step) {
  if (!(p >= 0.0 && p <= 1.0)) throw InvalidArgument(strf("%s: p = %g is not in 0 .. 1", who, p));
  if (reinterpret_cast<uintptr_t>(step) % 8) throw InvalidArgument(strf("%s: step is not aligned to its 8 bytes", who));
  const uint32_t bar = uint32_t(std::nearbyint(p * 65536.0));
  return {seed, offset, step, bar, bar >= 65536 ? 0.0f : float(65536.0 / (65536 - bar))};
}

}  // namespace op
}  // namespace cchip

using namespace cchip;
using namespace cchip::op;

extern "C" int cchip_dropout_run(const cchip_dropout *op, const cchip_dropout_io *io, void *stream) {
  return guarded([&] {
    const char *who = "dropout";
    if (!op || !io) throw InvalidArgument("dropout: no descriptor or tensors");
    check_rows_type(who, op->dtype);
    if (op->rows < 0 || op->cols < 0 || op->rows >= (int64_t(1) << 32) || op->cols >= (int64_t(1) << 35))
      throw InvalidArgument("dropout: rows are below 2^32 and columns below 2^35");
    if (!std::isfinite(op->scale)) throw InvalidArgument("dropout: scale is not finite");
    DropoutArgs a = {};
    a.drop = drop_of(who, op->p, io->seed, io->offset, io->step);
    if (op->rows == 0 || op->cols == 0) return;
    a.x = rows_of(who, "x", op->dtype, op->rows, op->cols, io->x, false, true);
    a.residual = rows_of(who, "residual", op->dtype, op->rows, op->cols, io->residual, false, false);
    a.out = rows_of(who, "out", op->dtype, op->rows, op->cols, io->out, true, true);
    check_place(who, op->dtype, op->rows, op->cols, "out", a.out, "x", a.x, true);
    check_place(who, op->dtype, op->rows, op->cols, "out", a.out, "residual", a.residual, true);
    a.per_row = uint64_t(op->cols + 7) / 8;
    if (a.per_row > (uint64_t(1) << 39) / uint64_t(op->rows)) throw InvalidArgument("dropout: more than 2^42 elements");
    a.groups = uint64_t(op->rows) * a.per_row;
    a.cols = op->cols;
    a.scale = op->scale;
    with_rows_type(op->dtype, [&](auto t) {
      typedef decltype(t) T;
      hipLaunchKernelGGL((dropout<T>), grid_of(int64_t((a.groups + 255) / 256)), dim3(256), 0, (hipStream_t)stream, a);
    });
    check_launch("dropout");
  });
}
