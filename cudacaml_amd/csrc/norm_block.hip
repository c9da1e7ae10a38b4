// The norm block: entry points, checks, and the sum over workgroups that
// ends the parameters' gradients.

#include "norm_block.hpp"

#include <cmath>
#include <utility>

namespace cchip {
namespace op {

extern template void norm_forward_launch<bf16>(const NormArgs &, hipStream_t);
extern template void norm_forward_launch<f16>(const NormArgs &, hipStream_t);
extern template void norm_forward_launch<float>(const NormArgs &, hipStream_t);
extern template void norm_backward_launch<bf16>(const NormArgs &, bool, int, hipStream_t);
extern template void norm_backward_launch<f16>(const NormArgs &, bool, int, hipStream_t);
extern template void norm_backward_launch<float>(const NormArgs &, bool, int, hipStream_t);

namespace {

struct ColumnArgs {
  const float *partial;
  void *to[kParams];
  int groups, sums, width;
  bool f32;
};

// 32 columns of one parameter a workgroup; 32 threads a column each sum
// every 32nd workgroup's share, and one of them those 32, in order.
template <typename T>
__global__ __launch_bounds__(1024) void norm_columns(const ColumnArgs a) {
  __shared__ float part[32][33];
  const int col = threadIdx.x % 32, turn = threadIdx.x / 32, s = blockIdx.y;
  const int c = int(blockIdx.x) * 32 + col;
  if (!a.to[s]) return;
  float q = 0.0f;
  if (c < a.width) {
#pragma unroll 8
    for (int g = turn; g < a.groups; g += 32) q += a.partial[(int64_t(g) * a.sums + s) * a.width + c];
  }
  part[turn][col] = q;
  __syncthreads();
  if (turn || c >= a.width) return;
  float x = 0.0f;
#pragma unroll
  for (int i = 0; i < 32; i++) x += part[i][col];
  if (a.f32) static_cast<float *>(a.to[s])[c] = x;
  else static_cast<T *>(a.to[s])[c] = T(x);
}

void check_op(const cchip_norm_block *op) {
  const char *who = "norm block";
  if (!op) throw InvalidArgument("norm block: no descriptor");
  check_rows_type(who, op->dtype);
  if (op->weight_dtype != op->dtype && op->weight_dtype != CCHIP_F32)
    throw InvalidArgument("norm block: parameters are of the operator's dtype or f32");
  if (op->rows < 0 || op->rows >= (int64_t(1) << 32)) throw InvalidArgument("norm block: rows are below 2^32");
  if (op->width < 1 || op->width > 32768)
    throw InvalidArgument(strf("norm block: width %lld is not in 1 .. 32768", (long long)op->width));
  for (int kind : {op->post, op->pre})
    if (kind != CCHIP_NORM_NONE && kind != CCHIP_NORM_RMS && kind != CCHIP_NORM_LAYER)
      throw InvalidArgument(strf("norm block: unknown norm %d", kind));
  if (op->gate != CCHIP_GATE_NONE && op->gate != CCHIP_GATE_SIGMOID && op->gate != CCHIP_GATE_SILU)
    throw InvalidArgument(strf("norm block: unknown gate %d", op->gate));
  if (!(op->p >= 0.0 && op->p <= 1.0)) throw InvalidArgument(strf("norm block: p = %g is not in 0 .. 1", op->p));
  if (!std::isfinite(op->scale) || !(op->eps >= 0.0f) || !std::isfinite(op->eps))
    throw InvalidArgument("norm block: scale is finite and eps finite and not negative");
}

NormArgs args_of(const cchip_norm_block &op, const cchip_norm_block_io *io) {
  if (!io) throw InvalidArgument("norm block: no tensors");
  NormArgs a = {};
  a.rows = uint32_t(op.rows);
  a.width = int(op.width);
  a.post = op.post;
  a.pre = op.pre;
  a.act = op.gate;
  a.scale = op.scale;
  a.eps = op.eps;
  a.weights_f32 = op.weight_dtype == CCHIP_F32;
  a.drop = drop_of("norm block", op.p, io->seed, io->offset, io->step);
  a.post_weight = io->params.post_weight;
  a.post_bias = io->params.post_bias;
  a.channel_scale = io->params.channel_scale;
  a.pre_weight = io->params.pre_weight;
  a.pre_bias = io->params.pre_bias;
  for (const void *p : {a.post_weight, a.post_bias, a.channel_scale, a.pre_weight, a.pre_bias})
    if (reinterpret_cast<uintptr_t>(p) % (a.weights_f32 ? 4 : 2))
      throw InvalidArgument("norm block: a parameter is not aligned to its elements");
  if (op.post == CCHIP_NORM_NONE && (a.post_weight || a.post_bias))
    throw InvalidArgument("norm block: parameters of a post norm that there is not");
  if (op.pre == CCHIP_NORM_NONE && (a.pre_weight || a.pre_bias))
    throw InvalidArgument("norm block: parameters of a pre norm that there is not");
  return a;
}

bool wide(const cchip_norm_block &op) { return op.width > 8192; }

// A backward pass leaves a workgroup's sums in memory: of 4 rows at least,
// so that they stay small beside the rows. Those of wide rows are of 2048
// columns each, four to a unit.
int backward_groups(const cchip_norm_block &op, bool bias) {
  if (wide(op)) return int(std::min<int64_t>((op.rows + 3) / 4, 1024 / ((op.width + 2047) / 2048)));
  int waves = 0;
  with_shape(int(op.width), [&](auto lanes, auto) {
    waves = waves_of(decltype(lanes)::value, op.gate != CCHIP_GATE_NONE, op.pre != CCHIP_NORM_NONE, bias);
  });
  return groups_of(op.rows, int(op.width), waves, 4);
}

// Sums of each workgroup, and wide rows' statistics after them.
size_t workspace_of(const cchip_norm_block &op, bool bias) {
  return size_t(backward_groups(op, bias)) * (bias ? 5 : 3) * op.width * sizeof(float) + (wide(op) ? size_t(op.rows) * sizeof(RowStat) : 0);
}

}  // namespace

int groups_of(int64_t rows, int width, int waves, int least) {
  const int64_t at_a_time = rows_at_a_time(width), sets = (rows + at_a_time - 1) / at_a_time;
  const int64_t most = 256 * (waves * 256 / threads_of(width));
  const int64_t each = std::max<int64_t>(least, (sets + most - 1) / most);
  return int((sets + each - 1) / each);
}

}  // namespace op
}  // namespace cchip

using namespace cchip;
using namespace cchip::op;

extern "C" {

int cchip_norm_block_forward(const cchip_norm_block *op, const cchip_norm_block_io *io, void *stream) {
  return guarded([&] {
    const char *who = "norm block";
    check_op(op);
    NormArgs a = args_of(*op, io);
    const bool pre = op->pre != CCHIP_NORM_NONE, gated = op->gate != CCHIP_GATE_NONE;
    if (op->rows == 0) return;
    if (pre != (io->n.data != nullptr)) throw InvalidArgument("norm block: n is given if and only if there is a pre norm");
    if (gated != (io->gate.data != nullptr)) throw InvalidArgument("norm block: a gate is given if and only if the operator has one");
    a.y = rows_of(who, "y", op->dtype, op->rows, op->width, io->y, false, true);
    a.gate = rows_of(who, "gate", op->dtype, op->rows, op->width, io->gate, false, false);
    a.residual = rows_of(who, "residual", op->dtype, op->rows, op->width, io->residual, false, false);
    a.h = rows_of(who, "h", op->dtype, op->rows, op->width, io->h, true, true);
    a.n = rows_of(who, "n", op->dtype, op->rows, op->width, io->n, true, false);
    const std::pair<const char *, const Rows &> in[] = {{"y", a.y}, {"gate", a.gate}, {"residual", a.residual}};
    for (auto &i : in) {
      check_place(who, op->dtype, op->rows, op->width, "h", a.h, i.first, i.second, true);
      check_place(who, op->dtype, op->rows, op->width, "n", a.n, i.first, i.second, true);
    }
    check_place(who, op->dtype, op->rows, op->width, "n", a.n, "h", a.h, false);
    with_rows_type(op->dtype, [&](auto t) { norm_forward_launch<decltype(t)>(a, (hipStream_t)stream); });
    check_launch(who);
  });
}

int cchip_norm_block_workspace(const cchip_norm_block *op, size_t *bytes) {
  return guarded([&] {
    check_op(op);
    if (bytes) *bytes = std::max(workspace_of(*op, false), workspace_of(*op, true));
  });
}

int cchip_norm_block_backward(const cchip_norm_block *op, const cchip_norm_block_io *io, void *workspace,
                              size_t workspace_bytes, void *stream) {
  return guarded([&] {
    const char *who = "norm block";
    check_op(op);
    NormArgs a = args_of(*op, io);
    const bool pre = op->pre != CCHIP_NORM_NONE, gated = op->gate != CCHIP_GATE_NONE;
    ColumnArgs c = {};
    c.to[kPostWeight] = io->grads.post_weight;
    c.to[kChannelScale] = io->grads.channel_scale;
    c.to[kPreWeight] = io->grads.pre_weight;
    c.to[kPostBias] = io->grads.post_bias;
    c.to[kPreBias] = io->grads.pre_bias;
    bool any = false;
    for (void *p : c.to) {
      any = any || p;
      if (reinterpret_cast<uintptr_t>(p) % (a.weights_f32 ? 4 : 2))
        throw InvalidArgument("norm block: a parameter's gradient is not aligned to its elements");
    }
    if ((c.to[kPostWeight] || c.to[kPostBias]) && op->post == CCHIP_NORM_NONE)
      throw InvalidArgument("norm block: gradients of a post norm that there is not");
    if ((c.to[kPreWeight] || c.to[kPreBias]) && !pre) throw InvalidArgument("norm block: gradients of a pre norm that there is not");
    const bool bias = c.to[kPostBias] || c.to[kPreBias] || a.post_bias;
    if (op->rows > 0) {
      if (pre != (io->dn.data != nullptr) || pre != (io->h.data != nullptr))
        throw InvalidArgument("norm block: h and dn are given if and only if there is a pre norm");
      if (gated != (io->gate.data != nullptr)) throw InvalidArgument("norm block: a gate is given if and only if the operator has one");
      if (!gated && io->dgate.data) throw InvalidArgument("norm block: the gradient of a gate that there is not");
      a.y = rows_of(who, "y", op->dtype, op->rows, op->width, io->y, false, true);
      a.gate = rows_of(who, "gate", op->dtype, op->rows, op->width, io->gate, false, false);
      a.h = rows_of(who, "h", op->dtype, op->rows, op->width, io->h, false, false);
      a.dh = rows_of(who, "dh", op->dtype, op->rows, op->width, io->dh, false, true);
      a.dn = rows_of(who, "dn", op->dtype, op->rows, op->width, io->dn, false, false);
      a.dy = rows_of(who, "dy", op->dtype, op->rows, op->width, io->dy, true, true);
      a.dgate = rows_of(who, "dgate", op->dtype, op->rows, op->width, io->dgate, true, false);
      a.dresidual = rows_of(who, "dresidual", op->dtype, op->rows, op->width, io->dresidual, true, false);
      // norm_sums reads its inputs after the others are written
      const std::pair<const char *, const Rows &> out[] = {{"dy", a.dy}, {"dgate", a.dgate}, {"dresidual", a.dresidual}},
                                                  in[] = {{"y", a.y}, {"gate", a.gate}, {"h", a.h}, {"dh", a.dh}, {"dn", a.dn}};
      for (auto &o : out) {
        for (auto &i : in) check_place(who, op->dtype, op->rows, op->width, o.first, o.second, i.first, i.second, false);
        for (auto *other = out; other != &o; other++)
          check_place(who, op->dtype, op->rows, op->width, o.first, o.second, other->first, other->second, false);
      }
    }
    const int groups = backward_groups(*op, bias);
    if (any) {
      const size_t need = workspace_of(*op, bias);
      if (workspace_bytes < need || (need && !workspace) || reinterpret_cast<uintptr_t>(workspace) % 4)
        throw InvalidArgument(strf("norm block: the workspace needs %zu bytes aligned to 4, has %zu", need, workspace ? workspace_bytes : 0));
      a.partial = static_cast<float *>(workspace);
      a.stats = reinterpret_cast<RowStat *>(a.partial + size_t(groups) * (bias ? 5 : 3) * op->width);
    }
    if (groups)
      with_rows_type(op->dtype, [&](auto t) { norm_backward_launch<decltype(t)>(a, bias, groups, (hipStream_t)stream); });
    check_launch(who);
    if (!any) return;
    c.partial = a.partial;
    c.groups = groups;
    c.sums = bias ? 5 : 3;
    c.width = a.width;
    c.f32 = a.weights_f32;
    with_rows_type(op->dtype, [&](auto t) {
      typedef decltype(t) T;
      hipLaunchKernelGGL((norm_columns<T>), dim3((a.width + 31) / 32, c.sums), dim3(1024), 0, (hipStream_t)stream, c);
    });
    check_launch(who);
  });
}

}  // extern "C"
