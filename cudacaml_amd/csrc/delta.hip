// Gated delta rule: the entry points of cchip_operators.h, their checks, and
// where a call's buffers lie in `saved` and the workspace.

#include "delta.hpp"

#include <cmath>
#include <utility>

using namespace cchip;
using namespace cchip::op;

namespace {

// Up to this many tokens a sequence the recurrence runs token by token, which
// grows with them while a chunk costs the same for 1 token and 64: 8 x 16
// heads of 128 x 128 take 17.6 us for 8 tokens, 30.2 for 16 and 55.9 for 32,
// the chunk's kernels 31; 256 x 32 heads 619 us for 8, 1085 for 16, the
// chunk's 1268.
constexpr int64_t kStepTokens = 16;

struct Layout {
  int64_t slots, slot_heads;
  size_t record, record_back, states, us, scales, powers, o_powers, dots;  // bytes, all slots and heads
};

void check_op(const cchip_gated_delta *op) {
  if (!op) throw InvalidArgument("gated delta: no descriptor");
  if (op->dtype != CCHIP_F32 && op->dtype != CCHIP_BF16 && op->dtype != CCHIP_F16)
    throw InvalidArgument(strf("gated delta: dtype %d is not f32, bf16 or f16", op->dtype));
  if (op->batch < 0 || op->tokens < 0 || op->sequences < 0 || op->tokens > (int64_t(1) << 31) - 64)
    throw InvalidArgument("gated delta: batch, tokens and sequences are not negative and tokens below 2^31 - 64");
  if (op->sequences > 0 && op->batch != 1) throw InvalidArgument("gated delta: packed sequences have a batch of 1");
  if (op->key_heads < 1 || op->value_heads < 1 || op->value_heads % op->key_heads)
    throw InvalidArgument(strf("gated delta: %d value heads are not a multiple of %d key heads", op->value_heads, op->key_heads));
  if (op->key_dim < 1 || op->key_dim > 128) throw InvalidArgument(strf("gated delta: key_dim %d is not in 1 .. 128", op->key_dim));
  if (op->value_dim < 1 || op->value_dim > 4096)
    throw InvalidArgument(strf("gated delta: value_dim %d is not in 1 .. 4096", op->value_dim));
  if (!std::isfinite(op->scale)) throw InvalidArgument("gated delta: scale is not finite");
}

int64_t count_sequences(const cchip_gated_delta &op) { return op.sequences ? op.sequences : op.batch; }

int padded_value_dim(const cchip_gated_delta &op) { return (op.value_dim + 31) / 32 * 32; }

Layout layout_of(const cchip_gated_delta &op) {
  Layout p;
  // batch and sequences below 2^31 and heads of all of them too, so nothing here overflows
  if (op.batch >= (int64_t(1) << 31) || op.sequences >= (int64_t(1) << 31) || count_sequences(op) * op.value_heads > INT32_MAX)
    throw InvalidArgument("gated delta: too many sequences and heads for a launch");
  p.slots = op.sequences ? op.tokens / kChunk + op.sequences : op.batch * ((op.tokens + kChunk - 1) / kChunk);
  if (p.slots > INT32_MAX) throw InvalidArgument("gated delta: more chunks than a launch can have");
  p.slot_heads = p.slots * op.value_heads;
  const int64_t blocks = padded_value_dim(op) / 16;
  if (p.slot_heads > INT32_MAX || (count_sequences(op) * op.value_heads + 8) * blocks > INT32_MAX)
    throw InvalidArgument("gated delta: more chunks, heads and value columns than a launch can have");
  with_mode(op, [&](auto m) {
    typedef decltype(m) M;
    p.record = size_t(p.slot_heads) * record_bytes<M>(false);
    p.record_back = size_t(p.slot_heads) * record_bytes<M>(true);
    p.states = size_t(p.slot_heads) * padded_key_dim(op.key_dim) * padded_value_dim(op) * sizeof(typename M::Saved);
    p.powers = sizeof(typename M::Saved) == 4 ? 0 : size_t(p.slot_heads) * 4 * (padded_value_dim(op) / 16);
    p.dots = sizeof(typename M::Saved) == 4 ? size_t(p.slot_heads) * (padded_value_dim(op) / 16) * 4 * sizeof(float) : 0;
    p.o_powers = sizeof(typename M::Saved) == 4 ? 0 : size_t(p.slot_heads) * kChunk * (padded_value_dim(op) / 16);
    p.us = size_t(p.slot_heads) * kChunk * padded_value_dim(op) * sizeof(typename M::Kept);
    p.scales = sizeof(typename M::Kept) == 4 ? 0 : size_t(p.slot_heads) * kChunk * (padded_value_dim(op) / 16) * sizeof(float);
  });
  return p;
}

bool steps(const cchip_gated_delta &op, bool saves) { return !op.sequences && !saves && op.tokens <= kStepTokens; }

int element_size(const cchip_gated_delta &op) { return op.dtype == CCHIP_F32 ? 4 : 2; }

Heads heads_of(const cchip_gated_delta &d, const cchip_heads &x, const char *name, bool written, int heads, int dim) {
  return cchip::op::heads_of("gated delta", name, d.dtype, d.batch, d.tokens, heads, dim, x, written);
}

// What a call writes is read by other workgroups of the same call, and in the
// backward pass by later kernels too. Of two tensors whose elements may lie
// between one another's, those of the first token and head are looked at.
void check_apart(const cchip_gated_delta &op, const cchip_gated_delta_io &io, bool back) {
  if (op.batch * op.tokens == 0) return;
  struct Head {
    const char *name;
    const void *data;
    size_t bytes;
  };
  const size_t size = element_size(op), key = size * op.key_dim, value = size * op.value_dim;
  const Head in[] = {{"q", io.q.data, key}, {"k", io.k.data, key}, {"v", io.v.data, value}, {"g", io.g.data, size},
                     {"beta", io.beta.data, size}, {"the gradient of o", io.d_o.data, value}};
  const Head forward[] = {{"o", io.o.data, value}};
  const Head backward[] = {{"dq", io.dq.data, key}, {"dk", io.dk.data, key}, {"dv", io.dv.data, value}, {"dg", io.dg.data, size},
                           {"dbeta", io.dbeta.data, size}};
  const Head *out = back ? backward : forward;
  for (int i = 0; i < (back ? 5 : 1); i++) {
    for (int j = 0; j < (back ? 6 : 5); j++)
      if (meet(out[i].data, out[i].bytes, in[j].data, in[j].bytes))
        throw InvalidArgument(strf("gated delta: %s is written over %s, which the call reads", out[i].name, in[j].name));
    for (int j = 0; j < i; j++)
      if (meet(out[i].data, out[i].bytes, out[j].data, out[j].bytes))
        throw InvalidArgument(strf("gated delta: %s and %s are written to one place", out[j].name, out[i].name));
  }
}

DeltaArgs args_of(const cchip_gated_delta &op, const cchip_gated_delta_io &io, const Layout &p, bool back) {
  DeltaArgs a = {};
  const int hk = op.key_heads, hv = op.value_heads, dk = op.key_dim, dv = op.value_dim;
  a.q = heads_of(op, io.q, "q", false, hk, dk);
  a.k = heads_of(op, io.k, "k", false, hk, dk);
  a.v = heads_of(op, io.v, "v", false, hv, dv);
  a.g = heads_of(op, io.g, "g", false, hv, 1);
  a.beta = heads_of(op, io.beta, "beta", false, hv, 1);
  if (op.sequences ? !io.offsets : io.offsets != nullptr)
    throw InvalidArgument(op.sequences ? "gated delta: packed sequences need offsets" : "gated delta: offsets without packed sequences");
  if (!op.states && (io.state || io.state_out || io.dstate || io.dstate_out))
    throw InvalidArgument("gated delta: a state for an operator made without states");
  if (back) {
    if (!io.saved && p.slots) throw InvalidArgument("gated delta: the backward pass needs what the forward pass saved");
    a.d_o = heads_of(op, io.d_o, "the gradient of o", false, hv, dv);
    a.gq = heads_of(op, io.dq, "dq", true, hk, dk);
    a.gk = heads_of(op, io.dk, "dk", true, hk, dk);
    a.gv = heads_of(op, io.dv, "dv", true, hv, dv);
    a.gg = heads_of(op, io.dg, "dg", true, hv, 1);
    a.gbeta = heads_of(op, io.dbeta, "dbeta", true, hv, 1);
    a.dstate_out = io.dstate_out;
    a.dstate = io.dstate;
  } else {
    a.o = heads_of(op, io.o, "o", true, hv, dv);
    a.state = io.state;
    a.state_out = io.state_out;
  }
  const std::pair<const char *, const void *> words[] = {{"offsets", io.offsets}, {"state", io.state}, {"state_out", io.state_out},
                                                        {"dstate", io.dstate}, {"dstate_out", io.dstate_out}};
  for (auto &w : words)
    if (reinterpret_cast<uintptr_t>(w.second) % 4) throw InvalidArgument(strf("gated delta: %s is not aligned to its elements", w.first));
  if (!aligned16(io.saved)) throw InvalidArgument("gated delta: saved is not aligned to 16 bytes");
  a.offsets = io.offsets;
  a.tokens = op.tokens;
  a.slots = p.slots;
  a.sequences = count_sequences(op);
  a.chunks = int((op.tokens + kChunk - 1) / kChunk);
  a.hk = hk;
  a.hv = hv;
  a.dk = dk;
  a.dv = dv;
  a.dvp = padded_value_dim(op);
  a.scale = op.scale;
  return a;
}

void check_workspace(const void *workspace, size_t have, size_t need) {
  if (have < need || (need && !workspace) || !aligned16(workspace))
    throw InvalidArgument(strf("gated delta: the workspace needs %zu bytes aligned to 16, has %zu", need, workspace ? have : 0));
}

size_t backward_bytes(const Layout &p) { return p.states + p.us + p.scales + p.dots + p.o_powers + p.powers; }

void lay_out(DeltaArgs &a, const Layout &p, char *saved) {
  a.records = saved;
  a.states = saved + p.record_back;
  a.us = a.states + p.states;
  a.u_scales = reinterpret_cast<float *>(a.us + p.us);
  a.state_powers = reinterpret_cast<uint8_t *>(a.us + p.us + p.scales);
}

}  // namespace

extern "C" {

int cchip_gated_delta_sizes(const cchip_gated_delta *op, size_t *forward, size_t *backward, size_t *saved) {
  return guarded([&] {
    check_op(op);
    const Layout p = layout_of(*op);
    if (forward) *forward = steps(*op, false) ? 0 : p.record;
    if (backward) *backward = backward_bytes(p);
    if (saved) *saved = p.record_back + p.states + p.us + p.scales + p.powers;
  });
}

int cchip_gated_delta_forward(const cchip_gated_delta *op, const cchip_gated_delta_io *io, void *workspace,
                              size_t workspace_bytes, void *stream) {
  return guarded([&] {
    check_op(op);
    if (!io) throw InvalidArgument("gated delta: no tensors");
    const Layout p = layout_of(*op);
    DeltaArgs a = args_of(*op, *io, p, false);
    if (a.sequences == 0) return;
    const bool step = steps(*op, io->saved != nullptr);
    if (io->saved) {
      lay_out(a, p, static_cast<char *>(io->saved));
    } else if (!step) {
      check_workspace(workspace, workspace_bytes, p.record);
      a.records = static_cast<char *>(workspace);
    }
    check_apart(*op, *io, false);
    if (step) return delta_step_launch(*op, a, (hipStream_t)stream);
    if (p.slots) delta_chunk_launch(*op, a, io->saved != nullptr, (hipStream_t)stream);
    delta_forward_launch(*op, a, io->saved != nullptr, (hipStream_t)stream);
  });
}

int cchip_gated_delta_backward(const cchip_gated_delta *op, const cchip_gated_delta_io *io, void *workspace,
                               size_t workspace_bytes, void *stream) {
  return guarded([&] {
    check_op(op);
    if (!io) throw InvalidArgument("gated delta: no tensors");
    const Layout p = layout_of(*op);
    DeltaArgs a = args_of(*op, *io, p, true);
    if (a.sequences == 0) return;
    lay_out(a, p, static_cast<char *>(io->saved));
    check_workspace(workspace, workspace_bytes, backward_bytes(p));
    check_apart(*op, *io, true);
    if (p.slots && workspace == io->saved) throw InvalidArgument("gated delta: the workspace is what the forward pass saved");
    a.grads = static_cast<char *>(workspace);
    a.ys = a.grads + p.states;
    a.y_scales = reinterpret_cast<float *>(a.ys + p.us);
    a.dots = reinterpret_cast<float *>(a.ys + p.us + p.scales);
    a.o_powers = reinterpret_cast<uint8_t *>(a.ys + p.us + p.scales + p.dots);
    a.grad_powers = a.o_powers + p.o_powers;
    delta_backward_launch(*op, a, (hipStream_t)stream);
  });
}

}  // extern "C"
