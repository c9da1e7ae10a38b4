// Attention: the entry points of cchip_operators.h, their checks, and how a
// call is cut into workgroups.

#include "attention_backward.hpp"

#include <algorithm>
#include <cmath>
#include <utility>

namespace cchip {
namespace op {

extern template void attend_launch<bf16>(const AttentionArgs &, int, hipStream_t);
extern template void attend_launch<f16>(const AttentionArgs &, int, hipStream_t);
extern template void attend_launch<float>(const AttentionArgs &, int, hipStream_t);

extern template void attend_back_launch<bf16>(const AttentionArgs &, hipStream_t);
extern template void attend_back_launch<f16>(const AttentionArgs &, hipStream_t);
extern template void attend_back_launch<float>(const AttentionArgs &, hipStream_t);

}  // namespace op
}  // namespace cchip

using namespace cchip;
using namespace cchip::op;

namespace {

const char *kWho = "attention";

void check_op(const cchip_attention *op) {
  if (!op) throw InvalidArgument("attention: no descriptor");
  if (op->dtype != CCHIP_F32 && op->dtype != CCHIP_BF16 && op->dtype != CCHIP_F16)
    throw InvalidArgument(strf("attention: dtype %d is not f32, bf16 or f16", op->dtype));
  const int64_t most = (int64_t(1) << 31) - 64;
  if (op->batch < 0 || op->tokens < 0 || op->sequences < 0 || op->keys < 0 || op->tokens > most || op->keys > most)
    throw InvalidArgument("attention: batch, tokens, sequences and keys are not negative, and tokens and keys below 2^31 - 64");
  if (op->sequences > 0 && op->batch != 1) throw InvalidArgument("attention: packed sequences have a batch of 1");
  if (op->sequences > 0 && op->keys > 0) throw InvalidArgument("attention: a cache's sequences are not packed");
  if (op->kv_heads < 1 || op->heads < 1 || op->heads % op->kv_heads)
    throw InvalidArgument(strf("attention: %d heads are not a multiple of %d key heads", op->heads, op->kv_heads));
  if (op->head_dim < 1 || op->head_dim > 128) throw InvalidArgument(strf("attention: head_dim %d is not in 1 .. 128", op->head_dim));
  if (!std::isfinite(op->scale)) throw InvalidArgument("attention: scale is not finite");
  // every count below is then under 2^31 times a small one
  if (op->batch > INT32_MAX || op->sequences > INT32_MAX || op->batch * op->kv_heads > INT32_MAX ||
      op->tokens * (op->heads / op->kv_heads) > (int64_t(1) << 34))
    throw InvalidArgument("attention: more sequences, heads and tokens than a launch can have");
}

struct Cut {
  int waves;  // 0: the kernel for few rows
  int slots, splits;
  int64_t workgroups;
  size_t bytes;  // of workspace
};

Cut cut_of(const cchip_attention &op) {
  Cut p = {};
  const int64_t group = op.heads / op.kv_heads, rows = op.tokens * group, keys = op.keys ? op.keys : op.tokens;
  const int64_t pairs = (op.sequences ? 1 : op.batch) * op.kv_heads, of_one = op.sequences ? rows / op.sequences : rows;
  const auto slots_of = [&](int height) { return (rows + height - 1) / height + op.sequences; };
  // Eight waves where there are rows for more than four: they share what is
  // read, and four would leave half of a unit's registers idle, as there is
  // LDS for one workgroup.
  p.waves = !op.sequences && rows <= 64 ? 0 : op.dtype != CCHIP_F32 && of_one > 128 ? 8 : 4;
  const int64_t slots = slots_of(p.waves ? 32 * p.waves : 32);
  if (slots > (int64_t(1) << 27) || pairs * slots > (int64_t(1) << 30))
    throw InvalidArgument("attention: more tokens and heads than a launch can have");
  p.slots = int(slots);
  p.splits = 1;
  // Keys are split where there are too few workgroups for the chip, but into
  // parts that are long beside what joining them costs. 512 are wanted: of the
  // kernel for few rows as many as run at once (with 1024 a step of 16
  // sequences over 2048 keys took 39.7 us in place of 32.7, of one over 32768 56.8 in
  // place of 41.8). Of the others 256 run at once, but parts follow each
  // sequence's own length: for sequences as long as one another 256 are better
  // (chunks of 512 tokens over 8192 keys 163 us in place of 174, four of 256
  // over 4096 98 in place of 114), for others 512 (512 over 8192 and 4352 keys
  // 145 in place of 158).
  const int64_t base = std::max<int64_t>(1, pairs * slots), least = !p.waves ? 128 : op.dtype == CCHIP_F32 ? 256 : 512, wanted = 512;
  if (!op.sequences && base < wanted) p.splits = int(std::max<int64_t>(1, std::min((wanted + base - 1) / base, keys / least)));
  p.workgroups = pairs * slots * p.splits;  // at most 2^30: splits are few where it is much
  if (p.splits > 1) p.bytes = size_t(op.batch) * op.tokens * op.heads * p.splits * (op.head_dim + 2) * sizeof(float);
  return p;
}

// What a forward pass saves: the lse of each row and, where o is rounded, what
// that leaves of it as bf16: do . o, which the backward pass subtracts from
// sums made in f32, would be off by o's rounding.
size_t lse_bytes(const cchip_attention &op) { return (size_t(op.batch) * op.tokens * op.heads * sizeof(float) + 15) / 16 * 16; }

size_t saved_bytes(const cchip_attention &op) {
  return lse_bytes(op) + (op.dtype == CCHIP_F32 ? 0 : size_t(op.batch) * op.tokens * op.heads * op.head_dim * 2);
}

struct BackCut {
  int64_t pairs, row_slots, key_slots;
  int chunks, chunk_tiles;
  BackSizes sizes;
};

BackCut back_cut_of(const cchip_attention &op) {
  BackCut c;
  c.pairs = (op.sequences ? 1 : op.batch) * op.kv_heads;
  c.row_slots = (op.tokens * (op.heads / op.kv_heads) + kUnit - 1) / kUnit + op.sequences;
  c.key_slots = (op.tokens + kUnit - 1) / kUnit + op.sequences;
  if (c.row_slots > (int64_t(1) << 24) || c.pairs * c.row_slots > (int64_t(1) << 27))
    throw InvalidArgument("attention: more tokens and heads than a launch can have");
  // Chunks of rows that there are four workgroups to a unit, of 2048 rows at
  // least: a chunk's sums cost what 30 of its rows do. Where all keys are too few
  // workgroups for the chip, what they leave idle costs more: of 256 rows.
  const int64_t high = op.dtype == CCHIP_F32 ? 32 : 64, tiles = (op.tokens * (op.heads / op.kv_heads) + high - 1) / high;
  const int64_t jobs = c.pairs * c.key_slots;
  c.chunks = int(std::max<int64_t>(1, std::min<int64_t>({8, (1024 + jobs - 1) / std::max<int64_t>(1, jobs), tiles * high / 2048})));
  if (jobs > 0 && jobs * c.chunks < 256) c.chunks = int(std::max<int64_t>(c.chunks, std::min<int64_t>({8, 256 / jobs, tiles * high / 256})));
  c.chunk_tiles = int((tiles + c.chunks - 1) / c.chunks);
  c.sizes = back_sizes(op.dtype, op.head_dim, c.pairs, c.row_slots, c.key_slots, c.chunks);
  return c;
}

AttentionArgs args_of(const cchip_attention &op, const cchip_attention_io &io, bool back) {
  AttentionArgs a = {};
  const int64_t b = op.batch, t = op.tokens, n = op.keys ? op.keys : op.tokens;
  const int h = op.heads, hk = op.kv_heads, d = op.head_dim;
  a.q = heads_of(kWho, "q", op.dtype, b, t, h, d, io.q, false);
  a.k = heads_of(kWho, "k", op.dtype, b, n, hk, d, io.k, false);
  a.v = heads_of(kWho, "v", op.dtype, b, n, hk, d, io.v, false);
  a.o = heads_of(kWho, "o", op.dtype, b, t, h, d, io.o, !back);
  if (back) {
    a.d_o = heads_of(kWho, "the gradient of o", op.dtype, b, t, h, d, io.d_o, false);
    a.gq = heads_of(kWho, "dq", op.dtype, b, t, h, d, io.dq, true);
    a.gk = heads_of(kWho, "dk", op.dtype, b, n, hk, d, io.dk, true);
    a.gv = heads_of(kWho, "dv", op.dtype, b, n, hk, d, io.dv, true);
  }
  // other workgroups read what one of a call writes
  struct Named {
    const char *name;
    const Heads *x;
    HeadCounts n;
  };
  const HeadCounts qs = {{b, t, h}}, ks = {{b, n, hk}};
  const Named in[] = {{"q", &a.q, qs}, {"k", &a.k, ks}, {"v", &a.v, ks}, {"the gradient of o", &a.d_o, qs}, {"o", &a.o, qs}};
  const Named out[] = {{"dq", &a.gq, qs}, {"dk", &a.gk, ks}, {"dv", &a.gv, ks}}, o = in[4];
  const int size = op.dtype == CCHIP_F32 ? 4 : 2;
  for (int i = 0; i < (back ? 3 : 1) && b * t; i++) {
    const Named &to = back ? out[i] : o;
    for (int j = 0; j < (back ? 5 : 3); j++)
      if (heads_meet(d, size, to.n, *to.x, in[j].n, *in[j].x))
        throw InvalidArgument(strf("attention: %s is written over %s, which the call reads", to.name, in[j].name));
    for (int j = 0; j < i; j++)
      if (heads_meet(d, size, to.n, *to.x, out[j].n, *out[j].x))
        throw InvalidArgument(strf("attention: %s and %s are written to one place", out[j].name, to.name));
  }
  if (op.sequences ? !io.offsets : io.offsets != nullptr)
    throw InvalidArgument(op.sequences ? "attention: packed sequences need offsets" : "attention: offsets without packed sequences");
  if (op.keys ? !io.lengths : io.lengths != nullptr)
    throw InvalidArgument(op.keys ? "attention: a cache needs lengths" : "attention: lengths without a cache");
  const std::pair<const char *, const void *> words[] = {{"offsets", io.offsets}, {"lengths", io.lengths}};
  for (auto &w : words)
    if (reinterpret_cast<uintptr_t>(w.second) % 4) throw InvalidArgument(strf("attention: %s is not aligned to its elements", w.first));
  a.offsets = io.offsets;
  a.lengths = io.lengths;
  if (!aligned16(io.saved)) throw InvalidArgument("attention: saved is not aligned to 16 bytes");
  a.lse = static_cast<float *>(io.saved);
  if (io.saved && op.dtype != CCHIP_F32) a.o_rest = reinterpret_cast<bf16 *>(static_cast<char *>(io.saved) + lse_bytes(op));
  a.batch = b;
  a.tokens = t;
  a.keys = n;
  a.sequences = op.sequences;
  a.kv_heads = hk;
  a.group = h / hk;
  a.dim = d;
  a.splits = 1;
  a.plain_scale = op.scale;
  a.negate = op.scale < 0.0f;
  // a scale of zero: scores that are masked have to stay -infinity
  a.scale = std::fmax(std::fabs(op.scale) * 1.44269504088896341f, 1e-37f);
  return a;
}

// The workspace is large enough, and neither it nor `saved` is where a tensor
// begins or the other is.
void check_workspace(const cchip_attention &op, const cchip_attention_io &io, const void *workspace, size_t have, size_t need) {
  if (have < need || (need && !workspace) || (need && !aligned16(workspace)))
    throw InvalidArgument(strf("attention: the workspace needs %zu bytes aligned to 16, has %zu", need, workspace ? have : 0));
  const size_t saved = io.saved ? saved_bytes(op) : 0, head = size_t(op.head_dim) * (op.dtype == CCHIP_F32 ? 4 : 2);
  if (meet(workspace, need, io.saved, saved)) throw InvalidArgument("attention: the workspace is what the forward pass saved");
  const std::pair<const char *, const void *> tensors[] = {{"q", io.q.data}, {"k", io.k.data}, {"v", io.v.data}, {"o", io.o.data},
                                                           {"the gradient of o", io.d_o.data}, {"dq", io.dq.data}, {"dk", io.dk.data}, {"dv", io.dv.data}};
  for (auto &x : tensors)
    if (x.second && (meet(workspace, need, x.second, head) || meet(io.saved, saved, x.second, head)))
      throw InvalidArgument(strf("attention: %s lies in %s", x.first, meet(workspace, need, x.second, head) ? "the workspace" : "what the forward pass saves"));
}

}  // namespace

extern "C" {

int cchip_attention_sizes(const cchip_attention *op, size_t *forward, size_t *backward, size_t *saved) {
  return guarded([&] {
    check_op(op);
    const Cut p = cut_of(*op);
    if (forward) *forward = p.bytes;
    if (backward) *backward = op->keys || op->batch * op->tokens == 0 ? 0 : back_cut_of(*op).sizes.bytes();
    if (saved) *saved = op->keys ? 0 : saved_bytes(*op);
  });
}

int cchip_attention_forward(const cchip_attention *op, const cchip_attention_io *io, void *workspace, size_t workspace_bytes,
                            void *stream) {
  return guarded([&] {
    check_op(op);
    if (!io) throw InvalidArgument("attention: no tensors");
    AttentionArgs a = args_of(*op, *io, false);
    if (op->keys && io->saved) throw InvalidArgument("attention: there is no backward pass over a cache");
    const Cut p = cut_of(*op);
    if (op->batch * op->tokens == 0) return;
    check_workspace(*op, *io, workspace, workspace_bytes, p.bytes);
    a.partial = static_cast<float *>(workspace);
    a.slots = p.slots;
    a.splits = p.splits;
    a.workgroups = uint32_t(p.workgroups);
    if (op->dtype == CCHIP_F32) attend_launch<float>(a, p.waves, (hipStream_t)stream);
    else if (op->dtype == CCHIP_F16) attend_launch<f16>(a, p.waves, (hipStream_t)stream);
    else attend_launch<bf16>(a, p.waves, (hipStream_t)stream);
  });
}

int cchip_attention_backward(const cchip_attention *op, const cchip_attention_io *io, void *workspace, size_t workspace_bytes,
                             void *stream) {
  return guarded([&] {
    check_op(op);
    if (!io) throw InvalidArgument("attention: no tensors");
    if (op->keys) throw InvalidArgument("attention: there is no backward pass over a cache");
    AttentionArgs a = args_of(*op, *io, true);
    if (op->batch * op->tokens == 0) return;
    if (!io->saved) throw InvalidArgument("attention: the backward pass needs what the forward pass saved");
    const BackCut c = back_cut_of(*op);
    check_workspace(*op, *io, workspace, workspace_bytes, c.sizes.bytes());
    char *at = static_cast<char *>(workspace);
    for (int i = 0; i < 4; i++) {
      a.tiles[i] = reinterpret_cast<u32x4 *>(at);
      at += c.sizes.tiles[i];
    }
    a.row_heads = reinterpret_cast<float *>(at);
    a.key_heads = reinterpret_cast<int32_t *>(at + c.sizes.row_heads);
    a.partial = reinterpret_cast<float *>(at + c.sizes.row_heads + c.sizes.key_heads);
    a.queues = reinterpret_cast<uint32_t *>(at + c.sizes.row_heads + c.sizes.key_heads + c.sizes.partial);
    a.chunks = c.chunks;
    a.chunk_tiles = c.chunk_tiles;
    a.pairs = uint32_t(c.pairs);
    a.row_slots = int(c.row_slots);
    a.key_slots = int(c.key_slots);
    const auto launch = op->dtype == CCHIP_F32 ? attend_back_launch<float> : op->dtype == CCHIP_F16 ? attend_back_launch<f16> : attend_back_launch<bf16>;
    launch(a, (hipStream_t)stream);
  });
}

}  // extern "C"
