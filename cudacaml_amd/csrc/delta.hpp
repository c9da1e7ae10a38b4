// The gated delta rule: arguments, chunk records and sequence lookup shared
// by its kernels (delta_chunk.hip, delta_forward.hip, delta_backward.hip,
// delta_step.hip) and their host side (delta.cpp).
//
// A sequence is cut into chunks of 64 tokens. With c the running sum of g in
// a chunk, D_ts = exp(c_t - c_s) for s <= t, Gam_t = exp(c_t), G_s =
// exp(c_63 - c_s) and S the state before it, the recurrence over a chunk is
//
//   A = strict lower of beta_t D_ts (k_t . k_s),   T = (I + A)^-1
//   P = lower of D_ts (q_t . k_s)
//   U = T (beta (V - Gam (K S))),   O = scale (Gam (Q S) + P U)
//   S' = Gam_63 S + K^T (G U)
//
// T and P depend on no state: one kernel makes them for all chunks at once
// (delta_chunk.hip), and what is left runs through the chunks in order, a
// workgroup for some value columns of one head (delta_forward.hip). Tokens
// past a sequence's end count as k = q = v = beta = g = 0, which leaves a
// state as it is.
#pragma once

#include "../../include/cchip_operators.h"
#include "operators.hpp"

namespace cchip {
namespace op {

constexpr int kChunk = 64;

struct Heads {
  char *p;  // elements of the operator's type
  int64_t b, t, h;
};

struct DeltaArgs {
  Heads q, k, v, g, beta, o;
  Heads d_o;                   // gradient of o
  Heads gq, gk, gv, gg, gbeta;  // gradients of the inputs
  const int *offsets;
  const float *state;
  float *state_out;
  const float *dstate_out;
  float *dstate;
  char *records;  // one a (slot, value head)
  char *states;   // saved S before each chunk, [key_dim][value_dim]; null if there is no backward pass
  char *us;       // saved U, [64][value_dim]
  char *grads;    // backward: dS after each chunk
  char *ys;       // backward: Y
  int64_t tokens, sequences;  // sequences: of the packed batch, or its rows
  int64_t slots;
  int chunks;  // of a row of the batch; unused where packed
  int hk, hv, dk, dv;
  float scale;
};

// What a chunk and value head have that depends on no state: matrices as
// fragments of 16 rows and 32 terms, [row block][term block][lane][8], in
// planes, and the decays.
template <int NS, int NO>
struct Record {
  static constexpr int kPlane = 64 * 64 * 2;
  static constexpr int T = 0, P = NS * kPlane, Decay = P + NO * kPlane;  // Gam, G, beta: 64 f32 each
  static constexpr int Tt = Decay + 768, Pt = Tt + NS * kPlane;          // transposed, for the backward pass
  static constexpr int64_t bytes(bool back) { return back ? Pt + NS * kPlane : Tt; }
};

// Element type, planes of an input, of what makes a state, of what makes
// only an output, and the type that states are saved in for the backward
// pass with the planes they are read back in.
template <typename T_, int NI_, int NS_, int NO_, typename Saved_, int NB_>
struct Mode {
  typedef T_ T;
  typedef Saved_ Saved;
  static constexpr int NI = NI_, NS = NS_, NO = NO_, NB = NB_;
};
typedef Mode<bf16, 1, 1, 1, bf16, 1> ModeBf16;    // bf16 in and out
typedef Mode<bf16, 1, 3, 1, bf16, 1> ModeBf16S;   // with f32 states in or out
typedef Mode<f16, 2, 3, 2, float, 2> ModeF16;
typedef Mode<float, 3, 3, 3, float, 3> ModeF32;

// A chunk: `first` is its first token, in the packed batch or in row `row`.
struct Chunk {
  int64_t row, first, sequence;
  int len;    // tokens in it, 0: there is no such chunk
};

__device__ __forceinline__ int64_t cut(const DeltaArgs &a, int64_t i) {
  const int64_t o = a.offsets[i];
  return o < 0 ? 0 : o > a.tokens ? a.tokens : o;
}

// Where sequence i begins, its length and its first slot. Sequence i of a
// packed batch has slots from offsets[i] / 64 + i on: as many as it can need,
// and never more than tokens / 64 + sequences in all.
struct Sequence {
  int64_t row, first, len, slot;
};

__device__ __forceinline__ Sequence sequence_of(const DeltaArgs &a, int64_t i) {
  if (!a.offsets) return {i, 0, a.tokens, i * a.chunks};
  const int64_t lo = cut(a, i), hi = cut(a, i + 1);
  return {0, lo, hi > lo ? hi - lo : 0, lo / kChunk + i};
}

__device__ __forceinline__ Chunk chunk_of(const DeltaArgs &a, int64_t slot) {
  int64_t i;
  if (!a.offsets) {
    i = slot / a.chunks;
  } else {
    int64_t lo = 0, hi = a.sequences;  // the last sequence whose first slot is not after this one
    while (hi - lo > 1) {
      const int64_t mid = (lo + hi) / 2;
      if (cut(a, mid) / kChunk + mid <= slot) lo = mid;
      else hi = mid;
    }
    i = lo;
  }
  const Sequence s = sequence_of(a, i);
  const int64_t at = (slot - s.slot) * kChunk;
  const int64_t left = at < 0 ? 0 : s.len - at;
  return {s.row, s.first + at, i, int(left < 0 ? 0 : left > kChunk ? kChunk : left)};
}

template <typename T>
__device__ __forceinline__ const T *at(const Heads &x, int64_t row, int64_t token, int head) {
  return reinterpret_cast<const T *>(x.p) + row * x.b + token * x.t + head * x.h;
}
template <typename T>
__device__ __forceinline__ T *out_at(const Heads &x, int64_t row, int64_t token, int head) {
  return reinterpret_cast<T *>(x.p) + row * x.b + token * x.t + head * x.h;
}

// Eight elements of token `t` of a chunk from element `d` on, of a head of
// `dim`; zeros past the chunk or the head.
template <typename T>
__device__ __forceinline__ Raw8<T> load_head8(const Heads &x, const Chunk &c, int head, int t, int d, int dim) {
  const int n = t < c.len ? (dim - d < 0 ? 0 : dim - d > 8 ? 8 : dim - d) : 0;
  return load8<T>(at<T>(x, c.row, c.first + t, head) + d, n);
}

template <typename Mode>
int64_t record_bytes(bool back) {
  return Record<Mode::NS, Mode::NO>::bytes(back);
}

void delta_chunk_launch(const cchip_gated_delta &op, const DeltaArgs &a, bool back, hipStream_t stream);
void delta_forward_launch(const cchip_gated_delta &op, const DeltaArgs &a, bool back, hipStream_t stream);
void delta_backward_launch(const cchip_gated_delta &op, const DeltaArgs &a, hipStream_t stream);
void delta_step_launch(const cchip_gated_delta &op, const DeltaArgs &a, hipStream_t stream);

// Calls f with the Mode of an operator.
template <typename F>
void with_mode(const cchip_gated_delta &op, F &&f) {
  if (op.dtype == CCHIP_F32) f(ModeF32());
  else if (op.dtype == CCHIP_F16) f(ModeF16());
  else if (op.states) f(ModeBf16S());
  else f(ModeBf16());
}

}  // namespace op
}  // namespace cchip
