// The gated delta rule: arguments, chunk records and sequence lookup shared
// by its kernels (delta_chunk.hip, delta_forward.hip, delta_backward.hip,
// delta_step.hip) and their host side (delta.hip).
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

#include <type_traits>

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
  // of each (slot, value head), in blocks of 32 value columns (put_block);
  // what pads a head is zero
  char *states;   // saved S before the chunk, DK rows; null if there is no backward pass
  char *us;       // saved U, 64 rows
  char *grads;    // backward: dS after the chunk
  char *ys;       // backward: Y
  float *u_scales, *y_scales;  // of U and Y in f16: [16 columns][64]
  float *dots;                  // backward: sums that make <S, dS>, four for each 16 value columns, where those are f32
  uint8_t *o_powers;            // backward: of the gradient of o, [16 columns][64]
  uint8_t *state_powers, *grad_powers;  // of S and dS in f16: [16 columns][4 blocks of DK / 4 rows], the exponents of f32
  int64_t tokens, sequences;  // sequences: of the packed batch, or its rows
  int64_t slots;
  int chunks;  // of a row of the batch; unused where packed
  int hk, hv, dk, dv;
  int dvp;     // dv rounded up to 32
  float scale;
};

// Element type, then the planes: NI of an input, NS of what makes a state
// (S, T, X and U in their products), NO of S, P, U and Y where they make only
// outputs. Saved is the type that S and dS are kept in for the backward pass
// and Kept that of U and Y: f32 or, with powers of two (half_exponent), f16,
// one for each token of U and Y and each DK / 4 rows of S and dS in the 16 or
// 32 columns of a workgroup. NB: planes of M and B and, in f32, of S and dS
// where the gradients of q and k are made.
//
// A product loses the most precise operand's worth of the other's rounding:
// 2^-9 of a value in one plane of bf16, 2^-17 in two; states in f32 take
// three. bf16 results are rounded to 2^-9 themselves, 1.7e-3 in the 2-norm.
// o adds nothing to that; in one plane it would be 2.4e-3 off, for 363 us in
// place of 376 (forward of 4 x 4096 tokens, 32 heads of 128). Nor do the
// gradients add to it: the 11 bits of f16 are exact on the f16 matrix
// instruction. S and dS as bf16, and M and B in one plane, made dq and dk 2.4e-3
// off, 3.5e-3 where keys are alike, and the four kernels of a training step
// there 1410 us in place of 1440. Value columns of a head that are more than
// 2^24 apart lose bits of the smaller ones' share in dq, dk, dg and dbeta.
template <typename T_, int NI_, int NS_, int NO_, typename Saved_, int NB_, typename Kept_>
struct Mode {
  typedef T_ T;
  typedef Saved_ Saved;
  typedef Kept_ Kept;
  static constexpr int NI = NI_, NS = NS_, NO = NO_, NB = NB_;
};
typedef Mode<bf16, 1, 2, 2, f16, 2, f16> ModeBf16;   // bf16 in and out
typedef Mode<bf16, 1, 3, 2, f16, 2, f16> ModeBf16S;  // with f32 states in or out
typedef Mode<f16, 2, 3, 2, float, 2, float> ModeF16;
typedef Mode<float, 3, 3, 3, float, 3, float> ModeF32;

// What a chunk and value head have that depends on no state: matrices as
// fragments of 16 rows and 32 terms, [row block][term block][lane][8], in
// planes, and the decays.
template <typename M>
struct Record {
  static constexpr int kPlane = 64 * 64 * 2;
  static constexpr int T = 0, P = M::NS * kPlane, Decay = P + M::NO * kPlane;  // Gam, G, beta: 64 f32 each
  static constexpr int Tt = Decay + 768, Pt = Tt + M::NS * kPlane;             // transposed, for the backward pass
  static constexpr int64_t bytes(bool back) { return back ? Pt + M::NS * kPlane : Tt; }
};

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

// How a head's elements are read. Whole: it is whole pieces of 16 bytes (of 4
// elements where a lane takes four at a time). Pieces: it is at least one
// piece; the last one is read so that it ends with the head, and shifted down
// when it is needed. Single: one element at a time.
enum Access { kSingle, kPieces, kWhole };

template <int Bytes>
__device__ __forceinline__ void shift_down(uint32_t *w, int elements, int size) {
  const uint32_t bits = elements <= 0 ? 0 : uint32_t(elements * size * 8);
  const uint64_t lo = w[0] | uint64_t(w[1]) << 32;
  if constexpr (Bytes == 8) {
    const uint64_t x = bits < 64 ? lo >> bits : 0;
    w[0] = uint32_t(x);
    w[1] = uint32_t(x >> 32);
  } else {
    const uint64_t hi = w[2] | uint64_t(w[3]) << 32;
    const uint64_t x = bits == 0 ? lo : bits < 64 ? lo >> bits | hi << (64 - bits) : bits < 128 ? hi >> (bits - 64) : 0;
    const uint64_t y = bits < 64 ? hi >> bits : 0;
    w[0] = uint32_t(x);
    w[1] = uint32_t(x >> 32);
    w[2] = uint32_t(y);
    w[3] = uint32_t(y >> 32);
  }
}

// Eight elements of token `t` of a chunk from element `d` on, of a head of
// `dim`: always loads, of elements that exist where those asked for do not,
// so that nothing branches and loads stay in flight; keep_head8 makes what
// is past the chunk or the head zero once they are needed.
template <int A, typename T>
__device__ __forceinline__ Raw8<T> load_head8(const Heads &x, const Chunk &c, int head, int t, int d, int dim) {
  constexpr int E = 16 / sizeof(T);
  const char *base = x.p + (c.row * x.b + c.first * x.t + head * x.h) * int64_t(sizeof(T));
  const uint32_t row = uint32_t(t < c.len ? t : c.len - 1) * uint32_t(x.t);
  Raw8<T> r;
  if (A != kSingle) {
#pragma unroll
    for (int i = 0; i < 8 / E; i++) {
      const int at = d + i * E + E <= dim ? d + i * E : dim - E;
      reinterpret_cast<u32x4 *>(&r)[i] = *reinterpret_cast<const u32x4_any *>(base + (row + uint32_t(at)) * uint32_t(sizeof(T)));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      r.x[i] = *reinterpret_cast<const T *>(base + (row + uint32_t(d + i < dim ? d + i : dim - 1)) * uint32_t(sizeof(T)));
  }
  return r;
}

template <int A, typename T>
__device__ __forceinline__ Raw8<T> keep_head8(Raw8<T> r, const Chunk &c, int t, int d, int dim) {
  constexpr int E = 16 / sizeof(T);
  if (A != kSingle) {
    u32x4 *x = reinterpret_cast<u32x4 *>(&r);
#pragma unroll
    for (int i = 0; i < 8 / E; i++) {
      if (A == kPieces) {
        uint32_t w[4] = {x[i][0], x[i][1], x[i][2], x[i][3]};
        shift_down<16>(w, d + i * E + E - dim, sizeof(T));
        x[i] = u32x4{w[0], w[1], w[2], w[3]};
      }
      x[i] = t < c.len && d + i * E < dim ? x[i] : u32x4{};
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) r.x[i] = t < c.len && d + i < dim ? r.x[i] : T(0.0f);
  }
  return r;
}

// Four in the same way, and the store of four.
template <typename T>
struct Raw4 {
  T x[4];
};
template <typename T>
struct Vector4;
template <>
struct Vector4<float> {
  typedef u32x4_any type;
};
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
template <>
struct Vector4<bf16> {
  typedef u32x2_any type;
};
template <>
struct Vector4<f16> {
  typedef u32x2_any type;
};

template <int A, typename T>
__device__ __forceinline__ Raw4<T> load_head4(const Heads &x, const Chunk &c, int head, int t, int d, int dim) {
  const char *base = x.p + (c.row * x.b + c.first * x.t + head * x.h) * int64_t(sizeof(T));
  const uint32_t row = uint32_t(t < c.len ? t : c.len - 1) * uint32_t(x.t);
  Raw4<T> r;
  if (A != kSingle) {
    typedef typename Vector4<T>::type V;
    *reinterpret_cast<V *>(&r) = *reinterpret_cast<const V *>(base + (row + uint32_t(d + 4 <= dim ? d : dim - 4)) * uint32_t(sizeof(T)));
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      r.x[i] = *reinterpret_cast<const T *>(base + (row + uint32_t(d + i < dim ? d + i : dim - 1)) * uint32_t(sizeof(T)));
  }
  return r;
}

template <int A, typename T>
__device__ __forceinline__ void store_head4(const Heads &x, const Chunk &c, int head, int t, int d, int dim, const f32x4 &v) {
  if (t >= c.len || d >= dim) return;
  char *base = x.p + (c.row * x.b + c.first * x.t + head * x.h) * int64_t(sizeof(T));
  char *to = base + (uint32_t(t) * uint32_t(x.t) + uint32_t(d)) * uint32_t(sizeof(T));
  Raw4<T> r;
#pragma unroll
  for (int i = 0; i < 4; i++) r.x[i] = T(v[i]);
  if (A == kWhole || d + 4 <= dim) {
    typedef typename Vector4<T>::type V;
    *reinterpret_cast<V *>(to) = *reinterpret_cast<const V *>(&r);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (d + i < dim) reinterpret_cast<T *>(to)[i] = r.x[i];
  }
}

// A lane of a transposed product has, of BV value columns, those from
// BV / 4 quad on: TV = BV / 16 fragments' worth of four, read with frag_v.
template <int N, int TV>
__device__ __forceinline__ Frag<N> frag_v(const bf16 *m, int plane, int ld, int j, int term0) {
  return frag_col<N, 4 * TV>(m, plane, ld, 4 * j, term0);
}

// A lane's 4 TV elements of token t of a tensor, and their store. Held as
// words: elements taken apart on the way round a loop would be waited for
// there.
template <typename T, int TV>
struct RawV {
  uint32_t w[TV * sizeof(T)];
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, w[i]);
    else if constexpr (std::is_same<T, bf16>::value) return i & 1 ? high_bf16(w[i / 2]) : low_bf16(w[i / 2]);
    else return float(__builtin_bit_cast(f16, uint16_t(w[i / 2] >> (i & 1 ? 16 : 0))));
  }
};

template <int A, typename T, int TV>
__device__ __forceinline__ RawV<T, TV> load_v(const Heads &x, const Chunk &c, int head, int t, int d, int dim) {
  if constexpr (TV == 2) return __builtin_bit_cast(RawV<T, TV>, load_head8<A, T>(x, c, head, t, d, dim));
  else return __builtin_bit_cast(RawV<T, TV>, load_head4<A, T>(x, c, head, t, d, dim));
}

// The lane's elements where they belong; those past the chunk or the head are
// of no meaning.
template <int A, typename T, int TV>
__device__ __forceinline__ RawV<T, TV> settle_v(RawV<T, TV> v, int d, int dim) {
  if constexpr (A == kPieces) {
    constexpr int kBytes = TV * 4 * sizeof(T) < 16 ? 8 : 16, E = kBytes / sizeof(T);
#pragma unroll
    for (int i = 0; i < 4 * TV / E; i++) shift_down<kBytes>(v.w + i * (kBytes / 4), d + i * E + E - dim, sizeof(T));
  }
  return v;
}

template <int A, typename T, int TV>
__device__ __forceinline__ void store_v(const Heads &x, const Chunk &c, int head, int t, int d, int dim, const f32x4 (&v)[TV]) {
  if (t >= c.len || d >= dim) return;
  char *base = x.p + (c.row * x.b + c.first * x.t + head * x.h) * int64_t(sizeof(T));
  char *to = base + (uint32_t(t) * uint32_t(x.t) + uint32_t(d)) * uint32_t(sizeof(T));
  union {
    T r[4 * TV];
    u32x4 w[sizeof(T) * TV >= 4 ? sizeof(T) * TV / 4 : 1];
    uint64_t half;
  } u;
#pragma unroll
  for (int i = 0; i < 4 * TV; i++) u.r[i] = T(v[i / 4][i % 4]);
  constexpr int kBytes = sizeof(u.r) < 16 ? 8 : 16, E = kBytes / sizeof(T);
#pragma unroll
  for (int i = 0; i < 4 * TV / E; i++) {
    if (A == kWhole ? d + i * E < dim : d + i * E + E <= dim) {
      if constexpr (kBytes == 16) reinterpret_cast<u32x4_any *>(to)[i] = u.w[i];
      else *reinterpret_cast<u32x2_any *>(to) = __builtin_bit_cast(u32x2_any, u.half);
    } else if (A != kWhole) {
#pragma unroll
      for (int j = 0; j < E; j++)
        if (d + i * E + j < dim) reinterpret_cast<T *>(to)[i * E + j] = u.r[i * E + j];
    }
  }
}

// Buffers between kernels hold value columns in blocks of 32, [block][row][32]:
// a workgroup writes whole lines, and a reader takes a block in one piece.
// `y`: the lane's first column of the block.
template <typename T, int TV>
__device__ __forceinline__ void put_block(char *rows, int row, int y, const f32x4 (&v)[TV]) {
  union {
    T r[4 * TV];
    u32x4 w[sizeof(T) * TV >= 4 ? sizeof(T) * TV / 4 : 1];
    uint64_t half;
  } u;
#pragma unroll
  for (int i = 0; i < 4 * TV; i++) u.r[i] = T(v[i / 4][i % 4]);
  char *to = rows + uint32_t(row * 32 + y) * uint32_t(sizeof(T));
  if constexpr (sizeof(u.r) >= 16) {
#pragma unroll
    for (int i = 0; i < int(sizeof(u.r) / 16); i++) reinterpret_cast<u32x4 *>(to)[i] = u.w[i];
  } else {
    *reinterpret_cast<uint64_t *>(to) = u.half;
  }
}

template <typename T, int TV>
__device__ __forceinline__ RawV<T, TV> load_block(const char *rows, int row, int y) {
  const char *from = rows + uint32_t(row * 32 + y) * uint32_t(sizeof(T));
  RawV<T, TV> r;
  if constexpr (sizeof(r) >= 16) {
#pragma unroll
    for (int i = 0; i < int(sizeof(r) / 16); i++) {
      const u32x4 x = reinterpret_cast<const u32x4 *>(from)[i];
#pragma unroll
      for (int j = 0; j < 4; j++) r.w[4 * i + j] = x[j];
    }
  } else {
    const uint2 x = *reinterpret_cast<const uint2 *>(from);
    r.w[0] = x.x;
    r.w[1] = x.y;
  }
  return r;
}

// What is kept in f16 is kept with a power of two, by which the largest of
// the values that share it becomes 2^14 .. 2^15: those down to 2^-28 of it
// have all of f16's 11 bits. `half_exponent` is the largest's, as f32 has it
// and in the range that the powers have; the values are multiplied by
// half_down of it and, read, by half_up.
__device__ __forceinline__ float power(uint32_t x) { return __builtin_bit_cast(float, x << 23); }
__device__ __forceinline__ uint32_t exponent(float x) { return __builtin_bit_cast(uint32_t, x) >> 23 & 0xFF; }
__device__ __forceinline__ uint32_t half_exponent(float largest) {
  const uint32_t e = exponent(largest);
  return e < 15 ? 15 : e > 254 ? 254 : e;
}
__device__ __forceinline__ float half_down(uint32_t x) { return power(268 - x); }
__device__ __forceinline__ float half_up(uint32_t x) { return power(x - 14); }
constexpr int kHalfZero = 127 + 14;  // the half_exponent whose half_up is 1

// A wave's rows of S or dS as they are kept, of a workgroup's columns from v0
// on: one power for all of them.
template <typename Saved, int DK, int TK, int TV>
__device__ __forceinline__ void keep_state(char *all, uint8_t *powers, int64_t slot_head, int dvp, int v0, int w, int row, int y,
                                           const f32x4 (&v)[TK][TV]) {
  char *rows = all + (slot_head * dvp + v0 / 32 * 32) * (DK * int64_t(sizeof(Saved)));
  if constexpr (sizeof(Saved) == 4) {
#pragma unroll
    for (int i = 0; i < TK; i++) put_block<float, TV>(rows, row + 16 * i, v0 % 32 + y, v[i]);
  } else {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < TK; i++)
#pragma unroll
      for (int j = 0; j < 4 * TV; j++) m = fmaxf(m, fabsf(v[i][j / 4][j % 4]));
    const uint32_t x = half_exponent(max_rows(max16(m)));
#pragma unroll
    for (int i = 0; i < TK; i++) {
      f32x4 s[TV];
#pragma unroll
      for (int j = 0; j < TV; j++) s[j] = v[i][j] * half_down(x);
      put_block<f16, TV>(rows, row + 16 * i, v0 % 32 + y, s);
    }
    const int l = threadIdx.x & 63;
    if (l < TV) powers[(slot_head * (dvp / 16) + v0 / 16 + l) * 4 + w] = uint8_t(x);
  }
}

// A token's share of U or Y as it is kept, of a workgroup's columns: one power
// for all of them. Every lane of the token takes part.
template <typename Kept, int TV>
__device__ __forceinline__ void keep_block(char *all, float *scales, int64_t slot_head, int dvp, int v0, int t, int quad, int y,
                                           const f32x4 (&v)[TV]) {
  char *rows = all + (slot_head * dvp + v0 / 32 * 32) * (kChunk * int64_t(sizeof(Kept)));
  if constexpr (sizeof(Kept) == 4) {
    put_block<float, TV>(rows, t, v0 % 32 + y, v);
  } else {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 4 * TV; i++) m = fmaxf(m, fabsf(v[i / 4][i % 4]));
    const uint32_t x = half_exponent(max_rows(m));
    f32x4 s[TV];
#pragma unroll
    for (int j = 0; j < TV; j++) s[j] = v[j] * half_down(x);
    put_block<f16, TV>(rows, t, v0 % 32 + y, s);
    if (quad < TV) scales[(slot_head * dvp + v0) * (kChunk / 16) + quad * kChunk + t] = half_up(x);
  }
}

template <typename T>
__device__ __forceinline__ Raw8<T> load_block8(const char *rows, uint32_t at) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < int(sizeof(T) * 8 / 16); i++)
    reinterpret_cast<u32x4 *>(&r)[i] = reinterpret_cast<const u32x4 *>(rows + at * uint32_t(sizeof(T)))[i];
  return r;
}

// Eight values that are kept in f16 with a power of two, or in f32.
template <typename Kept>
__device__ __forceinline__ Raw8<float> kept8(const Raw8<Kept> &r, float power) {
  Raw8<float> x;
#pragma unroll
  for (int i = 0; i < 8; i++) x.x[i] = sizeof(Kept) < 4 ? power * float(r.x[i]) : float(r.x[i]);
  return x;
}

// The first N planes of a fragment.
template <int N, int M>
__device__ __forceinline__ Frag<N> first_planes(const Frag<M> &f) {
  Frag<N> r;
#pragma unroll
  for (int i = 0; i < N; i++) r.p[i] = f.p[i];
  return r;
}

template <typename Mode>
int64_t record_bytes(bool back) {
  return Record<Mode>::bytes(back);
}

void delta_chunk_launch(const cchip_gated_delta &op, const DeltaArgs &a, bool back, hipStream_t stream);
void delta_forward_launch(const cchip_gated_delta &op, const DeltaArgs &a, bool back, hipStream_t stream);
void delta_backward_launch(const cchip_gated_delta &op, const DeltaArgs &a, hipStream_t stream);
void delta_step_launch(const cchip_gated_delta &op, const DeltaArgs &a, hipStream_t stream);

// Whether forward and reverse take 16 value columns a workgroup and not 32:
// where so many workgroups still find a unit each, as a chunk of 16 columns
// takes less time than one of 32 (forward of 16384 tokens, 32 bf16 heads of
// 128: 570 us in 256 workgroups, 878 in 128). Beyond that 32 do more at once:
// forward and reverse of 3 x 4096 tokens, 16 heads, take 533 us in 192
// workgroups and 573 in 384, of 4 x 4096 and 32 heads 767 and 1107.
inline bool narrow_blocks(const DeltaArgs &a) { return a.sequences * a.hv * ((a.dv + 31) / 32) <= 128; }

// Workgroups of delta_forward and delta_reverse a unit is to hold: two where
// their LDS leaves room. (With keys of up to 64 elements f32 and f16 would
// have it too, but not the registers: they spill, and run no faster.)
template <typename M>
constexpr int groups_a_unit(int dk, int bv) {
  return M::NI > 1 || (M::NS > 2 && dk * bv > 128 * 16) ? 1 : 2;
}

inline int padded_key_dim(int dk) { return dk <= 64 ? 64 : 128; }

template <typename F>
void with_bool(bool x, F &&f) {
  if (x) f(std::true_type());
  else f(std::false_type());
}

// Calls f with how the heads of an operator are read. The four kernels of an
// f32 training step of 2 x 2048 tokens, 8 heads of 70 x 90, take 461 us in
// pieces and 668 us an element at a time; of a bf16 step of 2 x 4096 tokens, 8
// heads of 100 x 100, 464 and over 1080. Whole heads spare the shifts: 8 heads of
// 72 x 100 of 5003 tokens in f32 take 497 us whole and 565 in pieces.
template <typename T, typename F>
void with_access(const DeltaArgs &a, F &&f) {
  constexpr int E = 16 / sizeof(T);
  if (a.dk % 8 == 0 && a.dv % E == 0) f(std::integral_constant<int, kWhole>());
  else if (a.dk >= E && a.dv >= E) f(std::integral_constant<int, kPieces>());
  else f(std::integral_constant<int, kSingle>());
}

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
