// Causal attention with grouped heads (attention*.hip).
//
// The heads of a group share keys, so the queries of a sequence and key head
// are one matrix of tokens x group rows: row r is head r % group of token
// r / group. A row sees the keys up to its token's own, counted from the end
// of both.
//
// Products are made transposed, on the 32 x 32 x 16 matrix instruction:
// S^T = K Q^T has a query a lane (two lanes, 32 apart, share its 32 keys), so
// a softmax's maximum and sum stay in the lane but for one exchange, and what
// a lane has of P^T is, packed, already the operand that O^T = V^T P^T takes:
// of each 16 keys lane half h has 4 h .. + 3 and 8 + 4 h .. + 3, and V's
// fragment is read in that order of keys.
#pragma once

#include <type_traits>

#include "heads.hpp"

namespace cchip {
namespace op {

typedef float f32x16 __attribute__((ext_vector_type(16)));

struct AttentionArgs {
  Heads q, k, v, o;
  Heads d_o, gq, gk, gv;
  const int32_t *offsets;  // packed sequences
  const int32_t *lengths;  // of a cache's sequences
  float *lse;              // log2 of a row's sum: [batch][key head][token][head of the group], or null
  bf16 *o_rest;            // what rounding o to 16 bits left, as lse with `dim` a row, or null
  // backward (attention_backward.hpp): tiles of q, the gradient of o, k and v,
  // and what belongs to a tile of rows and of keys
  u32x4 *tiles[4];
  float *row_heads;
  int32_t *key_heads;
  int row_slots, key_slots;
  int chunks;        // of the rows that see a key, kept apart until they are summed
  int chunk_tiles;   // tiles of rows in a chunk
  uint32_t *queues;  // kQueues of the rows' workgroups, then of the keys'
  uint32_t pairs;
  float *partial;          // of splits: [row][split][dim], then the maximum and sum of each; backward: of
                           // chunks, [slot of keys][chunk][dk, dv][kUnit][dim]
  int64_t tokens, keys;    // of a row of the batch; keys: of the cache, or the tokens
  int64_t sequences;       // packed; 0: the batch's rows
  int64_t batch;
  int kv_heads, group, dim;
  int slots;    // forward, tiles of rows: of a sequence, or of the packed batch
  int splits;   // of the keys
  uint32_t workgroups;
  float scale;  // times log2(e), positive
  float plain_scale;
  bool negate;  // the scale is negative: queries count negated
};

// ---- element types ------------------------------------------------------------

// N planes (operators.hpp) of 16 bits: bf16 and f16 as they are, f32 in three
// bf16 planes, of whose products those below 2^-24 are left out. Six bf16
// products are faster than one of f32: 2.5 PFLOP/s / 6 against 157 TFLOP/s.
template <typename T>
struct Planes {
  static constexpr int N = std::is_same<T, float>::value ? 3 : 1;
  static constexpr int kWaves = N == 1 ? 2 : 1;  // of a SIMD, by the registers that they need
  typedef typename std::conditional<std::is_same<T, f16>::value, f16, bf16>::type E;
};

template <int N>
struct Bits {
  u32x4 p[N];
};

template <typename T>
__device__ __forceinline__ f32x16 mma32(const u32x4 &a, const u32x4 &b, f32x16 c) {
  if constexpr (std::is_same<T, f16>::value)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// c += a b^T over 16 terms: lane l holds row (column) l % 32 of a (b), terms
// 8 (l / 32) .. + 7, and of c column l % 32, rows 8 (i / 4) + 4 (l / 32) + i % 4.
// Small products first.
template <typename T, int N>
__device__ __forceinline__ f32x16 product(f32x16 c, const Bits<N> &a, const Bits<N> &b) {
#pragma unroll
  for (int s = N - 1; s >= 0; s--)
#pragma unroll
    for (int i = 0; i <= s; i++) c = mma32<T>(a.p[i], b.p[s - i], c);
  return c;
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), f16x2));
}

// Eight values as an operand's; `first` is what the first of several planes is
// rounded from.
template <typename T>
__device__ __forceinline__ Bits<Planes<T>::N> planes_of(const float *x, const float *first) {
  Bits<Planes<T>::N> r;
  if constexpr (std::is_same<T, f16>::value) {
#pragma unroll
    for (int i = 0; i < 4; i++) r.p[0][i] = pack_f16(x[2 * i], x[2 * i + 1]);
  } else {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; i++) y[i] = x[i];
#pragma unroll
    for (int n = 0; n < Planes<T>::N; n++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const uint32_t u = n ? pack_bf16(y[2 * i], y[2 * i + 1]) : pack_bf16(first[2 * i], first[2 * i + 1]);
        r.p[n][i] = u;
        if (n + 1 < Planes<T>::N) y[2 * i] -= low_bf16(u), y[2 * i + 1] -= high_bf16(u);
      }
  }
  return r;
}

template <typename T>
__device__ __forceinline__ Bits<Planes<T>::N> operand_of(const float *x) {
  return planes_of<T>(x, x);
}

template <typename T>
__device__ __forceinline__ Bits<Planes<T>::N> bits_of(const Raw8<T> &r) {
  if constexpr (std::is_same<T, float>::value) {
    return operand_of<T>(r.x);
  } else {
    Bits<1> b;
    b.p[0] = *reinterpret_cast<const u32x4 *>(&r);
    return b;
  }
}

// The same of finite elements however large: what would round to an infinity
// has the largest bf16 as its first plane, and the others hold the rest.
template <typename T>
__device__ __forceinline__ Bits<Planes<T>::N> whole_bits_of(const Raw8<T> &r) {
  if constexpr (std::is_same<T, float>::value) {
    constexpr float kMost = 0x1.FEp127f;
    float first[8];
#pragma unroll
    for (int i = 0; i < 8; i++) first[i] = __builtin_amdgcn_fmed3f(r.x[i], -kMost, kMost);
    return planes_of<T>(r.x, first);
  } else {
    return bits_of<T>(r);
  }
}

template <typename T>
__device__ __forceinline__ Raw8<T> negated(Raw8<T> r) {
#pragma unroll
  for (int i = 0; i < 8; i++) r.x[i] = -r.x[i];
  return r;
}

// Made here, among the products that it stands between, and not where it is
// used.
__device__ __forceinline__ float stay(float x) {
  asm volatile("" : "+v"(x));
  return x;
}

// ---- tiles in LDS ---------------------------------------------------------------

// A tile of rows of D elements of 16 bits, a plane after another, a row's
// pieces of 16 bytes exchanged by a number of the row's. Rows lie in groups of
// 1 KB, which are 16 bytes apart: 16 rows' pieces of one column lie in banks of
// their own, as do four neighbouring rows' 64 bytes, which is what the two
// kinds of reads below take at a time, and groups of rows are a constant apart,
// so that few registers address them all.
constexpr int kGroup = 520;  // elements from group to group

template <int D>
__device__ __forceinline__ int twist(int row) {
  return D == 128 ? (row & 3) << 2 : (((row >> 1) & 1) << 2) | (((row >> 2) & 1) << 1);
}

template <int D>
__device__ __forceinline__ int piece_at(int row, int piece) {
  constexpr int kRows = 512 / D;
  return row / kRows * kGroup + (row % kRows * (D / 8) + (piece ^ twist<D>(row))) * 8;
}

template <int D>
constexpr int tile_elements(int rows) { return rows * D / 512 * kGroup; }

// A lane's places in a tile of the operands that it reads.
template <int D>
struct Places {
  int rows[4], columns[D / 32];
  __device__ __forceinline__ Places() {
    const int l = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < 4; i++) rows[i] = piece_at<D>(l & 31, (D == 128 ? 4 * i : 2 * i) + (l >> 5));
    const int row = 4 * (l >> 5) + ((l >> 2) & 3), col = (l & 16) + (l & 3) * 4;
#pragma unroll
    for (int i = 0; i < D / 32; i++) columns[i] = piece_at<D>(row, 4 * i + (col >> 3)) + (col & 4);
  }
};

// Rows row0 + l % 32, terms 16 step + 8 (l / 32) .. + 7.
template <int N, int D, typename E>
__device__ __forceinline__ Bits<N> rows_of_tile(const Places<D> &at, const E *m, int plane, int row0, int step) {
  const E *p = m + (D == 128 ? at.rows[step / 2] + step % 2 * 16 : at.rows[step]) + row0 * D / 512 * kGroup;
  Bits<N> f;
#pragma unroll
  for (int n = 0; n < N; n++) f.p[n] = *reinterpret_cast<const u32x4 *>(p + n * plane);
  return f;
}

// Columns col0 + l % 32 as rows; terms are the tile's rows row0 + 4 (l / 32)
// .. + 3 and row0 + 8 + 4 (l / 32) .. + 3: the transposing LDS read, which
// gives lane i of 16 column i of the four rows whose 4 elements each the 16
// lanes address.
template <int N, int D, typename E>
__device__ __forceinline__ Bits<N> columns_of_tile(const Places<D> &at, const E *m, int plane, int row0, int col0) {
  typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
  const E *a = m + at.columns[col0 / 32] + row0 * D / 512 * kGroup;
  Bits<N> f;
#pragma unroll
  for (int n = 0; n < N; n++) {
    union {
      i16x4 h[2];
      u32x4 v;
    } u;
    u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(a + n * plane));
    u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(a + n * plane + 8 * D / 512 * kGroup));
    f.p[n] = u.v;
  }
  return f;
}

// What is on its way from memory is there.
__device__ __forceinline__ void copies_done() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0F70);
  asm volatile("" ::: "memory");
}

// Rows of a tensor on their way to a tile: pieces of 8 elements, `Threads`
// threads that read a row one after another. Rows from `rows` on and elements
// from dim on are zero and not read.
template <typename T, int D, int Rows, int Threads>
struct Staged {
  static constexpr int kPieces = D / 8, kEach = Rows * kPieces / Threads;
  static_assert(Rows * kPieces % Threads == 0, "every thread has as many pieces");
  Raw8<T> r[kEach];

  static __device__ __forceinline__ int row(int t, int i) { return (t + i * Threads) / kPieces; }
  static __device__ __forceinline__ int piece(int t, int i) { return (t + i * Threads) % kPieces; }

  __device__ __forceinline__ void load(int t, const T *p, int64_t stride, int64_t rows, int dim) {
    if (rows >= Rows && dim == D) {
#pragma unroll
      for (int i = 0; i < kEach; i++) r[i] = load8<T>(p + row(t, i) * stride + piece(t, i) * 8, 8);
    } else if (dim % 8 == 0) {
#pragma unroll
      for (int i = 0; i < kEach; i++) {
        r[i] = Raw8<T>{};
        if (row(t, i) < rows && piece(t, i) * 8 < dim) r[i] = load8<T>(p + row(t, i) * stride + piece(t, i) * 8, 8);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kEach; i++) {
        const int left = dim - piece(t, i) * 8;
        r[i] = load8<T>(p + row(t, i) * stride + piece(t, i) * 8, row(t, i) < rows && left > 0 ? (left < 8 ? left : 8) : 0);
      }
      // the elements' registers are used otherwise where rows are whole: a
      // wait here, or there it would be for what is on its way
      copies_done();
    }
  }

  template <typename E>
  __device__ __forceinline__ void store(int t, E *m) const {
#pragma unroll
    for (int i = 0; i < kEach; i++) store_piece(t, i, m, bits_of<T>(r[i]));
  }
  template <typename E>
  __device__ __forceinline__ void store_whole(int t, E *m) const {
#pragma unroll
    for (int i = 0; i < kEach; i++) store_piece(t, i, m, whole_bits_of<T>(r[i]));
  }
  template <typename E>
  static __device__ __forceinline__ void store_piece(int t, int i, E *m, const Bits<Planes<T>::N> &b) {
#pragma unroll
    for (int n = 0; n < Planes<T>::N; n++)
      *reinterpret_cast<u32x4 *>(m + n * tile_elements<D>(Rows) + piece_at<D>(row(t, i), piece(t, i))) = b.p[n];
  }
};

// The wave of the workgroup, in a scalar register as all that follows from it.
__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)); }

// In a branch that most waves do not take: keeps the compiler from taking it
// always and selecting.
__device__ __forceinline__ void stay_branch() { asm volatile(""); }

// 16 bytes a lane from memory to LDS without registers, lane after lane from
// `to`, which is the wave's; `offset` bytes, below 2^32, are the lane's. As the
// compiler sees it every read of LDS after such a copy has to wait for all of
// them, also those that go to other tiles; an instruction that it does not see
// leaves the waiting to copies_left. It writes no vector register, so nothing
// that is in use can be overwritten by it, and m0, which the compiler keeps
// nothing in.
__device__ __forceinline__ void copy_lanes(const void *from, uint32_t offset, void *to) {
  // both are the wave's; the instruction takes them from scalar registers
  const uint64_t source = reinterpret_cast<uint64_t>(from);
  const uint64_t base = uint64_t(uint32_t(__builtin_amdgcn_readfirstlane(int(source >> 32)))) << 32 | uint32_t(__builtin_amdgcn_readfirstlane(int(source)));
  const uint32_t at = __builtin_amdgcn_readfirstlane(int(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char *)to)));
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(at), "v"(offset), "s"(base) : "memory");
}

// All but the last Left copies and loads of the wave are there.
template <int Left>
__device__ __forceinline__ void copies_left() {
  static_assert(Left < 64, "as many as the counter has");
  asm volatile("s_waitcnt vmcnt(%0)" ::"i"(Left) : "memory");
}

// The same rows, of 16-bit elements at 16-byte places, copied to a tile
// directly. Pieces behind dim are not written: the tile has zeros there from
// the start. Rows from `rows` on are the last one again: what they give has to
// be masked.
template <int D, int Rows, int Threads>
struct Copied {
  static constexpr int kPieces = D / 8, kEach = Rows * kPieces / Threads;
  uint32_t offset[kEach];  // bytes from the tile's first row
  bool live[kEach];

  static __device__ __forceinline__ int row(int i) { return (i * Threads + int(threadIdx.x)) / kPieces; }

  __device__ __forceinline__ void start(int64_t stride, int dim) {
#pragma unroll
    for (int i = 0; i < kEach; i++) {
      const int piece = (i * Threads + int(threadIdx.x)) % kPieces ^ twist<D>(row(i));
      live[i] = piece * 8 < dim;
      offset[i] = (uint32_t(row(i)) * uint32_t(stride) + piece * 8) * 2;
    }
  }
  __device__ __forceinline__ void copy(const char *from, uint32_t stride, int rows, int dim, char *to) const {
#pragma unroll
    for (int i = 0; i < kEach; i++) {
      uint32_t at = offset[i];
      if (rows < Rows) {
        stay_branch();
        if (row(i) >= rows) at -= uint32_t(row(i) - rows + 1) * stride * 2;
      }
      char *const there = to + (i * Threads / 64 + wave_index()) * (kGroup * 2);
      if (dim == D) {
        copy_lanes(from, at, there);
      } else if (live[i]) {
        copy_lanes(from, at, there);
      }
    }
  }
};

// ---- lanes ------------------------------------------------------------------------

// A kernel of so many threads whose registers are for exactly so many waves a
// SIMD: the compiler knows nothing of the LDS that a launch asks for, and would
// save registers, and keep loads next to their uses, for waves that never come.
#define CCHIP_WAVES(threads, waves) __launch_bounds__(threads, waves) __attribute__((amdgpu_waves_per_eu(waves, waves)))

// All waves are here, and what they wrote to LDS is there; loads from memory
// stay on their way.
__device__ __forceinline__ void phase_done() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// use(i, operand) for i below Count, each operand read(i) from LDS Depth of
// them ahead. The compiler would read each just before its product and wait.
template <int Count, int Depth, int N>
struct Ahead {
  static constexpr int kDepth = Depth < Count ? Depth : Count;
  Bits<N> f[kDepth];
  template <typename Read>
  __device__ __forceinline__ void start(const Read &read) {
#pragma unroll
    for (int i = 0; i < kDepth; i++) f[i] = read(i);
    __builtin_amdgcn_sched_barrier(0);
  }
  template <typename Read, typename Use>
  __device__ __forceinline__ void run(const Read &read, const Use &use) {
    run(read, use, [](int) {});
  }
  // With work(i) after each product: vector instructions while it is made.
  template <typename Read, typename Use, typename Work>
  __device__ __forceinline__ void run(const Read &read, const Use &use, const Work &work) {
#pragma unroll
    for (int i = 0; i < Count; i++) {
      use(i, f[i % kDepth]);
      if (i + kDepth < Count) f[i % kDepth] = read(i + kDepth);
      work(i);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

// x of the lane 32 on or before.
__device__ __forceinline__ float other_half(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t lo = a[0], hi = a[1];
  return __builtin_bit_cast(float, (threadIdx.x & 32) ? lo : hi);
}

__device__ __forceinline__ float max_halves(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t lo = a[0], hi = a[1];
  return fmaxf(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
}

__device__ __forceinline__ float sum_halves(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t lo = a[0], hi = a[1];
  return __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
}

// ---- which rows and keys a workgroup has --------------------------------------------

// A lane's value for all, in scalar registers.
__device__ __forceinline__ int of_lane(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }

struct Span {
  int64_t batch;       // row of the batch
  int64_t first;       // token its rows begin at
  int64_t rows;        // tokens x group
  int64_t keys;        // of the sequence
  int64_t ahead;       // key that token 0 sees last
  int64_t key0;        // row of k and v that the sequence's keys begin at
  int kv;
  int tile;            // of rows (or keys, backward), heavy ones first; < 0: nothing to do
  int chunk;
  int64_t row_base, key_base;  // tiles of rows and of keys of the pairs and sequences before, as tall as this one
};

// Workgroups go to the eight dies in turn, each with a second-level cache of
// its own: those of one sequence and key head, which read the same keys, run on
// one die; eight pairs at a time, each die all tiles of its own.
__device__ __forceinline__ void pair_a_die(uint32_t id, uint32_t pairs, uint32_t slots, uint32_t &pair, uint32_t &slot) {
  const uint32_t set = id / (8 * slots), in = id - set * 8 * slots;
  const uint32_t here = pairs - set * 8 < 8 ? pairs - set * 8 : 8;
  slot = in / here;
  pair = set * 8 + in - slot * here;
}

__device__ __forceinline__ int64_t clamped(int64_t x, int64_t most) { return x < 0 ? 0 : x > most ? most : x; }

// Tiles of `height` rows, `per_token` to a token; `last_first`: tiles of a
// sequence are counted from its end. `slots` are what the pair has tiles for;
// with `chunks` of each there are those of the first chunk first.
__device__ __forceinline__ Span span_of(const AttentionArgs &a, uint32_t id, uint32_t slots, int per_token, int height, bool last_first,
                                        uint32_t chunks = 1) {
  Span s;
  uint32_t pair, slot;
  pair_a_die(id, uint32_t((a.sequences ? 1 : a.batch) * a.kv_heads), slots * chunks, pair, slot);
  s.chunk = int(slot / slots);
  slot %= slots;
  int64_t tokens = a.tokens, tiles = slots;
  s.kv = int(pair % uint32_t(a.kv_heads));
  s.batch = pair / uint32_t(a.kv_heads);
  s.first = 0;
  s.key0 = 0;
  s.tile = int(slot);
  s.keys = a.keys;
  s.row_base = int64_t(pair) * a.row_slots;
  s.key_base = int64_t(pair) * a.key_slots;
  if (a.sequences) {
    // the sequence whose tiles this slot is among: 64 sequences at a time
    const int l = threadIdx.x & 63;
    int64_t before = 0;
    int tile = -1;
    for (int64_t s0 = 0; s0 < a.sequences; s0 += 64) {
      const int64_t i = s0 + l;
      int64_t lo = 0, hi = 0;
      if (i < a.sequences) {
        lo = clamped(a.offsets[i], a.tokens);
        hi = clamped(a.offsets[i + 1], a.tokens);
        if (hi < lo) hi = lo;
      }
      const int mine = int(((hi - lo) * per_token + height - 1) / height);
      const int rows = int(((hi - lo) * a.group + height - 1) / height), keys = int((hi - lo + height - 1) / height);
      int upto = mine, upto_rows = rows, upto_keys = keys;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const int x = __shfl_up(upto, d, 64), y = __shfl_up(upto_rows, d, 64), z = __shfl_up(upto_keys, d, 64);
        if (l >= d) upto += x, upto_rows += y, upto_keys += z;
      }
      const int64_t at = int64_t(slot) - before;
      const uint64_t found = __ballot(at < upto);
      if (found) {
        const int w = __ffsll((unsigned long long)found) - 1;
        s.first = of_lane(int(lo), w);
        tokens = of_lane(int(hi), w) - s.first;
        tiles = of_lane(mine, w);
        tile = int(at) - (of_lane(upto, w) - int(tiles));
        s.row_base += of_lane(upto_rows - rows, w);
        s.key_base += of_lane(upto_keys - keys, w);
        // offsets that decrease: what lies behind the tiles there is room for
        const int64_t past = int64_t(pair) + 1;
        if (a.row_slots && (s.row_base + of_lane(rows, w) > past * a.row_slots || s.key_base + of_lane(keys, w) > past * a.key_slots)) tile = -1;
        break;
      }
      before += of_lane(upto, 63);
      s.row_base += of_lane(upto_rows, 63);
      s.key_base += of_lane(upto_keys, 63);
    }
    s.tile = tile;
    s.batch = 0;
    s.key0 = s.first;
    s.keys = tokens;
  } else if (a.lengths) {
    s.keys = clamped(a.lengths[s.batch], a.keys);
  }
  s.rows = tokens * a.group;
  s.ahead = s.keys - tokens;
  if (s.tile >= 0 && last_first) s.tile = int(tiles) - 1 - s.tile;
  return s;
}

// Workgroups that take one job after another: the hardware hands its own out in
// order, each to the next of a die's four engines, so that one waits for a unit
// of its engine while others idle: up to half the time where jobs differ in
// length, and two thirds where engines differ in units. A die has a queue of
// every eighth job (see above) and goes on with the next one's when that is
// empty. What a job does is the same whoever has it. There are some more
// workgroups than units, as those of an engine that has no room find nothing
// left.
constexpr uint32_t kTakers = 320;
constexpr uint32_t kQueues = 8;

struct Jobs {
  uint32_t *queue;
  uint32_t count, tried, die;
  __device__ __forceinline__ Jobs(uint32_t *queues, uint32_t jobs) : queue(queues), count(jobs), tried(0), die(blockIdx.x % kQueues) {}
  // the next, or `count`; `place` is in LDS
  __device__ __forceinline__ uint32_t next(uint32_t &place) {
    __syncthreads();
    if (threadIdx.x == 0) {
      uint32_t job = count;
      while (tried < kQueues && job >= count) {
        const uint32_t q = (die + tried) % kQueues;
        job = q + kQueues * atomicAdd(&queue[q], 1u);
        if (job >= count) tried++;
      }
      place = job;
    }
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(place);
  }
};

__device__ __forceinline__ const char *element(const Heads &x, int64_t b, int64_t t, int64_t h, int size) {
  return x.p + (b * x.b + t * x.t + h * x.h) * size;
}

// Lse of a span's row 0.
__device__ __forceinline__ int64_t row_values(const AttentionArgs &a, const Span &s) {
  return ((s.batch * a.kv_heads + s.kv) * a.tokens + s.first) * a.group;
}

}  // namespace op
}  // namespace cchip
