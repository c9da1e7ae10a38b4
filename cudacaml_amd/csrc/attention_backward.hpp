// Attention, backward. With P = 2^(scores - lse) and D = do . o of each row,
//
//   dV = P^T dO,  dS = P (dO V^T - D),  dQ = scale dS K,  dK = scale dS^T Q
//
// One kernel goes over the keys for the rows' gradients and one over the rows
// for the keys' and values', so that every gradient is a sum in registers, in
// an order that does not change: what it costs is that scores and dO V^T are
// made twice, seven products in place of five. The rows of a group's heads are
// rows like others (attention.hpp), so the keys' gradients sum over them.
//
// A kernel before them lays q, dO, k and v out as both take them: tiles of
// kHigh rows as they lie in LDS, which are copied there without passing
// through registers, with zeros for rows and elements that there are not. 16-bit
// tensors become f16 times a power of two for each tile, exact but for what is
// 2^-28 of the tile's largest value and less: P and dS can then be f16 as well,
// whose 11 bits add little to the rounding of a bf16 gradient (in bf16 they
// would make it 1.5 times as much). f32 becomes three bf16 planes.
//
// 8192 packed tokens, 16 heads of 128 over 4, bf16, 407 GFLOP with the forward
// pass's 192 us: 45 us for laying out, 227 for the rows, 367 for the keys and
// 20 for the sums of chunks, 838 together. The rows' kernel has two waves a
// SIMD; the keys' has registers for one, with vector instructions in the way
// of its products: 2.5 us for 64 rows and 128 keys, of which the products are
// 0.9. Of some 540 vector instructions a tile and wave 192 read accumulators that only
// the seldom branch of `settle` uses: the compiler moves them before it.

#include <algorithm>

#include "attention_forward.hpp"

namespace cchip {
namespace op {

constexpr int kUnit = 128;  // rows or keys of a workgroup

// Terms are 2^kLift P in f16, normal down to 2^-29.
template <typename T>
struct Backward {
  static constexpr int N = Planes<T>::N;
  static constexpr bool kScaled = N == 1;
  static constexpr int kHigh = kScaled ? 64 : 32;  // rows of a tile
  static constexpr float kLift = 15.0f;
  typedef typename std::conditional<kScaled, f16, float>::type M;  // the products' type
};

// What belongs to a tile of rows: the lse and do . o of each and the powers of
// two of q and of the gradient of o; to one of keys: those of k and of v.
template <typename T>
constexpr int kRowHead = 2 * Backward<T>::kHigh + 4;
constexpr int kKeyHead = 2;

// Power of two of a tile without finite values other than zero.
constexpr int kNoPower = 100;

// 2^e, as far as that times a value of f16 is one of f32.
__device__ __forceinline__ float power_of_two(int e) {
  return __builtin_bit_cast(float, uint32_t((e < -126 ? -126 : e > 100 ? 100 : e) + 127) << 23);
}

// ---- laying out ---------------------------------------------------------------------

// A tile of a tensor: x's kHigh rows from row0, its power of two and, for the
// gradient of o, each row's product with o, as much of it as o's type has
// not rounded off, and its lse.
template <typename T, int D>
__device__ __forceinline__ void lay_tile(const AttentionArgs &a, const Heads &x, const Span &s, int64_t row0, int64_t rows, int per_token,
                                         u32x4 *to, int32_t *power, bool with_o, float *lse, float *dot) {
  typedef Backward<T> B;
  constexpr int kPieces = D / 8, kEach = B::kHigh * kPieces / 256;
  __shared__ uint32_t most[4];
  const int t = threadIdx.x, l = t & 63, piece = t % kPieces;
  Raw8<T> r[kEach];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kEach; i++) {
    const int at = (t + i * 256) / kPieces;
    const int64_t row = row0 + at;
    const bool live = row < rows;
    const uint32_t token = live ? uint32_t(uint64_t(row) / uint32_t(per_token)) : 0, in = live ? uint32_t(row - int64_t(token) * per_token) : 0;
    const int64_t head = per_token == 1 ? s.kv : int64_t(s.kv) * per_token + in;
    const int left = a.dim - piece * 8, n = live && left > 0 ? (left < 8 ? left : 8) : 0;
    r[i] = load8<T>(reinterpret_cast<const T *>(element(x, s.batch, s.first + token, head, sizeof(T))) + piece * 8, n);
    if constexpr (B::kScaled) {
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const uint32_t u = __builtin_bit_cast(uint32_t, float(r[i].x[j])) & 0x7FFFFFFFu;
        top = u < 0x7F800000u && u > top ? u : top;
      }
    }
    if (with_o) {
      const Raw8<T> y = load8<T>(reinterpret_cast<const T *>(element(a.o, s.batch, s.first + token, head, sizeof(T))) + piece * 8, n);
      float sum = 0.0f;
      if constexpr (B::kScaled) {
        const Raw8<bf16> z = load8<bf16>(a.o_rest + (row_values(a, s) + (live ? row : 0)) * a.dim + piece * 8, n);
#pragma unroll
        for (int j = 0; j < 8; j++) sum += float(r[i].x[j]) * (float(y.x[j]) + float(z.x[j]));
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++) sum += r[i].x[j] * y.x[j];
      }
#pragma unroll
      for (int d = 1; d < kPieces; d *= 2) sum += __shfl_xor(sum, d, 64);
      if (piece == 0) {
        dot[at] = sum;
        lse[at] = live ? a.lse[row_values(a, s) + row] : INFINITY;
      }
    }
  }
  if constexpr (B::kScaled) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const uint32_t u = __shfl_xor(top, d, 64);
      top = u > top ? u : top;
    }
    if (!l) most[t >> 6] = top;
    __syncthreads();
    top = most[0];
#pragma unroll
    for (int i = 1; i < 4; i++) top = most[i] > top ? most[i] : top;
    // the largest becomes 2^14 and more
    int e = top ? 14 + 127 - int(top >> 23) : kNoPower;
    if (e > kNoPower) e = kNoPower;
    const float up = power_of_two(e);
    if (!t) *power = e;
#pragma unroll
    for (int i = 0; i < kEach; i++) {
      u32x4 u;
#pragma unroll
      for (int j = 0; j < 4; j++) u[j] = pack_f16(float(r[i].x[2 * j]) * up, float(r[i].x[2 * j + 1]) * up);
      to[(t + i * 256) / kPieces * kPieces + (piece ^ twist<D>((t + i * 256) / kPieces))] = u;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kEach; i++) {
      const Bits<B::N> b = whole_bits_of<T>(r[i]);  // an infinity's are NaN
#pragma unroll
      for (int n = 0; n < B::N; n++) to[(n * B::kHigh + (t + i * 256) / kPieces) * kPieces + (piece ^ twist<D>((t + i * 256) / kPieces))] = b.p[n];
    }
  }
}

// 16-byte pieces of a tile.
template <typename T, int D>
constexpr int kTilePieces = Backward<T>::N *Backward<T>::kHigh *D / 8;

// Tiles of q, then of the gradient of o, then of k and of v.
template <typename T, int D>
__global__ __launch_bounds__(256) void lay_out(const AttentionArgs a) {
  typedef Backward<T> B;
  constexpr int kTiles = kUnit / B::kHigh;
  uint32_t id = block_index();
  if (id >= a.workgroups) return;
  if (id == 0 && threadIdx.x < 2 * kQueues) a.queues[threadIdx.x] = 0;
  const uint32_t pairs = a.pairs, row_tiles = pairs * uint32_t(a.row_slots) * kTiles, key_tiles = pairs * uint32_t(a.key_slots) * kTiles;
  int which = 0;
  if (id >= row_tiles) id -= row_tiles, which = 1;
  if (which == 1 && id >= row_tiles) id -= row_tiles, which = 2;
  if (which == 2 && id >= key_tiles) id -= key_tiles, which = 3;
  const bool rows = which < 2;
  const int per_token = rows ? a.group : 1;
  const Span s = span_of(a, id / kTiles, uint32_t(rows ? a.row_slots : a.key_slots), per_token, kUnit, false);
  if (s.tile < 0) return;
  const int64_t tile = (rows ? s.row_base : s.key_base) * kTiles + s.tile * kTiles + id % kTiles;
  const int64_t row0 = (int64_t(s.tile) * kTiles + id % kTiles) * B::kHigh, count = rows ? s.rows : s.keys;
  float *head = a.row_heads + tile * kRowHead<T>;
  int32_t *powers = rows ? reinterpret_cast<int32_t *>(head + 2 * B::kHigh) : a.key_heads + tile * kKeyHead;
  const Heads x = which == 0 ? a.q : which == 1 ? a.d_o : which == 2 ? a.k : a.v;
  u32x4 *to = which == 0 ? a.tiles[0] : which == 1 ? a.tiles[1] : which == 2 ? a.tiles[2] : a.tiles[3];
  lay_tile<T, D>(a, x, s, row0, count, per_token, to + tile * kTilePieces<T, D>, powers + which % 2, which == 1, head, head + B::kHigh);
}

// ---- products -------------------------------------------------------------------------

// A tile in memory to LDS, 1 KB an instruction and group of rows, which four
// waves share: the i-th of a wave's.
__device__ __forceinline__ void copy_group(const u32x4 *from, char *to, int i) {
  copy_lanes(from, (i * 256 + threadIdx.x) * 16, to + (i * 4 + wave_index()) * (kGroup * 2));
}

template <int Pieces>
__device__ __forceinline__ void copy_tile(const u32x4 *from, char *to) {
  static_assert(Pieces % 256 == 0, "every wave copies as much");
#pragma unroll
  for (int i = 0; i < Pieces / 256; i++) copy_group(from, to, i);
}

// Rows at + l % 32 of a tile in memory as an operand.
template <typename T, int D>
__device__ __forceinline__ void load_operand(Bits<Backward<T>::N> (&q)[D / 16], const u32x4 *tile, int at) {
  const int l = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < D / 16; i++)
#pragma unroll
    for (int n = 0; n < Backward<T>::N; n++)
      q[i].p[n] = tile[(n * Backward<T>::kHigh + at + (l & 31)) * (D / 8) + ((2 * i + (l >> 5)) ^ twist<D>(l & 31))];
}

// A column's dS in f16 has a power of two, so that the largest so far is
// below 2^15: what the column has is rescaled when that grows, as a running
// maximum's, to 2^10, so that this is seldom. Takes the largest of dS as it stands and the power that the
// product needs besides; powers are counted as exponents, as the first ones
// are far from any value's.
constexpr int kFirstPower = 100;

// The exponent of the larger of a column's two lanes' values.
__device__ __forceinline__ int exponent(float most) { return int(__builtin_bit_cast(uint32_t, max_halves(most)) >> 23) - 127; }

template <int D>
__device__ __forceinline__ void lower(int &power, f32x16 (&out)[D / 32], float most, int besides) {
  const int over = exponent(most) + power + besides - 14;
  if (__builtin_expect(!__ballot(over > 0), 1)) return;
  stay_branch();
  const int by = over > 0 ? over + 4 : 0;
  const float factor = power_of_two(-by);
  power -= by;
#pragma unroll
  for (int d = 0; d < D / 32; d++) out[d] *= factor;
}

__device__ __forceinline__ float largest(const f32x16 &x) {
  float most = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; i++) most = fmaxf(most, __builtin_fabsf(x[i]));
  return most;
}

template <typename M>
__device__ __forceinline__ void operands_of(Bits<Planes<M>::N> (&p)[2], const f32x16 &x) {
#pragma unroll
  for (int h = 0; h < 2; h++) {
    float z[8];
#pragma unroll
    for (int i = 0; i < 8; i++) z[i] = x[8 * h + i];
    p[h] = operand_of<M>(z);
  }
}

// Elements from `at` on are padding: here six products of f32 are worth a
// branch (heads of 72: 76 us in place of 82), one of 16 bits is not. The other
// kernels' instructions are in an order that branches would break (of the keys'
// gradients 74 us in place of 62).
template <int N>
__device__ __forceinline__ bool no_product(int at, int dim) { return N > 1 && at >= dim; }

// kUnit rows, 32 a wave, over the keys that they see.
template <typename T, int D>
__device__ __forceinline__ void back_rows_job(const AttentionArgs &a, uint32_t id, char *lds, int (&heads)[2][kKeyHead]) {
  typedef Backward<T> B;
  typedef typename B::M M;
  typedef typename Planes<M>::E E;
  constexpr int N = B::N, kHigh = B::kHigh, kPlane = tile_elements<D>(kHigh), kBytes = N * kPlane * 2, kPieces = kTilePieces<T, D>, kTiles = kUnit / kHigh;

  const int t = threadIdx.x, l = t & 63, half = l >> 5, w = wave_index();
  const Span s = span_of(a, id, uint32_t(a.row_slots), a.group, kUnit, true);
  if (s.tile < 0) return;
  const int64_t row0 = int64_t(s.tile) * kUnit, wave_row = row0 + w * 32, row = wave_row + (l & 31);
  const int64_t last_row = s.rows - 1 < row0 + kUnit - 1 ? s.rows - 1 : row0 + kUnit - 1;
  const int64_t wave_last = s.rows - 1 < wave_row + 31 ? s.rows - 1 : wave_row + 31;
  const int64_t to = last_row / a.group + 1;  // keys that rows see
  const int64_t wave_all = wave_row / a.group + 1;
  const int64_t wave_any = wave_row < s.rows ? wave_last / a.group + 1 : 0;
  const int64_t mine = row / a.group + 1;
  const int end = int((to + kHigh - 1) / kHigh);

  const int64_t row_tile = (s.row_base + s.tile) * kTiles + w * 32 / kHigh, key_tile = s.key_base * kTiles;
  const u32x4 *k = a.tiles[2] + key_tile * kPieces, *v = a.tiles[3] + key_tile * kPieces;
  const int32_t *head_of = a.key_heads + key_tile * kKeyHead;
  int head = 0;
  if (t < kKeyHead) heads[0][t] = head_of[t];
  copy_tile<kPieces>(k, lds);
  copy_tile<kPieces>(v, lds + kBytes);

  Bits<N> q[D / 16], g[D / 16];
  const int in_tile = w * 32 % kHigh;
  load_operand<T, D>(q, a.tiles[0] + row_tile * kPieces, in_tile);
  load_operand<T, D>(g, a.tiles[1] + row_tile * kPieces, in_tile);
  const float *row_head = a.row_heads + row_tile * kRowHead<T>;
  const float lse = row_head[in_tile + (l & 31)], dot = row_head[kHigh + in_tile + (l & 31)];
  const int qe = reinterpret_cast<const int *>(row_head)[2 * kHigh], ge = reinterpret_cast<const int *>(row_head)[2 * kHigh + 1];
  const float scale = a.negate ? -a.scale : a.scale;

  const Places<D> at;
  f32x16 out[D / 32] = {};
  int power = kFirstPower;
  copies_done();
  __syncthreads();
  copies_done();
  for (int tile = 0; tile < end; tile++) {
    const int ke = of_lane(heads[tile & 1][0], 0), ve = of_lane(heads[tile & 1][1], 0);
    const E *km = reinterpret_cast<const E *>(lds + (tile & 1) * 2 * kBytes), *vm = km + N * kPlane;
    if (tile + 1 < end) {
      char *next = lds + ((tile + 1) & 1) * 2 * kBytes;
      copy_tile<kPieces>(k + int64_t(tile + 1) * kPieces, next);
      copy_tile<kPieces>(v + int64_t(tile + 1) * kPieces, next + kBytes);
      if (t < kKeyHead) head = head_of[(tile + 1) * kKeyHead + t];
    }
    const int64_t key0 = int64_t(tile) * kHigh;
    if (key0 < wave_any) {
      float s_scale = scale, p_scale = 1.0f;
      if constexpr (B::kScaled) {
        s_scale = scale * power_of_two(-qe - ke);
        p_scale = power_of_two(-ge - ve);
      }
      const bool masked = key0 + kHigh > wave_all;
      const int left = int(clamped(mine - key0, kHigh)) - 4 * half;
#pragma unroll
      for (int part = 0; part < kHigh / 32; part++) {
        f32x16 x = {}, y = {};
        {
          const auto read = [&](int i) { return rows_of_tile<N, D>(at, i % 2 ? vm : km, kPlane, 32 * part, i / 2); };
          Ahead<D / 8, N == 1 ? 6 : 2, N> rows;
          rows.start(read);
          rows.run(read, [&](int i, const Bits<N> &f) {
            if (no_product<N>(16 * (i / 2), a.dim)) return;
            if (i % 2) y = product<M, N>(y, f, g[i / 2]);
            else x = product<M, N>(x, f, q[i / 2]);
          });
        }
        const auto read = [&](int i) { return columns_of_tile<N, D>(at, km, kPlane, 32 * part + 16 * (i / (D / 32)), 32 * (i % (D / 32))); };
        Ahead<D / 16, N == 1 ? 4 : 1, N> columns;
        columns.start(read);
#pragma unroll
        for (int i = 0; i < 16; i++)
          x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], s_scale, -lse)) * __builtin_fmaf(y[i], p_scale, -dot);
        if (masked) {
          stay_branch();
#pragma unroll
          for (int i = 0; i < 16; i++)
            if (part * 32 + 8 * (i / 4) + i % 4 >= left) x[i] = 0.0f;
        }
        if constexpr (B::kScaled) {
          lower<D>(power, out, largest(x), -ke);
          const float by = power_of_two(power - ke);
#pragma unroll
          for (int i = 0; i < 16; i++) x[i] *= by;
        }
        Bits<N> p[2];
        operands_of<M>(p, x);
        columns.run(read, [&](int i, const Bits<N> &f) {
          if (no_product<N>(32 * (i % (D / 32)), a.dim)) return;
          out[i % (D / 32)] = product<M, N>(out[i % (D / 32)], f, p[i / (D / 32)]);
        });
      }
    }
    if (tile + 1 < end && t < kKeyHead) heads[(tile + 1) & 1][t] = head;
    copies_done();
    __syncthreads();
  }
  const bool live = row < s.rows;
  const int64_t token = live ? row / a.group : 0, in = int64_t(s.kv) * a.group + (live ? int(row - token * a.group) : 0);
  T *p = reinterpret_cast<T *>(const_cast<char *>(element(a.gq, s.batch, s.first + token, in, sizeof(T))));
  store_row<T, D>(p, out, B::kScaled ? a.plain_scale * power_of_two(-power) : a.plain_scale, a.dim, live);
}

template <typename T, int D>
__global__ CCHIP_WAVES(256, Planes<T>::kWaves) void attend_back_rows(const AttentionArgs a) {
  extern __shared__ u32x4 lds[];  // [2][keys, values][tile]
  __shared__ int heads[2][kKeyHead];
  __shared__ uint32_t place;
  Jobs jobs(a.queues, a.workgroups);
  for (uint32_t job = jobs.next(place); job < a.workgroups; job = jobs.next(place))
    back_rows_job<T, D>(a, job, reinterpret_cast<char *>(lds), heads);
}

constexpr int kBackSlots = 3;  // tiles of rows in LDS: in use, the one before, and on its way

// Tiles of a chunk's rows that see keys from key0 on. Chunks are cut at the
// same rows for all keys; with several, each leaves its sums and sum_chunks
// adds them up: a key's gradient is long where it is early, and where there are
// few heads there would be as many workgroups as units, the first with twice
// the average's work.
struct Range {
  int first, end;
};

template <typename T>
__device__ __forceinline__ Range chunk_of(const AttentionArgs &a, const Span &s, int64_t key0, int chunk) {
  constexpr int kHigh = Backward<T>::kHigh;
  Range r = {int(key0 * a.group / kHigh), int((s.rows + kHigh - 1) / kHigh)};
  if (a.chunks > 1) {
    const int64_t from = int64_t(chunk) * a.chunk_tiles;
    if (r.first < from) r.first = int(from < r.end ? from : r.end);
    if (r.end > from + a.chunk_tiles) r.end = int(from + a.chunk_tiles);
  }
  return r;
}

// kUnit keys, 32 a wave, over the rows that see them, 32 at a time. Keys and
// values stay in registers as second operands, and the gradients of both: one
// wave a SIMD, which has to keep its matrix unit busy by itself. So three steps
// of rows are under way at once: the products that a step gives the gradients
// are made while the next one's terms are, and the scores of the one after
// while those are packed.
template <typename T, int D>
__device__ __forceinline__ void back_keys_job(const AttentionArgs &a, uint32_t job, char *lds, f32x4 (*heads)[(kRowHead<T> + 3) / 4]) {
  typedef Backward<T> B;
  typedef typename B::M M;
  typedef typename Planes<M>::E E;
  constexpr int N = B::N, kHigh = B::kHigh, kPlane = tile_elements<D>(kHigh), kBytes = N * kPlane * 2, kPieces = kTilePieces<T, D>, kTiles = kUnit / kHigh;
  constexpr int kParts = kHigh / 32, kSlots = kBackSlots;

  const int t = threadIdx.x, l = t & 63, half = l >> 5, w = wave_index();
  const Span s = span_of(a, job, uint32_t(a.key_slots), 1, kUnit, false, uint32_t(a.chunks));
  if (s.tile < 0) return;
  const int chunk = s.chunk;
  const int64_t key0 = int64_t(s.tile) * kUnit, wave_key = key0 + w * 32, key = wave_key + (l & 31);
  const bool live = key < s.keys;

  const int64_t key_tile = (s.key_base + s.tile) * kTiles + w * 32 / kHigh, row_tile = s.row_base * kTiles;
  const int in_tile = w * 32 % kHigh;
  const u32x4 *q = a.tiles[0] + row_tile * kPieces, *g = a.tiles[1] + row_tile * kPieces;
  const float *head_of = a.row_heads + row_tile * kRowHead<T>;
  // rows from the workgroup's first key's on; those that see all of the
  // wave's keys; the lane's
  const int64_t group = a.group;
  const Range range = chunk_of<T>(a, s, key0, chunk);
  const int first = range.first, end = range.end;
  const int64_t wave_full = (wave_key + 31) * group, mine = key * group;
  if (first >= end) return;

  // Behind the last tile it is copied again, so that what is on its way can
  // be counted.
  const auto copy = [&](int tile) {
    const int from = tile < end ? tile : end - 1;
    char *to = lds + tile % kSlots * 2 * kBytes;
    copy_tile<kPieces>(q + int64_t(from) * kPieces, to);
    copy_tile<kPieces>(g + int64_t(from) * kPieces, to + kBytes);
  };
  constexpr int kCopies = kPieces / 256;  // of a tensor's tile, an instruction each
  const auto copy_one = [&](int tile, int i) {
    const int from = tile < end ? tile : end - 1;
    char *to = lds + tile % kSlots * 2 * kBytes;
    if (i < kCopies) copy_group(q + int64_t(from) * kPieces, to, i);
    else copy_group(g + int64_t(from) * kPieces, to + kBytes, i - kCopies);
  };
  float head = 0.0f;
  const auto load_head = [&](int tile) {
    if (t < kRowHead<T>) head = head_of[int64_t(tile < end ? tile : end - 1) * kRowHead<T> + t];
  };
  const auto put_head = [&](int tile) {
    if (t < kRowHead<T>) reinterpret_cast<float *>(heads[tile % kSlots])[t] = head;
  };
  copy(first);
  load_head(first);

  Bits<N> k[D / 16], v[D / 16];
  load_operand<T, D>(k, a.tiles[2] + key_tile * kPieces, in_tile);
  load_operand<T, D>(v, a.tiles[3] + key_tile * kPieces, in_tile);
  int ke = 0, ve = 0;
  if constexpr (B::kScaled) ke = a.key_heads[key_tile * kKeyHead], ve = a.key_heads[key_tile * kKeyHead + 1];
  const float scale = a.negate ? -a.scale : a.scale;
  const Places<D> at;
  put_head(first);
  load_head(first + 1);
  copy(first + 1);
  copies_done();
  __syncthreads();

  f32x16 gk[D / 32] = {}, gv[D / 32] = {};
  f32x16 x[kParts], y[kParts];
  Bits<N> p[2] = {}, ds[2] = {};
  int power = kFirstPower;
  int lift = 127;  // terms are 2^lift P over the power of two of the gradients' tile
  const auto queries = [&](int tile) { return reinterpret_cast<const E *>(lds + tile % kSlots * 2 * kBytes); };

  // scores and products with the values of a part of a tile
  const auto read_rows = [&](int tile, int part, int i) {
    return rows_of_tile<N, D>(at, queries(tile) + i % 2 * N * kPlane, kPlane, 32 * part, i / 2);
  };
  const auto use_rows = [&](int part, int i, const Bits<N> &f) {
    if (i % 2) y[part] = product<M, N>(y[part], f, v[i / 2]);
    else x[part] = product<M, N>(x[part], f, k[i / 2]);
  };
  // what its terms give the gradients
  const auto read_columns = [&](int tile, int part, int i) {
    return columns_of_tile<N, D>(at, queries(tile) + (i % 2 ? 0 : N * kPlane), kPlane, 32 * part + 16 * (i / 2 % 2), 32 * (i / 4));
  };
  const auto use_columns = [&](int i, const Bits<N> &f) {
    const int d = i / 4, h = i / 2 % 2;
    if (i % 2) gk[d] = product<M, N>(gk[d], f, ds[h]);
    else gv[d] = product<M, N>(gv[d], f, p[h]);
  };
  constexpr int kRowOps = D / 8, kColumnOps = D / 8, kDepth = N == 1 ? 6 : 2;

  float s_scale = scale, p_scale = 1.0f, more = 0.0f;
  int besides = 0, fall = 0;
  // terms of a part, element i of the lane's 16
  f32x4 lse[4], dot[4];
  int qe = 0, ge = 0;
  const auto read_head = [&](int tile, int part) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      lse[j] = heads[tile % kSlots][8 * part + 2 * j + half];
      dot[j] = heads[tile % kSlots][kHigh / 4 + 8 * part + 2 * j + half];
    }
    if (B::kScaled && part == 0) {
      qe = reinterpret_cast<const int *>(heads[tile % kSlots])[2 * kHigh];
      ge = reinterpret_cast<const int *>(heads[tile % kSlots])[2 * kHigh + 1];
    }
  };
  float most = 0.0f;  // of dS
  const auto term = [&](int part, int i) {
    x[part][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[part][i], s_scale, more - lse[i / 4][i % 4]));
    y[part][i] = stay(x[part][i] * __builtin_fmaf(y[part][i], p_scale, -dot[i / 4][i % 4]));
    if constexpr (B::kScaled) most = fmaxf(most, __builtin_fabsf(y[part][i]));
  };
  // What is seldom, in one branch: rows that do not see all keys, the
  // gradients of v at a new power of two, those of k at theirs.
  const auto settle = [&](int tile, int part) {
    const int64_t row0 = int64_t(tile) * kHigh + 32 * part;
    bool some = row0 < wave_full;
    if constexpr (B::kScaled) some = some || fall || __ballot(exponent(most) + power + besides > 14);
    if (__builtin_expect(some, 0)) {
      stay_branch();
      const int from = int(clamped(mine - row0, 32)) - 4 * half;  // rows of the lane's from here on
#pragma unroll
      for (int i = 0; i < 16; i++)
        if (8 * (i / 4) + i % 4 < from) x[part][i] = y[part][i] = 0.0f;
      if constexpr (B::kScaled) {
        const float by = power_of_two(fall);
        fall = 0;
#pragma unroll
        for (int d = 0; d < D / 32; d++) gv[d] *= by;
        lower<D>(power, gk, largest(y[part]), besides);
      }
    }
    most = 0.0f;
  };
  float by = 1.0f;
  const auto pack = [&](int part, int h) {
    float z[8], u[8];
#pragma unroll
    for (int i = 0; i < 8; i++) z[i] = x[part][8 * h + i], u[i] = B::kScaled ? y[part][8 * h + i] * by : y[part][8 * h + i];
    p[h] = operand_of<M>(z);
    ds[h] = operand_of<M>(u);
  };
  const auto begin = [&]() {
    if constexpr (B::kScaled) {
      qe = of_lane(qe, 0);
      ge = of_lane(ge, 0);
      s_scale = scale * power_of_two(-qe - ke);
      p_scale = power_of_two(-ge - ve);
      const int now = lift < ge + int(B::kLift) ? lift : ge + int(B::kLift);
      fall = now - lift;
      lift = now;
      more = float(lift - ge);
      besides = ge - lift - qe;
    }
  };

  {
    Ahead<kRowOps, kDepth, N> rows;
    const auto read = [&](int i) { return read_rows(first, 0, i); };
    x[0] = y[0] = f32x16{};
    rows.start(read);
    rows.run(read, [&](int i, const Bits<N> &f) { use_rows(0, i, f); });
  }
  read_head(first, 0);
  // before the first part there are no terms, and behind the last one its tile
  // again: products that give nothing are less than a branch
  for (int tile = first; tile < end; tile++) {
    begin();
#pragma unroll
    for (int part = 0; part < kParts; part++) {
      const int before = part ? part - 1 : kParts - 1, before_tile = part || tile == first ? tile : tile - 1;
      const int after = part + 1 < kParts ? part + 1 : 0, after_tile = part + 1 < kParts ? tile : tile + 1;
      {
        Ahead<kColumnOps, kDepth, N> columns;
        const auto read = [&](int i) { return read_columns(before_tile, before, i); };
        columns.start(read);
        columns.run(read, use_columns, [&](int i) {
#pragma unroll
          for (int e = i * 16 / kColumnOps; e < (i + 1) * 16 / kColumnOps; e++) term(part, e);
        });
      }
      // the tile before is done with, and the next has been on its way for
      // as long as one takes
      if (part == 0) {
        copies_done();
        put_head(tile + 1);
        __syncthreads();
        load_head(tile + 2);
      }
      settle(tile, part);
      if constexpr (B::kScaled) by = power_of_two(power + besides);
      {
        read_head(after_tile, after);
        Ahead<kRowOps, kDepth, N> rows;
        const auto read = [&](int i) { return read_rows(after_tile, after, i); };
        if constexpr (kParts == 1) pack(part, 0), pack(part, 1);
        x[after] = y[after] = f32x16{};
        rows.start(read);
        rows.run(read, [&](int i, const Bits<N> &f) { use_rows(after, i, f); }, [&](int i) {
          if (kParts > 1 && (i == 1 || i == 5)) pack(part, i / 4);
          if (part == 0) {
#pragma unroll
            for (int c = i * 2 * kCopies / kRowOps; c < (i + 1) * 2 * kCopies / kRowOps; c++) copy_one(tile + 2, c);
          }
        });
      }
    }
  }
  {
    Ahead<kColumnOps, kDepth, N> columns;
    const auto read = [&](int i) { return read_columns(end - 1, kParts - 1, i); };
    columns.start(read);
    columns.run(read, use_columns);
  }
  copies_done();
  const float k_scale = B::kScaled ? a.plain_scale * power_of_two(-power) : a.plain_scale, v_scale = B::kScaled ? power_of_two(-lift) : 1.0f;
  if (a.chunks > 1) {
    float *to = a.partial + ((s.key_base + s.tile) * a.chunks + chunk) * 2 * kUnit * a.dim + (w * 32 + (l & 31)) * a.dim;
    store_row<float, D>(to, gk, k_scale, a.dim, true);
    store_row<float, D>(to + kUnit * a.dim, gv, v_scale, a.dim, true);
    return;
  }
  const int64_t place = s.key0 + (live ? key : 0);
  T *kp = reinterpret_cast<T *>(const_cast<char *>(element(a.gk, s.batch, place, s.kv, sizeof(T))));
  T *vp = reinterpret_cast<T *>(const_cast<char *>(element(a.gv, s.batch, place, s.kv, sizeof(T))));
  store_row<T, D>(kp, gk, k_scale, a.dim, live);
  store_row<T, D>(vp, gv, v_scale, a.dim, live);
}

template <typename T, int D>
__global__ CCHIP_WAVES(256, 1) void attend_back_keys(const AttentionArgs a) {
  extern __shared__ u32x4 lds[];  // [kBackSlots][queries, gradients of o][tile]
  __shared__ f32x4 heads[kBackSlots][(kRowHead<T> + 3) / 4];
  __shared__ uint32_t place;
  Jobs jobs(a.queues + kQueues, a.workgroups);
  for (uint32_t job = jobs.next(place); job < a.workgroups; job = jobs.next(place))
    back_keys_job<T, D>(a, job, reinterpret_cast<char *>(lds), heads);
}

// Chunks' sums of kUnit keys, in their order.
template <typename T>
__global__ __launch_bounds__(256) void sum_chunks(const AttentionArgs a) {
  const uint32_t block = block_index(), id = block / 8;  // an eighth of the keys a workgroup
  if (block >= a.workgroups) return;
  const Span s = span_of(a, id, uint32_t(a.key_slots), 1, kUnit, false);
  if (s.tile < 0) return;
  const int64_t key0 = int64_t(s.tile) * kUnit;
  int from = 0, to = 0;  // chunks that there are
  for (int c = 0; c < a.chunks; c++) {
    const Range r = chunk_of<T>(a, s, key0, c);
    if (r.first >= r.end) {
      if (to == 0) from = c + 1;
    } else {
      to = c + 1;
    }
  }
  if (to == 0) from = 0;
  const float *p = a.partial + (s.key_base + s.tile) * a.chunks * 2 * kUnit * a.dim;
  const int pieces = (a.dim + 3) / 4;
  for (int i = threadIdx.x; i < 2 * (kUnit / 8) * pieces; i += 256) {
    const int which = i / (kUnit / 8 * pieces), in = i - which * (kUnit / 8 * pieces), row = in / pieces, col = (in - row * pieces) * 4;
    const int64_t key = key0 + block % 8 * (kUnit / 8) + row;
    if (key >= s.keys) continue;
    float sum[4] = {};
    const float *x = p + int64_t(which) * kUnit * a.dim + (block % 8 * (kUnit / 8) + row) * a.dim + col;
    const int n = a.dim - col < 4 ? a.dim - col : 4;
    const int64_t step = int64_t(2) * kUnit * a.dim;
    if (n == 4 && a.dim % 4 == 0) {  // all on their way at once: there are eight at most
      f32x4 y[8];
#pragma unroll
      for (int c = 0; c < 8; c++) y[c] = *reinterpret_cast<const f32x4 *>(x + (from + c < to ? from + c : from) * step);
#pragma unroll
      for (int c = 0; c < 8; c++)
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (from + c < to) sum[j] += y[c][j];
    } else {
      for (int c = from; c < to; c++)
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (j < n) sum[j] += x[c * step + j];
    }
    T *out = reinterpret_cast<T *>(const_cast<char *>(element(which ? a.gv : a.gk, s.batch, s.key0 + key, s.kv, sizeof(T)))) + col;
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (j < n) out[j] = T(sum[j]);
  }
}

// ---- host -------------------------------------------------------------------------------

// Where a backward pass's tiles lie in its workspace.
struct BackSizes {
  size_t tiles[4], row_heads, key_heads, partial, queues;  // bytes
  size_t bytes() const {
    size_t n = row_heads + key_heads + partial + queues;
    for (int i = 0; i < 4; i++) n += tiles[i];
    return n;
  }
};

inline BackSizes back_sizes(int dtype, int dim, int64_t pairs, int64_t row_slots, int64_t key_slots, int chunks) {
  const int d = dim <= 64 ? 64 : 128, planes = dtype == CCHIP_F32 ? 3 : 1, high = dtype == CCHIP_F32 ? 32 : 64;
  BackSizes b = {};
  for (int i = 0; i < 4; i++) {
    const size_t rows = size_t(pairs) * (i < 2 ? row_slots : key_slots) * kUnit;
    b.tiles[i] = rows * d * planes * 2;
  }
  b.row_heads = size_t(pairs) * row_slots * kUnit / high * (2 * high + 4) * sizeof(float);
  b.key_heads = (size_t(pairs) * key_slots * kUnit / high * kKeyHead * sizeof(int32_t) + 15) / 16 * 16;
  b.partial = chunks > 1 ? size_t(pairs) * key_slots * chunks * 2 * kUnit * dim * sizeof(float) : 0;
  b.queues = 2 * kQueues * sizeof(uint32_t);
  return b;
}

template <typename T, int D>
void launch_attend_back(AttentionArgs a, hipStream_t stream) {
  constexpr size_t bytes = size_t(4) * Backward<T>::N * tile_elements<D>(Backward<T>::kHigh) * 2, key_bytes = bytes / 4 * 6;
  constexpr uint32_t kTiles = kUnit / Backward<T>::kHigh;
  allow_lds<&attend_back_rows<T, D>>(int(bytes), "attention");
  allow_lds<&attend_back_keys<T, D>>(int(key_bytes), "attention");
  a.workgroups = 2 * a.pairs * uint32_t(a.row_slots + a.key_slots) * kTiles;
  hipLaunchKernelGGL((lay_out<T, D>), grid_of(a.workgroups), dim3(256), 0, stream, a);
  check_launch("attention");
  a.workgroups = a.pairs * uint32_t(a.row_slots);
  hipLaunchKernelGGL((attend_back_rows<T, D>), dim3(std::min(a.workgroups, 2 * kTakers)), dim3(256), bytes, stream, a);
  check_launch("attention");
  a.workgroups = a.pairs * uint32_t(a.key_slots) * uint32_t(a.chunks);
  hipLaunchKernelGGL((attend_back_keys<T, D>), dim3(std::min(a.workgroups, kTakers)), dim3(256), key_bytes, stream, a);
  check_launch("attention");
  if (a.chunks == 1) return;
  a.workgroups = a.pairs * uint32_t(a.key_slots) * 8;
  hipLaunchKernelGGL((sum_chunks<T>), grid_of(a.workgroups), dim3(256), 0, stream, a);
  check_launch("attention");
}

template <typename T>
void attend_back_launch(const AttentionArgs &a, hipStream_t stream) {
  if (a.dim <= 64) launch_attend_back<T, 64>(a, stream);
  else launch_attend_back<T, 128>(a, stream);
}

}  // namespace op
}  // namespace cchip
