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
                                         u32x4 *to, int32_t *power, const Heads *o, float *lse, float *dot) {
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
    if (o) {
      const Raw8<T> y = load8<T>(reinterpret_cast<const T *>(element(*o, s.batch, s.first + token, head, sizeof(T))) + piece * 8, n);
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
      const Bits<B::N> b = bits_of<T>(r[i]);
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
  if (which == 0) lay_tile<T, D>(a, a.q, s, row0, count, per_token, a.tiles[0] + tile * kTilePieces<T, D>, a.powers[0] + tile, nullptr, nullptr, nullptr);
  else if (which == 1) lay_tile<T, D>(a, a.d_o, s, row0, count, per_token, a.tiles[1] + tile * kTilePieces<T, D>, a.powers[1] + tile, &a.o, a.lses + tile * B::kHigh, a.dots + tile * B::kHigh);
  else if (which == 2) lay_tile<T, D>(a, a.k, s, row0, count, 1, a.tiles[2] + tile * kTilePieces<T, D>, a.powers[2] + tile, nullptr, nullptr, nullptr);
  else lay_tile<T, D>(a, a.v, s, row0, count, 1, a.tiles[3] + tile * kTilePieces<T, D>, a.powers[3] + tile, nullptr, nullptr, nullptr);
}

// ---- products -------------------------------------------------------------------------

// A tile in memory to LDS, 1 KB an instruction and group of rows, which four
// waves share.
template <int Pieces>
__device__ __forceinline__ void copy_tile(const u32x4 *from, char *to) {
  static_assert(Pieces % 256 == 0, "every wave copies as much");
#pragma unroll
  for (int i = 0; i < Pieces / 256; i++) copy_lanes(from, (i * 256 + threadIdx.x) * 16, to + (i * 4 + wave_index()) * (kGroup * 2));
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
// maximum's. Takes the largest of dS as it stands and the power that the
// product needs besides; powers are counted as exponents, as the first ones
// are far from any value's.
constexpr int kFirstPower = 100;

template <int D>
__device__ __forceinline__ void lower(int &power, f32x16 (&out)[D / 32], float most, int besides) {
  const int e = int(__builtin_bit_cast(uint32_t, max_halves(most)) >> 23) - 127, over = e + power + besides - 14;
  if (!__ballot(over > 0)) return;
  const float factor = over > 0 ? power_of_two(-over) : 1.0f;
  if (over > 0) power -= over;
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

// kUnit rows, 32 a wave, over the keys that they see.
template <typename T, int D>
__global__ CCHIP_WAVES(256, Planes<T>::kWaves) void attend_back_rows(const AttentionArgs a) {
  typedef Backward<T> B;
  typedef typename B::M M;
  typedef typename Planes<M>::E E;
  constexpr int N = B::N, kHigh = B::kHigh, kPlane = tile_elements<D>(kHigh), kBytes = N * kPlane * 2, kPieces = kTilePieces<T, D>, kTiles = kUnit / kHigh;
  extern __shared__ u32x4 lds_[];  // [2][keys, values][tile]
  char *const lds = reinterpret_cast<char *>(lds_);

  const int t = threadIdx.x, l = t & 63, half = l >> 5, w = wave_index();
  const uint32_t id = block_index();
  if (id >= a.workgroups) return;
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
  const int32_t *ke = a.powers[2] + key_tile, *ve = a.powers[3] + key_tile;
  copy_tile<kPieces>(k, lds);
  copy_tile<kPieces>(v, lds + kBytes);

  Bits<N> q[D / 16], g[D / 16];
  const int in_tile = w * 32 % kHigh;
  load_operand<T, D>(q, a.tiles[0] + row_tile * kPieces, in_tile);
  load_operand<T, D>(g, a.tiles[1] + row_tile * kPieces, in_tile);
  const float lse = a.lses[row_tile * kHigh + in_tile + (l & 31)], dot = a.dots[row_tile * kHigh + in_tile + (l & 31)];
  int qe = 0, ge = 0;
  if constexpr (B::kScaled) qe = a.powers[0][row_tile], ge = a.powers[1][row_tile];
  const float scale = a.negate ? -a.scale : a.scale;

  const Places<D> at;
  f32x16 out[D / 32] = {};
  int power = kFirstPower;
  copies_done();
  __syncthreads();
  for (int tile = 0; tile < end; tile++) {
    const E *km = reinterpret_cast<const E *>(lds + (tile & 1) * 2 * kBytes), *vm = km + N * kPlane;
    if (tile + 1 < end) {
      char *next = lds + ((tile + 1) & 1) * 2 * kBytes;
      copy_tile<kPieces>(k + int64_t(tile + 1) * kPieces, next);
      copy_tile<kPieces>(v + int64_t(tile + 1) * kPieces, next + kBytes);
    }
    const int64_t key0 = int64_t(tile) * kHigh;
    if (key0 < wave_any) {
      float s_scale = scale, p_scale = 1.0f;
      if constexpr (B::kScaled) {
        s_scale = scale * power_of_two(-qe - ke[tile]);
        p_scale = power_of_two(-ge - ve[tile]);
      }
      const bool masked = key0 + kHigh > wave_all;
      const int left = int(clamped(mine - key0, kHigh)) - 4 * half;
#pragma unroll
      for (int part = 0; part < kHigh / 32; part++) {
        f32x16 x = {}, y = {};
#pragma unroll
        for (int j = 0; j < D / 16; j++) {
          x = product<M, N>(x, rows_of_tile<N, D>(at, km, kPlane, 32 * part, j), q[j]);
          y = product<M, N>(y, rows_of_tile<N, D>(at, vm, kPlane, 32 * part, j), g[j]);
        }
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
          lower<D>(power, out, largest(x), -ke[tile]);
          const float by = power_of_two(power - ke[tile]);
#pragma unroll
          for (int i = 0; i < 16; i++) x[i] *= by;
        }
        Bits<N> p[2];
        operands_of<M>(p, x);
#pragma unroll
        for (int d = 0; d < D / 32; d++)
#pragma unroll
          for (int h = 0; h < 2; h++)
            out[d] = product<M, N>(out[d], columns_of_tile<N, D>(at, km, kPlane, 32 * part + 16 * h, 32 * d), p[h]);
      }
    }
    copies_done();
    __syncthreads();
  }
  const bool live = row < s.rows;
  const int64_t token = live ? row / a.group : 0, head = int64_t(s.kv) * a.group + (live ? int(row - token * a.group) : 0);
  T *p = reinterpret_cast<T *>(const_cast<char *>(element(a.gq, s.batch, s.first + token, head, sizeof(T))));
  store_row<T, D>(p, out, B::kScaled ? a.plain_scale * power_of_two(-power) : a.plain_scale, a.dim, live);
}

// kUnit keys, 32 a wave, over the rows that see them. Keys and values stay in
// registers as second operands.
template <typename T, int D>
__global__ CCHIP_WAVES(256, 1) void attend_back_keys(const AttentionArgs a) {
  typedef Backward<T> B;
  typedef typename B::M M;
  typedef typename Planes<M>::E E;
  constexpr int N = B::N, kHigh = B::kHigh, kPlane = tile_elements<D>(kHigh), kBytes = N * kPlane * 2, kPieces = kTilePieces<T, D>, kTiles = kUnit / kHigh;
  extern __shared__ u32x4 lds_[];  // [2][queries, gradients of o][tile]
  char *const lds = reinterpret_cast<char *>(lds_);
  __shared__ f32x4 lses[2][kHigh / 4], dots[2][kHigh / 4];

  const int t = threadIdx.x, l = t & 63, half = l >> 5, w = wave_index();
  const uint32_t id = block_index();
  if (id >= a.workgroups) return;
  const Span s = span_of(a, id, uint32_t(a.key_slots), 1, kUnit, false);
  if (s.tile < 0) return;
  const int64_t key0 = int64_t(s.tile) * kUnit, wave_key = key0 + w * 32, key = wave_key + (l & 31);
  const bool live = key < s.keys;

  const int64_t key_tile = (s.key_base + s.tile) * kTiles + w * 32 / kHigh, row_tile = s.row_base * kTiles;
  const int in_tile = w * 32 % kHigh;
  const u32x4 *q = a.tiles[0] + row_tile * kPieces, *g = a.tiles[1] + row_tile * kPieces;
  const int32_t *qe = a.powers[0] + row_tile, *ge = a.powers[1] + row_tile;
  const float *lse_of = a.lses + row_tile * kHigh, *dot_of = a.dots + row_tile * kHigh;
  // the first row that sees the workgroup's, the wave's and the lane's keys
  const int64_t group = a.group;
  const int first = int(key0 * group / kHigh), end = int((s.rows + kHigh - 1) / kHigh);
  const int64_t wave_first = wave_key * group, wave_full = (wave_key + 31) * group, mine = key * group;

  float row_value = 0.0f;  // a thread's lse or dot of a tile
  const auto fetch = [&](int tile) {
    char *to = lds + (tile & 1) * 2 * kBytes;
    copy_tile<kPieces>(q + int64_t(tile) * kPieces, to);
    copy_tile<kPieces>(g + int64_t(tile) * kPieces, to + kBytes);
    if (t < 2 * kHigh) row_value = t < kHigh ? lse_of[int64_t(tile) * kHigh + t] : dot_of[int64_t(tile) * kHigh + t - kHigh];
  };
  const auto put = [&](int tile) {
    if (t < kHigh) reinterpret_cast<float *>(lses[tile & 1])[t] = row_value;
    else if (t < 2 * kHigh) reinterpret_cast<float *>(dots[tile & 1])[t - kHigh] = row_value;
  };
  if (first < end) fetch(first);

  Bits<N> k[D / 16], v[D / 16];
  load_operand<T, D>(k, a.tiles[2] + key_tile * kPieces, in_tile);
  load_operand<T, D>(v, a.tiles[3] + key_tile * kPieces, in_tile);
  int ke = 0, ve = 0;
  if constexpr (B::kScaled) ke = a.powers[2][key_tile], ve = a.powers[3][key_tile];
  const float scale = a.negate ? -a.scale : a.scale;

  const Places<D> at;
  f32x16 gk[D / 32] = {}, gv[D / 32] = {};
  int power = kFirstPower;
  int lift = 127;  // terms are 2^lift P over the power of two of the gradients' tile
  if (first < end) put(first);
  copies_done();
  __syncthreads();
  for (int tile = first; tile < end; tile++) {
    if (tile + 1 < end) fetch(tile + 1);
    const int64_t tile_row = int64_t(tile) * kHigh;
    if (tile_row + kHigh > wave_first && wave_key < s.keys) {
      const E *qm = reinterpret_cast<const E *>(lds + (tile & 1) * 2 * kBytes), *gm = qm + N * kPlane;
      float s_scale = scale, p_scale = 1.0f, more = 0.0f;
      int besides = 0;
      if constexpr (B::kScaled) {
        s_scale = scale * power_of_two(-qe[tile] - ke);
        p_scale = power_of_two(-ge[tile] - ve);
        if (lift > ge[tile] + int(B::kLift)) {
          const float factor = power_of_two(ge[tile] + int(B::kLift) - lift);
          lift = ge[tile] + int(B::kLift);
#pragma unroll
          for (int d = 0; d < D / 32; d++) gv[d] *= factor;
        }
        more = float(lift - ge[tile]);
        besides = ge[tile] - lift - qe[tile];
      }
#pragma unroll
      for (int part = 0; part < kHigh / 32; part++) {
        const int64_t row0 = tile_row + 32 * part;
        if (row0 + 32 <= wave_first) continue;
        f32x16 x = {}, y = {};
#pragma unroll
        for (int j = 0; j < D / 16; j++) {
          x = product<M, N>(x, rows_of_tile<N, D>(at, qm, kPlane, 32 * part, j), k[j]);
          y = product<M, N>(y, rows_of_tile<N, D>(at, gm, kPlane, 32 * part, j), v[j]);
        }
        const bool masked = row0 < wave_full;
        const int from = int(clamped(mine - row0, 32)) - 4 * half;  // rows of the lane's from here on
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const f32x4 lse = lses[tile & 1][8 * part + 2 * j + half], dot = dots[tile & 1][8 * part + 2 * j + half];
#pragma unroll
          for (int i = 0; i < 4; i++) {
            x[4 * j + i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[4 * j + i], s_scale, more - lse[i]));
            y[4 * j + i] = x[4 * j + i] * __builtin_fmaf(y[4 * j + i], p_scale, -dot[i]);
          }
        }
        if (masked) {
          stay_branch();
#pragma unroll
          for (int i = 0; i < 16; i++)
            if (8 * (i / 4) + i % 4 < from) x[i] = y[i] = 0.0f;
        }
        if constexpr (B::kScaled) {
          lower<D>(power, gk, largest(y), besides);
          const float by = power_of_two(power + besides);
#pragma unroll
          for (int i = 0; i < 16; i++) y[i] *= by;
        }
        Bits<N> p[2], ds[2];
        operands_of<M>(p, x);
        operands_of<M>(ds, y);
#pragma unroll
        for (int d = 0; d < D / 32; d++)
#pragma unroll
          for (int h = 0; h < 2; h++) {
            gv[d] = product<M, N>(gv[d], columns_of_tile<N, D>(at, gm, kPlane, 32 * part + 16 * h, 32 * d), p[h]);
            gk[d] = product<M, N>(gk[d], columns_of_tile<N, D>(at, qm, kPlane, 32 * part + 16 * h, 32 * d), ds[h]);
          }
      }
    }
    if (tile + 1 < end) put(tile + 1);
    copies_done();
    __syncthreads();
  }
  const int64_t place = s.key0 + (live ? key : 0);
  T *kp = reinterpret_cast<T *>(const_cast<char *>(element(a.gk, s.batch, place, s.kv, sizeof(T))));
  T *vp = reinterpret_cast<T *>(const_cast<char *>(element(a.gv, s.batch, place, s.kv, sizeof(T))));
  store_row<T, D>(kp, gk, B::kScaled ? a.plain_scale * power_of_two(-power) : a.plain_scale, a.dim, live);
  store_row<T, D>(vp, gv, B::kScaled ? power_of_two(-lift) : 1.0f, a.dim, live);
}

// ---- host -------------------------------------------------------------------------------

// Where a backward pass's tiles lie in its workspace.
struct BackSizes {
  size_t tiles[4], powers[4], values;  // bytes; values: of lse and of dots each
  size_t bytes() const {
    size_t n = 2 * values;
    for (int i = 0; i < 4; i++) n += tiles[i] + powers[i];
    return n;
  }
};

inline BackSizes back_sizes(int dtype, int dim, int64_t pairs, int64_t row_slots, int64_t key_slots) {
  const int d = dim <= 64 ? 64 : 128, planes = dtype == CCHIP_F32 ? 3 : 1, high = dtype == CCHIP_F32 ? 32 : 64;
  BackSizes b = {};
  for (int i = 0; i < 4; i++) {
    const size_t rows = size_t(pairs) * (i < 2 ? row_slots : key_slots) * kUnit;
    b.tiles[i] = rows * d * planes * 2;
    b.powers[i] = (rows / high * sizeof(int32_t) + 15) / 16 * 16;
  }
  b.values = size_t(pairs) * row_slots * kUnit * sizeof(float);
  return b;
}

template <typename T, int D>
void launch_attend_back(AttentionArgs a, hipStream_t stream) {
  constexpr size_t bytes = size_t(4) * Backward<T>::N * tile_elements<D>(Backward<T>::kHigh) * 2;
  constexpr uint32_t kTiles = kUnit / Backward<T>::kHigh;
  check_hip(hipFuncSetAttribute(reinterpret_cast<const void *>(&attend_back_rows<T, D>), hipFuncAttributeMaxDynamicSharedMemorySize, int(bytes)), "attention");
  check_hip(hipFuncSetAttribute(reinterpret_cast<const void *>(&attend_back_keys<T, D>), hipFuncAttributeMaxDynamicSharedMemorySize, int(bytes)), "attention");
  a.workgroups = 2 * a.pairs * uint32_t(a.row_slots + a.key_slots) * kTiles;
  hipLaunchKernelGGL((lay_out<T, D>), grid_of(a.workgroups), dim3(256), 0, stream, a);
  check_launch("attention");
  a.workgroups = a.pairs * uint32_t(a.row_slots);
  hipLaunchKernelGGL((attend_back_rows<T, D>), grid_of(a.workgroups), dim3(256), bytes, stream, a);
  check_launch("attention");
  a.workgroups = a.pairs * uint32_t(a.key_slots);
  hipLaunchKernelGGL((attend_back_keys<T, D>), grid_of(a.workgroups), dim3(256), bytes, stream, a);
  check_launch("attention");
}

template <typename T>
void attend_back_launch(const AttentionArgs &a, hipStream_t stream) {
  if (a.dim <= 64) launch_attend_back<T, 64>(a, stream);
  else launch_attend_back<T, 128>(a, stream);
}

}  // namespace op
}  // namespace cchip
