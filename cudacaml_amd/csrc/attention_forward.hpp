// Attention, forward: the kernel over tiles of rows, and the one for few rows
// whose waves share the keys out.

#include "attention.hpp"

namespace cchip {
namespace op {

// A row's maximum follows the largest score only when that is kSlack (a power
// of two) ahead of it: what the row has so far is rescaled in the first tile
// and hardly ever again. Terms are 2^(score - maximum + kLift): f16 has normal
// values from 2^-14, so that what is dropped there is below 2^-24 of the
// largest term, and nothing reaches 2^16.
template <typename T>
struct Powers {
  static constexpr float kSlack = std::is_same<T, f16>::value ? 4.0f : 8.0f;
  static constexpr float kLift = std::is_same<T, f16>::value ? 10.0f : 0.0f;
};

// The running maximum, sum (of this lane's keys) and transposed output of 32 rows.
template <int D>
struct Running {
  float top = -INFINITY, sum = 0.0f;
  f32x16 out[D / 32] = {};
};

// What a sum adds up of eight terms: for 16-bit types the terms as the
// product takes them, so that rows of equal values come out whole.
template <typename T>
__device__ __forceinline__ float sum_of(float sum, const float *x, const Bits<Planes<T>::N> &b) {
  if constexpr (std::is_same<T, float>::value) {
    return sum + (((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7])));
  } else if constexpr (std::is_same<T, f16>::value) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t u = b.p[0][i];
      sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, u), f16x2{_Float16(1.0f), _Float16(1.0f)}, sum, false);
    }
    return sum;
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t u = b.p[0][i], ones = 0x3F803F80u;
      sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, u), __builtin_bit_cast(bf16x2, ones), sum, false);
    }
    return sum;
  }
}

// Scores s of 32 Tiles keys become terms, and what the rows have so far is
// brought to their maximum. `left`: masked from this key of the lane's on.
template <typename T, int D, int Tiles>
__device__ __forceinline__ void terms_of(Running<D> &r, f32x16 (&s)[Tiles], Bits<Planes<T>::N> (&p)[2 * Tiles], float scale,
                                         bool masked, int left) {
  if (masked) {
    stay_branch();
#pragma unroll
    for (int t = 0; t < Tiles; t++)
#pragma unroll
      for (int i = 0; i < 16; i++)
        if (t * 32 + 8 * (i / 4) + i % 4 >= left) s[t][i] = -INFINITY;
  }
  float most = s[0][0];
#pragma unroll
  for (int t = 0; t < Tiles; t++)
#pragma unroll
    for (int i = t ? 0 : 1; i < 16; i++) most = fmaxf(most, s[t][i]);
  most = max_halves(most) * scale;
  if (__ballot(most > r.top + Powers<T>::kSlack)) {
    const float top = most > r.top ? most : r.top;
    const float factor = top == r.top ? 1.0f : __builtin_amdgcn_exp2f(r.top - top);
    r.top = top;
    r.sum *= factor;
#pragma unroll
    for (int d = 0; d < D / 32; d++) r.out[d] *= factor;
  }
  const float from = (r.top == -INFINITY ? 0.0f : r.top) - Powers<T>::kLift;
#pragma unroll
  for (int t = 0; t < Tiles; t++)
#pragma unroll
    for (int half = 0; half < 2; half++) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][half * 8 + i], scale, -from));
      p[2 * t + half] = operand_of<T>(x);
      r.sum = sum_of<T>(r.sum, x, p[2 * t + half]);
    }
}

// Queries of 32 rows as the second operand, zero behind the last row.
template <typename T, int D>
__device__ __forceinline__ void load_queries(Bits<Planes<T>::N> (&q)[D / 16], const AttentionArgs &a, const Heads &x, const Span &s,
                                             int64_t row, bool negate) {
  const int half = (threadIdx.x & 63) >> 5;
  const bool live = row < s.rows;
  const int64_t token = live ? row / a.group : 0;
  const int head = live ? int(row - token * a.group) : 0;
  const T *p = reinterpret_cast<const T *>(element(x, s.batch, s.first + token, int64_t(s.kv) * a.group + head, sizeof(T)));
#pragma unroll
  for (int i = 0; i < D / 16; i++) {
    const int at = 16 * i + 8 * half, left = a.dim - at;
    Raw8<T> r = load8<T>(p + at, live && left > 0 ? (left < 8 ? left : 8) : 0);
    if (negate) r = negated(r);
    q[i] = bits_of<T>(r);
  }
}

template <typename T>
__device__ __forceinline__ void store_some(T *p, const Raw8<T> &r, int n) {
  if (n >= 8) {
    const u32x4 *from = reinterpret_cast<const u32x4 *>(&r);
    u32x4_any *to = reinterpret_cast<u32x4_any *>(p);
#pragma unroll
    for (int i = 0; i < int(sizeof(T) * 8 / 16); i++) to[i] = from[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (i < n) p[i] = r.x[i];
  }
}

// A lane's columns of a row, out[d][4 j + i] being element 32 d + 8 j +
// 4 half + i: halves exchange them to have 8 neighbours.
// `rest`: where what is rounded off goes, or null.
template <typename T, int D>
__device__ __forceinline__ void store_row(T *p, const f32x16 (&out)[D / 32], float factor, int dim, bool live, bf16 *rest = nullptr) {
  const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int d = 0; d < D / 32; d++)
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      Raw8<T> r;
      Raw8<bf16> left_off;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float x = out[d][4 * j + i] * factor, y = out[d][4 * j + 4 + i] * factor;
        const auto z = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, y), false, false);
        const uint32_t lo = z[0], hi = z[1];
        r.x[i] = T(__builtin_bit_cast(float, lo));
        r.x[4 + i] = T(__builtin_bit_cast(float, hi));
        left_off.x[i] = bf16(__builtin_bit_cast(float, lo) - float(r.x[i]));
        left_off.x[4 + i] = bf16(__builtin_bit_cast(float, hi) - float(r.x[4 + i]));
      }
      const int at = 32 * d + 8 * (j + half), left = dim - at;
      if (!live || left <= 0) continue;
      if (rest) store_some<bf16>(rest + at, left_off, left);
      store_some<T>(p + at, r, left);
    }
}

// Rows' outputs: to o, or as they are for the sum over splits.
template <typename T, int D>
__device__ __forceinline__ void finish(const AttentionArgs &a, const Span &s, Running<D> &r, int64_t row, int split, float sum) {
  const bool live = row < s.rows;
  const int half = (threadIdx.x & 63) >> 5;
  if (a.splits > 1) {
    const int64_t rows = a.batch * a.kv_heads * a.tokens * a.group, at = row_values(a, s) + row;
    float *p = a.partial + (at * a.splits + split) * a.dim;
    store_row<float, D>(p, r.out, 1.0f, a.dim, live);
    if (live && !half) {
      float *m = a.partial + rows * a.splits * a.dim + (at * a.splits + split) * 2;
      m[0] = r.top;
      m[1] = sum;
    }
    return;
  }
  const int64_t token = live ? row / a.group : 0;
  const int head = live ? int(row - token * a.group) : 0;
  T *p = reinterpret_cast<T *>(const_cast<char *>(element(a.o, s.batch, s.first + token, int64_t(s.kv) * a.group + head, sizeof(T))));
  store_row<T, D>(p, r.out, sum == 0.0f ? 0.0f : 1.0f / sum, a.dim, live, a.o_rest ? a.o_rest + (row_values(a, s) + row) * a.dim : nullptr);
  if (a.lse && live && !half)
    a.lse[row_values(a, s) + row] = sum == 0.0f ? INFINITY : r.top - Powers<T>::kLift + __builtin_log2f(sum);
}

// Whether an element is infinite or NaN; and zero in its place.
template <typename T>
__device__ __forceinline__ bool take_finite(Raw8<T> &r) {
  bool all = true;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const bool finite = __builtin_fabsf(float(r.x[i])) < INFINITY;
    all = all && finite;
    if (!finite) r.x[i] = T(0.0f);
  }
  return all;
}

// Values of a tile that are not finite, and that the tile has zeros for,
// where a row sees them: an infinity or NaN times the term's sign. A product
// would bring them to the rows that do not, as zero times infinity.
template <typename T, int D>
__device__ __forceinline__ void add_infinite(Running<D> &r, const T *v, int64_t stride, int64_t keys, int64_t seen, int dim) {
  const int half = (threadIdx.x & 63) >> 5;
#pragma unroll 1
  for (int64_t j = 0; j < keys; j++) {
#pragma unroll
    for (int d = 0; d < D / 32; d++)
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const int at = 32 * d + 8 * (i / 4) + 4 * half + i % 4;
        if (at >= dim) continue;
        const float x = float(v[j * stride + at]);
        if (!(__builtin_fabsf(x) < INFINITY) && j < seen) r.out[d][i] += x;
      }
  }
}

// 32 Waves rows of a sequence and key head, a split of the keys they see.
// Tiles of Keys keys and values go from memory through registers to one half
// of LDS while the other is computed with; every wave reads all of both
// (32 KB a tile of 64 for D = 128), which at 128 bytes a cycle of the unit
// takes as long as the tile's products: waves are 8 where there are rows for
// them, as they share what is loaded.
template <typename T, int D, int Waves, int Keys>
__global__ __launch_bounds__(Waves * 64, Planes<T>::kWaves) void attend(const AttentionArgs a) {
  constexpr int N = Planes<T>::N, kTile = Keys * D, kBuffer = 2 * N * kTile;
  typedef typename Planes<T>::E E;
  extern __shared__ u32x4 lds[];
  E *tiles = reinterpret_cast<E *>(lds);  // [2][keys, values][plane][Keys][D]
  __shared__ int bad[2];                  // the tile, counted from 1, in a buffer some of whose values were not finite

  const int t = threadIdx.x, l = t & 63, half = l >> 5, w = wave_index();
  const uint32_t block = block_index(), id = block / uint32_t(a.splits);
  const int split = int(block - id * uint32_t(a.splits));
  if (block >= a.workgroups) return;
  const Span s = span_of(a, id, uint32_t(a.slots), a.group, 32 * Waves, true);
  if (s.tile < 0) return;
  const int64_t row0 = int64_t(s.tile) * 32 * Waves, wave_row = row0 + w * 32, row = wave_row + (l & 31);
  if (row0 >= s.rows) return;

  // keys that rows see: all of the workgroup's, all of the wave's, any of the
  // wave's, the lane's
  const int64_t last_row = s.rows - 1 < row0 + 32 * Waves - 1 ? s.rows - 1 : row0 + 32 * Waves - 1;
  const int64_t wave_last = s.rows - 1 < wave_row + 31 ? s.rows - 1 : wave_row + 31;
  const int64_t to = clamped(last_row / a.group + s.ahead + 1, s.keys);
  const int64_t all = clamped(row0 / a.group + s.ahead + 1, s.keys);
  const int64_t wave_all = clamped(wave_row / a.group + s.ahead + 1, s.keys);
  const int64_t wave_any = wave_row < s.rows ? clamped(wave_last / a.group + s.ahead + 1, s.keys) : 0;
  const int64_t mine = clamped(row / a.group + s.ahead + 1, s.keys);
  const int64_t count = (to + Keys - 1) / Keys;
  const int64_t first = count * split / a.splits, end = count * (split + 1) / a.splits;

  Bits<N> q[D / 16];
  load_queries<T, D>(q, a, a.q, s, row, a.negate);
  Running<D> r;
  const T *k = reinterpret_cast<const T *>(element(a.k, s.batch, s.key0 + first * Keys, s.kv, sizeof(T)));
  const T *v = reinterpret_cast<const T *>(element(a.v, s.batch, s.key0 + first * Keys, s.kv, sizeof(T)));
  if (t < 2) bad[t] = 0;

  Staged<T, D, Keys, Waves * 64> ks, vs;
  const auto put = [&](int64_t tile) {
    E *m = tiles + (tile & 1) * kBuffer;
    ks.store(t, m);
    if ((tile + 1) * Keys > all) {
      bool finite = true;
#pragma unroll
      for (int i = 0; i < vs.kEach; i++) finite = take_finite(vs.r[i]) && finite;
      if (!finite) bad[tile & 1] = int(tile) + 1;
    }
    vs.store(t, m + N * kTile);
  };
  if (first < end) {
    ks.load(t, k, a.k.t, to - first * Keys, a.dim);
    vs.load(t, v, a.v.t, to - first * Keys, a.dim);
    __syncthreads();
    put(first);
  }
  __syncthreads();
  for (int64_t tile = first; tile < end; tile++) {
    const int64_t key0 = tile * Keys;
    k += Keys * a.k.t;
    v += Keys * a.v.t;
    if (tile + 1 < end) {
      ks.load(t, k, a.k.t, to - key0 - Keys, a.dim);
      vs.load(t, v, a.v.t, to - key0 - Keys, a.dim);
    }
    if (key0 < wave_any) {
      const E *km = tiles + (tile & 1) * kBuffer, *vm = km + N * kTile;
      f32x16 x[Keys / 32];
#pragma unroll
      for (int i = 0; i < Keys / 32; i++) {
        x[i] = f32x16{};
#pragma unroll
        for (int j = 0; j < D / 16; j++) x[i] = product<T, N>(x[i], rows_of_tile<N, D>(km, kTile, 32 * i, j), q[j]);
      }
      Bits<N> p[Keys / 16];
      terms_of<T, D, Keys / 32>(r, x, p, a.scale, key0 + Keys > wave_all, int(clamped(mine - key0, Keys)) - 4 * half);
#pragma unroll
      for (int d = 0; d < D / 32; d++)
#pragma unroll
        for (int i = 0; i < Keys / 16; i++) r.out[d] = product<T, N>(r.out[d], columns_of_tile<N, D>(vm, kTile, 16 * i, 32 * d), p[i]);
      if (key0 + Keys > all && bad[tile & 1] == int(tile) + 1)
        add_infinite<T, D>(r, v - Keys * a.v.t, a.v.t, to - key0 < Keys ? to - key0 : Keys, mine - key0, a.dim);
    }
    if (tile + 1 < end) put(tile + 1);
    __syncthreads();
  }
  finish<T, D>(a, s, r, row, split, sum_halves(r.sum));
}

// Up to 32 rows of a sequence and key head: the tokens being decoded, bound
// by the keys and values, which are read once. A split's tiles of 32 keys go
// to four waves in turn, each with its own part of LDS and no barrier; what
// they have is joined at the end.
template <typename T, int D>
__global__ __launch_bounds__(256, Planes<T>::kWaves) void attend_few(const AttentionArgs a) {
  constexpr int N = Planes<T>::N, kTile = 32 * D, kWaves = 4;
  typedef typename Planes<T>::E E;
  extern __shared__ u32x4 lds[];
  const int t = threadIdx.x, l = t & 63, w = wave_index(), half = l >> 5;
  const uint32_t block = block_index(), id = block / uint32_t(a.splits);
  const int split = int(block - id * uint32_t(a.splits));
  if (block >= a.workgroups) return;
  const Span s = span_of(a, id, uint32_t(a.slots), a.group, 32, true);
  if (s.tile < 0) return;
  const int64_t row0 = int64_t(s.tile) * 32, row = row0 + (l & 31);
  if (row0 >= s.rows) return;
  const int64_t last_row = s.rows - 1 < row0 + 31 ? s.rows - 1 : row0 + 31;
  const int64_t to = clamped(last_row / a.group + s.ahead + 1, s.keys);
  const int64_t all = clamped(row0 / a.group + s.ahead + 1, s.keys);
  const int64_t mine = clamped(row / a.group + s.ahead + 1, s.keys);
  const int64_t count = (to + 31) / 32;
  const int64_t first = count * split / a.splits + w, end = count * (split + 1) / a.splits;

  Bits<N> q[D / 16];
  load_queries<T, D>(q, a, a.q, s, row, a.negate);
  Running<D> r;
  E *m = reinterpret_cast<E *>(lds) + w * N * kTile;
  Staged<T, D, 32, 64> ks, vs;
  const T *k = reinterpret_cast<const T *>(element(a.k, s.batch, s.key0 + first * 32, s.kv, sizeof(T)));
  const T *v = reinterpret_cast<const T *>(element(a.v, s.batch, s.key0 + first * 32, s.kv, sizeof(T)));
  if (first < end) {
    ks.load(l, k, a.k.t, to - first * 32, a.dim);
    vs.load(l, v, a.v.t, to - first * 32, a.dim);
  }
  for (int64_t tile = first; tile < end; tile += kWaves) {
    const int64_t key0 = tile * 32, next = key0 + 32 * kWaves;
    const bool masked = key0 + 32 > all, more = tile + kWaves < end;
    k += 32 * kWaves * a.k.t;
    ks.store(l, m);
    if (more) ks.load(l, k, a.k.t, to - next, a.dim);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    f32x16 x[1] = {};
#pragma unroll
    for (int j = 0; j < D / 16; j++) x[0] = product<T, N>(x[0], rows_of_tile<N, D>(m, kTile, 0, j), q[j]);
    Bits<N> p[2];
    terms_of<T, D, 1>(r, x, p, a.scale, masked, int(clamped(mine - key0, 32)) - 4 * half);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    bool finite = true;
    if (masked) {
#pragma unroll
      for (int i = 0; i < vs.kEach; i++) finite = take_finite(vs.r[i]) && finite;
    }
    vs.store(l, m);
    const bool some_bad = masked && __ballot(!finite);
    const T *here = v;
    v += 32 * kWaves * a.v.t;
    if (more) vs.load(l, v, a.v.t, to - next, a.dim);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int d = 0; d < D / 32; d++)
#pragma unroll
      for (int i = 0; i < 2; i++) r.out[d] = product<T, N>(r.out[d], columns_of_tile<N, D>(m, kTile, 16 * i, 32 * d), p[i]);
    if (some_bad) add_infinite<T, D>(r, here, a.v.t, to - key0 < 32 ? to - key0 : 32, mine - key0, a.dim);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }

  // the waves' maxima and sums, then their outputs at the largest maximum
  __syncthreads();
  __shared__ float tops[kWaves][32], sums[kWaves][32];
  float *outs = reinterpret_cast<float *>(lds);  // [wave][row][D]
  const float sum = sum_halves(r.sum);
  if (!half) tops[w][l] = r.top, sums[w][l] = sum;
  __syncthreads();
  float top = tops[0][l & 31], total = 0.0f;
#pragma unroll
  for (int i = 1; i < kWaves; i++) top = fmaxf(top, tops[i][l & 31]);
  const float from = top == -INFINITY ? 0.0f : top;
#pragma unroll
  for (int i = 0; i < kWaves; i++) total += sums[i][l & 31] * __builtin_amdgcn_exp2f(tops[i][l & 31] - from);
  const float factor = __builtin_amdgcn_exp2f(r.top - from);
  if (row < s.rows) {
#pragma unroll
    for (int d = 0; d < D / 32; d++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        f32x4 y;
#pragma unroll
        for (int i = 0; i < 4; i++) y[i] = r.out[d][4 * j + i] * factor;
        *reinterpret_cast<f32x4 *>(outs + (w * 32 + (l & 31)) * D + ((32 * d + 8 * j + 4 * half) ^ ((l & 7) * 4))) = y;
      }
  }
  __syncthreads();
  const int64_t left = s.rows - row0;
  const int rows = left < 32 ? int(left) : 32;
  const int64_t all_rows = a.batch * a.kv_heads * a.tokens * a.group;
  // eight elements a thread, D / 8 threads a row; every thread of a wave
  // goes on, as a row's sum comes from another lane
  for (int i = t; i < (rows * (D / 8) + 63) / 64 * 64; i += 256) {
    const int at_row = i / (D / 8), at = i % (D / 8) * 8;
    const float its = __shfl(total, at_row & 31, 64), its_top = __shfl(top, at_row & 31, 64);
    if (at_row >= rows || at >= a.dim) continue;
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int c = at_row * D + ((at + j) ^ ((at_row & 7) * 4));
      y[j] = 0.0f;
#pragma unroll
      for (int wave = 0; wave < kWaves; wave++) y[j] += outs[wave * 32 * D + c];
    }
    const int n = a.dim - at < 8 ? a.dim - at : 8;
    const int64_t all_at = row_values(a, s) + row0 + at_row;
    if (a.splits > 1) {
      float *p = a.partial + (all_at * a.splits + split) * a.dim + at;
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (j < n) p[j] = y[j];
      if (!at) {
        float *ms = a.partial + all_rows * a.splits * a.dim + (all_at * a.splits + split) * 2;
        ms[0] = its_top;
        ms[1] = its;
      }
      continue;
    }
    const int64_t token = (row0 + at_row) / a.group;
    const int head = int(row0 + at_row - token * a.group);
    T *p = reinterpret_cast<T *>(const_cast<char *>(element(a.o, s.batch, s.first + token, int64_t(s.kv) * a.group + head, sizeof(T)))) + at;
    const float up = its == 0.0f ? 0.0f : 1.0f / its;
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (j < n) {
        p[j] = T(y[j] * up);
        if (a.o_rest) a.o_rest[all_at * a.dim + at + j] = bf16(y[j] * up - float(p[j]));
      }
    if (a.lse && !at) a.lse[all_at] = its == 0.0f ? INFINITY : its_top - Powers<T>::kLift + __builtin_log2f(its);
  }
}

// The splits' outputs of a row joined, a wave a row.
template <typename T>
__global__ __launch_bounds__(256) void join_splits(const AttentionArgs a) {
  const int l = threadIdx.x & 63;
  const int64_t rows = a.batch * a.kv_heads * a.tokens * a.group, at = int64_t(block_index()) * 4 + (threadIdx.x >> 6);
  if (at >= rows) return;
  const float *ms = a.partial + rows * a.splits * a.dim + at * a.splits * 2;
  float top = -INFINITY;
  for (int i = 0; i < a.splits; i++) top = fmaxf(top, ms[2 * i]);
  const float from = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f, y[2] = {};
  for (int i = 0; i < a.splits; i++) {
    const float f = __builtin_amdgcn_exp2f(ms[2 * i] - from);
    sum += ms[2 * i + 1] * f;
    const float *p = a.partial + (at * a.splits + i) * a.dim;
#pragma unroll
    for (int j = 0; j < 2; j++)
      if (l + 64 * j < a.dim) y[j] += p[l + 64 * j] * f;
  }
  // at = ((batch x kv heads + kv) x tokens + token) x group + head of the group
  const int64_t per_head = a.tokens * a.group, pair = at / per_head, in = at - pair * per_head, token = in / a.group;
  const int64_t batch = pair / a.kv_heads, head = (pair - batch * a.kv_heads) * a.group + (in - token * a.group);
  T *p = reinterpret_cast<T *>(const_cast<char *>(element(a.o, batch, token, head, sizeof(T))));
  const float up = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int j = 0; j < 2; j++)
    if (l + 64 * j < a.dim) {
      p[l + 64 * j] = T(y[j] * up);
      if (a.o_rest) a.o_rest[at * a.dim + l + 64 * j] = bf16(y[j] * up - float(T(y[j] * up)));
    }
  if (a.lse && !l) a.lse[at] = sum == 0.0f ? INFINITY : top - Powers<T>::kLift + __builtin_log2f(sum);
}

template <typename T, int D, int Waves, int Keys>
void launch_attend(const AttentionArgs &a, hipStream_t stream) {
  constexpr size_t bytes = size_t(2) * 2 * Planes<T>::N * Keys * D * 2;
  check_hip(hipFuncSetAttribute(reinterpret_cast<const void *>(&attend<T, D, Waves, Keys>), hipFuncAttributeMaxDynamicSharedMemorySize, int(bytes)),
            "attention");
  hipLaunchKernelGGL((attend<T, D, Waves, Keys>), grid_of(a.workgroups), dim3(Waves * 64), bytes, stream, a);
}

template <typename T, int D>
void launch_attend_few(const AttentionArgs &a, hipStream_t stream) {
  constexpr size_t tiles = size_t(4) * Planes<T>::N * 32 * D * 2, outs = size_t(4) * 32 * D * 4, bytes = tiles > outs ? tiles : outs;
  check_hip(hipFuncSetAttribute(reinterpret_cast<const void *>(&attend_few<T, D>), hipFuncAttributeMaxDynamicSharedMemorySize, int(bytes)), "attention");
  hipLaunchKernelGGL((attend_few<T, D>), grid_of(a.workgroups), dim3(256), bytes, stream, a);
}

// `waves` 0: the kernel for few rows.
template <typename T>
void attend_launch(const AttentionArgs &a, int waves, hipStream_t stream) {
  constexpr int kKeys = std::is_same<T, float>::value ? 32 : 64;
  if (a.dim <= 64) {
    if (!waves) launch_attend_few<T, 64>(a, stream);
    else if (waves == 4) launch_attend<T, 64, 4, kKeys>(a, stream);
    else if constexpr (!std::is_same<T, float>::value) launch_attend<T, 64, 8, kKeys>(a, stream);
  } else {
    if (!waves) launch_attend_few<T, 128>(a, stream);
    else if (waves == 4) launch_attend<T, 128, 4, kKeys>(a, stream);
    else if constexpr (!std::is_same<T, float>::value) launch_attend<T, 128, 8, kKeys>(a, stream);
  }
  check_launch("attention");
  if (a.splits > 1) {
    const int64_t rows = a.batch * a.kv_heads * a.tokens * a.group;
    hipLaunchKernelGGL((join_splits<T>), grid_of((rows + 3) / 4), dim3(256), 0, stream, a);
    check_launch("attention");
  }
}

}  // namespace op
}  // namespace cchip
