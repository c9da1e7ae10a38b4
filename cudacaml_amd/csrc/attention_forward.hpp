// Attention, forward: the kernel over tiles of rows, and the one for few rows
// whose waves share the keys out.

#include "attention.hpp"

namespace cchip {
namespace op {

// A row's maximum follows the largest score only when that is kSlack (a power
// of two) ahead of it: what the row has so far is rescaled in the first tile
// and hardly ever again, and never for another row's sake, so that a row's
// result does not depend on its neighbours. Terms are 2^(score - maximum + kLift): f16 has normal
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
//
// Terms of 16-bit types are rounded to T, as the product takes operands of one
// type, which is the one rounding of an output besides its own: bf16 outputs
// are 2.0e-3 to 2.3e-3 off 64 bits (2-norm), f16 ones 2.6e-4. With a second
// operand for what rounding leaves off they are 1.6e-3 and 2.1e-4, their own
// rounding; that is half as many products again: 714 us in place of 577 for a prompt of
// 8192 tokens, 170 in place of 145 for chunks of 512, 313 in place of 260 for
// a token each of 64 sequences, f16 15.6 in place of 15.0 for four. f32 has all of its bits.
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
    const float top = most > r.top + Powers<T>::kSlack ? most : r.top;
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

// Planes of f32 cannot hold an infinity: the scores of 32 Tiles keys that came
// out as NaN are made again from q and k themselves.
template <int Tiles>
__device__ __forceinline__ void plain_scores(f32x16 (&s)[Tiles], const AttentionArgs &a, const Span &span, int64_t row, const float *k, int64_t keys) {
  bool some = false;
#pragma unroll
  for (int t = 0; t < Tiles; t++)
#pragma unroll
    for (int i = 0; i < 16; i++) some = some || s[t][i] != s[t][i];
  if (!__ballot(some)) return;
  stay_branch();
  if (row >= span.rows) return;
  const int half = (threadIdx.x & 63) >> 5;
  const int64_t token = row / a.group;
  const float *q = reinterpret_cast<const float *>(element(a.q, span.batch, span.first + token, int64_t(span.kv) * a.group + (row - token * a.group), sizeof(float)));
#pragma unroll
  for (int t = 0; t < Tiles; t++)
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const int key = t * 32 + 8 * (i / 4) + 4 * half + i % 4;
      if (s[t][i] == s[t][i] || key >= keys) continue;
      float sum = 0.0f;
#pragma unroll 1
      for (int d = 0; d < a.dim; d++) sum = __builtin_fmaf(a.negate ? -q[d] : q[d], k[key * a.k.t + d], sum);
      s[t][i] = sum;
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

// Whether an element is infinite or NaN; and zero in its place. Planes cannot
// hold one, so that values of f32 are looked at in all tiles, others only in
// those that some rows do not see all of.
template <typename T>
constexpr bool kPlanar = Planes<T>::N > 1;

template <typename T>
__device__ __forceinline__ bool take_finite(Raw8<T> &r) {
  if constexpr (kPlanar<T>) {
    float any = 0.0f;  // NaN: an element is not finite
#pragma unroll
    for (int i = 0; i < 8; i++) any = __builtin_fmaf(r.x[i], 0.0f, any);
    if (any == 0.0f) return true;
    stay_branch();
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (!(__builtin_fabsf(r.x[i]) < INFINITY)) r.x[i] = 0.0f;
    return false;
  } else {
    bool all = true;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const bool finite = __builtin_fabsf(float(r.x[i])) < INFINITY;
      all = all && finite;
      if (!finite) r.x[i] = T(0.0f);
    }
    return all;
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

// The same of eight 16-bit elements as they are: exponents of ones only.
template <typename T>
__device__ __forceinline__ bool some_infinite(uint32_t u) {
  const uint32_t e = std::is_same<T, f16>::value ? 0x7C007C00u : 0x7F807F80u, one = std::is_same<T, f16>::value ? 0x04000400u : 0x00800080u;
  return ((u & e) + one) & 0x80008000u;
}

template <typename T>
__device__ __forceinline__ u32x4 finite_only(u32x4 u) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if (some_infinite<T>(u[i] & 0xFFFFu)) u[i] &= 0xFFFF0000u;
    if (some_infinite<T>(u[i] & 0xFFFF0000u)) u[i] &= 0xFFFFu;
  }
  return u;
}

// Of a tile, without what lies between its groups, which nothing writes.
template <typename T>
__device__ __forceinline__ bool tile_finite(const u32x4 *tile, int groups) {
  bool some = false;
  for (int i = 0; i < groups; i++) {
    const u32x4 u = tile[i * (kGroup / 8) + (threadIdx.x & 63)];
    some = some || some_infinite<T>(u[0]) || some_infinite<T>(u[1]) || some_infinite<T>(u[2]) || some_infinite<T>(u[3]);
  }
  return __ballot(some) == 0;
}

// Values of a tile that are not finite, and that the tile has zeros for,
// where a row sees them: an infinity or NaN times the term's sign. A product
// would bring them to the rows that do not, as zero times infinity.
template <typename T, int D>
__device__ __forceinline__ void add_infinite(Running<D> &r, const T *v, int64_t stride, int64_t keys, int64_t seen, int dim) {
  const int l = threadIdx.x & 63, half = l >> 5;
#pragma unroll 1
  for (int64_t j0 = 0; j0 < keys; j0 += 8) {
    uint32_t rows = 0;  // of eight, that have any
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const T *row = v + (j0 + i < keys ? j0 + i : j0) * stride;
      bool some = false;
#pragma unroll
      for (int d = 0; d < D; d += 64) some = some || (l + d < dim && !(__builtin_fabsf(float(row[l + d])) < INFINITY));
      if (__ballot(some) && j0 + i < keys) rows |= 1u << i;
    }
    for (; rows; rows &= rows - 1) {
      const int64_t j = j0 + __builtin_ctz(rows);
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
}

// 32 Waves rows of a sequence and key head, a split of the keys they see, in
// tiles of Keys keys that go from memory to LDS, 16-bit ones of whole 16-byte
// pieces directly (Direct), others through registers. A wave goes
// through two phases a tile: products (what the terms of the tile before give
// of its values, and this tile's scores) and terms. Of eight waves, two a SIMD,
// four are a phase behind, so that the matrix units have one half's products
// while the vector units make the other half's terms; with all in step each
// would wait for the other. A tile of 64 keys and 256 rows of 128 takes 2.3 us, in
// which a SIMD's products are 0.9 and its two waves' terms, some 125 vector
// instructions each, 0.8 at most. As long as the products are the reads of LDS:
// each of eight waves reads the whole tile for its 32 rows, 256 KB. Between them
// stand the copies, some 90 scalar instructions a wave with reloads of scalars
// that the function, masked tail and all, spills (405). Which of these a tile
// waits for was not taken apart. 8192 tokens, 32 heads of 128 over 8, bf16: 589 us, 934 TFLOP/s of the
// products that masks leave (a library's product of 16384: 1363).
template <typename T, int D, int Waves, int Keys, bool Direct>
__global__ CCHIP_WAVES(Waves * 64, Planes<T>::kWaves) void attend(const AttentionArgs a) {
  constexpr int N = Planes<T>::N, kTile = tile_elements<D>(Keys), kBuffer = N * kTile;
  constexpr bool kTwo = Waves == 8;
  constexpr int kSlots = Direct ? 4 : 2;
  typedef typename Planes<T>::E E;
  extern __shared__ u32x4 lds[];
  __shared__ int bad[2];  // the tile, counted from 1, in a buffer some of whose values were not finite
  E *const kt = reinterpret_cast<E *>(lds), *const vt = kt + kSlots * kBuffer;  // [kSlots][plane][Keys][D] of keys and of values

  const int t = threadIdx.x, l = t & 63, half = l >> 5, w = wave_index();
  const uint32_t block = block_index(), id = block / uint32_t(a.splits);
  const int split = int(block - id * uint32_t(a.splits));
  if (block >= a.workgroups) return;
  const Span s = span_of(a, id, uint32_t(a.slots), a.group, 32 * Waves, true);
  if (s.tile < 0) return;
  const int64_t row0 = int64_t(s.tile) * 32 * Waves, wave_row = row0 + w * 32, row = wave_row + (l & 31);
  if (row0 >= s.rows) return;

  // keys that rows see: all of the workgroup's, all of the
  // wave's, the lane's
  const int64_t last_row = s.rows - 1 < row0 + 32 * Waves - 1 ? s.rows - 1 : row0 + 32 * Waves - 1;
  const int to = int(clamped(last_row / a.group + s.ahead + 1, s.keys));
  const int all = int(clamped(row0 / a.group + s.ahead + 1, s.keys));
  const int wave_all = int(clamped(wave_row / a.group + s.ahead + 1, s.keys));
  const int mine = int(clamped(row / a.group + s.ahead + 1, s.keys));
  const int count = (to + Keys - 1) / Keys;
  const int first = int(int64_t(count) * split / a.splits), end = int(int64_t(count) * (split + 1) / a.splits);

  Bits<N> q[D / 16];
  load_queries<T, D>(q, a, a.q, s, row, a.negate);
  Running<D> r;
  const T *const k = reinterpret_cast<const T *>(element(a.k, s.batch, s.key0, s.kv, sizeof(T)));
  const T *const v = reinterpret_cast<const T *>(element(a.v, s.batch, s.key0, s.kv, sizeof(T)));
  if (t < 2) bad[t] = 0;

  Staged<T, D, Keys, Waves * 64> ks, vs;
  const auto load = [&](int k_tile, int v_tile) {
    if (k_tile < end) ks.load(t, k + int64_t(k_tile) * Keys * a.k.t, a.k.t, to - k_tile * Keys, a.dim);
    if (v_tile < end) vs.load(t, v + int64_t(v_tile) * Keys * a.v.t, a.v.t, to - v_tile * Keys, a.dim);
  };
  const auto put = [&](int k_tile, int v_tile) {
    if (k_tile < end) ks.store(t, kt + (k_tile & 1) * kBuffer);
    if (v_tile < end) {
      if (kPlanar<T> || (v_tile + 1) * Keys > all) {
        stay_branch();
        bool finite = true;
#pragma unroll
        for (int i = 0; i < vs.kEach; i++) finite = take_finite(vs.r[i]) && finite;
        if (!finite) bad[v_tile & 1] = v_tile + 1;
      }
      vs.store_whole(t, vt + (v_tile & 1) * kBuffer);
    }
  };
  const Places<D> at;
  f32x16 x[Keys / 32];
  Bits<N> p[Keys / 16];
  constexpr int kValues = D / 32 * (Keys / 16), kScores = Keys / 32 * (D / 16);
  const auto read_values = [&](int tile, int i) {
    return columns_of_tile<N, D>(at, vt + tile % kSlots * kBuffer, kTile, 16 * (i / (D / 32)), 32 * (i % (D / 32)));
  };
  const auto read_keys = [&](int tile, int i) {
    return rows_of_tile<N, D>(at, kt + tile % kSlots * kBuffer, kTile, 32 * (i % (Keys / 32)), i / (Keys / 32));
  };
  const auto use_values = [&](int i, const Bits<N> &f) { r.out[i % (D / 32)] = product<T, N>(r.out[i % (D / 32)], f, p[i / (D / 32)]); };
  const auto use_keys = [&](int i, const Bits<N> &f) { x[i % (Keys / 32)] = product<T, N>(x[i % (Keys / 32)], f, q[i / (Keys / 32)]); };
  const auto scores = [&](int tile) {
#pragma unroll
    for (int i = 0; i < Keys / 32; i++) x[i] = f32x16{};
    const auto read = [&](int i) { return read_keys(tile, i); };
    Ahead<kScores, 6 / N, N> ahead;
    ahead.start(read);
    ahead.run(read, use_keys);
  };
  // products of the terms of tile - 1 and, between, the scores of tile
  const auto both = [&](int tile) {
#pragma unroll
    for (int i = 0; i < Keys / 32; i++) x[i] = f32x16{};
    const auto read = [&](int i) { return i < kValues ? read_values(tile - 1, i) : read_keys(tile, i - kValues); };
    Ahead<kValues + kScores, 6 / N, N> ahead;
    ahead.start(read);
    ahead.run(read, [&](int i, const Bits<N> &f) { i < kValues ? use_values(i, f) : use_keys(i - kValues, f); });
  };
  const auto values = [&](int tile) {
    const auto read = [&](int i) { return read_values(tile, i); };
    Ahead<kValues, 6 / N, N> ahead;
    ahead.start(read);
    ahead.run(read, use_values);
  };
  const auto infinite = [&](int tile) {
    stay_branch();
    add_infinite<T, D>(r, v + int64_t(tile) * Keys * a.v.t, a.v.t, to - tile * Keys < Keys ? to - tile * Keys : Keys, mine - tile * Keys, a.dim);
  };
  // `some` rows may not see all of the tile
  const auto terms = [&](int tile, bool some) {
    if constexpr (std::is_same<T, float>::value) plain_scores(x, a, s, row, k + int64_t(tile) * Keys * a.k.t, to - tile * Keys);
    terms_of<T, D, Keys / 32>(r, x, p, a.scale, some && (tile + 1) * Keys > wave_all, (mine - tile * Keys < Keys ? mine - tile * Keys : Keys) - 4 * half);
  };

  const bool behind = kTwo && w >= Waves / 2;
  if constexpr (Direct) {
    // Tiles are copied three ahead, in the first phase of a tile's two, and
    // are there when the second ends: the slot that one goes to was done with
    // then. Behind the last tile copies go on, so that those on their way can
    // be counted.
    Copied<D, Keys, Waves * 64> kc, vc;
    kc.start(a.k.t, a.dim);
    vc.start(a.v.t, a.dim);
    const auto copy_keys = [&](int tile) {
      const int at = tile < end ? tile : end - 1;
      kc.copy(reinterpret_cast<const char *>(k + int64_t(at) * Keys * a.k.t), uint32_t(a.k.t), to - at * Keys, a.dim,
              reinterpret_cast<char *>(kt + tile % kSlots * kBuffer));
    };
    const auto copy_values = [&](int tile) {
      const int at = tile < end ? tile : end - 1;
      vc.copy(reinterpret_cast<const char *>(v + int64_t(at) * Keys * a.v.t), uint32_t(a.v.t), to - at * Keys, a.dim,
              reinterpret_cast<char *>(vt + tile % kSlots * kBuffer));
    };
    const auto copy = [&](int tile) { copy_keys(tile + 3), copy_values(tile + 2); };
    constexpr int kLeft = 2 * (kc.kEach + vc.kEach);
    // values that rows see and others do not have to be finite for a product
    const auto values_of = [&](int tile) {
      if ((tile + 1) * Keys <= all || tile_finite<T>(reinterpret_cast<const u32x4 *>(vt + tile % kSlots * kBuffer), kTile / kGroup)) return values(tile);
      stay_branch();
#pragma unroll
      for (int i = 0; i < kValues; i++) {
        Bits<N> f = read_values(tile, i);
        f.p[0] = finite_only<T>(f.p[0]);
        use_values(i, f);
        __builtin_amdgcn_sched_barrier(0);
      }
      infinite(tile);
    };
    if (first < end) {
      if (a.dim < D) {
        for (int i = t; i < 2 * kSlots * kBuffer / 8; i += Waves * 64) lds[i] = u32x4{};
        __syncthreads();
      }
      copy_keys(first), copy_keys(first + 1), copy_values(first);
      copy_keys(first + 2), copy_values(first + 1);
      copies_left<kLeft>();
      __syncthreads();
      if (kTwo && behind) copy(first), phase_done();
      const auto step = [&](int tile, bool some) {
        if (behind) copies_left<kLeft>();
        if (kTwo) phase_done();
        if (behind) copy(tile + 1);
        terms(tile, some);
        if (!behind) copies_left<kLeft>();
        phase_done();
      };
      if (!behind) copy(first);
      scores(first);
      step(first, true);
      const int full = all / Keys < end ? all / Keys : end;  // tiles that all rows see
      int tile = first + 1;
      for (; tile < full; tile++) {
        if (!behind) copy(tile);
        both(tile);
        step(tile, false);
      }
      for (; tile < end; tile++) {
        if (!behind) copy(tile);
        values_of(tile - 1);
        scores(tile);
        step(tile, true);
      }
      values_of(end - 1);
      if (kTwo && !behind) phase_done();
      copies_done();
    }
  } else {
    // waves that are behind have the tiles after theirs on their way one phase
    // earlier, as all that a phase of the others needs is there at its start
    const int lead = behind ? 1 : 0;
    const auto step = [&](int tile) {
      if (kTwo) phase_done();
      terms(tile, true);
      put(tile + 1 + lead, tile + lead);
      phase_done();
    };
    const auto mend = [&](int tile) {
      if ((kPlanar<T> || (tile + 1) * Keys > all) && bad[tile & 1] == tile + 1) infinite(tile);
    };
    if (first < end) {
      load(first, end);
      copies_done();  // the queries too: a wait within the loop would be for the keys on their way as well
      if (kTwo) __syncthreads();  // `bad` is clear before a wave that is behind says what it found in the first values
      put(first, end);
      if (behind) {
        load(first + 1, first);
        put(first + 1, first);
      }
      __syncthreads();
      if (behind) phase_done();
      load(first + 1 + lead, first + lead);
      scores(first);
      step(first);
      for (int tile = first + 1; tile < end; tile++) {
        load(tile + 1 + lead, tile + lead);
        both(tile);
        mend(tile - 1);
        step(tile);
      }
      values(end - 1);
      mend(end - 1);
      if (kTwo && !behind) phase_done();
    }
  }
  finish<T, D>(a, s, r, row, split, sum_halves(r.sum));
}

// Up to 32 rows of a sequence and key head: the tokens being decoded, bound
// by the keys and values, which are read once. A split's tiles of 32 keys go
// to four waves in turn, each with its own part of LDS and no barrier; what
// they have is joined at the end. 64 sequences of up to 8192 keys, 8 key heads
// of 128, bf16: 255 us for 1.09 GB, 4.3 TB/s (a copy: 4.86; 5.8 where all are as
// long); four of 1024, f16: 12.4 us, a launch and one chain of memory's, LDS's and the
// join's latencies.
template <typename T, int D>
__global__ CCHIP_WAVES(256, Planes<T>::kWaves) void attend_few(const AttentionArgs a) {
  constexpr int N = Planes<T>::N, kTile = tile_elements<D>(32), kWaves = 4;
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
  const Places<D> at;
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
    for (int j = 0; j < D / 16; j++) x[0] = product<T, N>(x[0], rows_of_tile<N, D>(at, m, kTile, 0, j), q[j]);
    if constexpr (std::is_same<T, float>::value) plain_scores(x, a, s, row, k - 32 * kWaves * a.k.t, to - key0);
    Bits<N> p[2];
    terms_of<T, D, 1>(r, x, p, a.scale, masked, int(clamped(mine - key0, 32)) - 4 * half);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    bool finite = true;
    if (kPlanar<T> || masked) {
#pragma unroll
      for (int i = 0; i < vs.kEach; i++) finite = take_finite(vs.r[i]) && finite;
    }
    vs.store_whole(l, m);
    const bool some_bad = (kPlanar<T> || masked) && __ballot(!finite);
    const T *here = v;
    v += 32 * kWaves * a.v.t;
    if (more) vs.load(l, v, a.v.t, to - next, a.dim);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int d = 0; d < D / 32; d++)
#pragma unroll
      for (int i = 0; i < 2; i++) r.out[d] = product<T, N>(r.out[d], columns_of_tile<N, D>(at, m, kTile, 16 * i, 32 * d), p[i]);
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
    const int at_row = i / (D / 8), col = i % (D / 8) * 8;
    const float its = __shfl(total, at_row & 31, 64), its_top = __shfl(top, at_row & 31, 64);
    if (at_row >= rows || col >= a.dim) continue;
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int c = at_row * D + ((col + j) ^ ((at_row & 7) * 4));
      y[j] = 0.0f;
#pragma unroll
      for (int wave = 0; wave < kWaves; wave++) y[j] += outs[wave * 32 * D + c];
    }
    const int n = a.dim - col < 8 ? a.dim - col : 8;
    const int64_t all_at = row_values(a, s) + row0 + at_row;
    if (a.splits > 1) {
      float *p = a.partial + (all_at * a.splits + split) * a.dim + col;
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (j < n) p[j] = y[j];
      if (!col) {
        float *ms = a.partial + all_rows * a.splits * a.dim + (all_at * a.splits + split) * 2;
        ms[0] = its_top;
        ms[1] = its;
      }
      continue;
    }
    const int64_t token = (row0 + at_row) / a.group;
    const int head = int(row0 + at_row - token * a.group);
    T *p = reinterpret_cast<T *>(const_cast<char *>(element(a.o, s.batch, s.first + token, int64_t(s.kv) * a.group + head, sizeof(T)))) + col;
    const float up = its == 0.0f ? 0.0f : 1.0f / its;
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (j < n) {
        p[j] = T(y[j] * up);
        if (a.o_rest) a.o_rest[all_at * a.dim + col + j] = bf16(y[j] * up - float(p[j]));
      }
    if (a.lse && !col) a.lse[all_at] = its == 0.0f ? INFINITY : its_top - Powers<T>::kLift + __builtin_log2f(its);
  }
}

// The splits' outputs of a row joined, a wave a row, some splits' reads under
// way at a time: 3.9 us for 64 rows of 8 splits, 17.1 for 32768 of 2.
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
#pragma unroll 4
  for (int i = 0; i < a.splits; i++) {
    const float f = __builtin_amdgcn_exp2f(ms[2 * i] - from);
    sum += ms[2 * i + 1] * f;
    const float *p = a.partial + (at * a.splits + i) * a.dim;
#pragma unroll
    for (int j = 0; j < 2; j++) y[j] += p[l + 64 * j < a.dim ? l + 64 * j : 0] * f;
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

// Whether rows are of whole pieces of 16 bytes, at places of them.
inline bool whole_pieces(const AttentionArgs &a, const Heads &x) {
  return a.dim % 8 == 0 && aligned16(x.p) && x.t % 8 == 0 && (x.h % 8 == 0 || a.kv_heads == 1) && (x.b % 8 == 0 || a.batch == 1);
}

template <typename T, int D, int Waves, int Keys, bool Direct>
void launch_attend_as(const AttentionArgs &a, hipStream_t stream) {
  constexpr size_t bytes = size_t(Direct ? 4 : 2) * 2 * Planes<T>::N * tile_elements<D>(Keys) * 2;
  allow_lds<&attend<T, D, Waves, Keys, Direct>>(int(bytes), "attention");
  hipLaunchKernelGGL((attend<T, D, Waves, Keys, Direct>), grid_of(a.workgroups), dim3(Waves * 64), bytes, stream, a);
}

template <typename T, int D, int Waves, int Keys>
void launch_attend(const AttentionArgs &a, hipStream_t stream) {
  if constexpr (!std::is_same<T, float>::value) {
    if (whole_pieces(a, a.k) && whole_pieces(a, a.v)) return launch_attend_as<T, D, Waves, Keys, true>(a, stream);
  }
  launch_attend_as<T, D, Waves, Keys, false>(a, stream);
}

template <typename T, int D>
void launch_attend_few(const AttentionArgs &a, hipStream_t stream) {
  constexpr size_t tiles = size_t(4) * Planes<T>::N * tile_elements<D>(32) * 2, outs = size_t(4) * 32 * D * 4, bytes = tiles > outs ? tiles : outs;
  allow_lds<&attend_few<T, D>>(int(bytes), "attention");
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
