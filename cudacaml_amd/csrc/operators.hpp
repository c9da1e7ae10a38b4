// What the layer operators (delta*.hip, attention*.hip, head_norm.hip,
// embedding.hip, norm_block*.hip, dropout.hip) share: element types, raw loads at any alignment, matrix-core fragments held in
// one to three bf16 planes, and the counter-based generator.
#pragma once

#include <hip/hip_runtime.h>

#include <atomic>
#include <cstdint>
#include <type_traits>

#include "internal.hpp"

namespace cchip {
namespace op {

typedef __bf16 bf16;
typedef _Float16 f16;
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// Eight neighbouring elements as they lie in memory: 16-byte accesses at any
// alignment that the elements have (the hardware takes them; what counts is
// how many lines they touch) where all eight exist; otherwise the first
// `valid` one by one, the rest zero.
template <typename T>
struct Raw8 {
  T x[8];
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));

template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T *p, int valid) {
  Raw8<T> r;
  if (valid == 8) {
    const u32x4_any *s = reinterpret_cast<const u32x4_any *>(p);
    u32x4 *d = reinterpret_cast<u32x4 *>(&r);
#pragma unroll
    for (int i = 0; i < int(sizeof(T) * 8 / 16); i++) d[i] = s[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) r.x[i] = i < valid ? p[i] : T(0.0f);
  }
  return r;
}

// Two values rounded to bf16, and those as f32 again. By conversions of the
// language and not an asm instruction: what a product has just written must
// not be read for some cycles, and only instructions that the compiler knows
// are kept from it.
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), bf16x2));
}
__device__ __forceinline__ float low_bf16(uint32_t u) { return __builtin_bit_cast(float, u << 16); }
__device__ __forceinline__ float high_bf16(uint32_t u) { return __builtin_bit_cast(float, u & 0xFFFF0000u); }

// x as the sum of N bf16 values, each the rounding of what the ones before
// it leave: 8, 16 and 24 bits of x for N = 1, 2 and 3 (24 hold every f32, 11
// every f16).
template <int N>
__device__ __forceinline__ void split(float x, bf16 (&out)[N]) {
#pragma unroll
  for (int i = 0; i < N; i++) {
    out[i] = bf16(x);
    x -= float(out[i]);
  }
}

// A matrix-core operand of 16 rows (or columns) and 32 terms: lane l holds
// row l % 16, terms 8 (l / 16) .. + 7, in N planes.
template <int N>
struct Frag {
  bf16x8 p[N];
};

template <int N, typename T>
__device__ __forceinline__ Frag<N> frag_of(const Raw8<T> &r) {
  Frag<N> f;
  if constexpr (N == 1 && std::is_same<T, bf16>::value) {
    f.p[0] = *reinterpret_cast<const bf16x8 *>(&r);
  } else {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = float(r.x[i]);
#pragma unroll
    for (int n = 0; n < N; n++) {
      u32x4 u;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const uint32_t p = pack_bf16(x[2 * i], x[2 * i + 1]);
        u[i] = p;
        x[2 * i] -= low_bf16(p);
        x[2 * i + 1] -= high_bf16(p);
      }
      f.p[n] = __builtin_bit_cast(bf16x8, u);
    }
  }
  return f;
}

// Fragment of a matrix in LDS stored [row][term], rows of `ld` elements (a
// multiple of 8), planes `plane` elements apart: one 16-byte read a plane.
template <int N>
__device__ __forceinline__ Frag<N> frag_row(const bf16 *m, int plane, int ld, int row0, int term0) {
  const int l = threadIdx.x & 63;
  const bf16 *p = m + (row0 + (l & 15)) * ld + term0 + (l >> 4) * 8;
  Frag<N> f;
#pragma unroll
  for (int n = 0; n < N; n++) f.p[n] = *reinterpret_cast<const bf16x8 *>(p + n * plane);
  return f;
}

// The same of a matrix stored [term][row]: the transposing LDS read. Of 16
// lanes each gives the address of 4 neighbouring elements, 4 lanes to a
// stored row; lane i gets column i of those 4 rows of 16. Row 4 i + r of the
// fragment is stored column row0 + Apart i + r: with Apart 8 two fragments,
// row0 4 apart, are 32 columns of which a lane of their products has 8 side
// by side. 16 lanes read at a time: the four stored rows they touch lie in
// banks of their own if rows are 8 to 56 banks of 64 apart (16 or 48 with
// Apart 8).
template <int N, int Apart = 4>
__device__ __forceinline__ Frag<N> frag_col(const bf16 *m, int plane, int ld, int row0, int term0) {
  typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
  const int l = threadIdx.x & 63;
  const bf16 *p = m + (term0 + (l >> 4) * 8 + ((l >> 2) & 3)) * ld + row0 + (l & 3) * Apart;
  Frag<N> f;
#pragma unroll
  for (int n = 0; n < N; n++) {
    union {
      i16x4 h[2];
      bf16x8 v;
    } u;
    u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(p + n * plane));
    u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(p + n * plane + 4 * ld));
    f.p[n] = u.v;
  }
  return f;
}

// c += a b^T over 32 terms. Planes i and j are multiplied while i + j is
// below `Levels`: the larger count of planes unless given, which leaves out
// terms of at most 2^-18 of a product for two planes (as small as what two
// drop of an f32) and 2^-27 for three. Two planes hold an f16 whole, and with
// Levels 3 its products are exact too. Small terms first. Lane l holds rows
// 4 (l / 16) .. + 3 of column l % 16.
template <int Levels = 0, int NA, int NB>
__device__ __forceinline__ f32x4 mma(f32x4 c, const Frag<NA> &a, const Frag<NB> &b) {
  constexpr int M = Levels ? Levels : NA > NB ? NA : NB;
#pragma unroll
  for (int s = M - 1; s >= 0; s--)
#pragma unroll
    for (int i = 0; i < NA; i++) {
      const int j = s - i;
      if (j >= 0 && j < NB) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[i], b.p[j], c, 0, 0, 0);
    }
  return c;
}

// The four values that a lane has of a product into LDS, side by side.
template <int N>
__device__ __forceinline__ void put_four(bf16 *at, int plane, f32x4 x) {
#pragma unroll
  for (int n = 0; n < N; n++) {
    const uint32_t a = pack_bf16(x[0], x[1]), b = pack_bf16(x[2], x[3]);
    *reinterpret_cast<uint2 *>(at + n * plane) = make_uint2(a, b);
    x -= f32x4{low_bf16(a), high_bf16(a), low_bf16(b), high_bf16(b)};
  }
}

// A sum of products that no product waits long for: the planes' levels i + j
// (see mma) each have a sum of their own, added up at the end, small first.
template <int L>
struct Levels {
  f32x4 s[L] = {};
  template <int NA, int NB>
  __device__ __forceinline__ void add(const Frag<NA> &a, const Frag<NB> &b) {
    static_assert((NA > NB ? NA : NB) <= L, "a level has no sum");
#pragma unroll
    for (int k = (NA > NB ? NA : NB) - 1; k >= 0; k--)
#pragma unroll
      for (int i = 0; i < NA; i++) {
        const int j = k - i;
        if (j >= 0 && j < NB) s[k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[i], b.p[j], s[k], 0, 0, 0);
      }
  }
  __device__ __forceinline__ f32x4 sum() const {
    f32x4 x = s[L - 1];
#pragma unroll
    for (int k = L - 2; k >= 0; k--) x += s[k];
    return x;
  }
};

template <int N>
__device__ __forceinline__ void put_frag(bf16 *at, int plane, const Frag<N> &f) {
#pragma unroll
  for (int n = 0; n < N; n++) *reinterpret_cast<bf16x8 *>(at + n * plane) = f.p[n];
}

// Sum over the 16 lanes of a row of lanes by rotations within it, and over
// the wave by swapping its rows and then its halves: every lane gets it, and
// nothing goes through LDS.
#define CCHIP_ROTATED(x, n) __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x120 + n, 0xf, 0xf, true))
__device__ __forceinline__ float sum16(float x) {
  x += CCHIP_ROTATED(x, 8);
  x += CCHIP_ROTATED(x, 4);
  x += CCHIP_ROTATED(x, 2);
  x += CCHIP_ROTATED(x, 1);
  return x;
}

// The largest of the 16 lanes of a row.
__device__ __forceinline__ float max16(float x) {
  x = fmaxf(x, CCHIP_ROTATED(x, 8));
  x = fmaxf(x, CCHIP_ROTATED(x, 4));
  x = fmaxf(x, CCHIP_ROTATED(x, 2));
  return fmaxf(x, CCHIP_ROTATED(x, 1));
}
#undef CCHIP_ROTATED

// x of another lane of the same four: 0xB1 the neighbour's, 0x4E that two on.
#define CCHIP_QUAD(x, order) __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), order, 0xf, 0xf, true))

// x of the same column summed over the four rows of 16 lanes.
__device__ __forceinline__ float sum_rows(float x) {
  uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t a0 = a[0], a1 = a[1];
  x = __builtin_bit_cast(float, a0) + __builtin_bit_cast(float, a1);
  u = __builtin_bit_cast(uint32_t, x);
  const auto b = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t b0 = b[0], b1 = b[1];
  return __builtin_bit_cast(float, b0) + __builtin_bit_cast(float, b1);
}

// The largest of the four rows' x of a column.
__device__ __forceinline__ float max_rows(float x) {
  uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t a0 = a[0], a1 = a[1];
  x = fmaxf(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1));
  u = __builtin_bit_cast(uint32_t, x);
  const auto b = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t b0 = b[0], b1 = b[1];
  return fmaxf(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
}

__device__ __forceinline__ float sum64(float x) { return sum_rows(sum16(x)); }

// Philox-4x32-10 (Salmon, Moraes, Dror and Shaw, SC'11), the generator of
// cudacaml_amd/rng.py: ten rounds, the key bumped after the first nine.
__device__ __forceinline__ uint4 philox(uint4 c, uint2 k) {
#pragma unroll
  for (int r = 0; r < 10; r++) {
    const uint64_t a = uint64_t(0xD2511F53u) * c.x, b = uint64_t(0xCD9E8D57u) * c.z;
    c = make_uint4(uint32_t(b >> 32) ^ c.y ^ k.x, uint32_t(b), uint32_t(a >> 32) ^ c.w ^ k.y, uint32_t(a));
    k.x += 0x9E3779B9u;
    k.y += 0xBB67AE85u;
  }
  return c;
}

// Which of columns 8 group .. + 7 of a row dropout keeps, as bits: the
// 16-bit halves of philox((group, row, offset), seed), low half first,
// against `bar` = round(65536 p).
struct Drop {
  uint64_t seed, offset;
  const uint64_t *step;  // device counter added to offset, or null
  uint32_t bar;          // 0: everything is kept and nothing is drawn
  float up;              // 65536 / (65536 - bar), 0 if nothing is kept
};

__device__ __forceinline__ uint32_t keep_bits(const Drop &d, uint64_t offset, uint32_t row, uint32_t group) {
  const uint4 w = philox(make_uint4(group, row, uint32_t(offset), uint32_t(offset >> 32)),
                         make_uint2(uint32_t(d.seed), uint32_t(d.seed >> 32)));
  const uint32_t x[4] = {w.x, w.y, w.z, w.w};
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    bits |= uint32_t((x[i] & 0xFFFFu) >= d.bar) << (2 * i);
    bits |= uint32_t((x[i] >> 16) >= d.bar) << (2 * i + 1);
  }
  return bits;
}

// A launch has fewer than 2^32 work items along an axis: workgroups (of at
// most 512 here) past the first 2^22 go on along y. The last row of y may have
// some over.
constexpr uint32_t kGridRow = 1u << 22;

__device__ __forceinline__ uint32_t block_index() { return blockIdx.y * kGridRow + blockIdx.x; }

// ---- host side --------------------------------------------------------------

// Whether two stretches of memory share a byte.
inline bool meet(const void *a, size_t a_bytes, const void *b, size_t b_bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + b_bytes && y < x + a_bytes;
}

inline dim3 grid_of(int64_t workgroups) {
  const int64_t rows = (workgroups + kGridRow - 1) / kGridRow;
  return dim3(unsigned(rows > 1 ? kGridRow : workgroups), unsigned(rows));
}

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// More than 64 KB of LDS have to be allowed, once for a kernel and device.
template <auto Kernel>
void allow_lds(int bytes, const char *what) {
  static std::atomic<uint64_t> allowed{0};
  int device = 0;
  check_hip(hipGetDevice(&device), what);
  const uint64_t bit = uint64_t(1) << (device & 63);
  if (device < 64 && (allowed.load(std::memory_order_relaxed) & bit)) return;
  check_hip(hipFuncSetAttribute(reinterpret_cast<const void *>(Kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes), what);
  allowed.fetch_or(bit, std::memory_order_relaxed);
}

inline void check_launch(const char *what) { check_hip(hipGetLastError(), what); }

}  // namespace op
}  // namespace cchip
