// Gated delta rule, the part of a chunk that depends on no state: T, P and
// the decays of every chunk and value head (the formulas stand in delta.hpp).

#include "delta.hpp"

namespace cchip {
namespace op {
namespace {

constexpr int kPad = 68;  // f32 rows of 64 in LDS: 4 banks on from row to row

// One 16-byte piece a plane of a fragment of rows row0.., terms term0.. of
// an f32 matrix in LDS, stored [row][term] or, transposed, [term][row].
template <int N, bool Transposed>
__device__ __forceinline__ void write_fragment(char *to, const float *m, int row0, int term0) {
  const int l = threadIdx.x & 63;
  const int row = row0 + (l & 15), term = term0 + (l >> 4) * 8;
  bf16x8 v[N];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    bf16 s[N];
    split<N>(Transposed ? m[(term + i) * kPad + row] : m[row * kPad + term + i], s);
#pragma unroll
    for (int n = 0; n < N; n++) v[n][i] = s[n];
  }
#pragma unroll
  for (int n = 0; n < N; n++) reinterpret_cast<bf16x8 *>(to + n * 8192)[((row0 / 16) * 2 + term0 / 32) * 64 + l] = v[n];
}

// c -= x y for 16 x 16 blocks in LDS on the f32 matrix instruction (4 terms
// a step): lane l holds row l % 16 of x, column l % 16 of y, term l / 16.
__device__ __forceinline__ f32x4 block_product(f32x4 c, const float *x, const float *y) {
  const int l = threadIdx.x & 63, i = l & 15, k = l >> 4;
#pragma unroll
  for (int s = 0; s < 16; s += 4)
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i * kPad + s + k], y[(s + k) * kPad + i], c, 0, 0, 0);
  return c;
}

// What a wave's lanes have written to LDS is there for its other lanes.
__device__ __forceinline__ void wave_settles() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ void put_block(float *to, const f32x4 &c, float sign) {
  const int l = threadIdx.x & 63;
#pragma unroll
  for (int r = 0; r < 4; r++) to[((l >> 4) * 4 + r) * kPad + (l & 15)] = sign * c[r];
}

// A workgroup of four waves a chunk and value head; wave w makes rows 16 w
// to 16 w + 15 of KK^T and QK^T. The inverse goes by blocks of 16: the four
// on the diagonal by substitution, a column a lane, then with L the strict
// lower triangle T_ij = -T_ii sum_m A_im T_mj, a diagonal of blocks at a
// time. All of it is f32: entries of T add up 64 products deep, and every
// state after the chunk carries what they lose. The substitution's 15 steps,
// each on the last, bound it, and three workgroups a unit cover each other's:
// 163 us for 256 chunks of 32 bf16 heads of 128 with what the backward pass
// reads (0.67 GB, 4.1 TB/s), 142 us with f32 states and no backward pass.
template <typename M, int DK, bool Back, int A>
__global__ __launch_bounds__(256) void delta_chunk(const DeltaArgs a) {
  typedef typename M::T T;
  constexpr int NI = M::NI, LD = DK + 8, KPlane = 64 * LD;
  typedef Record<M> R;
  __shared__ __align__(16) bf16 ks[NI * KPlane];
  __shared__ __align__(16) float am[64 * kPad], tm[64 * kPad];
  __shared__ double cs[64];
  __shared__ float bs[64];

  const int64_t slot = block_index() / a.hv;
  if (slot >= a.slots) return;
  const int h = int(block_index() - slot * a.hv), hk = h / (a.hv / a.hk);
  const Chunk c = chunk_of(a, slot);
  if (c.len == 0) return;
  char *rec = a.records + (slot * a.hv + h) * R::bytes(Back);
  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, quad = l >> 4, col = l & 15;

  if (w == 0) {
    // The running sum in f64: differences of it are exponents, and an f32
    // sum of 64 would lose up to 6 bits of them. exp(-1000) is 0 in f32, so
    // a decay to nothing (g = -inf) loses nothing by the bound, and its
    // differences stay numbers.
    const float g = l < c.len ? float(*at<T>(a.g, c.row, c.first + l, h)) : 0.0f;
    const float beta = l < c.len ? float(*at<T>(a.beta, c.row, c.first + l, h)) : 0.0f;
    double s = g < -1000.0f ? -1000.0 : double(g);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const double up = __shfl_up(s, d, 64);
      if (l >= d) s += up;
    }
    cs[l] = s;
    bs[l] = beta;
    const double last = __shfl(s, 63, 64);
    float *dec = reinterpret_cast<float *>(rec + R::Decay);
    dec[l] = expf(float(s));
    dec[64 + l] = expf(float(last - s));
    dec[128 + l] = beta;
  }
  Raw8<T> rk[DK / 32], rq[DK / 32];
#pragma unroll
  for (int j = 0; j < DK / 32; j++) {
    const int i = tid + 256 * j;
    rk[j] = load_head8<A, T>(a.k, c, hk, i / (DK / 8), i % (DK / 8) * 8, a.dk);
    rq[j] = load_head8<A, T>(a.q, c, hk, 16 * w + col, 32 * j + quad * 8, a.dk);
  }
#pragma unroll
  for (int j = 0; j < DK / 32; j++) {
    const int i = tid + 256 * j, t = i / (DK / 8), d = i % (DK / 8) * 8;
    put_frag<NI>(ks + t * LD + d, KPlane, frag_of<NI>(keep_head8<A>(rk[j], c, t, d, a.dk)));
  }
  for (int i = tid; i < 64 * kPad; i += 256) tm[i] = 0.0f;
  __syncthreads();

  f32x4 kk[4] = {}, qk[4] = {};
#pragma unroll
  for (int d = 0; d < DK; d += 32) {
    const Frag<NI> fk = frag_row<NI>(ks, KPlane, LD, 16 * w, d);
    const Frag<NI> fq = frag_of<NI>(keep_head8<A>(rq[d / 32], c, 16 * w + col, d + quad * 8, a.dk));
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (j <= w) {
        const Frag<NI> fs = frag_row<NI>(ks, KPlane, LD, 16 * j, d);
        // T and P^T go into f32 states: products of f16 inputs are whole
        constexpr int kLevels = NI == 2 ? 3 : 0;
        kk[j] = mma<kLevels>(kk[j], fk, fs);
        qk[j] = mma<kLevels>(qk[j], fq, fs);
      }
  }
  float *pm = reinterpret_cast<float *>(ks);  // the keys are done with
  static_assert(sizeof(ks) >= sizeof(float) * 64 * kPad || DK < 128, "P does not fit where the keys were");
  __shared__ __align__(16) float own[DK < 128 ? 64 * kPad : 1];
  if (DK < 128) pm = own;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 4; j++)
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int t = 16 * w + 4 * quad + r, s = 16 * j + col;
      const float d = s <= t ? expf(float(cs[t] - cs[s])) : 0.0f;
      am[t * kPad + s] = s < t ? bs[t] * d * kk[j][r] : 0.0f;
      pm[t * kPad + s] = s <= t ? d * qk[j][r] : 0.0f;
    }
  __syncthreads();

  if (w == 0) {
    const float *blk = am + 16 * quad * (kPad + 1);
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; i++) {
      float v = i == col ? 1.0f : 0.0f;
#pragma unroll
      for (int m = 0; m < i; m++) v -= blk[i * kPad + m] * x[m];
      x[i] = v;
    }
#pragma unroll
    for (int i = 0; i < 16; i++) tm[(16 * quad + i) * kPad + 16 * quad + col] = x[i];
  } else {
    for (int f = w - 1; f < 8; f += 3) {
      write_fragment<M::NO, false>(rec + R::P, pm, f / 2 * 16, f % 2 * 32);
      if (Back) write_fragment<M::NS, true>(rec + R::Pt, pm, f / 2 * 16, f % 2 * 32);
    }
  }
  __syncthreads();
  // wave w goes down block row w; am's blocks above the diagonal are free
  // and hold the sums between the two products
#pragma unroll
  for (int d = 1; d < 4; d++) {
    if (w >= d) {
      f32x4 sum = {};
      for (int m = w - d; m < w; m++)
        sum = block_product(sum, am + 16 * w * kPad + 16 * m, tm + 16 * m * kPad + 16 * (w - d));
      float *tmp = am + 16 * (w - d) * kPad + 16 * w;
      put_block(tmp, sum, 1.0f);
      wave_settles();
      f32x4 t = {};
      t = block_product(t, tm + 16 * w * kPad + 16 * w, tmp);
      put_block(tm + 16 * w * kPad + 16 * (w - d), t, -1.0f);
    }
    __syncthreads();
  }
  for (int f = w; f < 8; f += 4) {
    write_fragment<M::NS, false>(rec + R::T, tm, f / 2 * 16, f % 2 * 32);
    if (Back) write_fragment<M::NS, true>(rec + R::Tt, tm, f / 2 * 16, f % 2 * 32);
  }
}

}  // namespace

void delta_chunk_launch(const cchip_gated_delta &op, const DeltaArgs &a, bool back, hipStream_t stream) {
  const int64_t grid = a.slots * a.hv;
  with_mode(op, [&](auto m) {
    typedef decltype(m) M;
    with_bool(back, [&](auto b) {
      with_access<typename M::T>(a, [&](auto f) {
        constexpr bool B = decltype(b)::value;
        constexpr int F = decltype(f)::value;
        auto *k = a.dk <= 64 ? delta_chunk<M, 64, B, F> : delta_chunk<M, 128, B, F>;
        hipLaunchKernelGGL(k, grid_of(grid), dim3(256), 0, stream, a);
      });
    });
  });
  check_launch("gated delta: chunks");
}

}  // namespace op
}  // namespace cchip
