// The norm block's kernels (cchip_operators.h states what they compute). One
// element type is instantiated a file: norm_block_bf16.hip and the like.
#pragma once

#include "rows.hpp"

namespace cchip {
namespace op {

// What a row's norms leave for norm_sums: xhat is (x - mean) inv, and the
// gradient through the pre norm (d - xhat along - share) inv.
struct RowStat {
  float pre_mean, pre_inv, along, share, post_mean, post_inv;
};

struct NormArgs {
  Rows y, gate, residual, h, n;                 // forward
  Rows dh, dn, dy, dgate, dresidual;            // backward (reads y, gate, h)
  const void *post_weight, *post_bias, *channel_scale, *pre_weight, *pre_bias;
  float *partial;  // backward: [workgroup][parameter][width]
  RowStat *stats;  // backward of wide rows: [row]
  uint32_t rows;
  int width, post, pre, act;
  bool weights_f32;
  float scale, eps;
  Drop drop;
};

// Row sums over LANES threads, or a workgroup of at most LANES: every one
// gets the sum. `at` is a scratch of a float a wave and set, two sets, used
// in turn, zero where there is no such wave.
template <int LANES>
struct RowSum {
  f32x2 (*at)[LANES > 64 ? LANES / 64 : 1];
  int set;
  __device__ __forceinline__ void begin() {
    if (LANES <= 64) return;
    set = 0;
    if (threadIdx.x < 2 * LANES / 64) at[0][threadIdx.x] = f32x2{};
    __syncthreads();
  }
  __device__ __forceinline__ float operator()(float x) {
    if (LANES == 16) return sum16(x);
    x = sum64(x);
    if (LANES == 64) return x;
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) at[set][w].x = x;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < (LANES > 64 ? LANES / 64 : 1); i++) s += at[set][i].x;
    set ^= 1;
    return s;
  }
  // Two at once.
  __device__ __forceinline__ void operator()(float &x, float &y) {
    if (LANES <= 64) {
      x = (*this)(x);
      y = (*this)(y);
      return;
    }
    x = sum64(x);
    y = sum64(y);
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) at[set][w] = f32x2{x, y};
    __syncthreads();
    f32x2 s = {};
#pragma unroll
    for (int i = 0; i < (LANES > 64 ? LANES / 64 : 1); i++) {
      s.x += at[set][i].x;
      s.y += at[set][i].y;
    }
    set ^= 1;
    x = s.x;
    y = s.y;
  }
};

// 1 / sqrt(x) by the instruction, which knows no subnormal x.
__device__ __forceinline__ float inverse_root(float x) {
  const bool small = x < 0x1p-100f;
  const float r = __builtin_amdgcn_rsqf(small ? x * 0x1p100f : x);
  return small ? r * 0x1p50f : r;
}

// Eight of a parameter vector; `none` where there is none.
template <typename T>
__device__ __forceinline__ void load_params(float (&w)[8], const void *p, bool f32, int at, int n, float none) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < 8; i++) w[i] = none;
  } else if (f32) {
    const Raw8<float> r = load8<float>(static_cast<const float *>(p) + at, n);
#pragma unroll
    for (int i = 0; i < 8; i++) w[i] = r.x[i];
  } else {
    const Raw8<T> r = load8<T>(static_cast<const T *>(p) + at, n);
#pragma unroll
    for (int i = 0; i < 8; i++) w[i] = float(r.x[i]);
  }
}

// x becomes (x - mean) / sqrt(mean of squares + eps); returns what it was
// multiplied by. Sums of squares are of centred values: nothing cancels.
template <int LANES, int V>
__device__ __forceinline__ float normalise(float (&x)[V][8], int kind, float inv_width, float eps, RowSum<LANES> &sum,
                                           int lane, int width, float *of = nullptr) {
  if (kind == CCHIP_NORM_LAYER) {
    float s = 0.0f;
#pragma unroll
    for (int v = 0; v < V; v++)
#pragma unroll
      for (int i = 0; i < 8; i++) s += x[v][i];
    const float mean = sum(s) * inv_width;
    if (of) *of = mean;
#pragma unroll
    for (int v = 0; v < V; v++)
#pragma unroll
      for (int i = 0; i < 8; i++) x[v][i] = (v * LANES + lane) * 8 + i < width ? x[v][i] - mean : 0.0f;
  }
  float q = 0.0f;
#pragma unroll
  for (int v = 0; v < V; v++)
#pragma unroll
    for (int i = 0; i < 8; i++) q += x[v][i] * x[v][i];
  const float inv = inverse_root(sum(q) * inv_width + eps);
#pragma unroll
  for (int v = 0; v < V; v++)
#pragma unroll
    for (int i = 0; i < 8; i++) x[v][i] *= inv;
  return inv;
}

// For 16-bit elements by the exponential and reciprocal instructions, 1e-7
// off for each unit of z where the element's rounding is 2e-4 or more.
template <typename T>
__device__ __forceinline__ float sigmoid(float z) {
  if (sizeof(T) == 4) return 1.0f / (1.0f + expf(-z));
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504f));
}

// A gate's value for z and its slope.
template <typename T>
__device__ __forceinline__ void gate_of(int kind, float z, float &act, float &slope) {
  const float s = sigmoid<T>(z);
  act = kind == CCHIP_GATE_SILU ? z * s : s;
  slope = kind == CCHIP_GATE_SILU ? s * (1.0f + z * (1.0f - s)) : s * (1.0f - s);
}

// A row to LANES threads, 8 neighbouring columns a thread and step, held in
// registers from the one read of it to the writes. A workgroup takes every
// gridDim-th set of rows and keeps the parameters of its columns.
template <typename T, int LANES, int V>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void norm_forward(const NormArgs a) {
  constexpr int kRows = LANES < 256 ? 256 / LANES : 1;
  __shared__ f32x2 scratch[2][LANES > 64 ? LANES / 64 : 1];
  RowSum<LANES> sum = {scratch, 0};
  sum.begin();
  const int lane = threadIdx.x % LANES;
  const float inv_width = 1.0f / float(a.width);
  const float up = a.scale * a.drop.up;
  const uint64_t offset = a.drop.bar ? offset_of(a.drop) : 0;

  // (yhat w + b) up t, as one product and sum. One row of parameters stays
  // in registers, more are read again for each row.
  float w[V][8], b[V][8], pw[V][8], pb[V][8];
  int n[V];
#pragma unroll
  for (int v = 0; v < V; v++) {
    const int c = (v * LANES + lane) * 8;
    n[v] = a.width - c < 0 ? 0 : a.width - c > 8 ? 8 : a.width - c;
  }
  auto post_params = [&](int v) {
    const int c = (v * LANES + lane) * 8;
    float t[8];
    load_params<T>(t, a.channel_scale, a.weights_f32, c, n[v], 1.0f);
    load_params<T>(w[v], a.post_weight, a.weights_f32, c, n[v], 1.0f);
    load_params<T>(b[v], a.post_bias, a.weights_f32, c, n[v], 0.0f);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      w[v][i] *= up * t[i];
      b[v][i] *= up * t[i];
    }
  };
  auto pre_params = [&](int v) {
    const int c = (v * LANES + lane) * 8;
    load_params<T>(pw[v], a.pre_weight, a.weights_f32, c, n[v], 1.0f);
    load_params<T>(pb[v], a.pre_bias, a.weights_f32, c, n[v], 0.0f);
  };
  if (V == 1) {
    post_params(0);
    pre_params(0);
  }
  for (int64_t row = int64_t(blockIdx.x) * kRows + threadIdx.x / LANES; row < a.rows; row += int64_t(gridDim.x) * kRows) {
    Raw8<T> y[V], z[V], x[V];
#pragma unroll
    for (int v = 0; v < V; v++) y[v] = load8<T>(row_at<T>(a.y, row) + (v * LANES + lane) * 8, n[v]);
    if (a.act != CCHIP_GATE_NONE)
#pragma unroll
      for (int v = 0; v < V; v++) z[v] = load8<T>(row_at<T>(a.gate, row) + (v * LANES + lane) * 8, n[v]);
    if (a.residual.p)
#pragma unroll
      for (int v = 0; v < V; v++) x[v] = load8<T>(row_at<T>(a.residual, row) + (v * LANES + lane) * 8, n[v]);
    uint32_t bits[V];  // drawn while the row is on its way
#pragma unroll
    for (int v = 0; v < V; v++)
      bits[v] = a.drop.bar ? keep_bits(a.drop, offset, uint32_t(row), v * LANES + lane) : 0xFFu;

    float h[V][8];
#pragma unroll
    for (int v = 0; v < V; v++)
#pragma unroll
      for (int i = 0; i < 8; i++) h[v][i] = float(y[v].x[i]);
    if (a.post != CCHIP_NORM_NONE) normalise<LANES, V>(h, a.post, inv_width, a.eps, sum, lane, a.width);
#pragma unroll
    for (int v = 0; v < V; v++) {
      if (V > 1) post_params(v);
#pragma unroll
      for (int i = 0; i < 8; i++) {
        float e = h[v][i] * w[v][i] + b[v][i];
        if (a.act != CCHIP_GATE_NONE) {
          const float zi = float(z[v].x[i]), s = sigmoid<T>(zi);
          e *= a.act == CCHIP_GATE_SILU ? zi * s : s;
        }
        e = bits[v] >> i & 1 ? e : 0.0f;
        if (a.residual.p) e += float(x[v].x[i]);
        h[v][i] = i < n[v] ? e : 0.0f;
      }
      store8<T>(row_at<T>(a.h, row) + (v * LANES + lane) * 8, h[v], n[v]);
    }
    if (a.pre == CCHIP_NORM_NONE) continue;
    normalise<LANES, V>(h, a.pre, inv_width, a.eps, sum, lane, a.width);
#pragma unroll
    for (int v = 0; v < V; v++) {
      if (V > 1) pre_params(v);
#pragma unroll
      for (int i = 0; i < 8; i++) h[v][i] = h[v][i] * pw[v][i] + pb[v][i];
      store8<T>(row_at<T>(a.n, row) + (v * LANES + lane) * 8, h[v], n[v]);
    }
  }
}

// d becomes the gradient of what `normalise` read, from that of what it
// gave: (d - mean(d) - xhat mean(d xhat)) inv, the first mean of a layer norm.
// Of a row of one value, or two centred ones, all of d lies along xhat and
// what is left is eps inv^2 of it: there the projection is taken off twice
// and that share put back, as the difference itself would be rounding.
template <int LANES, int V>
__device__ __forceinline__ void normalise_back(float (&d)[V][8], const float (&xhat)[V][8], int kind, float inv,
                                               float inv_width, float eps, int width, RowSum<LANES> &sum,
                                               RowStat *of = nullptr) {
  float p = 0.0f, q = 0.0f;
#pragma unroll
  for (int v = 0; v < V; v++)
#pragma unroll
    for (int i = 0; i < 8; i++) {
      p += d[v][i] * xhat[v][i];
      q += d[v][i];
    }
  if (kind == CCHIP_NORM_LAYER) sum(p, q);
  else p = sum(p);
  p *= inv_width;
  q = kind == CCHIP_NORM_LAYER ? q * inv_width : 0.0f;
  float back = 0.0f;
  if (width <= 2) {
    float s = 0.0f;
    for (int i = 0; i < 8; i++) s += xhat[0][i] * xhat[0][i];
    s = sum(s) * inv_width;  // mean of xhat^2, 1 - eps inv^2
    const float once = s > 0.0f ? p / s : 0.0f;
    float r = 0.0f;
    for (int i = 0; i < 8; i++) r += (d[0][i] - q - xhat[0][i] * once) * xhat[0][i];
    r = sum(r) * inv_width;
    const float twice = s > 0.0f ? r / s : 0.0f;
    for (int i = 0; i < 8; i++) d[0][i] = (d[0][i] - q - xhat[0][i] * once) - xhat[0][i] * twice;
    back = once * eps * inv * inv;
    p = q = 0.0f;
  }
  if (of) {
    of->along = p;
    of->share = q;
  }
#pragma unroll
  for (int v = 0; v < V; v++)
#pragma unroll
    for (int i = 0; i < 8; i++) d[v][i] = (d[v][i] - xhat[v][i] * (p - back) - q) * inv;
}

// The parameters' gradients in the order of their sums; without Bias there
// are no biases and the last two are not made.
enum Param { kPostWeight, kChannelScale, kPreWeight, kPostBias, kPreBias, kParams };

// Waves a SIMD holds of a backward pass: 4 of at most 128 registers; with two
// norms and a gate or biases, what a thread holds does not fit in those and
// is not spilled for a fourth wave: 16384 rows of 4096 with all of it take
// 347 us so and 593 spilled, without gate and biases 174 us of four waves and
// 228 of three. (bf16; floors of 220 and 165 us by the bytes.)
constexpr int waves_of(int lanes, bool gate, bool pre, bool bias) {
  return lanes > 512 || !(pre && (gate || bias)) ? 4 : lanes > 256 ? 2 : 3;
}

// As norm_forward, a workgroup taking every gridDim-th set of rows so that it
// can sum the parameters' gradients of its columns in registers; they are
// left in `partial` and added up by norm_columns. Rows of over 8192 columns
// (V > 1) leave no registers for that: each leaves its statistics, and
// norm_sums reads it again, 4096 rows of 16384 taking 357 us in both kernels
// where one that spilled its sums took 678. Up to 8192 columns one kernel is
// the faster: 16384 rows of 5000 with two norms and a gate take 567 us, and
// 715 in two.
template <typename T, int LANES, int V, bool Gate, bool Pre, bool Bias>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES, waves_of(LANES, Gate, Pre, Bias)) void norm_backward(const NormArgs a) {
  constexpr int kRows = LANES < 256 ? 256 / LANES : 1, kThreads = LANES < 256 ? 256 : LANES;
  constexpr int kSums = Bias ? 5 : 3;
  __shared__ f32x2 scratch[2][LANES > 64 ? LANES / 64 : 1];
  RowSum<LANES> sum = {scratch, 0};
  sum.begin();
  const int lane = threadIdx.x % LANES;
  const float inv_width = 1.0f / float(a.width);
  const float up = a.scale * a.drop.up;
  const uint64_t offset = a.drop.bar ? offset_of(a.drop) : 0;
  float acc[kSums][V][8] = {};  // of one step
  int n[V];
#pragma unroll
  for (int v = 0; v < V; v++) {
    const int c = (v * LANES + lane) * 8;
    n[v] = a.width - c < 0 ? 0 : a.width - c > 8 ? 8 : a.width - c;
  }
  // Parameters of this thread's columns: in LDS where a workgroup's fit.
  extern __shared__ f32x4 held[];
  const int lanes = LANES < 256 ? LANES : int(blockDim.x);
  auto from_memory = [&](int k, int v, float(&x)[8]) {
    const void *p = k == kPostWeight ? a.post_weight : k == kChannelScale ? a.channel_scale : k == kPreWeight ? a.pre_weight : a.post_bias;
    load_params<T>(x, p, a.weights_f32, (v * LANES + lane) * 8, n[v], k == kPostBias ? 0.0f : 1.0f);
  };
  auto param = [&](int k, int v, int half) {
    if (V == 1) return held[(k * 2 + half) * lanes + lane];
    float x[8];
    from_memory(k, v, x);
    return f32x4{x[4 * half], x[4 * half + 1], x[4 * half + 2], x[4 * half + 3]};
  };
  if (V == 1) {
#pragma unroll
    for (int k = 0; k < (Bias ? 4 : 3); k++) {
      float x[8];
      from_memory(k, 0, x);
      if (threadIdx.x < lanes)
#pragma unroll
        for (int i = 0; i < 2; i++) held[(k * 2 + i) * lanes + lane] = f32x4{x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]};
    }
    __syncthreads();
  }
  for (int64_t row = int64_t(blockIdx.x) * kRows + threadIdx.x / LANES; row < a.rows; row += int64_t(gridDim.x) * kRows) {
    Raw8<T> ry[V], rz[V], rh[V], rdh[V], rdn[V];
#pragma unroll
    for (int v = 0; v < V; v++) {
      const int c = (v * LANES + lane) * 8;
      if (Pre) rh[v] = load8<T>(row_at<T>(a.h, row) + c, n[v]);
      if (Pre) rdn[v] = load8<T>(row_at<T>(a.dn, row) + c, n[v]);
      rdh[v] = load8<T>(row_at<T>(a.dh, row) + c, n[v]);
      if (V < 4) ry[v] = load8<T>(row_at<T>(a.y, row) + c, n[v]);
      if (V < 4 && Gate) rz[v] = load8<T>(row_at<T>(a.gate, row) + c, n[v]);
    }
    RowStat stat = {0.0f, 1.0f, 0.0f, 0.0f, 0.0f, 1.0f};
    float d[V][8], x[V][8];
    if (Pre) {
#pragma unroll
      for (int v = 0; v < V; v++)
#pragma unroll
        for (int i = 0; i < 8; i++) x[v][i] = float(rh[v].x[i]);
      const float inv = normalise<LANES, V>(x, a.pre, inv_width, a.eps, sum, lane, a.width, &stat.pre_mean);
      stat.pre_inv = inv;
#pragma unroll
      for (int v = 0; v < V; v++) {
#pragma unroll
        for (int half = 0; half < 2; half++) {
          const f32x4 pw = param(kPreWeight, v, half);
#pragma unroll
          for (int i = 4 * half; i < 4 * half + 4; i++) {
            const float dn = float(rdn[v].x[i]);
            if (V == 1) acc[kPreWeight][v][i] += dn * x[v][i];
            if (V == 1 && Bias) acc[kPreBias][v][i] += dn;
            d[v][i] = i < n[v] ? dn * pw[i % 4] : 0.0f;
          }
        }
      }
      normalise_back<LANES, V>(d, x, a.pre, inv, inv_width, a.eps, a.width, sum, &stat);
#pragma unroll
      for (int v = 0; v < V; v++)
#pragma unroll
        for (int i = 0; i < 8; i++) d[v][i] += float(rdh[v].x[i]);
    } else {
#pragma unroll
      for (int v = 0; v < V; v++)
#pragma unroll
        for (int i = 0; i < 8; i++) d[v][i] = float(rdh[v].x[i]);
    }
    if (a.dresidual.p)
#pragma unroll
      for (int v = 0; v < V; v++) store8<T>(row_at<T>(a.dresidual, row) + (v * LANES + lane) * 8, d[v], n[v]);

    if (V == 4)
#pragma unroll
      for (int v = 0; v < V; v++) {
        ry[v] = load8<T>(row_at<T>(a.y, row) + (v * LANES + lane) * 8, n[v]);
        if (Gate) rz[v] = load8<T>(row_at<T>(a.gate, row) + (v * LANES + lane) * 8, n[v]);
      }
#pragma unroll
    for (int v = 0; v < V; v++)
#pragma unroll
      for (int i = 0; i < 8; i++) x[v][i] = float(ry[v].x[i]);
    float inv = 1.0f;
    if (a.post != CCHIP_NORM_NONE) inv = normalise<LANES, V>(x, a.post, inv_width, a.eps, sum, lane, a.width, &stat.post_mean);
    stat.post_inv = inv;
    if (V > 1 && a.partial && threadIdx.x == 0) a.stats[row] = stat;
#pragma unroll
    for (int v = 0; v < V; v++) {
      const int g = v * LANES + lane, c = g * 8;
      float dz[8];
      const uint32_t bits = a.drop.bar ? keep_bits(a.drop, offset, uint32_t(row), g) : 0xFFu;
#pragma unroll
      for (int half = 0; half < 2; half++) {
        __builtin_amdgcn_sched_barrier(0);  // four at a time: all eight hold more registers than there are
        const f32x4 w = param(kPostWeight, v, half), t = param(kChannelScale, v, half);
        const f32x4 b = Bias ? param(kPostBias, v, half) : f32x4{};
#pragma unroll
        for (int i = 4 * half; i < 4 * half + 4; i++) {
          const bool keep = bits >> i & 1 && i < n[v];
          const float e = Bias ? x[v][i] * w[i % 4] + b[i % 4] : x[v][i] * w[i % 4];
          float act = 1.0f, slope = 0.0f;
          if (Gate) gate_of<T>(a.act, float(rz[v].x[i]), act, slope);
          // selected last: what was dropped may be no number
          const float du = d[v][i] * up, db = du * t[i % 4], da = keep ? db * act : 0.0f;
          if (V == 1) acc[kChannelScale][v][i] += keep ? du * e * act : 0.0f;
          if (Gate) dz[i] = keep ? db * e * slope : 0.0f;
          if (V == 1) acc[kPostWeight][v][i] += da * x[v][i];
          if (V == 1 && Bias) acc[kPostBias][v][i] += da;
          d[v][i] = da * w[i % 4];
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      if (Gate && a.dgate.p) store8<T>(row_at<T>(a.dgate, row) + c, dz, n[v]);
    }
    if (a.post != CCHIP_NORM_NONE) normalise_back<LANES, V>(d, x, a.post, inv, inv_width, a.eps, a.width, sum);
#pragma unroll
    for (int v = 0; v < V; v++) store8<T>(row_at<T>(a.dy, row) + (v * LANES + lane) * 8, d[v], n[v]);
  }
  if (V > 1 || !a.partial) return;
  if (kRows > 1) {
    // the workgroup's rows side by side: sum them in the order of the rows
    __shared__ float side[kThreads * 8];
#pragma unroll
    for (int s = 0; s < kSums; s++)
#pragma unroll
      for (int v = 0; v < V; v++) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; i++) side[threadIdx.x * 8 + i] = acc[s][v][i];
        __syncthreads();
        for (int i = threadIdx.x; i < LANES * 8; i += kThreads) {
          float q = 0.0f;
          for (int r = 0; r < kRows; r++) q += side[r * LANES * 8 + i];
          const int c = v * LANES * 8 + i;
          if (c < a.width) a.partial[(int64_t(blockIdx.x) * kSums + s) * a.width + c] = q;
        }
      }
  } else {
#pragma unroll
    for (int s = 0; s < kSums; s++)
#pragma unroll
      for (int v = 0; v < V; v++)
#pragma unroll
        for (int i = 0; i < 8; i++)
          if (i < n[v]) a.partial[(int64_t(blockIdx.x) * kSums + s) * a.width + (v * LANES + lane) * 8 + i] = acc[s][v][i];
  }
}

// The parameters' gradients of wide rows: a workgroup sums 2048 columns of
// every gridDim.y-th row from what the rows' statistics make of them.
template <typename T, bool Gate, bool Pre, bool Bias>
__global__ __launch_bounds__(256, 4) void norm_sums(const NormArgs a) {
  constexpr int kSums = Bias ? 5 : 3;
  const int group = int(blockIdx.x) * 256 + int(threadIdx.x), c = group * 8;
  const int n = a.width - c < 0 ? 0 : a.width - c > 8 ? 8 : a.width - c;
  if (!n) return;
  const float up = a.scale * a.drop.up;
  const uint64_t offset = a.drop.bar ? offset_of(a.drop) : 0;
  float acc[kSums][8] = {};
  float w[8], t[8], b[8], pw[8];
  load_params<T>(w, a.post_weight, a.weights_f32, c, n, 1.0f);
  load_params<T>(t, a.channel_scale, a.weights_f32, c, n, 1.0f);
  if (Bias) load_params<T>(b, a.post_bias, a.weights_f32, c, n, 0.0f);
  if (Pre) load_params<T>(pw, a.pre_weight, a.weights_f32, c, n, 1.0f);
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    Raw8<T> ry, rz, rh, rdh, rdn;
    if (Pre) rh = load8<T>(row_at<T>(a.h, row) + c, n);
    if (Pre) rdn = load8<T>(row_at<T>(a.dn, row) + c, n);
    rdh = load8<T>(row_at<T>(a.dh, row) + c, n);
    ry = load8<T>(row_at<T>(a.y, row) + c, n);
    if (Gate) rz = load8<T>(row_at<T>(a.gate, row) + c, n);
    const RowStat s = a.stats[row];
    const uint32_t bits = a.drop.bar ? keep_bits(a.drop, offset, uint32_t(row), group) : 0xFFu;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      float d = float(rdh.x[i]);
      if (Pre) {
        const float dn = float(rdn.x[i]), xhat = (float(rh.x[i]) - s.pre_mean) * s.pre_inv;
        acc[kPreWeight][i] += dn * xhat;
        if (Bias) acc[kPreBias][i] += dn;
        d += (dn * pw[i] - xhat * s.along - s.share) * s.pre_inv;
      }
      const float x = (float(ry.x[i]) - s.post_mean) * s.post_inv, e = Bias ? x * w[i] + b[i] : x * w[i];
      float act = 1.0f, slope = 0.0f;
      if (Gate) gate_of<T>(a.act, float(rz.x[i]), act, slope);
      const float du = d * up, da = bits >> i & 1 ? du * t[i] * act : 0.0f;
      acc[kChannelScale][i] += bits >> i & 1 ? du * e * act : 0.0f;
      acc[kPostWeight][i] += da * x;
      if (Bias) acc[kPostBias][i] += da;
    }
  }
#pragma unroll
  for (int s = 0; s < kSums; s++)
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (i < n) a.partial[(int64_t(blockIdx.y) * kSums + s) * a.width + c + i] = acc[s][i];
}

template <typename T>
void norm_forward_launch(const NormArgs &a, hipStream_t stream);
template <typename T>
void norm_backward_launch(const NormArgs &a, bool bias, int groups, hipStream_t stream);

// Rows a workgroup takes at a time for a width.
inline int rows_at_a_time(int width) { return width <= 128 ? 16 : width <= 512 ? 4 : 1; }

// Threads of a workgroup: a wave for each 512 columns where a row is one's
// (the backward pass of 65536 rows of 1000 takes 404 us in two waves, 670 in
// four of which two have no columns).
inline int threads_of(int width) { return width <= 512 ? 256 : width <= 8192 ? (width + 511) / 512 * 64 : 1024; }

// Workgroups that take `rows` evenly, `least` at least each, as many as run
// at once with `waves` a SIMD.
int groups_of(int64_t rows, int width, int waves, int least);

// Calls f(lanes, steps) with the smallest shape that holds a row: few lanes
// for short rows, so that none idles, and 8 columns a thread up to 8192, so
// that a backward pass's sums stay in registers.
template <typename F>
void with_shape(int width, F &&f) {
  if (width <= 128) f(std::integral_constant<int, 16>(), std::integral_constant<int, 1>());
  else if (width <= 512) f(std::integral_constant<int, 64>(), std::integral_constant<int, 1>());
  else if (width <= 2048) f(std::integral_constant<int, 256>(), std::integral_constant<int, 1>());
  else if (width <= 4096) f(std::integral_constant<int, 512>(), std::integral_constant<int, 1>());
  else if (width <= 8192) f(std::integral_constant<int, 1024>(), std::integral_constant<int, 1>());
  else if (width <= 16384) f(std::integral_constant<int, 1024>(), std::integral_constant<int, 2>());
  else f(std::integral_constant<int, 1024>(), std::integral_constant<int, 4>());
}

// Calls f with whether there are a gate, a pre norm and biases.
template <typename F>
void with_parts(const NormArgs &a, bool bias, F &&f) {
  auto third = [&](auto gate, auto pre) {
    if (bias) f(gate, pre, std::true_type());
    else f(gate, pre, std::false_type());
  };
  auto second = [&](auto gate) {
    if (a.pre != CCHIP_NORM_NONE) third(gate, std::true_type());
    else third(gate, std::false_type());
  };
  if (a.act != CCHIP_GATE_NONE) second(std::true_type());
  else second(std::false_type());
}

#define CCHIP_NORM_BLOCK_LAUNCHERS(T)                                                                              \
  template <>                                                                                                      \
  void norm_forward_launch<T>(const NormArgs &a, hipStream_t stream) {                                             \
    with_shape(a.width, [&](auto lanes, auto steps) {                                                              \
      constexpr int L = decltype(lanes)::value, V = decltype(steps)::value;                                        \
      hipLaunchKernelGGL((norm_forward<T, L, V>), dim3(unsigned(groups_of(a.rows, a.width, 8, 1))),                \
                         dim3(threads_of(a.width)), 0, stream, a);                                                 \
    });                                                                                                            \
  }                                                                                                                \
  template <>                                                                                                      \
  void norm_backward_launch<T>(const NormArgs &a, bool bias, int groups, hipStream_t stream) {                     \
    with_shape(a.width, [&](auto lanes, auto steps) {                                                              \
      constexpr int L = decltype(lanes)::value, V = decltype(steps)::value;                                        \
      with_parts(a, bias, [&](auto g, auto p, auto b) {                                                            \
        constexpr bool G = decltype(g)::value, P = decltype(p)::value, B = decltype(b)::value;                     \
        const int threads = threads_of(a.width);                                                                   \
        if constexpr (V == 1) {                                                                                    \
          hipLaunchKernelGGL((norm_backward<T, L, V, G, P, B>), dim3(unsigned(groups)), dim3(threads),             \
                             (B ? 8 : 6) * 16 * (L < 256 ? L : threads), stream, a);                               \
        } else {                                                                                                   \
          hipLaunchKernelGGL((norm_backward<T, L, V, G, P, B>), dim3(unsigned(groups_of(a.rows, a.width, 4, 1))),  \
                             dim3(threads), 0, stream, a);                                                         \
          if (a.partial)                                                                                           \
            hipLaunchKernelGGL((norm_sums<T, G, P, B>), dim3(unsigned((a.width + 2047) / 2048), unsigned(groups)),     \
                               dim3(256), 0, stream, a);                                                           \
        }                                                                                                          \
      });                                                                                                          \
    });                                                                                                            \
  }

}  // namespace op
}  // namespace cchip
