// Gated delta rule for a few tokens of each sequence: the recurrence itself,
// the state read once and written once.

#include "delta.hpp"

namespace cchip {
namespace op {
namespace {

constexpr int kColumns = 32;

__device__ __forceinline__ f32x4 load_state4(const float *p, int n, bool vec) {
  f32x4 s = {};
  if (vec && n >= 4) return *reinterpret_cast<const f32x4 *>(p);
#pragma unroll
  for (int i = 0; i < 4; i++) s[i] = i < n ? p[i] : 0.0f;
  return s;
}

// A workgroup a sequence, value head and 32 value columns. A thread holds 4
// neighbouring columns of rows x = tid / 8 + 32 i, so that 8 lanes read 128
// neighbouring bytes of a row. S^T k and S^T q come out of one reduction:
// with u known, S_t^T q = exp(g) S^T q + (k . q) u. The states' bytes bound
// it: one token of 256 sequences, 32 heads of 128 x 128, moves 1.08 GB in 215
// us, 5.0 TB/s, as fast as a copy. With few states (8 sequences, 16 heads:
// 6.6 us) it is the time of a launch and one pass through memory.
template <typename T, int ROWS>
__global__ __launch_bounds__(256) void delta_step(const DeltaArgs a, int blocks, bool vec) {
  __shared__ float qs[2][ROWS * 32], ks[2][ROWS * 32], part[2][4][2 * kColumns + 1];
  const int64_t lane_id = block_index() / blocks;
  if (lane_id >= a.sequences * a.hv) return;
  const int64_t row = lane_id / a.hv;
  const int h = int(lane_id - row * a.hv), hk = h / (a.hv / a.hk);
  const int v0 = int(block_index() - lane_id * blocks) * kColumns;
  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, y = v0 + tid % 8 * 4, n = a.dv - y;

  f32x4 s[ROWS];
  const int64_t state_at = lane_id * a.dk * a.dv;
#pragma unroll
  for (int i = 0; i < ROWS; i++) {
    const int x = tid / 8 + 32 * i;
    s[i] = a.state && x < a.dk ? load_state4(a.state + state_at + int64_t(x) * a.dv + y, n, vec) : f32x4{};
  }
  for (int64_t t = 0; t < a.tokens; t++) {
    const int b = t & 1;
    if (tid < ROWS * 32) ks[b][tid] = tid < a.dk ? float(at<T>(a.k, row, t, hk)[tid]) : 0.0f;
    else if (tid - ROWS * 32 < ROWS * 32) {
      const int x = tid - ROWS * 32;
      qs[b][x] = x < a.dk ? float(at<T>(a.q, row, t, hk)[x]) : 0.0f;
    }
    const float alpha = expf(float(*at<T>(a.g, row, t, h))), beta = float(*at<T>(a.beta, row, t, h));
    f32x4 v;
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = i < n ? float(at<T>(a.v, row, t, h)[y + i]) : 0.0f;
    __syncthreads();
    f32x4 sk = {}, sq = {};
    float kq = 0.0f;
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      const float k = ks[b][tid / 8 + 32 * i], q = qs[b][tid / 8 + 32 * i];
      sk += s[i] * k;
      sq += s[i] * q;
      kq += k * q;
    }
#pragma unroll
    for (int d = 8; d < 64; d *= 2) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        sk[i] += __shfl_xor(sk[i], d, 64);
        sq[i] += __shfl_xor(sq[i], d, 64);
      }
      kq += __shfl_xor(kq, d, 64);
    }
    if (l < 8) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        part[b][w][l * 4 + i] = sk[i];
        part[b][w][kColumns + l * 4 + i] = sq[i];
      }
      if (l == 0) part[b][w][2 * kColumns] = kq;
    }
    __syncthreads();
    kq = part[b][0][2 * kColumns] + part[b][1][2 * kColumns] + part[b][2][2 * kColumns] + part[b][3][2 * kColumns];
    f32x4 u, o;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int c = tid % 8 * 4 + i;
      const float k4 = part[b][0][c] + part[b][1][c] + part[b][2][c] + part[b][3][c];
      const float q4 = part[b][0][kColumns + c] + part[b][1][kColumns + c] + part[b][2][kColumns + c] + part[b][3][kColumns + c];
      u[i] = beta * (v[i] - alpha * k4);
      o[i] = a.scale * (alpha * q4 + kq * u[i]);
    }
#pragma unroll
    for (int i = 0; i < ROWS; i++) s[i] = s[i] * alpha + u * ks[b][tid / 8 + 32 * i];
    if (tid < 8) {
      T *to = out_at<T>(a.o, row, t, h) + y;
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (i < n) to[i] = T(o[i]);
    }
  }
  if (a.state_out)
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      const int x = tid / 8 + 32 * i;
      if (x >= a.dk || n <= 0) continue;
      float *to = a.state_out + state_at + int64_t(x) * a.dv + y;
      if (vec && n >= 4) *reinterpret_cast<f32x4 *>(to) = s[i];
      else
        for (int j = 0; j < 4 && j < n; j++) to[j] = s[i][j];
    }
}

}  // namespace

void delta_step_launch(const cchip_gated_delta &op, const DeltaArgs &a, hipStream_t stream) {
  const int blocks = (a.dv + kColumns - 1) / kColumns;
  const bool vec = a.dv % 4 == 0 && aligned16(a.state) && aligned16(a.state_out);
  auto launch = [&](auto t) {
    typedef decltype(t) T;
    auto *k = a.dk <= 64 ? delta_step<T, 2> : delta_step<T, 4>;
    hipLaunchKernelGGL(k, grid_of(a.sequences * a.hv * blocks), dim3(256), 0, stream, a, blocks, vec);
  };
  if (op.dtype == CCHIP_F32) launch(float());
  else if (op.dtype == CCHIP_F16) launch(f16());
  else launch(bf16());
  check_launch("gated delta: step");
}

}  // namespace op
}  // namespace cchip
