// The norm of each head of q and k with the rotation by position, and the
// write of k and v to their caches.
//
// A head's elements are taken in pairs: the rotated ones as they are rotated,
// the others the first half with the second. A lane has 8 pairs, so that both
// elements of a pair are its own and it reads 16 bytes of a 16-bit head
// twice, and as many lanes have a head as that takes, rounded up to a power
// of two: 8 for 128 elements, 8 heads to a wave at a time. A wave goes through
// the heads of a token; the cosines and sines, which all of them share, are
// made by its lanes, one each, and handed round through LDS. Bound by memory:
// 16384 tokens, 32 and 8 heads of 128, bf16: 73.6 us for 336 MB forward, 107.1
// for 503 MB backward and 5.1 for the sums of the weights' gradients: 4.6 and 4.7 TB/s
// (a copy of 2 GiB: 4.86).

#include "heads.hpp"
#include "rows.hpp"

#include <algorithm>
#include <cmath>

namespace cchip {
namespace op {
namespace {

// One of q, k and v.
struct HeadPart {
  Heads x, y;         // read, written
  Heads g;            // backward: the gradient of what the forward pass wrote
  Heads cache;        // forward: written at the tokens' positions
  const void *weight;
  float *partial;     // backward: sums of a workgroup, or null
  int heads;
  uint32_t workgroups;
};

struct HeadArgs {
  HeadPart q, k, v;
  const int32_t *positions;
  const float *frequencies;
  int64_t keys;
  uint32_t tokens;   // of all rows of the batch
  uint32_t per_row;  // of a row of the batch
  uint32_t each;     // heads' iterations a wave takes at a time
  int dim, rotary, chunks;  // chunks: of 8 rotated pairs
  float eps;
  bool norm, weights_f32;
};

constexpr int kWaves = 4;

// Sum over the lanes of a head.
template <int Lanes>
__device__ __forceinline__ float sum_lanes(float x) {
#define CCHIP_MOVED(x, how) __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), how, 0xf, 0xf, true))
  x += CCHIP_MOVED(x, 0xB1);   // the neighbour
  x += CCHIP_MOVED(x, 0x4E);   // two on
  if (Lanes > 4) x += CCHIP_MOVED(x, 0x141);  // of 8 the other end's
  if (Lanes > 8) x += CCHIP_MOVED(x, 0x140);  // of 16
#undef CCHIP_MOVED
  if (Lanes > 16) x += __shfl_xor(x, 16, 64);
  if (Lanes > 32) x += __shfl_xor(x, 32, 64);
  return x;
}

// A lane's pairs: `count` elements from first on and `seconds` from second on,
// the elements of a pair side by side in both (alternate) or one in each. Those
// that are not rotated have nothing to do with one another: no turn of zero,
// in which an infinity in one would be a NaN in the other.
struct Pairs {
  int first, second, count, seconds;
  bool rotated, alternate;
};

__device__ __forceinline__ Pairs pairs_of(const HeadArgs &a, int chunk, bool interleaved) {
  Pairs p;
  p.rotated = chunk < a.chunks;
  p.alternate = interleaved && p.rotated;
  // the rest's pairs are its halves
  const int half = a.rotary / 2, rest = a.dim - a.rotary, lows = (rest + 1) / 2, at = 8 * (p.rotated ? chunk : chunk - a.chunks);
  int n = (p.rotated ? half : lows) - at, m = (p.rotated ? half : rest - lows) - at;
  p.first = (p.rotated ? 0 : a.rotary) + at;
  p.second = p.first + (p.rotated ? half : lows);
  if (p.alternate) {
    n *= 2;
    m = n - 8;
    p.first = 2 * at;
    p.second = p.first + 8;
  }
  p.count = n < 0 ? 0 : n < 8 ? n : 8;
  p.seconds = m < 0 ? 0 : m < 8 ? m : 8;
  return p;
}

template <typename T, bool Interleaved>
__device__ __forceinline__ void load_pairs(const T *p, const Pairs &at, bool live, float (&lo)[8], float (&hi)[8]) {
  const Raw8<T> x = load8<T>(p + at.first, live ? at.count : 0), y = load8<T>(p + at.second, live ? at.seconds : 0);
  float z[16];
#pragma unroll
  for (int i = 0; i < 8; i++) z[i] = float(x.x[i]), z[8 + i] = float(y.x[i]);
#pragma unroll
  for (int i = 0; i < 8; i++) {
    lo[i] = Interleaved && at.alternate ? z[2 * i] : z[i];
    hi[i] = Interleaved && at.alternate ? z[2 * i + 1] : z[8 + i];
  }
}

template <typename T, bool Interleaved>
__device__ __forceinline__ void store_pairs(T *p, const Pairs &at, const float (&lo)[8], const float (&hi)[8]) {
  float x[8], y[8];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const float a = i % 2 ? hi[i / 2] : lo[i / 2], b = i % 2 ? hi[4 + i / 2] : lo[4 + i / 2];
    x[i] = Interleaved && at.alternate ? a : lo[i];
    y[i] = Interleaved && at.alternate ? b : hi[i];
  }
  store8<T>(p + at.first, x, at.count);
  store8<T>(p + at.second, y, at.seconds);
}

// Workgroups of q, then of k, then of v.
template <typename T, int Lanes, bool Interleaved, bool Back>
__global__ __launch_bounds__(kWaves * 64) void head_norm(const HeadArgs a) {
  constexpr int kHeads = 64 / Lanes;
  __shared__ float turns[kWaves][2][256];
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6, chunk = l % Lanes;
  uint32_t id = blockIdx.x;
  HeadPart part = a.q;
  bool plain = false;  // v goes to its cache as it is
  if (id >= a.q.workgroups) {
    id -= a.q.workgroups;
    part = a.k;
    if (id >= a.k.workgroups) {
      id -= a.k.workgroups;
      part = a.v;
      plain = true;
    }
  }
  const Pairs at = pairs_of(a, chunk, Interleaved);

  float wl[8], wh[8];
#pragma unroll
  for (int i = 0; i < 8; i++) wl[i] = wh[i] = 1.0f;
  if (part.weight) {
    if (a.weights_f32) load_pairs<float, Interleaved>(static_cast<const float *>(part.weight), at, true, wl, wh);
    else load_pairs<T, Interleaved>(static_cast<const T *>(part.weight), at, true, wl, wh);
  }
  float dl[8] = {}, dh[8] = {}, cs[8], sn[8];
#pragma unroll
  for (int i = 0; i < 8; i++) cs[i] = 1.0f, sn[i] = 0.0f;

  const uint32_t rounds = uint32_t(part.heads + kHeads - 1) / kHeads, starts = (rounds + a.each - 1) / a.each;
  const uint64_t units = uint64_t(a.tokens) * starts, step = uint64_t(part.workgroups) * kWaves;
  for (uint64_t unit = uint64_t(id) * kWaves + w; unit < units; unit += step) {
    const uint32_t token = uint32_t(unit / starts), start = uint32_t(unit - uint64_t(token) * starts);
    const uint32_t batch = token / a.per_row, in = token - batch * a.per_row;
    const int32_t position = a.positions ? a.positions[token] : int32_t(in);
    if (a.chunks && !plain) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      for (int p = l; p < a.rotary / 2; p += 64) {
        // in turns, whole ones taken off while there are 64 bits
        const double turn = double(position) * double(a.frequencies[p]) * 0.15915494309189533577;
        float s, c;
        sincospif(2.0f * float(turn - __builtin_rint(turn)), &s, &c);
        turns[w][0][p] = c;
        turns[w][1][p] = s;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (at.rotated) {
#pragma unroll
        for (int i = 0; i < 8; i++)
          if (8 * chunk + i < a.rotary / 2) cs[i] = turns[w][0][8 * chunk + i], sn[i] = turns[w][1][8 * chunk + i];
      }
    }
    const uint32_t end = start * a.each + a.each < rounds ? start * a.each + a.each : rounds;
    for (uint32_t round = start * a.each; round < end; round++) {
      const int head = int(round) * kHeads + l / Lanes;
      const bool live = head < part.heads;
      const int64_t h = live ? head : 0;
      float lo[8], hi[8];
      load_pairs<T, Interleaved>(reinterpret_cast<const T *>(part.x.p) + batch * part.x.b + in * part.x.t + h * part.x.h, at, live, lo, hi);
      if constexpr (!Back) {
        if (a.norm && !plain) {
          float sum = 0.0f;
#pragma unroll
          for (int i = 0; i < 8; i++) sum += lo[i] * lo[i] + hi[i] * hi[i];
          const float inv = 1.0f / __builtin_sqrtf(sum_lanes<Lanes>(sum) / float(a.dim) + a.eps);
#pragma unroll
          for (int i = 0; i < 8; i++) lo[i] *= inv * wl[i], hi[i] *= inv * wh[i];
        }
        if (at.rotated && !plain) {
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const float x = lo[i] * cs[i] - hi[i] * sn[i];
            hi[i] = hi[i] * cs[i] + lo[i] * sn[i];
            lo[i] = x;
          }
        }
        if (!live) continue;
        if (part.y.p) store_pairs<T, Interleaved>(reinterpret_cast<T *>(part.y.p) + batch * part.y.b + in * part.y.t + h * part.y.h, at, lo, hi);
        if (part.cache.p && position >= 0 && position < a.keys)
          store_pairs<T, Interleaved>(reinterpret_cast<T *>(part.cache.p) + batch * part.cache.b + position * part.cache.t + h * part.cache.h, at, lo, hi);
      } else {
        float gl[8], gh[8];
        load_pairs<T, Interleaved>(reinterpret_cast<const T *>(part.g.p) + batch * part.g.b + in * part.g.t + h * part.g.h, at, live, gl, gh);
        if (at.rotated) {
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const float x = gl[i] * cs[i] + gh[i] * sn[i];
            gh[i] = gh[i] * cs[i] - gl[i] * sn[i];
            gl[i] = x;
          }
        }
        if (a.norm) {
          float sum = 0.0f, dot = 0.0f;
#pragma unroll
          for (int i = 0; i < 8; i++) {
            sum += lo[i] * lo[i] + hi[i] * hi[i];
            dot += gl[i] * wl[i] * lo[i] + gh[i] * wh[i] * hi[i];
          }
          // behind the last head there is nothing to add, with an eps of zero 0 times an infinity
          sum = sum_lanes<Lanes>(sum);
          const float inv = live ? 1.0f / __builtin_sqrtf(sum / float(a.dim) + a.eps) : 0.0f;
          const float mean = sum_lanes<Lanes>(dot) / float(a.dim) * inv * inv;
#pragma unroll
          for (int i = 0; i < 8; i++) {
            dl[i] += gl[i] * (lo[i] * inv);
            dh[i] += gh[i] * (hi[i] * inv);
            gl[i] = inv * (gl[i] * wl[i] - lo[i] * mean);
            gh[i] = inv * (gh[i] * wh[i] - hi[i] * mean);
          }
        }
        if (live) store_pairs<T, Interleaved>(reinterpret_cast<T *>(part.y.p) + batch * part.y.b + in * part.y.t + h * part.y.h, at, gl, gh);
      }
    }
  }
  if constexpr (Back) {
    if (!part.partial) return;
    // over the heads of a wave, then over the waves
#pragma unroll
    for (int i = 0; i < 8; i++)
#pragma unroll
      for (int d = Lanes; d < 64; d *= 2) {
        dl[i] += __shfl_xor(dl[i], d, 64);
        dh[i] += __shfl_xor(dh[i], d, 64);
      }
    __shared__ float sums[kWaves][512];
    if (l < Lanes) store_pairs<float, Interleaved>(sums[w], at, dl, dh);
    __syncthreads();
    for (int i = threadIdx.x; i < a.dim; i += kWaves * 64) {
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < kWaves; j++) sum += sums[j][i];
      part.partial[int64_t(id) * a.dim + i] = sum;
    }
  }
}

struct WeightArgs {
  const float *partial[2];
  void *to[2];
  uint32_t workgroups[2];
  int dim;
  bool f32;
};

// 32 elements of a weight's gradient a workgroup; 32 threads an element each
// sum every 32nd workgroup's share, and one of them those 32, in order.
template <typename T>
__global__ __launch_bounds__(1024) void head_weights(const WeightArgs a) {
  __shared__ float part[32][33];
  const int col = threadIdx.x % 32, turn = threadIdx.x / 32, s = blockIdx.y, c = int(blockIdx.x) * 32 + col;
  if (!a.to[s]) return;
  float q = 0.0f;
  if (c < a.dim) {
#pragma unroll 8
    for (uint32_t g = turn; g < a.workgroups[s]; g += 32) q += a.partial[s][int64_t(g) * a.dim + c];
  }
  part[turn][col] = q;
  __syncthreads();
  if (turn || c >= a.dim) return;
  float x = 0.0f;
#pragma unroll
  for (int i = 0; i < 32; i++) x += part[i][col];
  if (a.f32) static_cast<float *>(a.to[s])[c] = x;
  else static_cast<T *>(a.to[s])[c] = T(x);
}

// ---- host ----------------------------------------------------------------------------

const char *kWho = "head norm";

void check_op(const cchip_head_norm *op) {
  if (!op) throw InvalidArgument("head norm: no descriptor");
  check_rows_type(kWho, op->dtype);
  if (op->weight_dtype != op->dtype && op->weight_dtype != CCHIP_F32)
    throw InvalidArgument("head norm: weights are of the operator's dtype or f32");
  if (op->batch < 0 || op->tokens < 0 || op->keys < 0 || op->batch > INT32_MAX || op->tokens > INT32_MAX || op->keys > INT32_MAX ||
      op->batch * op->tokens > INT32_MAX)
    throw InvalidArgument("head norm: batch, tokens and keys are not negative, and batch times tokens and keys below 2^31");
  if (op->heads < 1 || op->kv_heads < 1 || op->heads > (1 << 20) || op->kv_heads > (1 << 20))
    throw InvalidArgument("head norm: heads and kv_heads are not in 1 .. 2^20");
  if (op->head_dim < 1 || op->head_dim > 512) throw InvalidArgument(strf("head norm: head_dim %d is not in 1 .. 512", op->head_dim));
  if (op->rotary < 0 || op->rotary % 2 || op->rotary > op->head_dim)
    throw InvalidArgument(strf("head norm: rotary %d is not even and at most head_dim %d", op->rotary, op->head_dim));
  if (op->norm != CCHIP_NORM_NONE && op->norm != CCHIP_NORM_RMS) throw InvalidArgument(strf("head norm: unknown norm %d", op->norm));
  if (!(op->eps >= 0.0f) || !std::isfinite(op->eps)) throw InvalidArgument("head norm: eps is finite and not negative");
}

int lanes_of(const cchip_head_norm &op) {
  const int need = (op.rotary / 2 + 7) / 8 + ((op.head_dim - op.rotary + 1) / 2 + 7) / 8;
  int lanes = 4;
  while (lanes < need) lanes *= 2;
  return lanes;
}

// Waves take a token's heads, which saves angles; few tokens are spread out.
// A backward pass has workgroups for a few rounds of the chip only, as each
// leaves a sum behind.
struct Cut {
  uint32_t each, workgroups[3];
};

Cut cut_of(const cchip_head_norm &op, bool back) {
  Cut c = {};
  const int64_t tokens = op.batch * op.tokens, at_a_time = 64 / lanes_of(op);
  c.each = tokens >= 2048 ? 1u << 20 : 1;
  for (int i = 0; i < (op.keys && !back ? 3 : 2); i++) {
    const int64_t rounds = ((i ? op.kv_heads : op.heads) + at_a_time - 1) / at_a_time, units = tokens * (c.each > 1 ? 1 : rounds);
    c.workgroups[i] = uint32_t(std::min<int64_t>((units + kWaves - 1) / kWaves, back ? (i ? 512 : 1536) : 1 << 20));
  }
  return c;
}

size_t partial_bytes(const cchip_head_norm &op) {
  const Cut c = cut_of(op, true);
  return op.norm == CCHIP_NORM_NONE ? 0 : size_t(c.workgroups[0] + c.workgroups[1]) * op.head_dim * sizeof(float);
}

void check_aligned(const char *name, const void *p, size_t to) {
  if (reinterpret_cast<uintptr_t>(p) % to) throw InvalidArgument(strf("head norm: %s is not aligned to its elements", name));
}

// Written over what is read: in one place only where `in_place` says that each
// head is read before it is written. Of caches, whose places are the
// positions', the first heads are looked at.
void check_place(const cchip_head_norm &op, const char *out, const Heads &y, int64_t y_heads, const char *in, const Heads &x, int64_t x_heads,
                 bool in_place, bool cache) {
  const int size = op.dtype == CCHIP_F32 ? 4 : 2;
  if (!y.p || !x.p) return;
  const size_t bytes = size_t(op.head_dim) * size;
  if (cache ? !meet(y.p, bytes, x.p, bytes)
            : !heads_meet(op.head_dim, size, {{op.batch, op.tokens, y_heads}}, y, {{op.batch, op.tokens, x_heads}}, x))
    return;
  if (in_place && y.p == x.p && (op.batch < 2 || y.b == x.b) && (op.tokens < 2 || y.t == x.t) && y.h == x.h) return;
  throw InvalidArgument(strf("head norm: %s is written over %s%s", out, in, in_place ? ", and not head for head" : ""));
}

HeadArgs args_of(const cchip_head_norm &op, const cchip_head_norm_io &io) {
  HeadArgs a = {};
  if (op.rotary && !io.frequencies) throw InvalidArgument("head norm: no frequencies");
  check_aligned("frequencies", io.frequencies, 4);
  check_aligned("positions", io.positions, 4);
  const size_t weight = op.weight_dtype == CCHIP_F32 ? 4 : 2;
  check_aligned("q_weight", io.q_weight, weight);
  check_aligned("k_weight", io.k_weight, weight);
  check_aligned("the gradient of q_weight", io.dq_weight, weight);
  check_aligned("the gradient of k_weight", io.dk_weight, weight);
  if (op.norm == CCHIP_NORM_NONE && (io.q_weight || io.k_weight || io.dq_weight || io.dk_weight))
    throw InvalidArgument("head norm: weights of a norm that there is not");
  a.positions = io.positions;
  a.frequencies = io.frequencies;
  a.keys = op.keys;
  a.tokens = uint32_t(op.batch * op.tokens);
  a.per_row = uint32_t(op.tokens);
  a.dim = op.head_dim;
  a.rotary = op.rotary;
  a.chunks = (op.rotary / 2 + 7) / 8;
  a.eps = op.eps;
  a.norm = op.norm == CCHIP_NORM_RMS;
  a.weights_f32 = op.weight_dtype == CCHIP_F32;
  a.q.weight = io.q_weight;
  a.k.weight = io.k_weight;
  a.q.heads = op.heads;
  a.k.heads = a.v.heads = op.kv_heads;
  return a;
}

Heads heads_of(const cchip_head_norm &op, const char *name, int64_t tokens, int heads, const cchip_heads &x, bool written, bool needed) {
  if (!x.data && !needed) return {};
  return cchip::op::heads_of(kWho, name, op.dtype, op.batch, tokens, heads, op.head_dim, x, written);
}

template <typename T, int Lanes>
void launch_lanes(const HeadArgs &a, bool interleaved, bool back, dim3 grid, hipStream_t stream) {
  const dim3 block(kWaves * 64);
  if (back) {
    if (interleaved) hipLaunchKernelGGL((head_norm<T, Lanes, true, true>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((head_norm<T, Lanes, false, true>), grid, block, 0, stream, a);
  } else {
    if (interleaved) hipLaunchKernelGGL((head_norm<T, Lanes, true, false>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((head_norm<T, Lanes, false, false>), grid, block, 0, stream, a);
  }
}

void launch(const cchip_head_norm &op, HeadArgs &a, const Cut &c, bool back, hipStream_t stream) {
  a.each = c.each;
  a.q.workgroups = c.workgroups[0];
  a.k.workgroups = c.workgroups[1];
  a.v.workgroups = c.workgroups[2];
  const dim3 grid(c.workgroups[0] + c.workgroups[1] + c.workgroups[2]);
  with_rows_type(op.dtype, [&](auto t) {
    typedef decltype(t) T;
    switch (lanes_of(op)) {
      case 4: return launch_lanes<T, 4>(a, op.interleaved, back, grid, stream);
      case 8: return launch_lanes<T, 8>(a, op.interleaved, back, grid, stream);
      case 16: return launch_lanes<T, 16>(a, op.interleaved, back, grid, stream);
      case 32: return launch_lanes<T, 32>(a, op.interleaved, back, grid, stream);
      default: return launch_lanes<T, 64>(a, op.interleaved, back, grid, stream);
    }
  });
  check_launch(kWho);
}

}  // namespace
}  // namespace op
}  // namespace cchip

using namespace cchip;
using namespace cchip::op;

extern "C" {

int cchip_head_norm_forward(const cchip_head_norm *op, const cchip_head_norm_io *io, void *stream) {
  return guarded([&] {
    check_op(op);
    if (!io) throw InvalidArgument("head norm: no tensors");
    HeadArgs a = args_of(*op, *io);
    if (op->batch * op->tokens == 0) return;
    HeadPart &q = a.q, &k = a.k, &v = a.v;
    q.x = heads_of(*op, "q", op->tokens, op->heads, io->q, false, true);
    k.x = heads_of(*op, "k", op->tokens, op->kv_heads, io->k, false, true);
    q.y = heads_of(*op, "q_out", op->tokens, op->heads, io->q_out, true, true);
    k.y = heads_of(*op, "k_out", op->tokens, op->kv_heads, io->k_out, true, op->keys == 0);
    if (op->keys) {
      v.x = heads_of(*op, "v", op->tokens, op->kv_heads, io->v, false, true);
      k.cache = heads_of(*op, "k_cache", op->keys, op->kv_heads, io->k_cache, true, true);
      v.cache = heads_of(*op, "v_cache", op->keys, op->kv_heads, io->v_cache, true, true);
    } else if (io->v.data || io->k_cache.data || io->v_cache.data) {
      throw InvalidArgument("head norm: a cache for an operator made without keys");
    }
    struct Named {
      const char *name;
      const Heads *x;
      int heads;
    };
    const int h = op->heads, hk = op->kv_heads;
    const Named in[] = {{"q", &q.x, h}, {"k", &k.x, hk}, {"v", &v.x, hk}},
                out[] = {{"q_out", &q.y, h}, {"k_out", &k.y, hk}, {"k_cache", &k.cache, hk}, {"v_cache", &v.cache, hk}};
    for (int i = 0; i < 4; i++) {
      for (int j = 0; j < 3; j++) check_place(*op, out[i].name, *out[i].x, out[i].heads, in[j].name, *in[j].x, in[j].heads, i == j && i < 2, i > 1);
      for (int j = 0; j < i; j++) check_place(*op, out[i].name, *out[i].x, out[i].heads, out[j].name, *out[j].x, out[j].heads, false, i > 1);
    }
    launch(*op, a, cut_of(*op, false), false, (hipStream_t)stream);
  });
}

int cchip_head_norm_workspace(const cchip_head_norm *op, size_t *bytes) {
  return guarded([&] {
    check_op(op);
    if (bytes) *bytes = partial_bytes(*op);
  });
}

int cchip_head_norm_backward(const cchip_head_norm *op, const cchip_head_norm_io *io, void *workspace, size_t workspace_bytes,
                             void *stream) {
  return guarded([&] {
    check_op(op);
    if (!io) throw InvalidArgument("head norm: no tensors");
    HeadArgs a = args_of(*op, *io);
    const Cut c = cut_of(*op, true);
    const bool any = io->dq_weight || io->dk_weight;
    if (op->batch * op->tokens) {
      HeadPart &q = a.q, &k = a.k;
      q.x = heads_of(*op, "q", op->tokens, op->heads, io->q, false, true);
      k.x = heads_of(*op, "k", op->tokens, op->kv_heads, io->k, false, true);
      q.g = heads_of(*op, "the gradient of q_out", op->tokens, op->heads, io->dq_out, false, true);
      k.g = heads_of(*op, "the gradient of k_out", op->tokens, op->kv_heads, io->dk_out, false, true);
      q.y = heads_of(*op, "dq", op->tokens, op->heads, io->dq, true, true);
      k.y = heads_of(*op, "dk", op->tokens, op->kv_heads, io->dk, true, true);
      struct Named {
        const char *name;
        const Heads *x;
        int heads;
      };
      const int h = op->heads, hk = op->kv_heads;
      const Named in[] = {{"the gradient of q_out", &q.g, h}, {"the gradient of k_out", &k.g, hk}, {"q", &q.x, h}, {"k", &k.x, hk}},
                  out[] = {{"dq", &q.y, h}, {"dk", &k.y, hk}};
      for (int i = 0; i < 2; i++)
        for (int j = 0; j < 4; j++) check_place(*op, out[i].name, *out[i].x, out[i].heads, in[j].name, *in[j].x, in[j].heads, i == j, false);
      check_place(*op, "dk", k.y, hk, "dq", q.y, h, false, false);
      if (any) {
        const size_t need = partial_bytes(*op);
        if (workspace_bytes < need || !workspace || !aligned16(workspace))
          throw InvalidArgument(strf("head norm: the workspace needs %zu bytes aligned to 16, has %zu", need, workspace ? workspace_bytes : 0));
        q.partial = static_cast<float *>(workspace);
        k.partial = q.partial + size_t(c.workgroups[0]) * op->head_dim;
      }
      launch(*op, a, c, true, (hipStream_t)stream);
    }
    if (!any) return;
    WeightArgs x = {};
    x.partial[0] = a.q.partial;
    x.partial[1] = a.k.partial;
    x.workgroups[0] = c.workgroups[0];
    x.workgroups[1] = c.workgroups[1];
    x.to[0] = io->dq_weight;
    x.to[1] = io->dk_weight;
    x.dim = op->head_dim;
    x.f32 = a.weights_f32;
    with_rows_type(op->dtype, [&](auto t) {
      hipLaunchKernelGGL((head_weights<decltype(t)>), dim3((op->head_dim + 31) / 32, 2), dim3(1024), 0, (hipStream_t)stream, x);
    });
    check_launch(kWho);
  });
}

}  // extern "C"
