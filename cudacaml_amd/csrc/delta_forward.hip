// Gated delta rule, forward: the chunks of a sequence in order, the state in
// registers (the formulas stand in delta.hpp).

#include "delta.hpp"

namespace cchip {
namespace op {
namespace {

// A workgroup of four waves runs BV value columns of one head through the
// chunks. Wave w holds rows w DK / 4 .. of S (f32, in the layout of a
// product's result) and makes rows 16 w .. of K S, U and O. Only K, S, beta X
// and U are shared through LDS: the rows of Q, T and P that a wave needs are
// its own and go from memory to registers as matrix operands. Each of them is
// asked for again for the next chunk as soon as this one has used it, so that
// memory answers while the chain of products, three waits for the other
// waves long, goes on.
template <typename M, int DK, int BV, bool Back, bool Fast>
__global__ __launch_bounds__(256, 2) void delta_forward(const DeltaArgs a, int blocks) {
  typedef typename M::T T;
  typedef typename M::Saved Saved;
  constexpr int NI = M::NI, NS = M::NS, NO = M::NO, NU = M::NU;
  constexpr int LDK = DK + 8, LDT = 72;
  constexpr int KP = 64 * LDK, SP = BV * LDK, XP = BV * LDT;
  constexpr int TK = DK / 64, TV = BV / 16;  // 16 x 16 tiles of S a wave holds
  typedef Record<M> R;
  __shared__ __align__(16) bf16 ks[NI * KP], st[NS * SP], xt[NS * XP], ut[NU * XP], gt[NS * XP];

  // heads 8 apart share a chiplet's L2: a head's column blocks, which read
  // the same q, k, T and P, are 8 workgroups apart
  const int64_t group = blockIdx.x / (8 * blocks);
  const int rest = int(blockIdx.x - group * 8 * blocks);
  const int64_t lane_id = group * 8 + rest % 8;
  if (lane_id >= a.sequences * a.hv) return;
  const int64_t sid = lane_id / a.hv;
  const int h = int(lane_id - sid * a.hv), hk = h / (a.hv / a.hk), dv0 = rest / 8 * BV;
  const Sequence sq = sequence_of(a, sid);
  const int chunks = int((sq.len + kChunk - 1) / kChunk);

  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, quad = l >> 4, col = l & 15;
  const int row0 = w * (DK / 4) + quad * 4;  // of S: this lane's rows are row0 + 16 i + r

  f32x4 s[TK][TV];
  const int64_t state_at = lane_id * a.dk * a.dv;
#pragma unroll
  for (int i = 0; i < TK; i++)
#pragma unroll
    for (int j = 0; j < TV; j++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int x = row0 + 16 * i + r, y = dv0 + 16 * j + col;
        s[i][j][r] = a.state && x < a.dk && y < a.dv ? a.state[state_at + int64_t(x) * a.dv + y] : 0.0f;
      }

  auto chunk = [&](int i) {
    const int64_t left = sq.len - int64_t(i) * kChunk;
    return Chunk{sq.row, sq.first + int64_t(i) * kChunk, sid, left > kChunk ? kChunk : int(left)};
  };
  auto record = [&](int i) { return a.records + ((sq.slot + i) * a.hv + h) * R::bytes(Back); };
  Raw8<T> rk[DK / 32], rq[DK / 32];
  T rv[TV][4];
  Frag<NS> ft[2];
  Frag<NO> fp[2];
  float gam[4], last[4], beta[4];
  auto fetch_k = [&](int i) {
    const Chunk c = chunk(i);
#pragma unroll
    for (int j = 0; j < DK / 32; j++) {
      const int at = tid + 256 * j;
      rk[j] = load_head8<Fast, T>(a.k, c, hk, at / (DK / 8), at % (DK / 8) * 8, a.dk);
    }
  };
  auto fetch_qv = [&](int i) {
    const Chunk c = chunk(i);
#pragma unroll
    for (int j = 0; j < DK / 32; j++) rq[j] = load_head8<Fast, T>(a.q, c, hk, 16 * w + col, 32 * j + 8 * quad, a.dk);
    const float *dec = reinterpret_cast<const float *>(record(i) + R::Decay);
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int t = 16 * w + 4 * quad + r;
#pragma unroll
      for (int j = 0; j < TV; j++) rv[j][r] = load_head1<T>(a.v, c, h, t, dv0 + 16 * j + col, a.dv);
      beta[r] = dec[128 + t];
    }
  };
  auto fetch_t = [&](int i) {
#pragma unroll
    for (int b = 0; b < 2; b++)
      if (b == 0 || w >= 2)  // T and P end at the diagonal
#pragma unroll
        for (int p = 0; p < NS; p++)
          ft[b].p[p] = reinterpret_cast<const bf16x8 *>(record(i) + R::T + p * 8192)[(w * 2 + b) * 64 + l];
  };
  auto fetch_p = [&](int i) {
#pragma unroll
    for (int b = 0; b < 2; b++)
      if (b == 0 || w >= 2)
#pragma unroll
        for (int p = 0; p < NO; p++)
          fp[b].p[p] = reinterpret_cast<const bf16x8 *>(record(i) + R::P + p * 8192)[(w * 2 + b) * 64 + l];
    const float *dec = reinterpret_cast<const float *>(record(i) + R::Decay);
#pragma unroll
    for (int r = 0; r < 4; r++) {
      gam[r] = dec[16 * w + 4 * quad + r];
      last[r] = dec[64 + 16 * w + 4 * quad + r];
    }
  };

  if (chunks > 0) {
    fetch_k(0);
    fetch_qv(0);
    fetch_t(0);
    fetch_p(0);
  }
  for (int ci = 0; ci < chunks; ci++) {
    const Chunk c = chunk(ci);
    const int next = ci + 1 < chunks ? ci + 1 : ci;
#pragma unroll
    for (int j = 0; j < DK / 32; j++) {
      const int at = tid + 256 * j, t = at / (DK / 8), d = at % (DK / 8) * 8;
      put_frag<NI>(ks + t * LDK + d, KP, frag_of<NI>(keep_head8<Fast>(rk[j], c, t, d, a.dk)));
    }
#pragma unroll
    for (int i = 0; i < TK; i++)
#pragma unroll
      for (int j = 0; j < TV; j++) put_column<NS>(st + (16 * j + col) * LDK + row0 + 16 * i, SP, s[i][j]);
    __syncthreads();
    fetch_k(next);
    if (Back) {
      Saved *to = reinterpret_cast<Saved *>(a.states) + ((sq.slot + ci) * a.hv + h) * DK * a.dvp + dv0;
#pragma unroll
      for (int i = 0; i < TK; i++)
#pragma unroll
        for (int j = 0; j < TV; j++)
#pragma unroll
          for (int r = 0; r < 4; r++) to[(row0 + 16 * i + r) * a.dvp + 16 * j + col] = Saved(s[i][j][r]);
    }

    f32x4 kS[TV] = {}, qS[TV] = {};
#pragma unroll
    for (int d = 0; d < DK; d += 32) {
      const Frag<NI> fk = frag_row<NI>(ks, KP, LDK, 16 * w, d);
      const Frag<NI> fq = frag_of<NI>(keep_head8<Fast>(rq[d / 32], c, 16 * w + col, d + 8 * quad, a.dk));
#pragma unroll
      for (int j = 0; j < TV; j++) {
        const Frag<NS> fs = frag_row<NS>(st, SP, LDK, 16 * j, d);
        kS[j] = mma(kS[j], fk, fs);
        qS[j] = mma(qS[j], fq, first_planes<NO>(fs));
      }
    }
#pragma unroll
    for (int j = 0; j < TV; j++) {
      f32x4 x;
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int t = 16 * w + 4 * quad + r, y = dv0 + 16 * j + col;
        const float v = t < c.len && y < a.dv ? float(rv[j][r]) : 0.0f;
        x[r] = beta[r] * (v - gam[r] * kS[j][r]);
      }
      put_column<NS>(xt + (16 * j + col) * LDT + 16 * w + 4 * quad, XP, x);
    }
    fetch_qv(next);
    __syncthreads();
    f32x4 u[TV] = {};
#pragma unroll
    for (int b = 0; b < 2; b++)
      if (b == 0 || w >= 2)
#pragma unroll
        for (int j = 0; j < TV; j++) u[j] = mma(u[j], ft[b], frag_row<NS>(xt, XP, LDT, 16 * j, 32 * b));
    fetch_t(next);
#pragma unroll
    for (int j = 0; j < TV; j++) {
      f32x4 g;
#pragma unroll
      for (int r = 0; r < 4; r++) g[r] = last[r] * u[j][r];
      put_column<NU>(ut + (16 * j + col) * LDT + 16 * w + 4 * quad, XP, u[j]);
      put_column<NS>(gt + (16 * j + col) * LDT + 16 * w + 4 * quad, XP, g);
    }
    if (Back) {
      float *to = a.us + ((sq.slot + ci) * a.hv + h) * kChunk * a.dvp + dv0;
#pragma unroll
      for (int j = 0; j < TV; j++)
#pragma unroll
        for (int r = 0; r < 4; r++) to[(16 * w + 4 * quad + r) * a.dvp + 16 * j + col] = u[j][r];
    }
    const float end = reinterpret_cast<const float *>(record(ci) + R::Decay)[63];
    __syncthreads();
    f32x4 o[TV];
#pragma unroll
    for (int j = 0; j < TV; j++)
#pragma unroll
      for (int r = 0; r < 4; r++) o[j][r] = gam[r] * qS[j][r];
#pragma unroll
    for (int b = 0; b < 2; b++)
      if (b == 0 || w >= 2)
#pragma unroll
        for (int j = 0; j < TV; j++) o[j] = mma(o[j], fp[b], frag_row<NU>(ut, XP, LDT, 16 * j, 32 * b));
    fetch_p(next);
#pragma unroll
    for (int i = 0; i < TK; i++)
#pragma unroll
      for (int j = 0; j < TV; j++) s[i][j] *= end;
#pragma unroll
    for (int b = 0; b < 2; b++) {
      Frag<NS> fg[TV];
#pragma unroll
      for (int j = 0; j < TV; j++) fg[j] = frag_row<NS>(gt, XP, LDT, 16 * j, 32 * b);
#pragma unroll
      for (int i = 0; i < TK; i++) {
        const Frag<NI> fk = frag_col<NI>(ks, KP, LDK, w * (DK / 4) + 16 * i, 32 * b);
#pragma unroll
        for (int j = 0; j < TV; j++) s[i][j] = mma(s[i][j], fk, fg[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < TV; j++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int t = 16 * w + 4 * quad + r, y = dv0 + 16 * j + col;
        if (t < c.len && y < a.dv) out_at<T>(a.o, c.row, c.first + t, h)[y] = T(a.scale * o[j][r]);
      }
    __syncthreads();
  }
  if (a.state_out)
#pragma unroll
    for (int i = 0; i < TK; i++)
#pragma unroll
      for (int j = 0; j < TV; j++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int x = row0 + 16 * i + r, y = dv0 + 16 * j + col;
          if (x < a.dk && y < a.dv) a.state_out[state_at + int64_t(x) * a.dv + y] = s[i][j][r];
        }
}

}  // namespace

void delta_forward_launch(const cchip_gated_delta &op, const DeltaArgs &a, bool back, hipStream_t stream) {
  const int64_t lanes = a.sequences * a.hv;
  auto launch = [&](auto m, auto dk, auto bv) {
    typedef decltype(m) M;
    constexpr int DK = decltype(dk)::value, BV = decltype(bv)::value;
    const int blocks = back ? a.dvp / BV : (a.dv + BV - 1) / BV;  // saved columns that pad a head are written too
    with_bool(back, [&](auto b) {
      with_bool(fast(a), [&](auto f) {
        hipLaunchKernelGGL((delta_forward<M, DK, BV, decltype(b)::value, decltype(f)::value>),
                           dim3(unsigned((lanes + 7) / 8 * 8 * blocks)), dim3(256), 0, stream, a, blocks);
      });
    });
  };
  typedef std::integral_constant<int, 16> C16;
  typedef std::integral_constant<int, 32> C32;
  typedef std::integral_constant<int, 64> C64;
  typedef std::integral_constant<int, 128> C128;
  with_mode(op, [&](auto m) {
    const bool narrow = lanes * ((a.dv + 31) / 32) < 256;
    if (a.dk <= 64) narrow ? launch(m, C64(), C16()) : launch(m, C64(), C32());
    else narrow ? launch(m, C128(), C16()) : launch(m, C128(), C32());
  });
  check_launch("gated delta: forward");
}

}  // namespace op
}  // namespace cchip
