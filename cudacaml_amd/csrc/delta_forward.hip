// Gated delta rule, forward: the chunks of a sequence in order, the state in
// registers (the formulas stand in delta.hpp).

#include "delta.hpp"

namespace cchip {
namespace op {
namespace {

// A workgroup of four waves runs BV value columns of one head through the
// chunks. Wave w holds columns w DK / 4 .. of S^T in the layout of a
// product's result (f32) and makes columns 16 w .. of (K S)^T, U^T and O^T:
// products are taken transposed, so that a lane has 4 neighbouring value
// columns of one token and reads and writes them at once. Only K, S, beta X
// and U are shared through LDS: the rows of Q, T and P that a wave needs are
// its own and go from memory to registers as matrix operands. Each of them is
// asked for again for the next chunk as soon as this one has used it, so that
// memory answers while the chain of products, three waits for the other
// waves long, goes on.
//
// That chain bounds it where workgroups have a unit each: 2.2 us a chunk (570
// us for 16384 tokens, 32 bf16 heads of 128 with f32 states; their bytes take
// 84). With two a unit (4 x 4096 tokens, saving for a backward pass, 376 us)
// it moves 0.95 GB of records, tokens, states and U at 2.5 TB/s and makes 8.4
// MFLOP of products a chunk and head, in planes over twice that, at a third of
// the matrix rate: neither is at its limit, the waits between are the rest.
template <typename M, int DK, int BV, bool Back, int A>
__global__ __launch_bounds__(256, groups_a_unit<M>(DK, BV)) void delta_forward(const DeltaArgs a, int blocks) {
  typedef typename M::T T;
  typedef typename M::Saved Saved;
  constexpr int NI = M::NI, NS = M::NS, NO = M::NO;
  constexpr int LDK = DK + 16, LDV = BV == 16 ? 24 : BV;
  constexpr int KP = 64 * LDK, SP = DK * LDV, XP = 64 * LDV;
  constexpr int TK = DK / 64, TV = BV / 16;  // 16 x 16 tiles of S a wave holds
  typedef Record<M> R;
  // two sets of keys where LDS has room: the next chunk's are written while
  // slower waves still read this one's
  constexpr int kSets = NI == 1 ? 2 : 1;
  __shared__ __align__(16) bf16 keys[kSets * NI * KP], ss[NS * SP], xs[NS * XP], us[NO * XP], gs[NS * XP];

  // heads 8 apart share a chiplet's L2: a head's column blocks, which read
  // the same q, k, T and P, are 8 workgroups apart
  const int64_t group = block_index() / (8 * blocks);
  const int rest = int(block_index() - group * 8 * blocks);
  const int64_t lane_id = group * 8 + rest % 8;
  if (lane_id >= a.sequences * a.hv) return;
  const int64_t sid = lane_id / a.hv;
  const int h = int(lane_id - sid * a.hv), hk = h / (a.hv / a.hk), dv0 = rest / 8 * BV;
  const Sequence sq = sequence_of(a, sid);
  const int chunks = int((sq.len + kChunk - 1) / kChunk);

  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, quad = l >> 4, col = l & 15;
  const int x0 = w * (DK / 4) + col, y0 = 4 * TV * quad;  // this lane's part of S: rows x0 + 16 i, columns dv0 + y0 + 4 j + r
  const int t = 16 * w + col;                        // and its token

  f32x4 s[TK][TV];
  const int64_t state_at = lane_id * a.dk * a.dv + dv0;
#pragma unroll
  for (int i = 0; i < TK; i++)
#pragma unroll
    for (int j = 0; j < TV; j++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int x = x0 + 16 * i, y = y0 + 4 * j + r;
        s[i][j][r] = a.state && x < a.dk && dv0 + y < a.dv ? a.state[state_at + int64_t(x) * a.dv + y] : 0.0f;
      }

  auto chunk = [&](int i) {
    const int64_t left = sq.len - int64_t(i) * kChunk;
    return Chunk{sq.row, sq.first + int64_t(i) * kChunk, sid, left > kChunk ? kChunk : int(left)};
  };
  auto record = [&](int i) { return a.records + ((sq.slot + i) * a.hv + h) * R::bytes(Back); };
  Raw8<T> rk[DK / 32], rq[DK / 32];
  RawV<T, TV> rv;
  Frag<NS> ft[2];
  Frag<NO> fp[2];
  float gam, last, beta, end;
  auto fetch_k = [&](int i) {
    const Chunk c = chunk(i);
#pragma unroll
    for (int j = 0; j < DK / 32; j++) {
      const int at = tid + 256 * j;
      rk[j] = load_head8<A, T>(a.k, c, hk, at / (DK / 8), at % (DK / 8) * 8, a.dk);
    }
  };
  auto fetch_qv = [&](int i) {
    const Chunk c = chunk(i);
#pragma unroll
    for (int j = 0; j < DK / 32; j++) rq[j] = load_head8<A, T>(a.q, c, hk, t, 32 * j + 8 * quad, a.dk);
    rv = load_v<A, T, TV>(a.v, c, h, t, dv0 + y0, a.dv);
  };
  auto fragment = [&](const char *from, int b) {  // rows 16 w .. of a matrix of the record, terms 32 b ..
    return *reinterpret_cast<const bf16x8 *>(from + uint32_t((w * 2 + b) * 1024 + l * 16));
  };
  auto fetch_t = [&](int i) {
#pragma unroll
    for (int b = 0; b < 2; b++)
      if (b == 0 || w >= 2)  // T and P end at the diagonal
#pragma unroll
        for (int p = 0; p < NS; p++) ft[b].p[p] = fragment(record(i) + R::T + p * 8192, b);
  };
  auto fetch_p = [&](int i) {
#pragma unroll
    for (int b = 0; b < 2; b++)
      if (b == 0 || w >= 2)
#pragma unroll
        for (int p = 0; p < NO; p++) fp[b].p[p] = fragment(record(i) + R::P + p * 8192, b);
    const float *dec = reinterpret_cast<const float *>(record(i) + R::Decay);
    gam = dec[t];
    last = dec[64 + t];
    beta = dec[128 + t];
    end = dec[63];
  };

  if (chunks > 0) {
    fetch_k(0);
    fetch_qv(0);
    fetch_t(0);
    fetch_p(0);
  }
  auto put_keys = [&](int i) {
    const Chunk c = chunk(i);
    bf16 *const to = keys + i % kSets * NI * KP;
#pragma unroll
    for (int j = 0; j < DK / 32; j++) {
      const int at = tid + 256 * j, kt = at / (DK / 8), d = at % (DK / 8) * 8;
      put_frag<NI>(to + kt * LDK + d, KP, frag_of<NI>(keep_head8<A>(rk[j], c, kt, d, a.dk)));
    }
  };
  auto put_state = [&]() {
#pragma unroll
    for (int i = 0; i < TK; i++)
#pragma unroll
      for (int j = 0; j < TV; j++) put_four<NS>(ss + (x0 + 16 * i) * LDV + y0 + 4 * j, SP, s[i][j]);
  };
  if (chunks > 0) {
    put_keys(0);
    put_state();
  }
  for (int ci = 0; ci < chunks; ci++) {
    const Chunk c = chunk(ci);
    const int next = ci + 1 < chunks ? ci + 1 : ci;
    const bf16 *const ks = keys + ci % kSets * NI * KP;
    __syncthreads();
    fetch_k(next);
    if (Back) {
      keep_state<Saved, DK, TK, TV>(a.states, a.state_powers, (sq.slot + ci) * a.hv + h, a.dvp, dv0, w, x0, y0, s);
    }

    f32x4 kS[TV], o[TV] = {};
    {
      Levels<NS> sum[TV];
      // operands first, products after: one wait for LDS, not one a product
      Frag<NI> fk[DK / 32];
      Frag<NS> fs[DK / 32][TV];
#pragma unroll
      for (int d = 0; d < DK / 32; d++) {
        fk[d] = frag_row<NI>(ks, KP, LDK, 16 * w, 32 * d);
#pragma unroll
        for (int j = 0; j < TV; j++) fs[d][j] = frag_v<NS, TV>(ss, SP, LDV, j, 32 * d);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int d = 0; d < DK / 32; d++) {
        const Frag<NI> fq = frag_of<NI>(keep_head8<A>(rq[d], c, t, 32 * d + 8 * quad, a.dk));
#pragma unroll
        for (int j = 0; j < TV; j++) {
          sum[j].add(fs[d][j], fk[d]);
          o[j] = mma(o[j], first_planes<NO>(fs[d][j]), fq);
        }
      }
#pragma unroll
      for (int j = 0; j < TV; j++) kS[j] = sum[j].sum();
    }
    const RawV<T, TV> v4 = settle_v<A>(rv, dv0 + y0, a.dv);
#pragma unroll
    for (int j = 0; j < TV; j++) {
      f32x4 x;
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const float v = t < c.len && dv0 + y0 + 4 * j + r < a.dv ? v4[4 * j + r] : 0.0f;
        x[r] = beta * (v - gam * kS[j][r]);
      }
      put_four<NS>(xs + t * LDV + y0 + 4 * j, XP, x);
    }
    fetch_qv(next);
    __syncthreads();
    f32x4 u[TV];
    {
      Levels<NS> sum[TV];
      Frag<NS> fx[2][TV];
#pragma unroll
      for (int b = 0; b < 2; b++)
#pragma unroll
        for (int j = 0; j < TV; j++) fx[b][j] = frag_v<NS, TV>(xs, XP, LDV, j, 32 * b);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int b = 0; b < 2; b++)
        if (b == 0 || w >= 2)
#pragma unroll
          for (int j = 0; j < TV; j++) sum[j].add(fx[b][j], ft[b]);
#pragma unroll
      for (int j = 0; j < TV; j++) u[j] = sum[j].sum();
    }
    fetch_t(next);
#pragma unroll
    for (int j = 0; j < TV; j++) {
      put_four<NO>(us + t * LDV + y0 + 4 * j, XP, u[j]);
      put_four<NS>(gs + t * LDV + y0 + 4 * j, XP, last * u[j]);
    }
    if (Back) keep_block<typename M::Kept, TV>(a.us, a.u_scales, (sq.slot + ci) * a.hv + h, a.dvp, dv0, t, quad, y0, u);
    __syncthreads();
    {
      Frag<NS> fg[2][TV];
      Frag<NI> fk[2][TK];
      Frag<NO> fu[2][TV];
#pragma unroll
      for (int b = 0; b < 2; b++) {
#pragma unroll
        for (int j = 0; j < TV; j++) fg[b][j] = frag_v<NS, TV>(gs, XP, LDV, j, 32 * b);
#pragma unroll
        for (int i = 0; i < TK; i++) fk[b][i] = frag_col<NI>(ks, KP, LDK, w * (DK / 4) + 16 * i, 32 * b);
#pragma unroll
        for (int j = 0; j < TV; j++) fu[b][j] = frag_v<NO, TV>(us, XP, LDV, j, 32 * b);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < TK; i++)
#pragma unroll
        for (int j = 0; j < TV; j++) s[i][j] *= end;
#pragma unroll
      for (int j = 0; j < TV; j++) o[j] *= gam;
#pragma unroll
      for (int b = 0; b < 2; b++)
#pragma unroll
        for (int i = 0; i < TK; i++)
#pragma unroll
          for (int j = 0; j < TV; j++) s[i][j] = mma(s[i][j], fg[b][j], fk[b][i]);
      // the next chunk waits for S only: O comes after it
      if (kSets == 2 && ci + 1 < chunks) {
        put_state();
        put_keys(ci + 1);
      }
#pragma unroll
      for (int b = 0; b < 2; b++)
        if (b == 0 || w >= 2)
#pragma unroll
          for (int j = 0; j < TV; j++) o[j] = mma(o[j], fu[b][j], fp[b]);
    }
    fetch_p(next);
#pragma unroll
    for (int j = 0; j < TV; j++) o[j] *= a.scale;
    store_v<A, T, TV>(a.o, c, h, t, dv0 + y0, a.dv, o);
    if (kSets == 1) {
      __syncthreads();
      if (ci + 1 < chunks) {
        put_state();
        put_keys(ci + 1);
      }
    }
  }
  if (a.state_out)
#pragma unroll
    for (int i = 0; i < TK; i++)
#pragma unroll
      for (int j = 0; j < TV; j++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int x = x0 + 16 * i, y = y0 + 4 * j + r;
          if (x < a.dk && dv0 + y < a.dv) a.state_out[state_at + int64_t(x) * a.dv + y] = s[i][j][r];
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
      with_access<typename M::T>(a, [&](auto f) {
        hipLaunchKernelGGL((delta_forward<M, DK, BV, decltype(b)::value, decltype(f)::value>),
                           grid_of((lanes + 7) / 8 * 8 * blocks), dim3(256), 0, stream, a, blocks);
      });
    });
  };
  typedef std::integral_constant<int, 16> C16;
  typedef std::integral_constant<int, 32> C32;
  typedef std::integral_constant<int, 64> C64;
  typedef std::integral_constant<int, 128> C128;
  with_mode(op, [&](auto m) {
    const bool narrow = narrow_blocks(a);
    if (a.dk <= 64) narrow ? launch(m, C64(), C16()) : launch(m, C64(), C32());
    else narrow ? launch(m, C128(), C16()) : launch(m, C128(), C32());
  });
  check_launch("gated delta: forward");
}

}  // namespace op
}  // namespace cchip
