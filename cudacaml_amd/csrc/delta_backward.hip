// Gated delta rule, backward. With dO' = scale dO and E the gradient of the
// state after a chunk, going through the chunks from the last to the first:
//
//   dU = P^T dO' + G (K E),   Y = T^T dU,   dV = beta Y
//   dS = Gam_63 E + Q^T (Gam dO') - K^T (Gam beta Y)       (E of the chunk before)
//
// (delta_reverse). What is left needs only a chunk's own S, U, E and Y, and
// goes over all chunks at once (delta_gradients), with D as in delta.hpp,
// L = strict lower of D (k_t . k_s), M = lower of D dO' U^T, F = Y U^T and
// B = - strict lower of beta D F:
//
//   dQ = Gam (dO' S^T) + M K
//   dK = M^T Q + G (U E^T) - Gam beta (Y S^T) + (B + B^T) K
//   dbeta_t = y_t . v_t - Gam_t (Y S^T)_t . k_t - sum_s F_ts L_ts
//
// and the gradient of c, from which dg_t is the sum over t' >= t in the
// chunk: a pair (t, s) of M (Q K^T) + B (K K^T) adds to c_t and takes from
// c_s, Gam_t q_t . (dO' S^T)_t - Gam_t beta_t k_t . (Y S^T)_t adds to c_t,
// G_s k_s . (U E^T)_s takes from c_s and adds to c_63, as does Gam_63 <S, E>.
// A sum over t' >= t of those is a sum over what spans t: nothing large
// cancels in it.

#include "delta.hpp"

namespace cchip {
namespace op {
namespace {

// The counterpart of delta_forward, laid out like it: BV value columns of a
// head, E in registers, each chunk's rows asked for while the one after it is
// computed. Where they are kept as f32, <S, E> is summed here, with E at hand.
// Bounded as delta_forward is, with one more wait a chunk: 375 us for 4 x 4096
// tokens, 32 bf16 heads of 128, 1.0 GB at 2.7 TB/s.
template <typename M, int DK, int BV, int A>
__global__ __launch_bounds__(256, groups_a_unit<M>(DK, BV)) void delta_reverse(const DeltaArgs a, int blocks) {
  typedef typename M::T T;
  typedef typename M::Saved Saved;
  constexpr int NI = M::NI, NS = M::NS;
  constexpr int LDK = DK + 16, LDV = BV == 16 ? 24 : BV;
  constexpr int KP = 64 * LDK, EP = DK * LDV, XP = 64 * LDV;
  constexpr int TK = DK / 64, TV = BV / 16;
  constexpr bool kDots = sizeof(Saved) == 4;
  typedef Record<M> R;
  __shared__ __align__(16) bf16 ks[NI * KP], qs[NI * KP], es[NS * EP], xs[NS * XP], os[NI * XP], gs[NS * XP];
  bf16 *const zs = es;  // E is done with when Z is made

  const int64_t group = block_index() / (8 * blocks);
  const int rest = int(block_index() - group * 8 * blocks);
  const int64_t lane_id = group * 8 + rest % 8;
  if (lane_id >= a.sequences * a.hv) return;
  const int64_t sid = lane_id / a.hv;
  const int h = int(lane_id - sid * a.hv), hk = h / (a.hv / a.hk), dv0 = rest / 8 * BV;
  const Sequence sq = sequence_of(a, sid);
  const int chunks = int((sq.len + kChunk - 1) / kChunk);

  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, quad = l >> 4, col = l & 15;
  const int x0 = w * (DK / 4) + col, y0 = 4 * TV * quad, t = 16 * w + col;
  const int ot = tid / (BV / 8), od = tid % (BV / 8) * 8;  // this thread's piece of dO, if it has one
  const bool has_o = tid < 64 * (BV / 8);

  f32x4 e[TK][TV];
  const int64_t state_at = lane_id * a.dk * a.dv + dv0;
#pragma unroll
  for (int i = 0; i < TK; i++)
#pragma unroll
    for (int j = 0; j < TV; j++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int x = x0 + 16 * i, y = y0 + 4 * j + r;
        e[i][j][r] = a.dstate_out && x < a.dk && dv0 + y < a.dv ? a.dstate_out[state_at + int64_t(x) * a.dv + y] : 0.0f;
      }

  auto chunk = [&](int i) {
    const int64_t left = sq.len - int64_t(i) * kChunk;
    return Chunk{sq.row, sq.first + int64_t(i) * kChunk, sid, left > kChunk ? kChunk : int(left)};
  };
  auto record = [&](int i) { return a.records + ((sq.slot + i) * a.hv + h) * R::bytes(true); };
  Raw8<T> rk[DK / 32], rq[DK / 32], ro;
  RawV<float, TV> rs[kDots ? TK : 1];
  Frag<NS> tt[2], pt[2];  // rows 16 w .. of T^T and P^T: terms from the diagonal on
  float og, gam, last, beta, end;
  auto fetch = [&](int i) {
    const Chunk c = chunk(i);
#pragma unroll
    for (int j = 0; j < DK / 32; j++) {
      const int at = tid + 256 * j;
      rk[j] = load_head8<A, T>(a.k, c, hk, at / (DK / 8), at % (DK / 8) * 8, a.dk);
      rq[j] = load_head8<A, T>(a.q, c, hk, at / (DK / 8), at % (DK / 8) * 8, a.dk);
    }
    if constexpr (kDots) {
      const char *from = a.states + (((sq.slot + i) * a.hv + h) * a.dvp + dv0 / 32 * 32) * DK * int64_t(sizeof(Saved));
#pragma unroll
      for (int j = 0; j < TK; j++) rs[j] = load_block<float, TV>(from, x0 + 16 * j, dv0 % 32 + y0);
    }
    if (has_o) {
      ro = load_head8<A, T>(a.d_o, c, h, ot, dv0 + od, a.dv);
      og = reinterpret_cast<const float *>(record(i) + R::Decay)[ot];
    }
  };
  auto fetch_end = [&](int i) { end = reinterpret_cast<const float *>(record(i) + R::Decay)[63]; };
  auto fragment = [&](const char *from, int b) {
    return *reinterpret_cast<const bf16x8 *>(from + uint32_t((w * 2 + b) * 1024 + l * 16));
  };
  auto fetch_p = [&](int i) {
#pragma unroll
    for (int b = 0; b < 2; b++)
      if (b == 1 || w < 2)
#pragma unroll
        for (int p = 0; p < NS; p++) pt[b].p[p] = fragment(record(i) + R::Pt + p * 8192, b);
  };
  auto fetch_t = [&](int i) {
#pragma unroll
    for (int b = 0; b < 2; b++)
      if (b == 1 || w < 2)
#pragma unroll
        for (int p = 0; p < NS; p++) tt[b].p[p] = fragment(record(i) + R::Tt + p * 8192, b);
    const float *dec = reinterpret_cast<const float *>(record(i) + R::Decay);
    gam = dec[t];
    last = dec[64 + t];
    beta = dec[128 + t];
  };
  if (chunks > 0) {
    fetch(chunks - 1);
    fetch_p(chunks - 1);
    fetch_t(chunks - 1);
    fetch_end(chunks - 1);
  }
  for (int ci = chunks - 1; ci >= 0; ci--) {
    const Chunk c = chunk(ci);
    const int next = ci ? ci - 1 : 0;
    const int64_t slot_head = (sq.slot + ci) * a.hv + h;
#pragma unroll
    for (int j = 0; j < DK / 32; j++) {
      const int at = tid + 256 * j, kt = at / (DK / 8), d = at % (DK / 8) * 8;
      put_frag<NI>(ks + kt * LDK + d, KP, frag_of<NI>(keep_head8<A>(rk[j], c, kt, d, a.dk)));
      put_frag<NI>(qs + kt * LDK + d, KP, frag_of<NI>(keep_head8<A>(rq[j], c, kt, d, a.dk)));
    }
    if (has_o) {
      const Raw8<T> raw = keep_head8<A>(ro, c, ot, dv0 + od, a.dv);
      put_frag<NI>(os + ot * LDV + od, XP, frag_of<NI>(raw));
      if (sizeof(Saved) < 4) {  // the largest of a token's in these columns, for delta_gradients
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(float(raw.x[i])));
        m = fmaxf(m, CCHIP_QUAD(m, 0xB1));
        if (TV == 2) m = fmaxf(m, CCHIP_QUAD(m, 0x4E));
        if (od < 8 * TV) a.o_powers[(slot_head * (a.dvp / 16) + dv0 / 16 + od / 8) * kChunk + ot] = uint8_t(half_exponent(m));
      }
      const float f = a.scale * og;
      Raw8<float> up;
#pragma unroll
      for (int i = 0; i < 8; i++) up.x[i] = f * float(raw.x[i]);
      put_frag<NS>(gs + ot * LDV + od, XP, frag_of<NS>(up));
    }
#pragma unroll
    for (int i = 0; i < TK; i++)
#pragma unroll
      for (int j = 0; j < TV; j++) put_four<NS>(es + (x0 + 16 * i) * LDV + y0 + 4 * j, EP, e[i][j]);
    if constexpr (kDots) {
      float dot = 0.0f;
#pragma unroll
      for (int i = 0; i < TK; i++)
#pragma unroll
        for (int j = 0; j < 4 * TV; j++) dot += rs[i][j] * e[i][j / 4][j % 4];
      dot = sum64(dot);
      if (l == 0) {
        float *dots = a.dots + (slot_head * (a.dvp / 16) + dv0 / 16) * 4;
        dots[w] = dot;
        if (TV == 2) dots[4 + w] = 0.0f;
      }
    }
    __syncthreads();
    fetch(next);
    keep_state<Saved, DK, TK, TV>(a.grads, a.grad_powers, slot_head, a.dvp, dv0, w, x0, y0, e);

    Levels<NS> ke[TV], po[TV];
    {
      // operands first, products after: one wait for LDS, not one a product
      Frag<NI> fk[DK / 32], fo[2][TV];
      Frag<NS> fe[DK / 32][TV];
#pragma unroll
      for (int d = 0; d < DK / 32; d++) {
        fk[d] = frag_row<NI>(ks, KP, LDK, 16 * w, 32 * d);
#pragma unroll
        for (int j = 0; j < TV; j++) fe[d][j] = frag_v<NS, TV>(es, EP, LDV, j, 32 * d);
      }
#pragma unroll
      for (int b = 0; b < 2; b++)
#pragma unroll
        for (int j = 0; j < TV; j++) fo[b][j] = frag_v<NI, TV>(os, XP, LDV, j, 32 * b);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int d = 0; d < DK / 32; d++)
#pragma unroll
        for (int j = 0; j < TV; j++) ke[j].add(fe[d][j], fk[d]);
#pragma unroll
      for (int b = 0; b < 2; b++)
        if (b == 1 || w < 2)
#pragma unroll
          for (int j = 0; j < TV; j++) po[j].add(fo[b][j], pt[b]);
    }
    fetch_p(next);
#pragma unroll
    for (int j = 0; j < TV; j++) {
      put_four<NS>(xs + t * LDV + y0 + 4 * j, XP, a.scale * po[j].sum() + last * ke[j].sum());
    }
    __syncthreads();
    f32x4 y[TV];
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
        if (b == 1 || w < 2)
#pragma unroll
          for (int j = 0; j < TV; j++) sum[j].add(fx[b][j], tt[b]);
#pragma unroll
      for (int j = 0; j < TV; j++) y[j] = sum[j].sum();
    }
    keep_block<typename M::Kept, TV>(a.ys, a.y_scales, slot_head, a.dvp, dv0, t, quad, y0, y);
#pragma unroll
    for (int j = 0; j < TV; j++) {
      put_four<NS>(zs + t * LDV + y0 + 4 * j, EP, (-gam * beta) * y[j]);
      y[j] *= beta;
    }
    store_v<A, T, TV>(a.gv, c, h, t, dv0 + y0, a.dv, y);
    fetch_t(next);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TK; i++)
#pragma unroll
      for (int j = 0; j < TV; j++) e[i][j] *= end;
    fetch_end(next);
#pragma unroll
    for (int b = 0; b < 2; b++) {
      Frag<NS> fg[TV], fz[TV];
      Frag<NI> fq[TK], fk[TK];
#pragma unroll
      for (int j = 0; j < TV; j++) {
        fg[j] = frag_v<NS, TV>(gs, XP, LDV, j, 32 * b);
        fz[j] = frag_v<NS, TV>(zs, EP, LDV, j, 32 * b);
      }
#pragma unroll
      for (int i = 0; i < TK; i++) {
        fq[i] = frag_col<NI>(qs, KP, LDK, w * (DK / 4) + 16 * i, 32 * b);
        fk[i] = frag_col<NI>(ks, KP, LDK, w * (DK / 4) + 16 * i, 32 * b);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < TK; i++)
#pragma unroll
        for (int j = 0; j < TV; j++) e[i][j] = mma(e[i][j], fg[j], fq[i]);
#pragma unroll
      for (int i = 0; i < TK; i++)
#pragma unroll
        for (int j = 0; j < TV; j++) e[i][j] = mma(e[i][j], fz[j], fk[i]);
    }
    __syncthreads();
  }
  if (a.dstate)
#pragma unroll
    for (int i = 0; i < TK; i++)
#pragma unroll
      for (int j = 0; j < TV; j++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int x = x0 + 16 * i, y = y0 + 4 * j + r;
          if (x < a.dk && dv0 + y < a.dv) a.dstate[state_at + int64_t(x) * a.dv + y] = e[i][j][r];
        }
}

// Eight values in f16 into LDS, times 2^n for n <= 0.
__device__ __forceinline__ void put_lower(bf16 *to, const Raw8<f16> &x, int n) {
  const f16 down = f16(n < -126 ? 0.0f : power(uint32_t(127 + n)));
  *reinterpret_cast<f16x8 *>(to) = __builtin_bit_cast(f16x8, x) * down;
}
template <typename T>
__device__ __forceinline__ void put_lower(bf16 *, const Raw8<T> &, int) {}

// The operand of 16 rows from row0 on of f16 rows in LDS, and a product of two.
__device__ __forceinline__ f16x8 half_row(const bf16 *m, int ld, int row0) {
  const int l = threadIdx.x & 63;
  return *reinterpret_cast<const f16x8 *>(m + (row0 + (l & 15)) * ld + (l >> 4) * 8);
}
__device__ __forceinline__ f32x4 mma_half(f32x4 c, f16x8 a, f16x8 b) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// A workgroup of eight waves a chunk and key head, its value heads one after
// another (so dQ and dK of a shared head are summed in registers, in an order
// that is always the same). Products are taken transposed, as in the forward
// pass: wave w has tokens 16 (w % 4) .. of each and part w / 4 of the rest,
// and a lane one token. S, E, U, Y and dO pass through LDS 32 value columns
// at a time, the next 32 being read while the products of these are made.
// Where they are f16 (kHalf, dO made so), the values of a token or of a block
// of rows of S and E are brought to the largest power of two that they have in
// any columns, so that products add up over all columns and are scaled once
// for a head: 525 us for 256 chunks of 32 bf16 heads of 128, 1.3 GB at 2.5
// TB/s, where the same accuracy from pairs of bf16 planes took 555 and single
// ones 480. Four parts and 16 waves would hide more but do not fit in 128
// registers (790 us with single planes). One workgroup a unit is what
// registers allow, so its waits for LDS and memory are not covered by
// another's work.
template <typename M, int DK, int A>
__global__ __launch_bounds__(512, 2) void delta_gradients(const DeltaArgs a) {
  typedef typename M::T T;
  typedef typename M::Saved Saved;
  typedef typename M::Kept Kept;
  constexpr int NI = M::NI, NB = M::NB, NO = M::NO, P = 2, kThreads = 256 * P;
  constexpr int LDK = DK + 16, KP = 64 * LDK, LDS = 40, SP = DK * LDS, UP = 64 * LDS, LDM = 72, MP = 64 * LDM;
  constexpr int JK = DK / 16 / P, JS = 4 / P;  // 16-wide tiles of a part: of a key, of the tokens
  constexpr bool kAll = NB < 3;               // everything in LDS at a time; else E after S, and Y and dO not
  constexpr bool kHalf = sizeof(Saved) == 2;  // slices as f16 with powers of two, on the f16 matrix instruction
  constexpr int PB = kHalf ? 1 : NB, PO = kHalf ? 1 : NO, PI = kHalf ? 1 : NI;  // planes of a slice
  typedef Record<M> R;
  constexpr int kSlices = (kAll ? 2 : 1) * PB * SP + PO * UP + (kAll ? (PO + PI) * UP : 0), kMs = (kAll ? 2 : 1) * NB * MP;
  __shared__ __align__(16) bf16 ks[NI * KP], qs[NI * KP], slice[kSlices > kMs ? kSlices : kMs];
  __shared__ double cs[64];
  __shared__ __align__(16) float down[4][64];
  __shared__ float row_c[P][64], row_b[P][64], row_y[64], total[4 * P];
  // kHalf: the powers that hold in all columns of a head, of the tokens and of the blocks of DK / 4 rows of S and E
  __shared__ __align__(16) uint32_t u_top[64], y_top[64], o_top[64], s_top[8];
  bf16 *const us = slice, *const ss = slice + PO * UP, *const es = kAll ? ss + PB * SP : ss;
  bf16 *const yl = es + PB * SP, *const ol = yl + PO * UP;  // Y and dO if kAll
  bf16 *const ms = slice, *const bs = kAll ? slice + NB * MP : slice;

  const int64_t slot = block_index() / a.hk;
  if (slot >= a.slots) return;
  const int hk = int(block_index() - slot * a.hk), per = a.hv / a.hk;
  const Chunk c = chunk_of(a, slot);
  if (c.len == 0) return;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, quad = l >> 4, col = l & 15;
  const int wr = w & 3, part = w >> 2;
  const int t = 16 * wr + col;                    // this lane's token
  const int x0 = 16 * JK * part + 4 * quad;       // its part of a key: x0 + 16 j + r
  const int s0 = 16 * JS * part + 4 * quad;       // and of the tokens before it: s0 + 16 j + r

  {
    constexpr int kRows = 64 * (DK / 8) / kThreads > 0 ? 64 * (DK / 8) / kThreads : 1;
    const bool has = tid < 64 * (DK / 8);
    Raw8<T> rk[kRows], rq[kRows];
#pragma unroll
    for (int j = 0; j < kRows; j++)
      if (has) {
        const int at = tid + kThreads * j;
        rk[j] = load_head8<A, T>(a.k, c, hk, at / (DK / 8), at % (DK / 8) * 8, a.dk);
        rq[j] = load_head8<A, T>(a.q, c, hk, at / (DK / 8), at % (DK / 8) * 8, a.dk);
      }
#pragma unroll
    for (int j = 0; j < kRows; j++)
      if (has) {
        const int at = tid + kThreads * j, kt = at / (DK / 8), d = at % (DK / 8) * 8;
        put_frag<NI>(ks + kt * LDK + d, KP, frag_of<NI>(keep_head8<A>(rk[j], c, kt, d, a.dk)));
        put_frag<NI>(qs + kt * LDK + d, KP, frag_of<NI>(keep_head8<A>(rq[j], c, kt, d, a.dk)));
      }
  }
  // four elements of this lane's row of K or Q as their planes add up
  auto value4 = [&](const bf16 *m, int d) {
    f32x4 x = {};
#pragma unroll
    for (int p = NI - 1; p >= 0; p--) {
      const bf16x4 v = *reinterpret_cast<const bf16x4 *>(m + p * KP + t * LDK + d);
#pragma unroll
      for (int r = 0; r < 4; r++) x[r] += float(v[r]);
    }
    return x;
  };
  // this thread's pieces of a slice, 8 columns from sv on: row sx of S and E,
  // and row ux of U and dO or, in the second half of the waves, of Y and v
  const int sv = tid % 4 * 8, sx = tid / 4, ux = (tid & 255) / 4;
  const bool has_s = sx < DK, second = w >= 4;

  f32x4 dq[JK] = {}, dk[JK] = {};
  for (int h = hk * per; h < (hk + 1) * per; h++) {
    const int64_t slot_head = slot * a.hv + h;
    const float *dec = reinterpret_cast<const float *>(a.records + slot_head * R::bytes(true) + R::Decay);
    const char *S = a.states + slot_head * DK * a.dvp * int64_t(sizeof(Saved));
    const char *E = a.grads + slot_head * DK * a.dvp * int64_t(sizeof(Saved));
    const char *U = a.us + slot_head * kChunk * a.dvp * int64_t(sizeof(Kept));
    const char *Y = a.ys + slot_head * kChunk * a.dvp * int64_t(sizeof(Kept));
    const float *u_scales = a.u_scales + slot_head * (kChunk / 16) * a.dvp, *y_scales = a.y_scales + slot_head * (kChunk / 16) * a.dvp;

    const int groups = a.dvp / 16;
    const uint8_t *s_powers = a.state_powers + slot_head * groups * 4, *e_powers = a.grad_powers + slot_head * groups * 4;
    const uint8_t *o_powers = a.o_powers + slot_head * groups * kChunk;

    Raw8<Saved> rs, re;
    Raw8<Kept> ru;
    Raw8<float> ry;
    Raw8<T> ro, rv;
    float scale = 1.0f;
    uint8_t ps = 0, pe = 0;  // S and E's exponents
    auto fetch = [&](int v0) {
      if (has_s) {
        rs = load_block8<Saved>(S, uint32_t(v0 * DK + sx * 32 + sv));
        re = load_block8<Saved>(E, uint32_t(v0 * DK + sx * 32 + sv));
        if (kHalf) {
          ps = s_powers[(v0 + sv) / 16 * 4 + sx / (DK / 4)];
          pe = e_powers[(v0 + sv) / 16 * 4 + sx / (DK / 4)];
        }
      }
      if (kAll) {
        ru = load_block8<Kept>(second ? Y : U, uint32_t(v0 * 64 + ux * 32 + sv));
        if (sizeof(Kept) < 4) scale = (second ? y_scales : u_scales)[(v0 + sv) / 16 * kChunk + ux];
        ro = load_head8<A, T>(second ? a.v : a.d_o, c, h, ux, v0 + sv, a.dv);
      } else {
        if (!second) ru = load_block8<Kept>(U, uint32_t(v0 * 64 + ux * 32 + sv));
        ry = load_block8<float>(Y, uint32_t(v0 * 64 + t * 32 + 8 * quad));
        ro = load_head8<A, T>(a.d_o, c, h, t, v0 + 8 * quad, a.dv);
        rv = load_head8<A, T>(a.v, c, h, t, v0 + 8 * quad, a.dv);
      }
    };
    fetch(0);
    double run = 0.0;  // the running sum of g, as delta_chunk makes it
    if (w == 0) {
      const float g = l < c.len ? float(*at<T>(a.g, c.row, c.first + l, h)) : 0.0f;
      run = g < -1000.0f ? -1000.0 : double(g);
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const double up = __shfl_up(run, d, 64);
        if (l >= d) run += up;
      }
    }
    if (kHalf && w >= 4) {
      // eight groups' at a time, so that they are waited for at once
      auto largest = [&](auto of) {
        uint32_t top = 1;
        for (int g = 0; g < groups; g += 8) {
          uint32_t x[8];
#pragma unroll
          for (int i = 0; i < 8; i++) x[i] = of(min(g + i, groups - 1));
#pragma unroll
          for (int i = 0; i < 8; i++) top = max(top, x[i]);
        }
        return top;
      };
      if (w < 6) {
        const float *scales = (w == 4 ? u_scales : y_scales) + l;
        (w == 4 ? u_top : y_top)[l] = largest([&](int g) { return exponent(scales[g * kChunk]); });
      } else if (w == 6) {
        o_top[l] = largest([&](int g) { return uint32_t(o_powers[g * kChunk + l]); });
      } else if (l < 8) {
        const uint8_t *powers = l < 4 ? s_powers + l : e_powers + l - 4;
        s_top[l] = largest([&](int g) { return uint32_t(powers[g * 4]); });
      }
    }
    __syncthreads();  // the head before is done with LDS
    if (w == 0) cs[l] = run;

    f32x4 os[JK] = {}, ys[JK] = {}, ue[JK] = {}, ou[JS] = {}, yu[JS] = {};
    float yv = 0.0f, se = 0.0f;  // yv: of row ux (kAll) or t, this thread's columns
    if (!kHalf)
      for (int i = tid; i < a.dvp / 4; i += kThreads) se += a.dots[slot_head * (a.dvp / 4) + i];
    for (int v0 = 0; v0 < a.dvp; v0 += 32) {
      Frag<NI> fo;
      Frag<NO> fy;
      const Raw8<Saved> late = re;
      if constexpr (kHalf) {
        if (has_s) {
          const int at = sx / (DK / 4);
          float dot = 0.0f;
#pragma unroll
          for (int i = 0; i < 8; i++) dot += float(rs.x[i]) * float(re.x[i]);
          se += ldexpf(dot, int(ps) + int(pe) - 2 * kHalfZero);
          put_lower(ss + sx * LDS + sv, rs, int(ps) - int(s_top[at]));
          put_lower(es + sx * LDS + sv, re, int(pe) - int(s_top[4 + at]));
        }
        put_lower((second ? yl : us) + ux * LDS + sv, ru, int(exponent(scale)) - int((second ? y_top : u_top)[ux]));
        const Raw8<T> x = keep_head8<A>(ro, c, ux, v0 + sv, a.dv);
        if (second) {
          const Raw8<float> u = kept8(ru, scale);
#pragma unroll
          for (int i = 0; i < 8; i++) yv += u.x[i] * float(x.x[i]);
        } else {
          const float down = half_down(o_top[ux]);
          f16x8 o;
#pragma unroll
          for (int i = 0; i < 8; i++) o[i] = f16(float(x.x[i]) * down);
          *reinterpret_cast<f16x8 *>(ol + ux * LDS + sv) = o;
        }
      } else {
        if (has_s) {
          put_frag<NB>(ss + sx * LDS + sv, SP, frag_of<NB>(rs));
          if (kAll) put_frag<NB>(es + sx * LDS + sv, SP, frag_of<NB>(re));
        }
        if (kAll) {
          put_frag<NO>((second ? yl : us) + ux * LDS + sv, UP, frag_of<NO>(ru));
          const Raw8<T> x = keep_head8<A>(ro, c, ux, v0 + sv, a.dv);
          if (second) {
#pragma unroll
            for (int i = 0; i < 8; i++) yv += ru.x[i] * float(x.x[i]);
          } else {
            put_frag<NI>(ol + ux * LDS + sv, UP, frag_of<NI>(x));
          }
        } else {
          if (!second) put_frag<NO>(us + ux * LDS + sv, UP, frag_of<NO>(ru));
          fo = frag_of<NI>(keep_head8<A>(ro, c, t, v0 + 8 * quad, a.dv));
          fy = frag_of<NO>(ry);
          const Raw8<T> v = keep_head8<A>(rv, c, t, v0 + 8 * quad, a.dv);
#pragma unroll
          for (int i = 0; i < 8; i++) yv += ry.x[i] * float(v.x[i]);
        }
      }
      __syncthreads();
      if (v0 + 32 < a.dvp) fetch(v0 + 32);
      if constexpr (kHalf) {
        const f16x8 ho = half_row(ol, LDS, 16 * wr), hy = half_row(yl, LDS, 16 * wr), hu = half_row(us, LDS, 16 * wr);
#pragma unroll
        for (int j = 0; j < JK; j++) {
          const int x = 16 * (JK * part + j);
          const f16x8 hs = half_row(ss, LDS, x);
          os[j] = mma_half(os[j], hs, ho);
          ys[j] = mma_half(ys[j], hs, hy);
          ue[j] = mma_half(ue[j], half_row(es, LDS, x), hu);
        }
#pragma unroll
        for (int j = 0; j < JS; j++)
          if (JS * part + j <= wr) {
            const f16x8 h = half_row(us, LDS, 16 * (JS * part + j));
            ou[j] = mma_half(ou[j], h, ho);
            yu[j] = mma_half(yu[j], h, hy);
          }
        __syncthreads();
      } else {
        if (kAll) {
          fo = frag_row<NI>(ol, UP, LDS, 16 * wr, 0);
          fy = frag_row<NO>(yl, UP, LDS, 16 * wr, 0);
        }
        const Frag<NO> fu = frag_row<NO>(us, UP, LDS, 16 * wr, 0);
#pragma unroll
        for (int j = 0; j < JK; j++) {
          const int x = 16 * (JK * part + j);
          const Frag<NB> fs = frag_row<NB>(ss, SP, LDS, x, 0);
          os[j] = mma(os[j], fs, fo);
          ys[j] = mma(ys[j], fs, fy);
          if (kAll) ue[j] = mma(ue[j], frag_row<NB>(es, SP, LDS, x, 0), fu);
        }
#pragma unroll
        for (int j = 0; j < JS; j++)
          if (JS * part + j <= wr) {
            const Frag<NO> f = frag_row<NO>(us, UP, LDS, 16 * (JS * part + j), 0);
            ou[j] = mma(ou[j], f, fo);
            yu[j] = mma(yu[j], f, fy);
          }
        __syncthreads();
        if (!kAll) {
          if (has_s) put_frag<NB>(es + sx * LDS + sv, SP, frag_of<NB>(late));
          __syncthreads();
#pragma unroll
          for (int j = 0; j < JK; j++) ue[j] = mma(ue[j], frag_row<NB>(es, SP, LDS, 16 * (JK * part + j), 0), fu);
          __syncthreads();
        }
      }
    }
    if constexpr (kHalf) {
      const int u = int(u_top[t]) - 127, y = int(y_top[t]) - 127, o = int(o_top[t]) - kHalfZero;
#pragma unroll
      for (int j = 0; j < JK; j++) {
        const int at = 16 * (JK * part + j) / (DK / 4);
        const int sn = int(s_top[at]) - kHalfZero, en = int(s_top[4 + at]) - kHalfZero;
#pragma unroll
        for (int r = 0; r < 4; r++) {
          os[j][r] = ldexpf(os[j][r], sn + o);
          ys[j][r] = ldexpf(ys[j][r], sn + y);
          ue[j][r] = ldexpf(ue[j][r], en + u);
        }
      }
#pragma unroll
      for (int j = 0; j < JS; j++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int n = int(u_top[s0 + 16 * j + r]) - 127;
          ou[j][r] = ldexpf(ou[j][r], n + o);
          yu[j][r] = ldexpf(yu[j][r], n + y);
        }
    }
    if (kAll) {
      yv += __shfl_xor(yv, 1, 64);
      yv += __shfl_xor(yv, 2, 64);
      if (second && tid % 4 == 0) row_y[ux] = yv;
    } else {
      yv = sum_rows(yv);
      if (part == 0 && quad == 0) row_y[t] = yv;
    }

    const float gam = dec[t], last = dec[64 + t], beta = dec[128 + t];
    float dc = 0.0f, db = 0.0f, end = 0.0f;
#pragma unroll
    for (int j = 0; j < JK; j++) {
      const f32x4 kv = value4(ks, x0 + 16 * j), qv = value4(qs, x0 + 16 * j);
      const f32x4 o = (a.scale * gam) * os[j], y = gam * ys[j], u = last * ue[j];
      dq[j] += o;
      dk[j] += u - beta * y;
#pragma unroll
      for (int r = 0; r < 4; r++) {
        dc += qv[r] * o[r] - kv[r] * (beta * y[r] + u[r]);
        db -= kv[r] * y[r];
        end += kv[r] * u[r];
      }
    }
    f32x4 kk[JS] = {}, qk[JS] = {};
#pragma unroll
    for (int d = 0; d < DK; d += 32) {
      const Frag<NI> fk = frag_row<NI>(ks, KP, LDK, 16 * wr, d), fq = frag_row<NI>(qs, KP, LDK, 16 * wr, d);
#pragma unroll
      for (int j = 0; j < JS; j++)
        if (JS * part + j <= wr) {
          const Frag<NI> fs = frag_row<NI>(ks, KP, LDK, 16 * (JS * part + j), d);
          kk[j] = mma(kk[j], fs, fk);
          qk[j] = mma(qk[j], fs, fq);
        }
    }
    f32x4 b[JS];
#pragma unroll
    for (int j = 0; j < JS; j++) {
      f32x4 m, across;
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int s = s0 + 16 * j + r;
        const float d = s <= t ? expf(float(cs[t] - cs[s])) : 0.0f;
        m[r] = s <= t ? a.scale * d * ou[j][r] : 0.0f;
        b[j][r] = s < t ? -beta * d * yu[j][r] : 0.0f;
        const float pair = m[r] * qk[j][r] + b[j][r] * kk[j][r];
        dc += pair;
        across[r] = sum16(pair);
        db -= s < t ? yu[j][r] * d * kk[j][r] : 0.0f;
      }
      if (col == 0) *reinterpret_cast<f32x4 *>(&down[wr][s0 + 16 * j]) = across;
      put_four<NB>(ms + t * LDM + s0 + 16 * j, MP, m);
      if (kAll) put_four<NB>(bs + t * LDM + s0 + 16 * j, MP, b[j]);
    }
    dc = sum_rows(dc);
    db = sum_rows(db);
    if (quad == 0) {
      row_c[part][t] = dc;
      row_b[part][t] = db;
    }
    end = sum64(end + se * dec[63]);
    if (l == 0) total[w] = end;
    __syncthreads();
    if (w == 0) {
      float x = -(down[0][l] + down[1][l] + down[2][l] + down[3][l]), y = row_y[l], all = 0.0f;
#pragma unroll
      for (int p = 0; p < P; p++) {
        x += row_c[p][l];
        y += row_b[p][l];
      }
#pragma unroll
      for (int i = 0; i < 4 * P; i++) all += total[i];
      if (l == 63) x += all;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const float up = __shfl_down(x, d, 64);
        if (l + d < 64) x += up;
      }
      if (l < c.len) {
        *out_at<T>(a.gg, c.row, c.first + l, h) = T(x);
        *out_at<T>(a.gbeta, c.row, c.first + l, h) = T(y);
      }
    }
#pragma unroll
    for (int t0 = 0; t0 < 64; t0 += 32) {
      if (t0 == 0 || wr >= 2) {  // M ends at the diagonal
        const Frag<NB> f = frag_row<NB>(ms, MP, LDM, 16 * wr, t0);
#pragma unroll
        for (int j = 0; j < JK; j++) dq[j] = mma(dq[j], frag_col<NI>(ks, KP, LDK, 16 * (JK * part + j), t0), f);
      }
      if (t0 != 0 || wr < 2) {
        const Frag<NB> f = frag_col<NB>(ms, MP, LDM, 16 * wr, t0);
#pragma unroll
        for (int j = 0; j < JK; j++) dk[j] = mma(dk[j], frag_col<NI>(qs, KP, LDK, 16 * (JK * part + j), t0), f);
      }
    }
    if (!kAll) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < JS; j++) put_four<NB>(bs + t * LDM + s0 + 16 * j, MP, b[j]);
      __syncthreads();
    }
#pragma unroll
    for (int t0 = 0; t0 < 64; t0 += 32) {
      const Frag<NB> fb = frag_row<NB>(bs, MP, LDM, 16 * wr, t0), ft = frag_col<NB>(bs, MP, LDM, 16 * wr, t0);
#pragma unroll
      for (int j = 0; j < JK; j++) {
        const Frag<NI> fk = frag_col<NI>(ks, KP, LDK, 16 * (JK * part + j), t0);
        if (t0 == 0 || wr >= 2) dk[j] = mma(dk[j], fk, fb);
        if (t0 != 0 || wr < 2) dk[j] = mma(dk[j], fk, ft);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < JK; j++) {
    store_head4<A, T>(a.gq, c, hk, t, x0 + 16 * j, a.dk, dq[j]);
    store_head4<A, T>(a.gk, c, hk, t, x0 + 16 * j, a.dk, dk[j]);
  }
}

}  // namespace

void delta_backward_launch(const cchip_gated_delta &op, const DeltaArgs &a, hipStream_t stream) {
  const int64_t lanes = a.sequences * a.hv;
  typedef std::integral_constant<int, 16> C16;
  typedef std::integral_constant<int, 32> C32;
  typedef std::integral_constant<int, 64> C64;
  typedef std::integral_constant<int, 128> C128;
  auto launch = [&](auto m, auto dk, auto bv) {
    typedef decltype(m) M;
    constexpr int DK = decltype(dk)::value, BV = decltype(bv)::value;
    const int blocks = a.dvp / BV;  // what pads a head is written too
    with_access<typename M::T>(a, [&](auto f) {
      constexpr int F = decltype(f)::value;
      hipLaunchKernelGGL((delta_reverse<M, DK, BV, F>), grid_of((lanes + 7) / 8 * 8 * blocks), dim3(256), 0, stream,
                         a, blocks);
      if (a.slots) hipLaunchKernelGGL((delta_gradients<M, DK, F>), grid_of(a.slots * a.hk), dim3(512), 0, stream, a);
    });
  };
  with_mode(op, [&](auto m) {
    constexpr bool wide = decltype(m)::NI < 3;  // three planes of K and Q leave no LDS for 32 columns
    if constexpr (wide) {
      if (!narrow_blocks(a)) {
        if (a.dk <= 64) launch(m, C64(), C32());
        else launch(m, C128(), C32());
        return;
      }
    }
    if (a.dk <= 64) launch(m, C64(), C16());
    else launch(m, C128(), C16());
  });
  check_launch("gated delta: backward");
}

}  // namespace op
}  // namespace cchip
