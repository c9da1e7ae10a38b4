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

// The counterpart of delta_forward: BV value columns of a head, E in
// registers, each chunk's rows asked for while the one after it is computed.
template <typename M, int DK, int BV, bool Fast>
__global__ __launch_bounds__(256, 2) void delta_reverse(const DeltaArgs a, int blocks) {
  typedef typename M::T T;
  typedef typename M::Saved Saved;
  constexpr int NI = M::NI, NS = M::NS;
  constexpr int LDK = DK + 8, LDT = 72, LDV = BV + 8;
  constexpr int KP = 64 * LDK, SP = BV * LDK, XP = BV * LDT, VP = 64 * LDV;
  constexpr int TK = DK / 64, TV = BV / 16;
  typedef Record<M> R;
  __shared__ __align__(16) bf16 ks[NI * KP], qs[NI * KP], et[NS * SP], xt[NS * XP], os[NI * VP], gs[NS * VP];
  static_assert(SP >= XP || DK < 128, "Z does not fit where E was");
  __shared__ __align__(16) bf16 own[DK < 128 ? NS * XP : 8];
  bf16 *const zt = DK < 128 ? own : et;  // E is done with when Z is made

  const int64_t group = blockIdx.x / (8 * blocks);
  const int rest = int(blockIdx.x - group * 8 * blocks);
  const int64_t lane_id = group * 8 + rest % 8;
  if (lane_id >= a.sequences * a.hv) return;
  const int64_t sid = lane_id / a.hv;
  const int h = int(lane_id - sid * a.hv), hk = h / (a.hv / a.hk), dv0 = rest / 8 * BV;
  const Sequence sq = sequence_of(a, sid);
  const int chunks = int((sq.len + kChunk - 1) / kChunk);

  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, quad = l >> 4, col = l & 15;
  const int row0 = w * (DK / 4) + quad * 4;
  const int ot = tid / (BV / 8), od = tid % (BV / 8) * 8;  // this thread's piece of dO, if it has one
  const bool has_o = tid < 64 * (BV / 8);

  f32x4 e[TK][TV];
  const int64_t state_at = lane_id * a.dk * a.dv;
#pragma unroll
  for (int i = 0; i < TK; i++)
#pragma unroll
    for (int j = 0; j < TV; j++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int x = row0 + 16 * i + r, y = dv0 + 16 * j + col;
        e[i][j][r] = a.dstate_out && x < a.dk && y < a.dv ? a.dstate_out[state_at + int64_t(x) * a.dv + y] : 0.0f;
      }

  auto chunk = [&](int i) {
    const int64_t left = sq.len - int64_t(i) * kChunk;
    return Chunk{sq.row, sq.first + int64_t(i) * kChunk, sid, left > kChunk ? kChunk : int(left)};
  };
  auto record = [&](int i) { return a.records + ((sq.slot + i) * a.hv + h) * R::bytes(true); };
  Raw8<T> rk[DK / 32], rq[DK / 32], ro;
  Frag<NS> tt[2], pt[2];  // rows 16 w .. of T^T and P^T: terms from the diagonal on
  float og;
  auto fetch = [&](int i) {
    const Chunk c = chunk(i);
#pragma unroll
    for (int j = 0; j < DK / 32; j++) {
      const int at = tid + 256 * j;
      rk[j] = load_head8<Fast, T>(a.k, c, hk, at / (DK / 8), at % (DK / 8) * 8, a.dk);
      rq[j] = load_head8<Fast, T>(a.q, c, hk, at / (DK / 8), at % (DK / 8) * 8, a.dk);
    }
    if (has_o) {
      ro = load_head8<Fast, T>(a.d_o, c, h, ot, dv0 + od, a.dv);
      og = reinterpret_cast<const float *>(record(i) + R::Decay)[ot];
    }
  };
  auto fetch_p = [&](int i) {
#pragma unroll
    for (int b = 0; b < 2; b++)
      if (b == 1 || w < 2)
#pragma unroll
        for (int p = 0; p < NS; p++)
          pt[b].p[p] = reinterpret_cast<const bf16x8 *>(record(i) + R::Pt + p * 8192)[(w * 2 + b) * 64 + l];
  };
  auto fetch_t = [&](int i) {
#pragma unroll
    for (int b = 0; b < 2; b++)
      if (b == 1 || w < 2)
#pragma unroll
        for (int p = 0; p < NS; p++)
          tt[b].p[p] = reinterpret_cast<const bf16x8 *>(record(i) + R::Tt + p * 8192)[(w * 2 + b) * 64 + l];
  };
  if (chunks > 0) {
    fetch(chunks - 1);
    fetch_p(chunks - 1);
    fetch_t(chunks - 1);
  }
  for (int ci = chunks - 1; ci >= 0; ci--) {
    const Chunk c = chunk(ci);
    const int next = ci ? ci - 1 : 0;
    const int64_t slot_head = (sq.slot + ci) * a.hv + h;
    const float *dec = reinterpret_cast<const float *>(record(ci) + R::Decay);
#pragma unroll
    for (int j = 0; j < DK / 32; j++) {
      const int at = tid + 256 * j, t = at / (DK / 8), d = at % (DK / 8) * 8;
      put_frag<NI>(ks + t * LDK + d, KP, frag_of<NI>(keep_head8<Fast>(rk[j], c, t, d, a.dk)));
      put_frag<NI>(qs + t * LDK + d, KP, frag_of<NI>(keep_head8<Fast>(rq[j], c, t, d, a.dk)));
    }
    if (has_o) {
      const Raw8<T> raw = keep_head8<Fast>(ro, c, ot, dv0 + od, a.dv);
      put_frag<NI>(os + ot * LDV + od, VP, frag_of<NI>(raw));
      const float f = a.scale * og;
      Raw8<float> up;
#pragma unroll
      for (int i = 0; i < 8; i++) up.x[i] = f * float(raw.x[i]);
      put_frag<NS>(gs + ot * LDV + od, VP, frag_of<NS>(up));
    }
#pragma unroll
    for (int i = 0; i < TK; i++)
#pragma unroll
      for (int j = 0; j < TV; j++) put_column<NS>(et + (16 * j + col) * LDK + row0 + 16 * i, SP, e[i][j]);
    float gam[4], last[4], beta[4];
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int t = 16 * w + 4 * quad + r;
      gam[r] = dec[t];
      last[r] = dec[64 + t];
      beta[r] = dec[128 + t];
    }
    const float end = dec[63];
    __syncthreads();
    fetch(next);
    Saved *es = reinterpret_cast<Saved *>(a.grads) + slot_head * DK * a.dvp + dv0;
#pragma unroll
    for (int i = 0; i < TK; i++)
#pragma unroll
      for (int j = 0; j < TV; j++)
#pragma unroll
        for (int r = 0; r < 4; r++) es[(row0 + 16 * i + r) * a.dvp + 16 * j + col] = Saved(e[i][j][r]);

    f32x4 ke[TV] = {}, du[TV] = {};
#pragma unroll
    for (int d = 0; d < DK; d += 32) {
      const Frag<NI> fk = frag_row<NI>(ks, KP, LDK, 16 * w, d);
#pragma unroll
      for (int j = 0; j < TV; j++) ke[j] = mma(ke[j], fk, frag_row<NS>(et, SP, LDK, 16 * j, d));
    }
#pragma unroll
    for (int b = 0; b < 2; b++)
      if (b == 1 || w < 2)
#pragma unroll
        for (int j = 0; j < TV; j++) du[j] = mma(du[j], pt[b], frag_col<NI>(os, VP, LDV, 16 * j, 32 * b));
    fetch_p(next);
#pragma unroll
    for (int j = 0; j < TV; j++) {
#pragma unroll
      for (int r = 0; r < 4; r++) du[j][r] = a.scale * du[j][r] + last[r] * ke[j][r];
      put_column<NS>(xt + (16 * j + col) * LDT + 16 * w + 4 * quad, XP, du[j]);
    }
    __syncthreads();
    f32x4 y[TV] = {};
#pragma unroll
    for (int b = 0; b < 2; b++)
      if (b == 1 || w < 2)
#pragma unroll
        for (int j = 0; j < TV; j++) y[j] = mma(y[j], tt[b], frag_row<NS>(xt, XP, LDT, 16 * j, 32 * b));
    fetch_t(next);
    float *ys = a.ys + slot_head * kChunk * a.dvp + dv0;
#pragma unroll
    for (int j = 0; j < TV; j++) {
      f32x4 z;
#pragma unroll
      for (int r = 0; r < 4; r++) z[r] = -gam[r] * beta[r] * y[j][r];
      put_column<NS>(zt + (16 * j + col) * LDT + 16 * w + 4 * quad, XP, z);
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int t = 16 * w + 4 * quad + r, v = 16 * j + col;
        ys[t * a.dvp + v] = y[j][r];
        if (t < c.len && dv0 + v < a.dv) out_at<T>(a.gv, c.row, c.first + t, h)[dv0 + v] = T(beta[r] * y[j][r]);
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TK; i++)
#pragma unroll
      for (int j = 0; j < TV; j++) e[i][j] *= end;
#pragma unroll
    for (int b = 0; b < 2; b++) {
      Frag<NS> fg[TV], fz[TV];
#pragma unroll
      for (int j = 0; j < TV; j++) {
        fg[j] = frag_col<NS>(gs, VP, LDV, 16 * j, 32 * b);
        fz[j] = frag_row<NS>(zt, XP, LDT, 16 * j, 32 * b);
      }
#pragma unroll
      for (int i = 0; i < TK; i++) {
        const Frag<NI> fq = frag_col<NI>(qs, KP, LDK, w * (DK / 4) + 16 * i, 32 * b);
        const Frag<NI> fk = frag_col<NI>(ks, KP, LDK, w * (DK / 4) + 16 * i, 32 * b);
#pragma unroll
        for (int j = 0; j < TV; j++) e[i][j] = mma(mma(e[i][j], fq, fg[j]), fk, fz[j]);
      }
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
          const int x = row0 + 16 * i + r, y = dv0 + 16 * j + col;
          if (x < a.dk && y < a.dv) a.dstate[state_at + int64_t(x) * a.dv + y] = e[i][j][r];
        }
}

// Eight neighbouring elements of an inner buffer, which has no ragged edges.
template <typename T>
__device__ __forceinline__ Raw8<T> load_inner8(const T *p) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < int(sizeof(T) * 8 / 16); i++) reinterpret_cast<u32x4 *>(&r)[i] = reinterpret_cast<const u32x4 *>(p)[i];
  return r;
}

// A workgroup of eight waves a chunk and key head, its value heads one after
// another (so dQ and dK of a shared head are summed in registers, in an order
// that is always the same). Wave w has rows 16 (w % 4) .. of every product
// and half w / 4 of its columns; S, E and U pass through LDS 32 value columns
// at a time, the next 32 being read while the products of these are made.
template <typename M, int DK, bool Fast>
__global__ __launch_bounds__(512, 2) void delta_gradients(const DeltaArgs a) {
  typedef typename M::T T;
  typedef typename M::Saved Saved;
  constexpr int NI = M::NI, NB = M::NB, NU = M::NU;
  constexpr int LDK = DK + 8, KP = 64 * LDK, LDS = 40, SP = DK * LDS, UP = 64 * LDS, LDM = 72, MP = 64 * LDM;
  constexpr int JK = DK / 32;        // 16-column tiles of a half of the keys' dimension
  constexpr bool kBoth = NB < 3;     // S and E in LDS at a time, M and B too
  typedef Record<M> R;
  constexpr int kSlices = (kBoth ? 2 : 1) * NB * SP + NU * UP, kMs = (kBoth ? 2 : 1) * NB * MP;
  __shared__ __align__(16) bf16 ks[NI * KP], qs[NI * KP], slice[kSlices > kMs ? kSlices : kMs];
  __shared__ double cs[64];
  __shared__ float down[4][64], row_c[2][64], row_b[2][64], total[8];
  bf16 *const us = slice, *const ss = slice + NU * UP, *const es = kBoth ? ss + NB * SP : ss;
  bf16 *const ms = slice, *const bs = kBoth ? slice + NB * MP : slice;

  const int64_t slot = blockIdx.x / a.hk;
  const int hk = int(blockIdx.x - slot * a.hk), per = a.hv / a.hk;
  const Chunk c = chunk_of(a, slot);
  if (c.len == 0) return;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, quad = l >> 4, col = l & 15;
  const int wr = w & 3, half = w >> 2;

  {
    Raw8<T> rk[DK / 64], rq[DK / 64];
#pragma unroll
    for (int j = 0; j < DK / 64; j++) {
      const int at = tid + 512 * j;
      rk[j] = load_head8<Fast, T>(a.k, c, hk, at / (DK / 8), at % (DK / 8) * 8, a.dk);
      rq[j] = load_head8<Fast, T>(a.q, c, hk, at / (DK / 8), at % (DK / 8) * 8, a.dk);
    }
#pragma unroll
    for (int j = 0; j < DK / 64; j++) {
      const int at = tid + 512 * j, t = at / (DK / 8), d = at % (DK / 8) * 8;
      put_frag<NI>(ks + t * LDK + d, KP, frag_of<NI>(keep_head8<Fast>(rk[j], c, t, d, a.dk)));
      put_frag<NI>(qs + t * LDK + d, KP, frag_of<NI>(keep_head8<Fast>(rq[j], c, t, d, a.dk)));
    }
  }
  // element (t, d) of K or Q as its planes add up
  auto value = [&](const bf16 *m, int t, int d) {
    float x = 0.0f;
#pragma unroll
    for (int p = NI - 1; p >= 0; p--) x += float(m[p * KP + t * LDK + d]);
    return x;
  };
  // this thread's pieces of a slice: of S and E (row sx), and of U (row ux)
  const int sx = tid / 4, sv = tid % 4 * 8, ux = (tid & 255) / 4, uv = tid % 4 * 8;
  const bool has_s = sx < DK, has_u = tid < 256;
  const int t_own = 16 * wr + col;

  f32x4 dq[JK] = {}, dk[JK] = {};
  for (int h = hk * per; h < (hk + 1) * per; h++) {
    const int64_t slot_head = slot * a.hv + h;
    const float *dec = reinterpret_cast<const float *>(a.records + slot_head * R::bytes(true) + R::Decay);
    const Saved *S = reinterpret_cast<const Saved *>(a.states) + slot_head * DK * a.dvp;
    const Saved *E = reinterpret_cast<const Saved *>(a.grads) + slot_head * DK * a.dvp;
    const float *U = a.us + slot_head * kChunk * a.dvp, *Y = a.ys + slot_head * kChunk * a.dvp;

    Raw8<Saved> rs, re;
    Raw8<float> ru, ry;
    Raw8<T> ro, rv;
    auto fetch = [&](int v0) {
      if (has_s) {
        rs = load_inner8(S + sx * a.dvp + v0 + sv);
        re = load_inner8(E + sx * a.dvp + v0 + sv);
      }
      if (has_u) ru = load_inner8(U + ux * a.dvp + v0 + uv);
      ry = load_inner8(Y + t_own * a.dvp + v0 + 8 * quad);
      ro = load_head8<Fast, T>(a.d_o, c, h, t_own, v0 + 8 * quad, a.dv);
      rv = load_head8<Fast, T>(a.v, c, h, t_own, v0 + 8 * quad, a.dv);
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
    __syncthreads();  // the head before is done with LDS
    if (w == 0) cs[l] = run;

    f32x4 os[JK] = {}, ys[JK] = {}, ue[JK] = {}, ou[2] = {}, yu[2] = {};
    float yv = 0.0f, se = 0.0f;  // yv: of row t_own, this lane's columns
    for (int v0 = 0; v0 < a.dvp; v0 += 32) {
      const Frag<NI> fo = frag_of<NI>(keep_head8<Fast>(ro, c, t_own, v0 + 8 * quad, a.dv));
      const Frag<NU> fy = frag_of<NU>(ry);
      const Raw8<T> v = keep_head8<Fast>(rv, c, t_own, v0 + 8 * quad, a.dv);
#pragma unroll
      for (int i = 0; i < 8; i++) yv += ry.x[i] * float(v.x[i]);
      if (has_u) put_frag<NU>(us + ux * LDS + uv, UP, frag_of<NU>(ru));
      Raw8<Saved> late = re;
      if (has_s) {
#pragma unroll
        for (int i = 0; i < 8; i++) se += float(rs.x[i]) * float(re.x[i]);
        put_frag<NB>(ss + sx * LDS + sv, SP, frag_of<NB>(rs));
        if (kBoth) put_frag<NB>(es + sx * LDS + sv, SP, frag_of<NB>(re));
      }
      __syncthreads();
      if (v0 + 32 < a.dvp) fetch(v0 + 32);
      const Frag<NU> fu = frag_row<NU>(us, UP, LDS, 16 * wr, 0);
#pragma unroll
      for (int j = 0; j < JK; j++) {
        const int x = 16 * (JK * half + j);
        const Frag<NB> fs = frag_row<NB>(ss, SP, LDS, x, 0);
        os[j] = mma(os[j], fo, fs);
        ys[j] = mma(ys[j], fy, fs);
        if (kBoth) ue[j] = mma(ue[j], fu, frag_row<NB>(es, SP, LDS, x, 0));
      }
#pragma unroll
      for (int j = 0; j < 2; j++)
        if (2 * half + j <= wr) {
          const Frag<NU> f = frag_row<NU>(us, UP, LDS, 16 * (2 * half + j), 0);
          ou[j] = mma(ou[j], fo, f);
          yu[j] = mma(yu[j], fy, f);
        }
      __syncthreads();
      if (!kBoth) {
        if (has_s) put_frag<NB>(es + sx * LDS + sv, SP, frag_of<NB>(late));
        __syncthreads();
#pragma unroll
        for (int j = 0; j < JK; j++) ue[j] = mma(ue[j], fu, frag_row<NB>(es, SP, LDS, 16 * (JK * half + j), 0));
        __syncthreads();
      }
    }

    // this lane's rows t = 16 wr + 4 quad + r
    float gam[4], last[4], beta[4], dc[4], db[4], end = 0.0f;
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int t = 16 * wr + 4 * quad + r;
      gam[r] = dec[t];
      last[r] = dec[64 + t];
      beta[r] = dec[128 + t];
      dc[r] = db[r] = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < JK; j++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int t = 16 * wr + 4 * quad + r, d = 16 * (JK * half + j) + col;
        const float kv = value(ks, t, d), qv = value(qs, t, d);
        const float o = a.scale * gam[r] * os[j][r], y = gam[r] * ys[j][r], u = last[r] * ue[j][r];
        dq[j][r] += o;
        dk[j][r] += u - beta[r] * y;
        dc[r] += qv * o - beta[r] * kv * y - kv * u;
        db[r] -= kv * y;
        end += kv * u;
      }
    f32x4 kk[2] = {}, qk[2] = {};
#pragma unroll
    for (int d = 0; d < DK; d += 32) {
      const Frag<NI> fk = frag_row<NI>(ks, KP, LDK, 16 * wr, d), fq = frag_row<NI>(qs, KP, LDK, 16 * wr, d);
#pragma unroll
      for (int j = 0; j < 2; j++)
        if (2 * half + j <= wr) {
          const Frag<NI> fs = frag_row<NI>(ks, KP, LDK, 16 * (2 * half + j), d);
          kk[j] = mma(kk[j], fk, fs);
          qk[j] = mma(qk[j], fq, fs);
        }
    }
    f32x4 b[2];
#pragma unroll
    for (int j = 0; j < 2; j++) {
      float across = 0.0f;
      f32x4 m;
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int t = 16 * wr + 4 * quad + r, s = 16 * (2 * half + j) + col;
        const float d = s <= t ? expf(float(cs[t] - cs[s])) : 0.0f;
        m[r] = s <= t ? a.scale * d * ou[j][r] : 0.0f;
        b[j][r] = s < t ? -beta[r] * d * yu[j][r] : 0.0f;
        const float pair = m[r] * qk[j][r] + b[j][r] * kk[j][r];
        dc[r] += pair;
        across += pair;
        db[r] -= s < t ? yu[j][r] * d * kk[j][r] : 0.0f;
      }
      across = sum_rows(across);
      if (quad == 0) down[wr][16 * (2 * half + j) + col] = across;
      // M is stored [s][t]
      put_column<NB>(ms + (16 * (2 * half + j) + col) * LDM + 16 * wr + 4 * quad, MP, m);
      if (kBoth) put_column<NB>(bs + (16 * (2 * half + j) + col) * LDM + 16 * wr + 4 * quad, MP, b[j]);
    }
    yv = half == 0 ? sum_rows(yv) : 0.0f;  // lane i: of row 16 wr + i % 16
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int t = 16 * wr + 4 * quad + r;
      const float x = sum16(dc[r]), y = sum16(db[r]) + __shfl(yv, 4 * quad + r, 64);
      if (col == 0) {
        row_c[half][t] = x;
        row_b[half][t] = y;
      }
    }
    end = sum64(end + se * dec[63]);
    if (l == 0) total[w] = end;
    __syncthreads();
    if (w == 0) {
      float x = row_c[0][l] + row_c[1][l] - (down[0][l] + down[1][l] + down[2][l] + down[3][l]);
      if (l == 63) x += ((total[0] + total[1]) + (total[2] + total[3])) + ((total[4] + total[5]) + (total[6] + total[7]));
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const float up = __shfl_down(x, d, 64);
        if (l + d < 64) x += up;
      }
      if (l < c.len) {
        *out_at<T>(a.gg, c.row, c.first + l, h) = T(x);
        *out_at<T>(a.gbeta, c.row, c.first + l, h) = T(row_b[0][l] + row_b[1][l]);
      }
    }
#pragma unroll
    for (int t0 = 0; t0 < 64; t0 += 32) {
      if (t0 == 0 || wr >= 2) {  // M ends at the diagonal
        const Frag<NB> f = frag_col<NB>(ms, MP, LDM, 16 * wr, t0);
#pragma unroll
        for (int j = 0; j < JK; j++) dq[j] = mma(dq[j], f, frag_col<NI>(ks, KP, LDK, 16 * (JK * half + j), t0));
      }
      if (t0 != 0 || wr < 2) {
        const Frag<NB> f = frag_row<NB>(ms, MP, LDM, 16 * wr, t0);
#pragma unroll
        for (int j = 0; j < JK; j++) dk[j] = mma(dk[j], f, frag_col<NI>(qs, KP, LDK, 16 * (JK * half + j), t0));
      }
    }
    if (!kBoth) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 2; j++)
        put_column<NB>(bs + (16 * (2 * half + j) + col) * LDM + 16 * wr + 4 * quad, MP, b[j]);
      __syncthreads();
    }
#pragma unroll
    for (int t0 = 0; t0 < 64; t0 += 32) {
      const Frag<NB> fb = frag_col<NB>(bs, MP, LDM, 16 * wr, t0), ft = frag_row<NB>(bs, MP, LDM, 16 * wr, t0);
#pragma unroll
      for (int j = 0; j < JK; j++) {
        const Frag<NI> fk = frag_col<NI>(ks, KP, LDK, 16 * (JK * half + j), t0);
        if (t0 == 0 || wr >= 2) dk[j] = mma(dk[j], fb, fk);
        if (t0 != 0 || wr < 2) dk[j] = mma(dk[j], ft, fk);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < JK; j++)
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int t = 16 * wr + 4 * quad + r, d = 16 * (JK * half + j) + col;
      if (t < c.len && d < a.dk) {
        out_at<T>(a.gq, c.row, c.first + t, hk)[d] = T(dq[j][r]);
        out_at<T>(a.gk, c.row, c.first + t, hk)[d] = T(dk[j][r]);
      }
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
    with_bool(fast(a), [&](auto f) {
      constexpr bool F = decltype(f)::value;
      hipLaunchKernelGGL((delta_reverse<M, DK, BV, F>), dim3(unsigned((lanes + 7) / 8 * 8 * blocks)), dim3(256), 0, stream,
                         a, blocks);
      if (a.slots) hipLaunchKernelGGL((delta_gradients<M, DK, F>), dim3(unsigned(a.slots * a.hk)), dim3(512), 0, stream, a);
    });
  };
  with_mode(op, [&](auto m) {
    constexpr bool wide = decltype(m)::NI < 3;  // three planes of K and Q leave no LDS for 32 columns
    const bool narrow = !wide || lanes * ((a.dv + 31) / 32) < 256;
    if constexpr (wide) {
      if (!narrow) {
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
