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
// registers.
template <typename M, int DK, int BV>
__global__ __launch_bounds__(256) void delta_reverse(const DeltaArgs a, int blocks) {
  typedef typename M::T T;
  typedef typename M::Saved Saved;
  constexpr int NI = M::NI, NS = M::NS, NO = M::NO;
  constexpr int LDK = DK + 8, LDT = 72, LDV = BV + 8;
  constexpr int KP = 64 * LDK, SP = BV * LDK, XP = BV * LDT, VP = 64 * LDV;
  constexpr int TK = DK / 64, TV = BV / 16;
  typedef Record<NS, NO> R;
  __shared__ __align__(16) bf16 ks[NI * KP], qs[NI * KP], et[NS * SP], xt[NS * XP], zt[NS * XP], os[NI * VP], gs[NS * VP];

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

  for (int ci = chunks - 1; ci >= 0; ci--) {
    const int64_t left = sq.len - int64_t(ci) * kChunk;
    const Chunk c = {sq.row, sq.first + int64_t(ci) * kChunk, sid, left > kChunk ? kChunk : int(left)};
    const int64_t slot_head = (sq.slot + ci) * a.hv + h;
    const char *rec = a.records + slot_head * R::bytes(true);
    const float *dec = reinterpret_cast<const float *>(rec + R::Decay);
    for (int at = tid; at < 64 * (DK / 8); at += 256) {
      const int t = at / (DK / 8), d = at % (DK / 8) * 8;
      put_frag<NI>(ks + t * LDK + d, KP, frag_of<NI>(load_head8<T>(a.k, c, hk, t, d, a.dk)));
      put_frag<NI>(qs + t * LDK + d, KP, frag_of<NI>(load_head8<T>(a.q, c, hk, t, d, a.dk)));
    }
    for (int at = tid; at < 64 * (BV / 8); at += 256) {
      const int t = at / (BV / 8), d = at % (BV / 8) * 8;
      const Raw8<T> raw = load_head8<T>(a.d_o, c, h, t, dv0 + d, a.dv);
      put_frag<NI>(os + t * LDV + d, VP, frag_of<NI>(raw));
      const float f = a.scale * dec[t];
      Raw8<float> up;
#pragma unroll
      for (int i = 0; i < 8; i++) up.x[i] = f * float(raw.x[i]);
      put_frag<NS>(gs + t * LDV + d, VP, frag_of<NS>(up));
    }
    Saved *es = reinterpret_cast<Saved *>(a.grads) + slot_head * a.dk * a.dv;
#pragma unroll
    for (int i = 0; i < TK; i++)
#pragma unroll
      for (int j = 0; j < TV; j++) {
        put_column<NS>(et + (16 * j + col) * LDK + row0 + 16 * i, SP, e[i][j]);
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int x = row0 + 16 * i + r, y = dv0 + 16 * j + col;
          if (x < a.dk && y < a.dv) es[int64_t(x) * a.dv + y] = Saved(e[i][j][r]);
        }
      }
    Frag<NS> tt[2], pt[2];  // rows 16 w .. of T^T and P^T: terms from the diagonal on
#pragma unroll
    for (int b = 0; b < 2; b++)
      if (b == 1 || w < 2)
#pragma unroll
        for (int p = 0; p < NS; p++) {
          tt[b].p[p] = reinterpret_cast<const bf16x8 *>(rec + R::Tt + p * 8192)[(w * 2 + b) * 64 + l];
          pt[b].p[p] = reinterpret_cast<const bf16x8 *>(rec + R::Pt + p * 8192)[(w * 2 + b) * 64 + l];
        }
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
    Saved *ys = reinterpret_cast<Saved *>(a.ys) + slot_head * kChunk * a.dv;
#pragma unroll
    for (int j = 0; j < TV; j++) {
      f32x4 z;
      const int v = dv0 + 16 * j + col;
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int t = 16 * w + 4 * quad + r;
        const float by = beta[r] * y[j][r];
        z[r] = -gam[r] * by;
        if (v < a.dv) {
          ys[int64_t(t) * a.dv + v] = Saved(y[j][r]);
          if (t < c.len) out_at<T>(a.gv, c.row, c.first + t, h)[v] = T(by);
        }
      }
      put_column<NS>(zt + (16 * j + col) * LDT + 16 * w + 4 * quad, XP, z);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TK; i++)
#pragma unroll
      for (int j = 0; j < TV; j++) e[i][j] *= end;
#pragma unroll
    for (int b = 0; b < 2; b++)
#pragma unroll
      for (int i = 0; i < TK; i++) {
        const Frag<NI> fq = frag_col<NI>(qs, KP, LDK, w * (DK / 4) + 16 * i, 32 * b);
        const Frag<NI> fk = frag_col<NI>(ks, KP, LDK, w * (DK / 4) + 16 * i, 32 * b);
#pragma unroll
        for (int j = 0; j < TV; j++) {
          e[i][j] = mma(e[i][j], fq, frag_col<NS>(gs, VP, LDV, 16 * j, 32 * b));
          e[i][j] = mma(e[i][j], fk, frag_row<NS>(zt, XP, LDT, 16 * j, 32 * b));
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

// A workgroup of four waves a chunk and key head, its value heads one after
// another (so dQ and dK of a shared head are summed in registers, in an order
// that is always the same). Wave w has rows 16 w .. 16 w + 15 of every
// product; S, E and U pass through LDS 32 value columns at a time.
template <typename M, int DK>
__global__ __launch_bounds__(256) void delta_gradients(const DeltaArgs a) {
  typedef typename M::T T;
  typedef typename M::Saved Saved;
  constexpr int NI = M::NI, NB = M::NB;
  constexpr int LDK = DK + 8, KP = 64 * LDK, LDS = 40, SP = DK * LDS, UP = 64 * LDS, LDM = 72, MP = 64 * LDM;
  constexpr int JK = DK / 16;
  typedef Record<M::NS, M::NO> R;
  constexpr int kSlice = NB * (SP + UP) > NB * MP ? NB * (SP + UP) : NB * MP;
  __shared__ __align__(16) bf16 ks[NI * KP], qs[NI * KP], slice[kSlice];
  __shared__ double cs[64];
  __shared__ float down[4][64], total[4];
  bf16 *const ss = slice, *const us = slice + NB * SP, *const mt = slice;

  const int64_t slot = blockIdx.x / a.hk;
  const int hk = int(blockIdx.x - slot * a.hk), per = a.hv / a.hk;
  const Chunk c = chunk_of(a, slot);
  if (c.len == 0) return;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, quad = l >> 4, col = l & 15;

  for (int at = tid; at < 64 * (DK / 8); at += 256) {
    const int t = at / (DK / 8), d = at % (DK / 8) * 8;
    put_frag<NI>(ks + t * LDK + d, KP, frag_of<NI>(load_head8<T>(a.k, c, hk, t, d, a.dk)));
    put_frag<NI>(qs + t * LDK + d, KP, frag_of<NI>(load_head8<T>(a.q, c, hk, t, d, a.dk)));
  }
  // element (t, d) of K or Q as its planes add up
  auto value = [&](const bf16 *m, int t, int d) {
    float x = 0.0f;
#pragma unroll
    for (int p = NI - 1; p >= 0; p--) x += float(m[p * KP + t * LDK + d]);
    return x;
  };

  f32x4 dq[JK] = {}, dk[JK] = {};
  for (int h = hk * per; h < (hk + 1) * per; h++) {
    const int64_t slot_head = slot * a.hv + h;
    const float *dec = reinterpret_cast<const float *>(a.records + slot_head * R::bytes(true) + R::Decay);
    const Saved *S = reinterpret_cast<const Saved *>(a.states) + slot_head * a.dk * a.dv;
    const Saved *E = reinterpret_cast<const Saved *>(a.grads) + slot_head * a.dk * a.dv;
    const Saved *U = reinterpret_cast<const Saved *>(a.us) + slot_head * kChunk * a.dv;
    const Saved *Y = reinterpret_cast<const Saved *>(a.ys) + slot_head * kChunk * a.dv;
    __syncthreads();
    if (w == 0) {
      const float g = l < c.len ? float(*at<T>(a.g, c.row, c.first + l, h)) : 0.0f;
      double s = g < -1000.0f ? -1000.0 : double(g);
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const double up = __shfl_up(s, d, 64);
        if (l >= d) s += up;
      }
      cs[l] = s;
    }

    f32x4 os[JK] = {}, ys[JK] = {}, ue[JK] = {}, ou[4] = {}, yu[4] = {};
    float yv = 0.0f, se = 0.0f;  // yv: of row 16 w + col, this lane's columns
    for (int v0 = 0; v0 < a.dv; v0 += 32) {
      const int v = v0 + 8 * quad, t = 16 * w + col;
      const int nv = a.dv - v < 0 ? 0 : a.dv - v > 8 ? 8 : a.dv - v;
      const Raw8<T> ro = load_head8<T>(a.d_o, c, h, t, v, a.dv), rv = load_head8<T>(a.v, c, h, t, v, a.dv);
      const Raw8<Saved> ry = load8<Saved>(Y + int64_t(t) * a.dv + v, nv), ru = load8<Saved>(U + int64_t(t) * a.dv + v, nv);
#pragma unroll
      for (int i = 0; i < 8; i++) yv += float(ry.x[i]) * float(rv.x[i]);
      const Frag<NI> fo = frag_of<NI>(ro);
      const Frag<NB> fy = frag_of<NB>(ry), fu = frag_of<NB>(ru);
      __syncthreads();
      put_frag<NB>(us + t * LDS + 8 * quad, UP, fu);
      for (int i = tid; i < DK * 4; i += 256) {
        const int x = i / 4, y = v0 + i % 4 * 8;
        const int n = x < a.dk && y < a.dv ? (a.dv - y > 8 ? 8 : a.dv - y) : 0;
        const Raw8<Saved> rs = load8<Saved>(S + int64_t(x) * a.dv + y, n), re = load8<Saved>(E + int64_t(x) * a.dv + y, n);
#pragma unroll
        for (int j = 0; j < 8; j++) se += float(rs.x[j]) * float(re.x[j]);
        put_frag<NB>(ss + x * LDS + i % 4 * 8, SP, frag_of<NB>(rs));
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < JK; j++) {
        const Frag<NB> fs = frag_row<NB>(ss, SP, LDS, 16 * j, 0);
        os[j] = mma(os[j], fo, fs);
        ys[j] = mma(ys[j], fy, fs);
      }
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (j <= w) {
          const Frag<NB> f = frag_row<NB>(us, UP, LDS, 16 * j, 0);
          ou[j] = mma(ou[j], fo, f);
          yu[j] = mma(yu[j], fy, f);
        }
      __syncthreads();
      for (int i = tid; i < DK * 4; i += 256) {
        const int x = i / 4, y = v0 + i % 4 * 8;
        const int n = x < a.dk && y < a.dv ? (a.dv - y > 8 ? 8 : a.dv - y) : 0;
        put_frag<NB>(ss + x * LDS + i % 4 * 8, SP, frag_of<NB>(load8<Saved>(E + int64_t(x) * a.dv + y, n)));
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < JK; j++) ue[j] = mma(ue[j], fu, frag_row<NB>(ss, SP, LDS, 16 * j, 0));
    }

    f32x4 kk[4] = {}, qk[4] = {};
#pragma unroll
    for (int d = 0; d < DK; d += 32) {
      const Frag<NI> fk = frag_row<NI>(ks, KP, LDK, 16 * w, d), fq = frag_row<NI>(qs, KP, LDK, 16 * w, d);
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (j <= w) {
          const Frag<NI> fs = frag_row<NI>(ks, KP, LDK, 16 * j, d);
          kk[j] = mma(kk[j], fk, fs);
          qk[j] = mma(qk[j], fq, fs);
        }
    }

    // this lane's rows t = 16 w + 4 quad + r
    float gam[4], last[4], beta[4], dc[4], db[4], from_last[4];
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int t = 16 * w + 4 * quad + r;
      gam[r] = dec[t];
      last[r] = dec[64 + t];
      beta[r] = dec[128 + t];
      dc[r] = db[r] = from_last[r] = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < JK; j++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int t = 16 * w + 4 * quad + r, d = 16 * j + col;
        const float kv = value(ks, t, d), qv = value(qs, t, d);
        const float o = a.scale * gam[r] * os[j][r], y = gam[r] * ys[j][r], u = last[r] * ue[j][r];
        dq[j][r] += o;
        dk[j][r] += u - beta[r] * y;
        dc[r] += qv * o - beta[r] * kv * y - kv * u;
        db[r] -= kv * y;
        from_last[r] += kv * u;
      }
    f32x4 m[4], b[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      float across = 0.0f;
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int t = 16 * w + 4 * quad + r, s = 16 * j + col;
        const float d = s <= t ? expf(float(cs[t] - cs[s])) : 0.0f;
        m[j][r] = s <= t ? a.scale * d * ou[j][r] : 0.0f;
        b[j][r] = s < t ? -beta[r] * d * yu[j][r] : 0.0f;
        const float pair = m[j][r] * qk[j][r] + b[j][r] * kk[j][r];
        dc[r] += pair;
        across += pair;
        db[r] -= s < t ? yu[j][r] * d * kk[j][r] : 0.0f;
      }
      across = sum_rows(across);
      if (quad == 0) down[w][16 * j + col] = across;
    }
    yv = sum_rows(yv);  // lane c: of row 16 w + c % 16
    float end = 0.0f;
#pragma unroll
    for (int r = 0; r < 4; r++) {
      dc[r] = sum16(dc[r]);
      db[r] = sum16(db[r]) + __shfl(yv, 4 * quad + r, 64);
      const float f = sum16(from_last[r]);
      end += f;
    }
    end = sum_rows(end);
    se = sum64(se);
    if (l == 0) total[w] = end + se * dec[63];
    __syncthreads();  // every wave is done with the slice; down and total are there
    // row sums to one lane a token, then suffix sums over the chunk
    __shared__ float rows[64];
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int t = 16 * w + 4 * quad + r;
      if (col == 0) {
        rows[t] = dc[r] - (down[0][t] + down[1][t] + down[2][t] + down[3][t]);
        if (t < c.len) *out_at<T>(a.gbeta, c.row, c.first + t, h) = T(db[r]);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; j++) put_column<NB>(mt + (16 * j + col) * LDM + 16 * w + 4 * quad, MP, m[j]);
    __syncthreads();
    if (w == 0) {
      float x = rows[l] + (l == 63 ? total[0] + total[1] + total[2] + total[3] : 0.0f);
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const float up = __shfl_down(x, d, 64);
        if (l + d < 64) x += up;
      }
      if (l < c.len) *out_at<T>(a.gg, c.row, c.first + l, h) = T(x);
    }
    // M is stored [s][t]
#pragma unroll
    for (int t0 = 0; t0 < 64; t0 += 32) {
      const Frag<NB> fm = frag_col<NB>(mt, MP, LDM, 16 * w, t0), ft = frag_row<NB>(mt, MP, LDM, 16 * w, t0);
#pragma unroll
      for (int j = 0; j < JK; j++) {
        dq[j] = mma(dq[j], fm, frag_col<NI>(ks, KP, LDK, 16 * j, t0));
        dk[j] = mma(dk[j], ft, frag_col<NI>(qs, KP, LDK, 16 * j, t0));
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; j++) put_column<NB>(mt + (16 * j + col) * LDM + 16 * w + 4 * quad, MP, b[j]);
    __syncthreads();
#pragma unroll
    for (int t0 = 0; t0 < 64; t0 += 32) {
      const Frag<NB> fm = frag_col<NB>(mt, MP, LDM, 16 * w, t0), ft = frag_row<NB>(mt, MP, LDM, 16 * w, t0);
#pragma unroll
      for (int j = 0; j < JK; j++) {
        const Frag<NI> fk = frag_col<NI>(ks, KP, LDK, 16 * j, t0);
        dk[j] = mma(dk[j], fm, fk);
        dk[j] = mma(dk[j], ft, fk);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < JK; j++)
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int t = 16 * w + 4 * quad + r, d = 16 * j + col;
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
    const int blocks = (a.dv + BV - 1) / BV;
    hipLaunchKernelGGL((delta_reverse<M, DK, BV>), dim3(unsigned((lanes + 7) / 8 * 8 * blocks)), dim3(256), 0, stream, a, blocks);
    if (a.slots) hipLaunchKernelGGL((delta_gradients<M, DK>), dim3(unsigned(a.slots * a.hk)), dim3(256), 0, stream, a);
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
