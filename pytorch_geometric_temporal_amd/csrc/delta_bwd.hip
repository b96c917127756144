// Gated delta rule, whole sequences, adjoint (delta_common.h has the forward formulas).  With dS the gradient of a chunk's end state,
// everything per chunk and q already scaled:
//   dU = P^T dO + diag(leave) K dS;      dR = (I + A)^-T dU,  A_ij = beta_i D_ij (k_i . k_j) (j < i);      dY = diag(beta) dR = dV
//   M1_ij = D_ij (dO_i . u_j) (j <= i);      M2_ij = -D_ij (dY_i . u_j) (j < i)
//   dQ = Gamma dO S0^T + M1 K
//   dK = -Gamma dY S0^T + diag(leave) U dS^T + (M2 + M2^T) K + M1^T Q
//   dbeta_i = dR_i . e_i
//   dS0 = exp(c_C) dS + Q^T Gamma dO - K^T Gamma dY
//   dg_l = sum_{i >= l > j} (M1_ij q_i.k_j + M2_ij k_i.k_j) + sum_{i >= l} z_i + sum_{j < l} w_j + exp(c_C) <S0, dS>,
//          z_i = q_i . (Gamma dO S0^T)_i + k_i . (-Gamma dY S0^T)_i,   w_j = k_j . (diag(leave) U dS^T)_j
// (the terms of dg that cancel exactly, i and j on the same side of l, are never formed).  E and the state before each chunk come
// from the forward pass, so the adjoint solves one triangular tile a chunk and runs no forward recurrence.
#include "delta_common.h"

using namespace gd;

namespace {

struct BwdArgs {
  Shape s;
  View q, k, g, beta;
  const void* d_o;               // [B, T, N, H, V]
  const float* e;                // [B, T, N, H, V]
  const float* start;            // [P, K, V] or null
  const float* states;           // [P, chunks - 1, K, V]
  const float* d_last;           // [P, K, V] or null
  void* dq; void* dk;            // [B, T, N, H / rep, K] in the inputs' type; rep > 1: fp32 [B, T, N, H, K], to be added over the heads
  void* dv;                      // [B, T, N, H, V]
  float* dg; float* dbeta;       // [B, T, N, H]
  float* d_start;                // [P, K, V] or null
  float* seg_end;                // [P, segs - 1, K, V]: the gradient of the state behind every segment but the last
  int vec, vec_do, vec_e, vec_s; // q, k / d_o / e / states can be read four values at a time
};

// One team per sequence and segment, chunks from the last to the first.  STATE: only the gradient of the state before the segment, from a
// zero gradient behind it (the last segment: from d_last).
template <class IO, int D, bool STATE>
__global__ __launch_bounds__(Team<D>::THREADS) void delta_bwd_kernel(BwdArgs a) {
  using TM = Team<D>;
  constexpr int NW = TM::NW, LD = TM::LD, TL = TM::TL, QD = D / 4, EPL = TM::EPL, NP = STATE ? 2 : 3;
  struct Lds {
    float k[16 * LD], q[16 * LD], o[16 * LD], e[STATE ? 4 : 16 * LD], y[16 * LD];
    float x[STATE ? 4 : D * LD];                           // dS, for the products that contract over its columns
    float part[NW][NP][TILE];
    float at[TILE], pm[TILE], m1[TILE], m2[TILE], xm[TILE];
    float red[NW][4][16];                                  // row sums by wavefront: dbeta, z, w, <S0, dS>
    float hi[16], lo[16], enter[16], leave[16], beta[16], whole[4];
  };
  __shared__ __attribute__((aligned(16))) char smem[sizeof(Lds) * TM::TEAMS];
  const Shape& s = a.s;
  const int tid = (int)threadIdx.x, team = tid / TL, tl = tid % TL, w = PGT_UNIFORM(tl / 64), lane = tid & 63, col = lane & 15, cg = lane >> 4;
  Lds& L = reinterpret_cast<Lds*>(smem)[team];
  const int64_t first = s.p0 + (int64_t)blockIdx.x * TM::TEAMS;
  const Seq sq = seq_of(s, first + team);
  const int seg = (int)blockIdx.y + (STATE ? 1 : 0);
  const int c0 = seg * s.cps, c1 = c0 + s.cps < s.chunks ? c0 + s.cps : s.chunks;
  const int reach = chunks_of_block<TM::TEAMS>(s, first), ce = reach < c1 ? reach : c1;
  const int kh = sq.h / s.rep;
  const IO* kp = at<IO>(a.k, sq, kh);
  const IO* qp = at<IO>(a.q, sq, kh);
  const float* gp = at<float>(a.g, sq, sq.h);
  const float* bp = at<float>(a.beta, sq, sq.h);
  const int n = 16 * w + col;                             // this lane's column: of the state (values) and, in the dQ / dK products, of the keys
  const bool vcols = 16 * w < s.V, kcols = 16 * w < s.K;
  const int64_t row_h = (int64_t)s.N * s.H, seq_h = (int64_t)sq.b * s.T * row_h + (int64_t)sq.n * s.H + sq.h;     // rows of [B, T, N, H]

  gd_f4 S[QD / 4];                                        // dS
  {
    const float* from = seg == s.segs - 1 ? a.d_last : STATE ? nullptr : a.seg_end;
    if (from) from += seg == s.segs - 1 ? sq.p * s.K * s.V : (sq.p * (s.segs - 1) + seg) * s.K * s.V;
#pragma unroll
    for (int t = 0; t < QD / 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * t + 4 * cg + r;
        S[t][r] = from && sq.live && row < s.K && n < s.V ? from[(int64_t)row * s.V + n] : 0.f;
      }
  }
  const int tok = tl / QD, qd = 4 * (tl % QD);
  gd_f4 nk = zero4(), nq = zero4(), no = zero4(), ne = zero4();
  float ng = 0.f, nb = 0.f;
  auto fetch = [&](int c) {
    const int t = 16 * c + tok;
    const bool in = t < sq.len;
    nk = load4(kp + (int64_t)t * a.k.st + qd, in ? s.K - qd : 0, a.vec != 0);
    nq = load4(qp + (int64_t)t * a.q.st + qd, in ? s.K - qd : 0, a.vec != 0);
    const int64_t off = (seq_h + t * row_h) * s.V + qd;
    no = load4(reinterpret_cast<const IO*>(a.d_o) + off, in ? s.V - qd : 0, a.vec_do != 0);
    if (!STATE) ne = load4(a.e + off, in ? s.V - qd : 0, a.vec_e != 0);
    if (w == 0) {
      const int tg = 16 * c + col;
      ng = tg < sq.len ? gp[(int64_t)tg * a.g.st] : 0.f;
      nb = tg < sq.len ? bp[(int64_t)tg * a.beta.st] : 0.f;
    }
  };
  if (c0 < ce) fetch(ce - 1);
  for (int c = ce - 1; c >= c0; --c) {
    put4(&L.k[tok * LD + qd], nk);
#pragma unroll
    for (int r = 0; r < 4; ++r) nq[r] *= s.scale;
    put4(&L.q[tok * LD + qd], nq);
    put4(&L.o[tok * LD + qd], no);
    if (!STATE) put4(&L.e[tok * LD + qd], ne);
    if (w == 0) {
      const Decay d = chunk_decay(ng);
      if (lane < 16) {
        L.hi[lane] = d.hi; L.lo[lane] = d.lo; L.enter[lane] = d.enter; L.leave[lane] = d.leave; L.beta[lane] = nb;
        if (lane == 0) L.whole[0] = d.whole;
      }
    }
    if (c > c0) fetch(c - 1);
    gd_f4 s0[STATE ? 1 : QD / 4];                         // S0, rows = this wavefront's sixteen key columns, along the values
    if (!STATE) {
      const float* from = c > 0 ? a.states + (sq.p * (s.chunks - 1) + c - 1) * s.K * s.V : a.start ? a.start + sq.p * s.K * s.V : nullptr;
#pragma unroll
      for (int t = 0; t < QD / 4; ++t)
        s0[t] = load4(from + (int64_t)n * s.V + 16 * t + 4 * cg, from && sq.live && n < s.K ? s.V - 16 * t - 4 * cg : 0, a.vec_s != 0);
    }
    team_sync<D>();
    {   // this wavefront's sixteen columns of K K^T, Q K^T (keys) and dO U^T (values)
      const gd_f4 kk = lds4(&L.k[col * LD + 16 * w + 4 * cg]);
      const gd_f4 x = mma16(kk, kk, zero4()), y = mma16(lds4(&L.q[col * LD + 16 * w + 4 * cg]), kk, zero4());
      gd_f4 z = zero4();
      if (!STATE) {
        gd_f4 u = lds4(&L.e[col * LD + 16 * w + 4 * cg]);
        const float b = L.beta[col];
#pragma unroll
        for (int r = 0; r < 4; ++r) u[r] *= b;
        z = mma16(lds4(&L.o[col * LD + 16 * w + 4 * cg]), u, z);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        L.part[w][0][(4 * cg + r) * TS + col] = x[r];
        L.part[w][1][(4 * cg + r) * TS + col] = y[r];
        if (!STATE) L.part[w][NP - 1][(4 * cg + r) * TS + col] = z[r];
      }
    }
    team_sync<D>();
    float el_d[EPL], el_kd[EPL], el_x[EPL];
    if (tl < 256) {
#pragma unroll
      for (int m = 0; m < EPL; ++m) {
        const int el = tl + m * TL, i = el >> 4, j = el & 15;
        float kk = 0.f, qk = 0.f, ou = 0.f;
#pragma unroll
        for (int u = 0; u < NW; ++u) {
          kk += L.part[u][0][i * TS + j];
          qk += L.part[u][1][i * TS + j];
          if (!STATE) ou += L.part[u][NP - 1][i * TS + j];
        }
        const float d = j <= i ? expf((L.hi[i] - L.hi[j]) + (L.lo[i] - L.lo[j])) : 0.f;
        L.at[j * TS + i] = j < i ? L.beta[i] * d * kk : 0.f;
        L.pm[i * TS + j] = j <= i ? d * qk : 0.f;
        if (!STATE) {
          const float m1 = j <= i ? d * ou : 0.f;
          L.m1[i * TS + j] = m1;
          el_d[m] = j < i ? d : 0.f;
          el_kd[m] = j < i ? d * kk : 0.f;
          el_x[m] = j < i ? m1 * qk : 0.f;
        }
      }
    }
    team_sync<D>();
    const gd_f4 enter = lds4(&L.enter[4 * cg]), leave = lds4(&L.leave[4 * cg]), beta = lds4(&L.beta[4 * cg]);
    gd_f4 dy = zero4();
    if (vcols) {
      gd_f4 ks = zero4();
#pragma unroll
      for (int t = 0; t < QD / 4; ++t) ks = mma16(lds4(&L.k[col * LD + 16 * t + 4 * cg]), S[t], ks);
      gd_f4 dout, pt;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        dout[r] = L.o[(4 * cg + r) * LD + n];
        pt[r] = L.pm[(4 * cg + r) * TS + col];
        ks[r] *= leave[r];
      }
      const gd_f4 du = mma16(pt, dout, ks);
      float arow[16];
      row16(&L.at[col * TS], arow);
      gd_f4 inv = unit_row(lane);
      solve_up<15>(arow, inv);
      const gd_f4 dr = mma16(inv, du, zero4());
      float db[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        dy[r] = beta[r] * dr[r];
        if (!STATE) {
          L.y[(4 * cg + r) * LD + n] = dy[r];
          db[r] = sum16(dr[r] * L.e[(4 * cg + r) * LD + n]);
          if (col == 0) L.red[w][0][4 * cg + r] = db[r];
          const int t = 16 * c + 4 * cg + r;
          if (sq.live && t < s.T && n < s.V) reinterpret_cast<IO*>(a.dv)[(seq_h + t * row_h) * s.V + n] = from_f32<IO>(dy[r]);
        }
      }
      const float whole = L.whole[0];
      gd_f4 eo, ey;
#pragma unroll
      for (int r = 0; r < 4; ++r) { eo[r] = enter[r] * dout[r]; ey[r] = -(enter[r] * dy[r]); }
#pragma unroll
      for (int t = 0; t < QD / 4; ++t) {
        gd_f4 kt, qt;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          kt[r] = L.k[(4 * cg + r) * LD + 16 * t + col];
          qt[r] = L.q[(4 * cg + r) * LD + 16 * t + col];
          if (!STATE) L.x[(16 * t + 4 * cg + r) * LD + n] = S[t][r];
          S[t][r] *= whole;
        }
        S[t] = mma16(kt, ey, mma16(qt, eo, S[t]));
      }
    } else if (!STATE) {                                  // columns behind the values' width: the products below read them
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        L.y[(4 * cg + r) * LD + n] = 0.f;
        if (col == 0) L.red[w][0][4 * cg + r] = 0.f;
      }
#pragma unroll
      for (int t = 0; t < QD / 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) L.x[(16 * t + 4 * cg + r) * LD + n] = 0.f;
    }
    if (!STATE) {
      gd_wave_sync();
      {   // dY U^T over this wavefront's sixteen value columns
        gd_f4 u = lds4(&L.e[col * LD + 16 * w + 4 * cg]);
        const float b = L.beta[col];
#pragma unroll
        for (int r = 0; r < 4; ++r) u[r] *= b;
        const gd_f4 z = mma16(lds4(&L.y[col * LD + 16 * w + 4 * cg]), u, zero4());
#pragma unroll
        for (int r = 0; r < 4; ++r) L.part[w][0][(4 * cg + r) * TS + col] = z[r];
      }
      team_sync<D>();
      if (tl < 256) {
#pragma unroll
        for (int m = 0; m < EPL; ++m) {
          const int el = tl + m * TL, i = el >> 4, j = el & 15;
          float yu = 0.f;
#pragma unroll
          for (int u = 0; u < NW; ++u) yu += L.part[u][0][i * TS + j];
          L.m2[i * TS + j] = -(yu * el_d[m]);
          L.xm[i * TS + j] = el_x[m] - yu * el_kd[m];
        }
      }
      team_sync<D>();
      if (kcols) {
        gd_f4 aq = zero4(), ak = zero4(), al = zero4();
        float dot = 0.f;
#pragma unroll
        for (int t = 0; t < QD / 4; ++t) {
          aq = mma16(lds4(&L.o[col * LD + 16 * t + 4 * cg]), s0[t], aq);
          ak = mma16(lds4(&L.y[col * LD + 16 * t + 4 * cg]), s0[t], ak);
          const gd_f4 x = lds4(&L.x[n * LD + 16 * t + 4 * cg]);
          gd_f4 u = lds4(&L.e[col * LD + 16 * t + 4 * cg]);
          const float b = L.beta[col];
#pragma unroll
          for (int r = 0; r < 4; ++r) { u[r] *= b; dot = fmaf(s0[t][r], x[r], dot); }
          al = mma16(u, x, al);
        }
        gd_f4 kc, qc, m1 = lds4(&L.m1[col * TS + 4 * cg]), m1t, m2 = lds4(&L.m2[col * TS + 4 * cg]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          kc[r] = L.k[(4 * cg + r) * LD + n];
          qc[r] = L.q[(4 * cg + r) * LD + n];
          m1t[r] = L.m1[(4 * cg + r) * TS + col];
          m2[r] += L.m2[(4 * cg + r) * TS + col];
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          aq[r] *= enter[r];
          ak[r] *= -enter[r];
          al[r] *= leave[r];
          const float z = sum16(qc[r] * aq[r] + kc[r] * ak[r]), wj = sum16(kc[r] * al[r]);
          if (col == 0) { L.red[w][1][4 * cg + r] = z; L.red[w][2][4 * cg + r] = wj; }
          ak[r] += al[r];
        }
        dot = sum16(dot);
        if (col == 0) L.red[w][3][cg] = dot;
        aq = mma16(m1, kc, aq);
        ak = mma16(m2, kc, ak);
        ak = mma16(m1t, qc, ak);
        if (sq.live && n < s.K) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int t = 16 * c + 4 * cg + r;
            if (t < s.T) {
              const int64_t off = (s.rep > 1 ? seq_h + t * row_h : (((int64_t)sq.b * s.T + t) * s.N + sq.n) * s.H + kh) * s.K + n;
              if (s.rep > 1) {
                reinterpret_cast<float*>(a.dq)[off] = aq[r] * s.scale;
                reinterpret_cast<float*>(a.dk)[off] = ak[r];
              } else {
                reinterpret_cast<IO*>(a.dq)[off] = from_f32<IO>(aq[r] * s.scale);
                reinterpret_cast<IO*>(a.dk)[off] = from_f32<IO>(ak[r]);
              }
            }
          }
        }
      } else if (lane < 16) {
        L.red[w][1][lane] = 0.f;
        L.red[w][2][lane] = 0.f;
        L.red[w][3][lane] = 0.f;
      }
      team_sync<D>();
      if (w == 0) {
        // lane l (of the first sixteen): dbeta_l; dg_l = c_l + sum_{i >= l} z_i + sum_{j < l} w_j + whole <S0, dS>
        float db = 0.f, z = 0.f, wj = 0.f, dot = 0.f;
#pragma unroll
        for (int u = 0; u < NW; ++u) {
          db += L.red[u][0][col];
          z += L.red[u][1][col];
          wj += L.red[u][2][col];
#pragma unroll
          for (int i = 0; i < 4; ++i) dot += L.red[u][3][i];
        }
        float dg = dot * L.whole[0];
        for (int i = 0; i < 16; ++i) {
          const float zi = __shfl(z, i, 16), wi = __shfl(wj, i, 16);
          dg += i >= col ? zi : wi;
        }
        float c_l = 0.f;                                  // the tile's entries left of column l in the rows from l on
        for (int i = 1; i < 16; ++i)
          for (int jj = 0; jj < 4; ++jj) {
            const int j = 4 * cg + jj;
            c_l += i >= col && j < col ? L.xm[i * TS + j] : 0.f;
          }
        c_l += __shfl_xor(c_l, 16);
        c_l += __shfl_xor(c_l, 32);
        dg += c_l;
        const int t = 16 * c + col;
        if (sq.live && cg == 0 && t < s.T) {
          a.dbeta[seq_h + t * row_h] = t < sq.len ? db : 0.f;
          a.dg[seq_h + t * row_h] = t < sq.len ? dg : 0.f;
        }
      }
    } else {
      team_sync<D>();
    }
  }

  if (sq.live) {
    float* to = STATE ? a.seg_end + (sq.p * (s.segs - 1) + seg - 1) * s.K * s.V : seg == 0 && a.d_start ? a.d_start + sq.p * s.K * s.V : nullptr;
    if (to) {
#pragma unroll
      for (int t = 0; t < QD / 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = 16 * t + 4 * cg + r;
          if (row < s.K && n < s.V) to[(int64_t)row * s.V + n] = S[t][r];
        }
    }
    if (!STATE) {                                         // rows behind the sequence: zero
      const int lo = 16 * (ce > c0 ? ce : c0), hi = 16 * c1 < s.T ? 16 * c1 : s.T;
      for (int t = lo + tok; t < hi; t += 16) {
        const int64_t row = seq_h + t * row_h, krow = s.rep > 1 ? row : (((int64_t)sq.b * s.T + t) * s.N + sq.n) * s.H + kh;
        for (int r = 0; r < 4; ++r) {
          if (qd + r < s.V) reinterpret_cast<IO*>(a.dv)[row * s.V + qd + r] = from_f32<IO>(0.f);
          if (qd + r < s.K) {
            if (s.rep > 1) {
              reinterpret_cast<float*>(a.dq)[krow * s.K + qd + r] = 0.f;
              reinterpret_cast<float*>(a.dk)[krow * s.K + qd + r] = 0.f;
            } else {
              reinterpret_cast<IO*>(a.dq)[krow * s.K + qd + r] = from_f32<IO>(0.f);
              reinterpret_cast<IO*>(a.dk)[krow * s.K + qd + r] = from_f32<IO>(0.f);
            }
          }
        }
        if (qd == 0) { a.dbeta[row] = 0.f; a.dg[row] = 0.f; }
      }
    }
  }
}

// y[row, kh, :] = sum over the key head's value heads of x[row, kh rep + i, :], in head order
template <class IO>
__global__ __launch_bounds__(256) void delta_heads_kernel(const float* x, IO* y, int64_t n, int rep, int K) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const int64_t head = i / K;
  const float* p = x + head * rep * K + (i - head * K);
  float acc = 0.f;
  for (int r = 0; r < rep; ++r) acc += p[(int64_t)r * K];
  y[i] = from_f32<IO>(acc);
}

template <class IO, int D, bool STATE> void go(const BwdArgs& a0, pgt_stream_t stream) {
  using TM = Team<D>;
  BwdArgs a = a0;
  const int64_t most = (int64_t)1 << 21;
  for (int64_t p0 = 0; p0 < a.s.P; p0 += most * TM::TEAMS) {
    a.s.p0 = p0;
    const int64_t wgs = pgt_cdiv(a.s.P - p0, TM::TEAMS);
    const dim3 grid((unsigned)(wgs < most ? wgs : most), (unsigned)(STATE ? a.s.segs - 1 : a.s.segs));
    PGT_LAUNCH((delta_bwd_kernel<IO, D, STATE>), grid, dim3(TM::THREADS), stream, a);
  }
}
template <class IO, int D> int all(const BwdArgs& a, const float* seg_trans, pgt_stream_t stream) {
  if (a.s.segs > 1) {
    go<IO, D, true>(a, stream);
    if (a.s.segs > 2)
      if (int e = pgt_delta_join_up(seg_trans, a.seg_end, a.s.P, a.s.segs, a.s.K, a.s.V, stream)) return e;
  }
  go<IO, D, false>(a, stream);
  return pgt_check_launch("pgt_gated_delta_bwd");
}
template <class IO> int by_width(const BwdArgs& a0, void* dq, void* dk, const float* seg_trans, pgt_stream_t stream) {
  const BwdArgs& a = a0;
  const int d = a.s.K > a.s.V ? a.s.K : a.s.V;
  int e;
  if (d <= 16) e = all<IO, 16>(a, seg_trans, stream);
  else if (d <= 32) e = all<IO, 32>(a, seg_trans, stream);
  else if (d <= 64) e = all<IO, 64>(a, seg_trans, stream);
  else e = all<IO, 128>(a, seg_trans, stream);
  if (e || a.s.rep == 1) return e;
  const int64_t n = (a.s.P / a.s.rep) * a.s.T * a.s.K;
  if (n == 0) return PGT_OK;
  const dim3 grid((unsigned)pgt_cdiv(n, 256));
  PGT_LAUNCH((delta_heads_kernel<IO>), grid, dim3(256), stream, (const float*)a.dq, (IO*)dq, n, a.s.rep, a.s.K);
  PGT_LAUNCH((delta_heads_kernel<IO>), grid, dim3(256), stream, (const float*)a.dk, (IO*)dk, n, a.s.rep, a.s.K);
  return pgt_check_launch("pgt_gated_delta_bwd");
}

}  // namespace

extern "C" int pgt_gated_delta_bwd(const pgt_delta_dims* d, const pgt_seq_view* q, const pgt_seq_view* k, const pgt_seq_view* g,
                                   const pgt_seq_view* beta, const float* start, const float* e, const float* states,
                                   const float* seg_trans, const void* d_o, const float* d_last, void* dq, void* dk, void* dv,
                                   float* dg, float* dbeta, float* d_start, float* head_ws, float* seg_end, pgt_stream_t stream) {
  BwdArgs a;
  if (int rc = pgt_delta_shape(d, "pgt_gated_delta_bwd", &a.s)) return rc;
  if (a.s.P == 0) return PGT_OK;
  if (a.s.T > 0) {
    PGT_REQUIRE(q && k && g && beta && q->data && k->data && g->data && beta->data && e && d_o && dq && dk && dv && dg && dbeta,
                "pgt_gated_delta_bwd: null pointer");
    PGT_REQUIRE(a.s.chunks == 1 || states, "pgt_gated_delta_bwd: %d chunks need the forward pass's states", a.s.chunks);
    a.q = pgt_delta_view(q); a.k = pgt_delta_view(k); a.g = pgt_delta_view(g); a.beta = pgt_delta_view(beta);
    a.vec = pgt_delta_vec(q, a.s.K, d->dtype) && pgt_delta_vec(k, a.s.K, d->dtype);
  } else {
    a.q = a.k = a.g = a.beta = View{nullptr, 0, 0, 0, 0};
    a.vec = 0;
  }
  PGT_REQUIRE(a.s.segs == 1 || (seg_trans && seg_end), "pgt_gated_delta_bwd: a sequence in %d segments needs seg_trans and seg_end", a.s.segs);
  PGT_REQUIRE(a.s.rep == 1 || head_ws || a.s.T == 0, "pgt_gated_delta_bwd: shared key heads need head_ws");
  const int64_t n = a.s.P * a.s.T * a.s.K;
  PGT_REQUIRE(n / 256 < ((int64_t)1 << 24) * a.s.rep || a.s.rep == 1, "pgt_gated_delta_bwd: size out of range");
  a.d_o = d_o; a.e = e; a.start = start; a.states = states; a.d_last = d_last;
  a.dq = a.s.rep > 1 ? (void*)head_ws : dq;
  a.dk = a.s.rep > 1 ? (void*)(head_ws + n) : dk;
  a.dv = dv; a.dg = dg; a.dbeta = dbeta; a.d_start = d_start; a.seg_end = seg_end;
  a.vec_do = a.s.V % 4 == 0 && pgt_aligned(d_o, d->dtype == PGT_DT_F32 ? 16 : 8);
  a.vec_e = a.s.V % 4 == 0 && pgt_aligned(e, 16);
  a.vec_s = a.s.V % 4 == 0 && pgt_aligned(states, 16) && pgt_aligned(start, 16);
  if (d->dtype == PGT_DT_F32) return by_width<float>(a, dq, dk, seg_trans, stream);
  if (d->dtype == PGT_DT_BF16) return by_width<bf16>(a, dq, dk, seg_trans, stream);
  return by_width<f16>(a, dq, dk, seg_trans, stream);
}
