// Gated delta rule, whole sequences, forward (delta_common.h has the formulas).
#include "delta_common.h"

using namespace gd;

namespace {

struct FwdArgs {
  Shape s;
  View q, k, v, g, beta;
  const float* start;            // [P, K, V] or null
  void* o;                       // [B, T, N, H, V]
  float* last;                   // [P, K, V]: the state behind the last step
  float* e;                      // [B, T, N, H, V] or null: the misses e_t, kept for the adjoint
  float* states;                 // [P, chunks - 1, K, V] or null: the state before every chunk but the first, kept for the adjoint
  float* seg_start;              // [P, segs - 1, K, V]: the state before every segment but the first
  float* seg_trans;              // [P, segs - 2, K, K]: what the inner segments multiply their start state by
  int vec;                       // q, k, v rows can be read four values at a time
};

// One team per sequence and segment of chunks.  PASS 0: outputs.  PASS 1: only the state behind the segment, from a zero start
// (the first segment: from the sequence's); PASS 2: the segment's transition matrix, i.e. the same recurrence with v = 0 from the unit
// matrix.  Passes 1 and 2 are what a long sequence with few heads is split with; one launch runs both (blockIdx.z).
template <class IO, int D, bool TRANS>
__global__ __launch_bounds__(Team<D>::THREADS) void delta_fwd_kernel(FwdArgs a) {
  using TM = Team<D>;
  constexpr int NW = TM::NW, LD = TM::LD, TL = TM::TL, QD = D / 4, EPL = TM::EPL;
  struct Lds {
    float k[16 * LD], q[16 * LD], v[16 * LD];
    float part[NW][2][TILE];
    float am[TILE], pm[TILE];
    float hi[16], lo[16], enter[16], leave[16], beta[16], whole[4];
  };
  __shared__ __attribute__((aligned(16))) char smem[sizeof(Lds) * TM::TEAMS];
  const Shape& s = a.s;
  const int tid = (int)threadIdx.x, team = tid / TL, tl = tid % TL, w = PGT_UNIFORM(tl / 64), lane = tid & 63, col = lane & 15, cg = lane >> 4;
  Lds& L = reinterpret_cast<Lds*>(smem)[team];
  const int64_t first = s.p0 + (int64_t)blockIdx.x * TM::TEAMS;
  const Seq sq = seq_of(s, first + team);
  const int seg = (int)blockIdx.y;
  const bool unit = TRANS && blockIdx.z == 1;             // the transition matrix
  if (TRANS && unit && seg == 0) return;
  const int c0 = seg * s.cps, c1 = c0 + s.cps < s.chunks ? c0 + s.cps : s.chunks;
  const int reach = chunks_of_block<TM::TEAMS>(s, first), ce = reach < c1 ? reach : c1;
  const int kh = sq.h / s.rep, cols = unit ? s.K : s.V;
  const IO* kp = at<IO>(a.k, sq, kh);
  const IO* qp = at<IO>(a.q, sq, kh);
  const IO* vp = at<IO>(a.v, sq, sq.h);
  const float* gp = at<float>(a.g, sq, sq.h);
  const float* bp = at<float>(a.beta, sq, sq.h);
  const bool vec = a.vec != 0;
  const int n = 16 * w + col;                             // this lane's column of the state
  const bool mine = 16 * w < cols;                        // a wavefront behind the width only helps with the tiles

  gd_f4 S[QD / 4];
#pragma unroll
  for (int t = 0; t < QD / 4; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 16 * t + 4 * cg + r;
      float x = 0.f;
      if (unit) {
        x = row == n ? 1.f : 0.f;
      } else if (sq.live && row < s.K && n < s.V) {
        if (seg == 0) { if (a.start) x = a.start[(sq.p * s.K + row) * s.V + n]; }
        else if (!TRANS) x = a.seg_start[((sq.p * (s.segs - 1) + seg - 1) * s.K + row) * s.V + n];
      }
      S[t][r] = x;
    }

  const int tok = tl / QD, qd = 4 * (tl % QD);
  gd_f4 nk = zero4(), nq = zero4(), nv = zero4();
  float ng = 0.f, nb = 0.f;
  auto fetch = [&](int c) {
    const int t = 16 * c + tok;
    const bool in = t < sq.len;
    nk = load4(kp + (int64_t)t * a.k.st + qd, in ? s.K - qd : 0, vec);
    if (!TRANS) nq = load4(qp + (int64_t)t * a.q.st + qd, in ? s.K - qd : 0, vec);
    if (!unit) nv = load4(vp + (int64_t)t * a.v.st + qd, in ? s.V - qd : 0, vec);
    if (w == 0) {
      const int tg = 16 * c + col;
      ng = tg < sq.len ? gp[(int64_t)tg * a.g.st] : 0.f;
      nb = tg < sq.len ? bp[(int64_t)tg * a.beta.st] : 0.f;
    }
  };
  if (c0 < ce) fetch(c0);
  for (int c = c0; c < ce; ++c) {
    put4(&L.k[tok * LD + qd], nk);
    if (!TRANS) {
#pragma unroll
      for (int r = 0; r < 4; ++r) nq[r] *= s.scale;
      put4(&L.q[tok * LD + qd], nq);
    }
    put4(&L.v[tok * LD + qd], nv);
    if (w == 0) {
      const Decay d = chunk_decay(ng);
      if (lane < 16) {
        L.hi[lane] = d.hi; L.lo[lane] = d.lo; L.enter[lane] = d.enter; L.leave[lane] = d.leave; L.beta[lane] = nb;
        if (lane == 0) L.whole[0] = d.whole;
      }
    }
    if (c + 1 < ce) fetch(c + 1);
    if (!TRANS && a.states && c > 0 && sq.live) {
      float* to = a.states + (sq.p * (s.chunks - 1) + c - 1) * s.K * s.V;
#pragma unroll
      for (int t = 0; t < QD / 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = 16 * t + 4 * cg + r;
          if (row < s.K && n < s.V) to[(int64_t)row * s.V + n] = S[t][r];
        }
    }
    team_sync<D>();
    {   // this wavefront's sixteen key columns of K K^T and Q K^T
      const gd_f4 kk = lds4(&L.k[col * LD + 16 * w + 4 * cg]);
      gd_f4 x = mma16(kk, kk, zero4()), y = zero4();
      if (!TRANS) y = mma16(lds4(&L.q[col * LD + 16 * w + 4 * cg]), kk, zero4());
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        L.part[w][0][(4 * cg + r) * TS + col] = x[r];
        if (!TRANS) L.part[w][1][(4 * cg + r) * TS + col] = y[r];
      }
    }
    team_sync<D>();
    if (tl < 256) {
#pragma unroll
      for (int m = 0; m < EPL; ++m) {
        const int el = tl + m * TL, i = el >> 4, j = el & 15;
        float kk = 0.f, qk = 0.f;
#pragma unroll
        for (int u = 0; u < NW; ++u) {
          kk += L.part[u][0][i * TS + j];
          if (!TRANS) qk += L.part[u][1][i * TS + j];
        }
        const float d = j <= i ? expf((L.hi[i] - L.hi[j]) + (L.lo[i] - L.lo[j])) : 0.f;
        L.am[i * TS + j] = j < i ? d * kk * L.beta[j] : 0.f;
        if (!TRANS) L.pm[i * TS + j] = j <= i ? d * qk : 0.f;
      }
    }
    team_sync<D>();
    if (mine) {
      float arow[16];
      row16(&L.am[col * TS], arow);
      gd_f4 inv = unit_row(lane);
      solve_down<0>(arow, inv);
      gd_f4 ks = zero4(), qs = zero4();
#pragma unroll
      for (int t = 0; t < QD / 4; ++t) {
        ks = mma16(lds4(&L.k[col * LD + 16 * t + 4 * cg]), S[t], ks);
        if (!TRANS) qs = mma16(lds4(&L.q[col * LD + 16 * t + 4 * cg]), S[t], qs);
      }
      const gd_f4 enter = lds4(&L.enter[4 * cg]), leave = lds4(&L.leave[4 * cg]), beta = lds4(&L.beta[4 * cg]);
      gd_f4 y, u, ul;
#pragma unroll
      for (int r = 0; r < 4; ++r) y[r] = (unit ? 0.f : L.v[(4 * cg + r) * LD + n]) - enter[r] * ks[r];
      const gd_f4 e = mma16(inv, y, zero4());
#pragma unroll
      for (int r = 0; r < 4; ++r) { u[r] = beta[r] * e[r]; ul[r] = leave[r] * u[r]; }
      if (!TRANS) {
#pragma unroll
        for (int r = 0; r < 4; ++r) qs[r] *= enter[r];
        const gd_f4 o = mma16(lds4(&L.pm[col * TS + 4 * cg]), u, qs);
        if (sq.live && n < s.V) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int t = 16 * c + 4 * cg + r;
            if (t < s.T) {
              const int64_t off = ((((int64_t)sq.b * s.T + t) * s.N + sq.n) * s.H + sq.h) * s.V + n;
              reinterpret_cast<IO*>(a.o)[off] = from_f32<IO>(o[r]);
              if (a.e) a.e[off] = e[r];
            }
          }
        }
      }
      const float whole = L.whole[0];
#pragma unroll
      for (int t = 0; t < QD / 4; ++t) {
        gd_f4 kt;
#pragma unroll
        for (int r = 0; r < 4; ++r) { kt[r] = L.k[(4 * cg + r) * LD + 16 * t + col]; S[t][r] *= whole; }
        S[t] = mma16(kt, ul, S[t]);
      }
    }
    team_sync<D>();
  }

  if (sq.live) {
    float* to;
    int64_t ld = s.V;
    if (unit) { to = a.seg_trans + (sq.p * (s.segs - 2) + seg - 1) * s.K * s.K; ld = s.K; }
    else if (TRANS) to = a.seg_start + (sq.p * (s.segs - 1) + seg) * s.K * s.V;
    else to = seg == s.segs - 1 ? a.last + sq.p * s.K * s.V : nullptr;
    if (to) {
#pragma unroll
      for (int t = 0; t < QD / 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = 16 * t + 4 * cg + r;
          if (row < s.K && n < cols) to[(int64_t)row * ld + n] = S[t][r];
        }
    }
    if (!TRANS) {                                         // rows behind the sequence: zero
      const int lo = 16 * (ce > c0 ? ce : c0), hi = 16 * c1 < s.T ? 16 * c1 : s.T;
      for (int t = lo + tok; t < hi; t += 16) {
        const int64_t off = ((((int64_t)sq.b * s.T + t) * s.N + sq.n) * s.H + sq.h) * s.V;
        for (int r = 0; r < 4; ++r)
          if (qd + r < s.V) reinterpret_cast<IO*>(a.o)[off + qd + r] = from_f32<IO>(0.f);
      }
    }
  }
}

// Joins the segments: the state before segment j + 1 is (transition of segment j) (state before segment j) + (what segment j adds), where
// x [P, segs - 1, K, V] holds the second summand and takes the sum (its entry 0 is complete already).  UP (the adjoint): from the last
// entry down with the transposed transitions.  A workgroup owns sixteen columns of a sequence's state; a wavefront sixteen rows.
template <int D, bool UP>
__global__ __launch_bounds__(64 * (D / 16)) void delta_join_kernel(const float* trans, float* x, int segs, int K, int V) {
  constexpr int LD = D + 4;
  __shared__ __attribute__((aligned(16))) float st[2][16 * LD];     // [column][row], two buffers
  const int w = (int)threadIdx.x / 64, lane = (int)threadIdx.x & 63, col = lane & 15, cg = lane >> 4;
  const int64_t p = blockIdx.x;
  const int n = 16 * (int)blockIdx.y + col, row0 = 16 * w + 4 * cg;
  const int entries = segs - 1;
  auto value = [&](int j, int r) -> float* { return x + ((p * entries + j) * K + row0 + r) * V + n; };
  gd_f4 s;
#pragma unroll
  for (int r = 0; r < 4; ++r) s[r] = row0 + r < K && n < V ? *value(UP ? entries - 1 : 0, r) : 0.f;
  for (int j = 1; j < entries; ++j) {
    const int to = UP ? entries - 1 - j : j;              // entry `to` takes the transition of segment `tr`
    const int tr = UP ? entries - j : j;
    const float* m = trans + (p * (segs - 2) + tr - 1) * K * K;
    float* buf = st[j & 1];
    put4(&buf[col * LD + row0], s);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 4; ++r) s[r] = row0 + r < K && n < V ? *value(to, r) : 0.f;
#pragma unroll
    for (int t = 0; t < D / 16; ++t) {
      gd_f4 am;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * w + col, k = 16 * t + 4 * cg + r;
        am[r] = i < K && k < K ? (UP ? m[(int64_t)k * K + i] : m[(int64_t)i * K + k]) : 0.f;
      }
      s = mma16(am, lds4(&buf[col * LD + 16 * t + 4 * cg]), s);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (row0 + r < K && n < V) *value(to, r) = s[r];
  }
}

template <class IO, int D, bool TRANS> void go(const FwdArgs& a0, pgt_stream_t stream) {
  using TM = Team<D>;
  FwdArgs a = a0;
  const int64_t most = (int64_t)1 << 21;                  // workgroups of a launch: the grid's threads stay below 2^32
  for (int64_t p0 = 0; p0 < a.s.P; p0 += most * TM::TEAMS) {
    a.s.p0 = p0;
    const int64_t wgs = pgt_cdiv(a.s.P - p0, TM::TEAMS);
    const dim3 grid((unsigned)(wgs < most ? wgs : most), (unsigned)(TRANS ? a.s.segs - 1 : a.s.segs), TRANS && a.s.segs > 2 ? 2 : 1);
    PGT_LAUNCH((delta_fwd_kernel<IO, D, TRANS>), grid, dim3(TM::THREADS), stream, a);
  }
}
template <class IO, int D> void all(const FwdArgs& a, pgt_stream_t stream) {
  if (a.s.segs > 1) {
    go<IO, D, true>(a, stream);
    if (a.s.segs > 2) {
      const dim3 grid((unsigned)a.s.P, (unsigned)((a.s.V + 15) / 16));
      PGT_LAUNCH((delta_join_kernel<D, false>), grid, dim3(64 * (D / 16)), stream, (const float*)a.seg_trans, a.seg_start, a.s.segs, a.s.K, a.s.V);
    }
  }
  go<IO, D, false>(a, stream);
}
template <class IO> void by_width(const FwdArgs& a, pgt_stream_t stream) {
  const int d = a.s.K > a.s.V ? a.s.K : a.s.V;
  if (d <= 16) all<IO, 16>(a, stream);
  else if (d <= 32) all<IO, 32>(a, stream);
  else if (d <= 64) all<IO, 64>(a, stream);
  else all<IO, 128>(a, stream);
}

}  // namespace

int pgt_delta_join_up(const float* trans, float* x, int64_t P, int segs, int K, int V, pgt_stream_t stream) {
  const dim3 grid((unsigned)P, (unsigned)((V + 15) / 16));
  const int d = K > V ? K : V;
  if (d <= 16) PGT_LAUNCH((delta_join_kernel<16, true>), grid, dim3(64), stream, trans, x, segs, K, V);
  else if (d <= 32) PGT_LAUNCH((delta_join_kernel<32, true>), grid, dim3(128), stream, trans, x, segs, K, V);
  else if (d <= 64) PGT_LAUNCH((delta_join_kernel<64, true>), grid, dim3(256), stream, trans, x, segs, K, V);
  else PGT_LAUNCH((delta_join_kernel<128, true>), grid, dim3(512), stream, trans, x, segs, K, V);
  return pgt_check_launch("pgt_gated_delta_bwd");
}

// the shape's kernel arguments and plan, checked; 0 or an error code
int pgt_delta_shape(const pgt_delta_dims* d, const char* who, gd::Shape* s) {
  PGT_REQUIRE(d, "%s: null dims", who);
  PGT_REQUIRE(d->batch >= 0 && d->steps >= 0 && d->nodes >= 0, "%s: negative size", who);
  PGT_REQUIRE(d->dtype == PGT_DT_F32 || d->dtype == PGT_DT_BF16 || d->dtype == PGT_DT_F16, "%s: unknown dtype %d", who, d->dtype);
  PGT_REQUIRE(d->key >= 1 && d->key <= 128 && d->value >= 1 && d->value <= 128, "%s: head widths 1 .. 128 (key %d, value %d)", who, d->key, d->value);
  PGT_REQUIRE(d->k_heads >= 1 && d->heads >= 1 && d->heads % d->k_heads == 0, "%s: %d value heads do not divide over %d key heads", who, d->heads, d->k_heads);
  PGT_REQUIRE(d->steps < ((int64_t)1 << 30) && d->nodes < ((int64_t)1 << 31) && d->heads <= 65536, "%s: size out of range", who);
  PGT_REQUIRE(d->batch == 0 || d->nodes == 0 || d->batch <= ((int64_t)1 << 31) / d->nodes / d->heads, "%s: more than 2^31 sequences", who);
  s->P = d->batch * d->nodes * d->heads;
  s->p0 = 0;
  s->N = (int)d->nodes; s->H = d->heads; s->rep = d->heads / d->k_heads; s->T = (int)d->steps; s->K = d->key; s->V = d->value;
  s->chunks = (int)((d->steps + 15) / 16);
  s->lengths = d->lengths;
  s->scale = d->scale;
  // Segments: a sequence is walked chunk by chunk; with few sequences most of the 256 CUs idle.  Splitting it costs two more
  // recurrences (a segment's own addition and its transition matrix) but divides the walk.
  const int width = s->K > s->V ? s->K : s->V;
  const int64_t teams_per_wg = width <= 16 ? 4 : width <= 32 ? 2 : 1;
  const int64_t wgs = pgt_cdiv(s->P, teams_per_wg);
  int segs = 1;
  if (wgs > 0 && wgs < 128 && s->chunks >= 16) {
    const int64_t most = 512 / wgs, by_length = s->chunks / 4;
    segs = (int)(most < by_length ? most : by_length);
    if (segs > 64) segs = 64;
    if (segs < 3) segs = 1;
  }
  s->cps = segs > 1 ? (s->chunks + segs - 1) / segs : (s->chunks > 0 ? s->chunks : 1);
  s->segs = s->chunks > 0 ? (s->chunks + s->cps - 1) / s->cps : 1;
  if (s->segs < 3) { s->segs = 1; s->cps = s->chunks > 0 ? s->chunks : 1; }
  return PGT_OK;
}
gd::View pgt_delta_view(const pgt_seq_view* v) { return gd::View{v->data, v->batch, v->step, v->node, v->head}; }
bool pgt_delta_vec(const pgt_seq_view* v, int width, int dtype) {
  const int64_t strides = v->batch | v->step | v->node | v->head;
  return width % 4 == 0 && strides % 4 == 0 && pgt_aligned(v->data, dtype == PGT_DT_F32 ? 16 : 8);
}

extern "C" int pgt_gated_delta_segments(const pgt_delta_dims* d) {
  gd::Shape s;
  if (int e = pgt_delta_shape(d, "pgt_gated_delta_segments", &s)) return e;
  return s.segs;
}

extern "C" int pgt_gated_delta_fwd(const pgt_delta_dims* d, const pgt_seq_view* q, const pgt_seq_view* k, const pgt_seq_view* v,
                                   const pgt_seq_view* g, const pgt_seq_view* beta, const float* start, void* o, float* last,
                                   float* e, float* states, float* seg_start, float* seg_trans, pgt_stream_t stream) {
  FwdArgs a;
  if (int rc = pgt_delta_shape(d, "pgt_gated_delta_fwd", &a.s)) return rc;
  if (a.s.P == 0) return PGT_OK;
  PGT_REQUIRE(last, "pgt_gated_delta_fwd: null pointer");
  if (a.s.T > 0) {
    PGT_REQUIRE(q && k && v && g && beta && q->data && k->data && v->data && g->data && beta->data && o, "pgt_gated_delta_fwd: null pointer");
    a.q = pgt_delta_view(q); a.k = pgt_delta_view(k); a.v = pgt_delta_view(v); a.g = pgt_delta_view(g); a.beta = pgt_delta_view(beta);
    a.vec = pgt_delta_vec(q, a.s.K, d->dtype) && pgt_delta_vec(k, a.s.K, d->dtype) && pgt_delta_vec(v, a.s.V, d->dtype);
  } else {
    a.q = a.k = a.v = a.g = a.beta = View{nullptr, 0, 0, 0, 0};
    a.vec = 0;
  }
  PGT_REQUIRE(a.s.segs == 1 || (seg_start && seg_trans), "pgt_gated_delta_fwd: a sequence in %d segments needs seg_start and seg_trans", a.s.segs);
  a.start = start; a.o = o; a.last = last; a.e = e; a.states = states; a.seg_start = seg_start; a.seg_trans = seg_trans;
  if (d->dtype == PGT_DT_F32) by_width<float>(a, stream);
  else if (d->dtype == PGT_DT_BF16) by_width<bf16>(a, stream);
  else by_width<f16>(a, stream);
  return pgt_check_launch("pgt_gated_delta_fwd");
}
