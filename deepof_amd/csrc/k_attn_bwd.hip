// Attention over packed documents, backward: two kernels that recompute the probabilities from the forward's log-sum-exp.
//
//   p = exp(s - lse) ; dp_ij = g_i.v_j ; ds = p (dp - delta_i) c_ij, delta_i = sum_d g_id o_id, c = 1 - tanh^2 under a cap, else 1
//   dq_i = scale sum_j ds_ij k_j        (k_attn_dq:  a workgroup per query tile, walks the keys as the forward does)
//   dv_j = sum_i p_ij g_i, dk_j = scale sum_i ds_ij q_i   (k_attn_dkv: a workgroup per key tile, walks the query rows that see it,
//                                                          through all query heads of its group)
//
// Every gradient element is summed by one workgroup in a fixed order: no atomics, the same bits on every run.  The price is that S
// and dP are computed twice (seven products of the size of S instead of five).  Both kernels keep their own rows' operands in
// registers and stream the other side through LDS (two images); the second products take P and dS straight from the registers the
// first ones left them in, as in the forward.  P and dS are rounded to the elements' type for their products; everything that is
// summed is fp32.  fp16 has 5 exponent bits: there P is carried as 2^12 P and dS as 2^6 dS (exact factors, taken out at the end), so
// that weights of long documents and small gradients stay out of its subnormals.
#include <cmath>

#include "deepof_hip.h"
#include "dof_rt.h"
#include "launchers.h"
#include "seq_attn.h"
#include "seq_attn_args.h"

namespace {

template <class T> struct Lift {
  static constexpr float p2 = 0.0f, p = 1.0f, ds = 1.0f;  // log2 of P's factor, P's factor, dS's factor
};
template <> struct Lift<DofF16> {
  static constexpr float p2 = 12.0f, p = 4096.0f, ds = 64.0f;
};

// PLAIN: neither cap nor bias (as in the forward)
template <class T, int DP, int NW, bool PLAIN>
__global__ void __launch_bounds__(64 * NW, sizeof(T) == 4 && DP > 32 ? 1 : 2) k_attn_dq(DofAttnBwd B) {
  const DofAttnFwd& A = B.f;
  // keys per step: 64 where two wavefronts per SIMD still fit (heads of 96: 162 us with 64, 174 with 32; of 128: 2.4 ms and 1.77)
  constexpr int KU = NW == 4 && DP == 96 ? 2 : 1, kKeys = 32 * KU;
  using Tile = DofTile<T, kKeys, DP>;
  using Stage = DofStage<T, kKeys, DP, 64 * NW>;
  __shared__ Tile sk[2], sv[2];
  constexpr int KS = DP / 16, DT = DP / 32;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, half = lane >> 5;
  int tile, h;
  dof_attn_item(blockIdx.x, A.n_tiles, A.q_heads, &tile, &h);
  const DofAttnTile t = A.tiles[tile];
  const int hk = h / (A.q_heads / A.k_heads);

  const int first = t.row0 + 32 * wave, row = first + col;
  const bool live = row < t.lq;
  const int last_wg = (t.row0 + 32 * NW < t.lq ? t.row0 + 32 * NW : t.lq) - 1;
  const int last = (first + 32 < t.lq ? first + 32 : t.lq) - 1;
  const int kmax = dof_attn_kend(t, A.causal, last_wg);
  const int wmax = first < t.lq ? dof_attn_kend(t, A.causal, last) : 0;
  const int wmin = first < t.lq ? dof_attn_kend(t, A.causal, first) : 0;
  const int kend = live ? dof_attn_kend(t, A.causal, row) : 0;
  const int pos = row + t.lk - t.lq;
  DofScore sc = A.score;
  if (A.slopes) sc.slope_l2 = A.slopes[h] * kLog2e;

  DofFrag<T> q[KS], g[KS];
  const T* qp = static_cast<const T*>(A.q) + (t.q0 + row) * A.qs[0] + h * A.qs[1];
  const T* gp = static_cast<const T*>(B.g) + (t.q0 + row) * B.gs[0] + h * B.gs[1];
  const T* op = static_cast<const T*>(A.o) + (t.q0 + row) * A.os[0] + h * A.os[1];
  float delta = 0.0f;
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int e = 16 * s + 8 * half;
    q[s] = g[s] = dof_frag_zero<T>();
    if (live && e < A.dim) {
      q[s] = dof_frag_load<T>(qp + e);
      g[s] = dof_frag_load<T>(gp + e);
      float a[8], b[8];
      dof_frag_unpack<T>(g[s], a);
      dof_frag_unpack<T>(dof_frag_load<T>(op + e), b);
#pragma unroll
      for (int i = 0; i < 8; ++i) delta = fmaf(a[i], b[i], delta);
    }
  }
  delta += dof_swap32(delta);
  const int64_t srow = (t.q0 + row) * A.q_heads + h;
  if (live && half == 0) B.delta[srow] = delta;
  float lse2 = live ? A.lse[srow] * kLog2e : 0.0f;
  if (lse2 == -INFINITY) lse2 = 0.0f;  // a row without keys: every score is masked below
  lse2 -= Lift<T>::p2;
  const T* kp = static_cast<const T*>(A.k) + t.k0 * A.ks[0] + hk * A.ks[1];
  const T* vp = static_cast<const T*>(A.v) + t.k0 * A.vs[0] + hk * A.vs[1];

  dof_f32x16 dq[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) dq[d] = dof_zero16();
  Stage rk, rv;
  if (kmax > 0) {
    rk.load(kp, A.ks[0], t.lk, A.dim, tid);
    rv.load(vp, A.vs[0], t.lk, A.dim, tid);
    rk.store(sk[0], tid);
    rv.store(sv[0], tid);
  }
  for (int j0 = 0, buf = 0; j0 < kmax; j0 += kKeys, buf ^= 1) {
    __syncthreads();
    const int next = j0 + kKeys;
    if (next < kmax) {
      rk.load(kp + next * A.ks[0], A.ks[0], t.lk - next, A.dim, tid);
      rv.load(vp + next * A.vs[0], A.vs[0], t.lk - next, A.dim, tid);
    }
    if (j0 < wmax) {
      const bool partial = j0 + kKeys > wmin;
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        dof_f32x16 x = dof_zero16(), y = dof_zero16();
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          x = dof_mma32<T>(sk[buf].rowfrag(32 * u + col, 2 * s + half), q[s], x);
          y = dof_mma32<T>(sv[buf].rowfrag(32 * u + col, 2 * s + half), g[s], y);
        }
        float ds[16];
        const float base = (float)(pos - j0 - 32 * u - 4 * half);
        const int left = kend - j0 - 32 * u - 4 * half;
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int r = 8 * (v / 4) + v % 4;
          float c = Lift<T>::ds / Lift<T>::p, p;
          if constexpr (PLAIN) {
            p = dof_exp2(fmaf(x[v], sc.mul, -lse2));
          } else {
            float w = x[v] * sc.mul;
            if (sc.cap_l2 != 0.0f) {
              const float th = dof_cap_tanh<T>(x[v], sc.mul);
              w = sc.cap_l2 * th;
              c *= fmaf(-th, th, 1.0f);
            }
            if (A.slopes) w -= sc.slope_l2 * fabsf(base - (float)r);
            p = dof_exp2(w - lse2);
          }
          ds[v] = p * c * (y[v] - delta);
          if (partial && r >= left) ds[v] = 0.0f;  // not 0 x (what a masked key holds)
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const DofFrag<T> f = dof_frag_pack<T>(ds + 8 * s);
          const int r = 32 * u + 16 * s + 4 * half;
#pragma unroll
          for (int d = 0; d < DT; ++d) dq[d] = dof_mma32<T>(sk[buf].colfrag(r, r + 8, 32 * d + col), f, dq[d]);
        }
      }
    }
    if (next < kmax) {
      rk.store(sk[buf ^ 1], tid);
      rv.store(sv[buf ^ 1], tid);
    }
  }
  if (!live) return;
  const float out = B.scale / Lift<T>::ds;
  T* dqp = static_cast<T*>(B.dq) + (t.q0 + row) * B.dqs[0] + h * B.dqs[1];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int v = 0; v < 16; v += 4) {
      const int e = 32 * d + 2 * v + 4 * half;
      if (e < A.dim) {
        const float r[4] = {dq[d][v] * out, dq[d][v + 1] * out, dq[d][v + 2] * out, dq[d][v + 3] * out};
        dof_store_vec<T, 4>(dqp + e, r);
      }
    }
}

// Documents of at most 32 query rows and 32 keys: all three gradients from one pass of one wavefront per document and key head.  S and dP
// are computed once (five products), q, k, v, o and g are read once and delta never leaves the workgroup.  dS turns from "lane = key"
// to "lane = query" through LDS for dq; dk and dv add up over the group's query heads in registers.
template <class T, int DP, bool PLAIN>
__global__ void __launch_bounds__(64, DP <= 32 ? 2 : 1) k_attn_bwd_one(DofAttnBwd B) {
  const DofAttnFwd& A = B.f;
  constexpr int KS = DP / 16, DT = (DP + 31) / 32;
  using Tile = DofTile<T, 32, 32 * DT>;
  using Stage = DofStage<T, 32, 32 * DT, 64>;
  __shared__ Tile sq, sg, sk;
  __shared__ DofTile<T, 32, 32> sds;  // dS, [query][key]
  alignas(16) __shared__ float sl[32];
  alignas(16) __shared__ float sd[32];
  const int lane = threadIdx.x, col = lane & 31, half = lane >> 5;
  const int group = A.q_heads / A.k_heads;
  int tile, hk;
  dof_attn_item(blockIdx.x, A.n_tiles, A.k_heads, &tile, &hk);
  const DofAttnTile t = A.tiles[tile];
  const int off = t.lk - t.lq;
  const bool live = col < t.lk, row = col < t.lq;

  const T* kp = static_cast<const T*>(A.k) + t.k0 * A.ks[0] + hk * A.ks[1];
  const T* vp = static_cast<const T*>(A.v) + (t.k0 + col) * A.vs[0] + hk * A.vs[1];
  Stage rq, rg, rk;
  rk.load(kp, A.ks[0], t.lk, A.dim, lane);
  DofFrag<T> vf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int e = 16 * s + 8 * half;
    vf[s] = dof_frag_zero<T>();
    if (live && e < A.dim) vf[s] = dof_frag_load<T>(vp + e);
  }
  rk.store(sk, lane);
  dof_f32x16 dk[DT], dv[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) dk[d] = dv[d] = dof_zero16();
  // the first row that sees the lane's key
  const int mine = !A.causal || col < t.prefix || col - off < 0 ? 0 : col - off;

  for (int h = hk * group; h < (hk + 1) * group; ++h) {
    rq.load(static_cast<const T*>(A.q) + t.q0 * A.qs[0] + h * A.qs[1], A.qs[0], t.lq, A.dim, lane);
    rg.load(static_cast<const T*>(B.g) + t.q0 * B.gs[0] + h * B.gs[1], B.gs[0], t.lq, A.dim, lane);
    const T* op = static_cast<const T*>(A.o) + (t.q0 + col) * A.os[0] + h * A.os[1];
    DofFrag<T> of[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int e = 16 * s + 8 * half;
      of[s] = dof_frag_zero<T>();
      if (row && e < A.dim) of[s] = dof_frag_load<T>(op + e);
    }
    float lse2 = INFINITY;
    if (row) lse2 = A.lse[(t.q0 + col) * A.q_heads + h] * kLog2e;
    if (lse2 == -INFINITY) lse2 = INFINITY;  // a row without keys takes no part
    __syncthreads();  // the previous head's reads are done
    rq.store(sq, lane);
    rg.store(sg, lane);
    __syncthreads();
    float delta = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      float a[8], b[8];
      dof_frag_unpack<T>(sg.rowfrag(col, 2 * s + half), a);
      dof_frag_unpack<T>(of[s], b);
#pragma unroll
      for (int i = 0; i < 8; ++i) delta = fmaf(a[i], b[i], delta);
    }
    delta += dof_swap32(delta);
    if (half == 0) {
      sl[col] = lse2 - Lift<T>::p2;
      sd[col] = delta;
    }
    __syncthreads();
    dof_f32x16 x = dof_zero16(), y = dof_zero16();
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      x = dof_mma32<T>(sq.rowfrag(col, 2 * s + half), sk.rowfrag(col, 2 * s + half), x);
      y = dof_mma32<T>(sg.rowfrag(col, 2 * s + half), vf[s], y);
    }
    float p[16], ds[16];
    const float slope = !PLAIN && A.slopes ? A.slopes[h] * kLog2e : 0.0f;
    const float base = (float)(off + 4 * half - col);
    const int left = live ? mine - 4 * half : 32;
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      const int r = 8 * (v / 4) + v % 4;
      float c = Lift<T>::ds / Lift<T>::p;
      const float ls = sl[r + 4 * half];
      if constexpr (PLAIN) {
        p[v] = dof_exp2(fmaf(x[v], A.score.mul, -ls));
      } else {
        float w = x[v] * A.score.mul;
        if (A.score.cap_l2 != 0.0f) {
          const float th = dof_cap_tanh<T>(x[v], A.score.mul);
          w = A.score.cap_l2 * th;
          c *= fmaf(-th, th, 1.0f);
        }
        if (A.slopes) w -= slope * fabsf(base + (float)r);
        p[v] = dof_exp2(w - ls);
      }
      ds[v] = p[v] * c * (y[v] - sd[r + 4 * half]);
      if (r < left) p[v] = ds[v] = 0.0f;
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const DofFrag<T> pf = dof_frag_pack<T>(p + 8 * s), df = dof_frag_pack<T>(ds + 8 * s);
      const int r = 16 * s + 4 * half;
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        dv[d] = dof_mma32<T>(sg.colfrag(r, r + 8, 32 * d + col), pf, dv[d]);
        dk[d] = dof_mma32<T>(sq.colfrag(r, r + 8, 32 * d + col), df, dk[d]);
      }
    }
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      const int r = 8 * (v / 4) + v % 4 + 4 * half;
      DofElem<T>::put(reinterpret_cast<T*>(sds.mem + sds.offset(r, col / Tile::EPC)) + col % Tile::EPC, ds[v]);
    }
    __syncthreads();
    // dq (queries in registers, d over the lanes) = dS K
    dof_f32x16 dq[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) dq[d] = dof_zero16();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      // the eight keys of an operand are rows 16 s + 8 half .. of K, four and four
      const DofFrag<T> f = sds.rowfrag(col, 2 * s + half);
      const int r = 16 * s + 8 * half;
#pragma unroll
      for (int d = 0; d < DT; ++d) dq[d] = dof_mma32<T>(f, sk.colfrag(r, r + 4, 32 * d + col), dq[d]);
    }
    const float out = B.scale / Lift<T>::ds;
    T* dqp = static_cast<T*>(B.dq) + t.q0 * B.dqs[0] + h * B.dqs[1];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const int r = 8 * (v / 4) + v % 4 + 4 * half, e = 32 * d + col;
        if (r < t.lq && e < A.dim) DofElem<T>::put(dqp + r * B.dqs[0] + e, dq[d][v] * out);
      }
  }
  if (!live) return;
  T* dkp = static_cast<T*>(B.dk) + (t.k0 + col) * B.dks[0] + hk * B.dks[1];
  T* dvp = static_cast<T*>(B.dv) + (t.k0 + col) * B.dvs[0] + hk * B.dvs[1];
  const float ok = B.scale / Lift<T>::ds, ov = 1.0f / Lift<T>::p;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int v = 0; v < 16; v += 4) {
      const int e = 32 * d + 2 * v + 4 * half;
      if (e >= A.dim) continue;
      const float a[4] = {dk[d][v] * ok, dk[d][v + 1] * ok, dk[d][v + 2] * ok, dk[d][v + 3] * ok};
      const float b[4] = {dv[d][v] * ov, dv[d][v + 1] * ov, dv[d][v + 2] * ov, dv[d][v + 3] * ov};
      dof_store_vec<T, 4>(dkp + e, a);
      dof_store_vec<T, 4>(dvp + e, b);
    }
}

// WANT: 1 = dv, 2 = dk, 3 = both in one pass.  Heads over 64 take two passes: with both accumulators (and their operands) in
// registers only one wavefront fits a SIMD, and one alone does not hide its own latencies (16384 frames, heads of 128: 6.4 ms in one
// pass, 4 products; the two passes run 5).
// A workgroup takes `heads_per` query heads of the group; several workgroups of one key tile leave fp32 parts for k_attn_join.
template <class T, int DP, int NW, bool PLAIN, int WANT>
__global__ void __launch_bounds__(64 * NW, sizeof(T) == 4 && DP > 32 ? 1 : 2) k_attn_dkv(DofAttnBwd B) {
  const DofAttnFwd& A = B.f;
  constexpr bool DV = (WANT & 1) != 0, DK = (WANT & 2) != 0;
  constexpr int kRows = 32;  // query rows per step
  using Tile = DofTile<T, kRows, DP>;
  using Stage = DofStage<T, kRows, DP, 64 * NW>;
  __shared__ Tile sq[2], sg[2];
  alignas(16) __shared__ float sl[2][kRows];  // log-sum-exp in units of log 2 (+inf: the row takes no part)
  alignas(16) __shared__ float sd[2][kRows];  // delta
  constexpr int KS = DP / 16, DT = DP / 32;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, half = lane >> 5;
  const int group = A.q_heads / A.k_heads;
  int tile, unit;
  dof_attn_item(blockIdx.x, A.n_tiles, A.k_heads * B.splits, &tile, &unit);
  const DofAttnTile t = A.tiles[tile];
  const int hk = unit / B.splits, split = unit - hk * B.splits;
  const int h_lo = hk * group + split * B.heads_per;
  const int heads = split * B.heads_per + B.heads_per < group ? B.heads_per : group - split * B.heads_per;
  const int off = t.lk - t.lq;

  const int first = t.row0 + 32 * wave, key = first + col;
  const bool live = key < t.lk;
  // the first query row that sees key j: keys below the prefix are seen by all, key j by the rows from j - off on
  auto row_from = [&](int j) {
    if (!A.causal || j < t.prefix) return 0;
    return j - off > 0 ? j - off : 0;
  };
  const int i_lo = row_from(t.row0) & ~(kRows - 1);
  const int w_lo = first < t.lk ? row_from(first) : t.lq;
  const int w_full = row_from(first + 31 < t.lk ? first + 31 : t.lk - 1);  // from here on every row sees every key of the wavefront
  const int mine = row_from(key);

  DofFrag<T> kf[KS], vf[DK ? KS : 1];
  const T* kp = static_cast<const T*>(A.k) + (t.k0 + key) * A.ks[0] + hk * A.ks[1];
  const T* vp = static_cast<const T*>(A.v) + (t.k0 + key) * A.vs[0] + hk * A.vs[1];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int e = 16 * s + 8 * half;
    kf[s] = dof_frag_zero<T>();
    if (live && e < A.dim) kf[s] = dof_frag_load<T>(kp + e);
    if constexpr (DK) {
      vf[s] = dof_frag_zero<T>();
      if (live && e < A.dim) vf[s] = dof_frag_load<T>(vp + e);
    }
  }
  dof_f32x16 dk[DK ? DT : 1], dv[DV ? DT : 1];
#pragma unroll
  for (int d = 0; d < DT; ++d) {
    if constexpr (DK) dk[d] = dof_zero16();
    if constexpr (DV) dv[d] = dof_zero16();
  }

  Stage rq, rg;
  float rl = 0.0f, rd = 0.0f;
  auto load = [&](int h, int i0) {
    rq.load(static_cast<const T*>(A.q) + (t.q0 + i0) * A.qs[0] + h * A.qs[1], A.qs[0], t.lq - i0, A.dim, tid);
    rg.load(static_cast<const T*>(B.g) + (t.q0 + i0) * B.gs[0] + h * B.gs[1], B.gs[0], t.lq - i0, A.dim, tid);
    if (tid < kRows) {
      rl = INFINITY;
      rd = 0.0f;
      if (i0 + tid < t.lq) {
        const int64_t srow = (t.q0 + i0 + tid) * A.q_heads + h;
        rl = A.lse[srow] * kLog2e;
        rd = B.delta[srow];
        rl = rl == -INFINITY ? INFINITY : rl - Lift<T>::p2;
      }
    }
  };
  auto store = [&](int buf) {
    rq.store(sq[buf], tid);
    rg.store(sg[buf], tid);
    if (tid < kRows) {
      sl[buf][tid] = rl;
      sd[buf][tid] = rd;
    }
  };
  const bool any = t.lq > i_lo && heads > 0;
  if (any) {
    load(h_lo, i_lo);
    store(0);
  }
  int buf = 0;
  for (int h = h_lo, i0 = i_lo; any && h < h_lo + heads; buf ^= 1) {
    __syncthreads();
    const bool wrap = i0 + kRows >= t.lq;
    const int next_h = wrap ? h + 1 : h, next_i = wrap ? i_lo : i0 + kRows;
    if (next_h < h_lo + heads) load(next_h, next_i);
    if (i0 + kRows > w_lo) {
      dof_f32x16 x = dof_zero16(), y = dof_zero16();
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        x = dof_mma32<T>(sq[buf].rowfrag(col, 2 * s + half), kf[s], x);
        if constexpr (DK) y = dof_mma32<T>(sg[buf].rowfrag(col, 2 * s + half), vf[s], y);
      }
      float p[16], ds[16];
      const float slope = !PLAIN && A.slopes ? A.slopes[h] * kLog2e : 0.0f;
      const float base = (float)(i0 + off + 4 * half - key);
      const bool partial = i0 < w_full;
      const int left = mine - i0 - 4 * half;  // rows before this one do not see the lane's key
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const int r = 8 * (v / 4) + v % 4;
        float c = Lift<T>::ds / Lift<T>::p;
        const float lse2 = sl[buf][r + 4 * half];
        if constexpr (PLAIN) {
          p[v] = dof_exp2(fmaf(x[v], A.score.mul, -lse2));
        } else {
          float w = x[v] * A.score.mul;
          if (A.score.cap_l2 != 0.0f) {
            const float th = dof_cap_tanh<T>(x[v], A.score.mul);
            w = A.score.cap_l2 * th;
            c *= fmaf(-th, th, 1.0f);
          }
          if (A.slopes) w -= slope * fabsf(base + (float)r);
          p[v] = dof_exp2(w - lse2);
        }
        if constexpr (DK) ds[v] = p[v] * c * (y[v] - sd[buf][r + 4 * half]);
      }
      if (partial) {
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const bool hidden = 8 * (v / 4) + v % 4 < left;
          if constexpr (DV) p[v] = hidden ? 0.0f : p[v];
          if constexpr (DK) ds[v] = hidden ? 0.0f : ds[v];
        }
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int r = 16 * s + 4 * half;
        if constexpr (DV) {
          const DofFrag<T> f = dof_frag_pack<T>(p + 8 * s);
#pragma unroll
          for (int d = 0; d < DT; ++d) dv[d] = dof_mma32<T>(sg[buf].colfrag(r, r + 8, 32 * d + col), f, dv[d]);
        }
        if constexpr (DK) {
          const DofFrag<T> f = dof_frag_pack<T>(ds + 8 * s);
#pragma unroll
          for (int d = 0; d < DT; ++d) dk[d] = dof_mma32<T>(sq[buf].colfrag(r, r + 8, 32 * d + col), f, dk[d]);
        }
      }
    }
    if (next_h < h_lo + heads) store(buf ^ 1);
    h = next_h;
    i0 = next_i;
  }
  if (!live) return;
  const float ok = B.scale / Lift<T>::ds, ov = 1.0f / Lift<T>::p;
  auto write = [&](const dof_f32x16* acc, float f, void* out, const int64_t* st, float* part) {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int v = 0; v < 16; v += 4) {
        const int e = 32 * d + 2 * v + 4 * half;
        if (e >= A.dim) continue;
        const float r[4] = {acc[d][v] * f, acc[d][v + 1] * f, acc[d][v + 2] * f, acc[d][v + 3] * f};
        if (B.splits == 1) dof_store_vec<T, 4>(static_cast<T*>(out) + (t.k0 + key) * st[0] + hk * st[1] + e, r);
        else dof_store_vec<float, 4>(part + ((split * B.k_rows + t.k0 + key) * A.k_heads + hk) * A.dim + e, r);
      }
  };
  if constexpr (DK) write(dk, ok, B.dk, B.dks, B.part);
  if constexpr (DV) write(dv, ov, B.dv, B.dvs, B.part + B.splits * B.k_rows * A.k_heads * A.dim);
}

// dk and dv (blockIdx.y) from the parts of several workgroups per key tile, added in order.  Four elements a thread, rows of the tiles.
template <class T>
__global__ void __launch_bounds__(256) k_attn_join(DofAttnBwd B) {
  const DofAttnFwd& A = B.f;
  const int quads = A.dim / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t rh = i / quads, row = rh / A.k_heads;
  if (row >= B.k_rows) return;
  const int e = (int)(i - rh * quads) * 4, hk = (int)(rh - row * A.k_heads);
  const float* part = B.part + (blockIdx.y ? B.splits * B.k_rows * A.k_heads * A.dim : 0);
  float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int k = 0; k < B.splits; ++k) {
    float v[4];
    dof_load_vec<float, 4>(part + ((k * B.k_rows + row) * A.k_heads + hk) * A.dim + e, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] += v[j];
  }
  const int64_t* st = blockIdx.y ? B.dvs : B.dks;
  dof_store_vec<T, 4>(static_cast<T*>(blockIdx.y ? B.dv : B.dk) + row * st[0] + hk * st[1] + e, s);
}

template <class T, int DP, bool PLAIN>
void launch_dq_as(const DofAttnBwd& B, int flat, hipStream_t stream) {
  const unsigned blocks = (unsigned)((int64_t)B.f.n_tiles * B.f.q_heads);
  if (flat) DOF_LAUNCH((k_attn_dq<T, DP, 1, PLAIN>), (blocks, 1, 1), (64, 1, 1), stream, B);
  else DOF_LAUNCH((k_attn_dq<T, DP, 4, PLAIN>), (blocks, 1, 1), (256, 1, 1), stream, B);
}
template <class T, int DP, bool PLAIN, int WANT>
void launch_dkv_want(const DofAttnBwd& B, int flat, hipStream_t stream) {
  const unsigned blocks = (unsigned)((int64_t)B.f.n_tiles * B.f.k_heads * B.splits);
  if (flat) DOF_LAUNCH((k_attn_dkv<T, DP, 1, PLAIN, WANT>), (blocks, 1, 1), (64, 1, 1), stream, B);
  else DOF_LAUNCH((k_attn_dkv<T, DP, 4, PLAIN, WANT>), (blocks, 1, 1), (256, 1, 1), stream, B);
}
template <class T, int DP, bool PLAIN>
void launch_dkv_as(const DofAttnBwd& B, int flat, hipStream_t stream) {
  if constexpr (DP <= 64) {
    launch_dkv_want<T, DP, PLAIN, 3>(B, flat, stream);
  } else {
    launch_dkv_want<T, DP, PLAIN, 1>(B, flat, stream);
    launch_dkv_want<T, DP, PLAIN, 2>(B, flat, stream);
  }
}
template <class T, int DP>
void launch_dq(const DofAttnBwd& B, int flat, hipStream_t stream) {
  if (dof_attn_plain(B.f)) launch_dq_as<T, DP, true>(B, flat, stream);
  else launch_dq_as<T, DP, false>(B, flat, stream);
}
template <class T, int DP>
void launch_dkv(const DofAttnBwd& B, int flat, hipStream_t stream) {
  if (dof_attn_plain(B.f)) launch_dkv_as<T, DP, true>(B, flat, stream);
  else launch_dkv_as<T, DP, false>(B, flat, stream);
}

template <class T, int DP>
void launch_one(const DofAttnBwd& B, hipStream_t stream) {
  const unsigned blocks = (unsigned)((int64_t)B.f.n_tiles * B.f.k_heads);
  if (dof_attn_plain(B.f)) DOF_LAUNCH((k_attn_bwd_one<T, DP, true>), (blocks, 1, 1), (64, 1, 1), stream, B);
  else DOF_LAUNCH((k_attn_bwd_one<T, DP, false>), (blocks, 1, 1), (64, 1, 1), stream, B);
}

}  // namespace

int dof_launch_attn_dq(const DofAttnBwd& B, int dtype, int flat, hipStream_t stream) {
  DOF_SEQ_DISPATCH(dtype, T, {
    if (B.f.dim <= 32) launch_dq<T, 32>(B, flat, stream);
    else if (B.f.dim <= 64) launch_dq<T, 64>(B, flat, stream);
    else if (B.f.dim <= 96) launch_dq<T, 96>(B, flat, stream);
    else launch_dq<T, 128>(B, flat, stream);
  });
  return dof_check_launch("k_attn_dq");
}

int dof_launch_attn_dkv(const DofAttnBwd& B, int dtype, int flat, hipStream_t stream) {
  DOF_SEQ_DISPATCH(dtype, T, {
    if (B.f.dim <= 32) launch_dkv<T, 32>(B, flat, stream);
    else if (B.f.dim <= 64) launch_dkv<T, 64>(B, flat, stream);
    else if (B.f.dim <= 96) launch_dkv<T, 96>(B, flat, stream);
    else launch_dkv<T, 128>(B, flat, stream);
    if (B.splits > 1)
      DOF_LAUNCH((k_attn_join<T>), (dof_cdiv(B.k_rows * B.f.k_heads * (B.f.dim / 4), 256), 2, 1), (256, 1, 1), stream, B);
  });
  return dof_check_launch("k_attn_dkv");
}

int dof_launch_attn_bwd_one(const DofAttnBwd& B, int dtype, hipStream_t stream) {
  DOF_SEQ_DISPATCH(dtype, T, {
    if (B.f.dim <= 16) launch_one<T, 16>(B, stream);
    else if (B.f.dim <= 32) launch_one<T, 32>(B, stream);
    else launch_one<T, 64>(B, stream);
  });
  return dof_check_launch("k_attn_bwd_one");
}
