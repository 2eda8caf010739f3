// Attention over packed documents, backward: kernels that recompute the probabilities from the forward's log-sum-exp.
//
//   p = exp(s - lse) ; dp_ij = g_i.v_j ; ds = p (dp - delta_i) c_ij, delta_i = sum_d g_id o_id, c = 1 - tanh^2 under a cap, else 1
//   dq_i = scale sum_j ds_ij k_j        (k_attn_dq:  a workgroup per query tile, walks the keys as the forward does)
//   dv_j = sum_i p_ij g_i, dk_j = scale sum_i ds_ij q_i   (k_attn_dkv: a workgroup per key tile, walks the query rows that see it,
//                                                          through all query heads of its group)
//
// Every gradient element is summed in a fixed order, by one workgroup or in parts that k_attn_join adds up: no atomics, the same bits on
// every run.  The price is that S and dP are computed again: heads up to 64 take nine products of the size of S with 16-bit elements (S and dP
// twice, dv, dq and dk with their rests), larger ones ten (dv has a pass of its own, with S a third time).  The kernels keep their own rows'
// operands in registers and stream the other side through LDS (two images); the second products take P and dS straight from the
// registers the first ones left them in, as in the forward.
//
// P is rounded to the elements' type for its product with g, as in the forward (dv's error: 1.4 times that of rounding it).  dS goes into
// its products as two 16-bit numbers, value and rest: rounded once, its error alone would be as large as that of rounding dq and dk
// themselves (of short documents it came to 1.8 times that, together with delta from the rounded o).  The second product costs a fifth:
// 16384 causal frames, 16 / 4 heads of 128, bf16: dq 1.75 -> 2.25 ms, dk 1.83 -> 2.16 ms.  The dq kernel starts from delta = g.o, sums the
// unrounded P dP on its way and leaves that delta to the dk kernel.  Everything that is summed is fp32.
// fp16 has 5 exponent bits: there P is carried as 2^12 P (an exact factor, taken out at the end), so that the weights of long
// documents stay out of its subnormals, and dS with a power of two that follows its largest value (Range): gradients of any size
// reach dq and dk as they would without the rounding.
#include <cmath>

#include "deepof_hip.h"
#include "dof_rt.h"
#include "launchers.h"
#include "seq_attn.h"
#include "seq_attn_args.h"

namespace {

template <class T> struct Lift {
  static constexpr float p2 = 0.0f, p = 1.0f;  // log2 of P's factor, P's factor
};
template <> struct Lift<DofF16> {
  static constexpr float p2 = 12.0f, p = 4096.0f;
};

// The power of two that dS takes into its fp16 products.  A lane holds values of one query row (dq) or one key (dk), and so does its half
// of the accumulators: the factor is the lane's own (and that of the lane 32 away), found as a running maximum is.  The largest value
// lies between 2^13 and 2^15 when it is set; what a value and its rest lose is at most 2^-25 then, 2^-38 of the largest.
// Values arrive times P's factor.
template <class T> struct Range {
  static constexpr bool kOn = std::is_same<T, DofF16>::value;
  float f = kOn ? 1.2676506e30f : 1.0f;  // 2^100
  // mx 2^k in [2^13, 2^14), k at most 100
  __device__ __forceinline__ static float fit(float mx) {
    const int k = 267 - (int)(__builtin_bit_cast(uint32_t, mx) >> 23);
    return __builtin_bit_cast(float, (uint32_t)(k < 227 ? k : 227) << 23);
  }
  __device__ __forceinline__ static float top(const float* ds) {
    float mx = 0.0f;
#pragma unroll
    for (int v = 0; v < 16; ++v) mx = fmaxf(mx, fabsf(ds[v]));
    return fmaxf(mx, dof_swap32(mx));
  }
  template <int N> __device__ __forceinline__ void follow(float mx, dof_f32x16 (&acc)[N]) {
    const bool up = mx * f > 32768.0f;
    if (!dof_wave_any(up)) return;
    const float to = up ? fit(mx) : f, a = to / f;
    f = to;
#pragma unroll
    for (int d = 0; d < N; ++d)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[d][v] *= a;
  }
  __device__ __forceinline__ void apply(float* ds) const {
    if constexpr (kOn) {
#pragma unroll
      for (int v = 0; v < 16; ++v) ds[v] *= f;
    }
  }
};

// A row's log-sum-exp in log 2, as the value and (fp32 elements) what its rounding left: there the weights are to be good to fp32, and
// one rounding of a number near 10 is not.  The lift is taken off.  +inf: the row takes no part (it has no keys).
struct Lse { float value, rest; };
template <class T> __device__ __forceinline__ Lse lse_of(float lse) {
  Lse r = {INFINITY, 0.0f};
  if (lse == -INFINITY) return r;
  r.value = lse * kLog2e;
  if constexpr (sizeof(T) == 4) r.rest = fmaf(lse, kLog2e, -r.value) + lse * 1.925963033500e-8f;  // log2(e) - kLog2e
  r.value -= Lift<T>::p2;
  return r;
}
// the weight: 2^(w - lse), w = x mul for plain scores
template <class T, int KIND> __device__ __forceinline__ float weight(float x, float mul, float w, float value, float rest) {
  const float e = KIND == 0 ? fmaf(x, mul, -value) : w - value;
  return dof_exp2(sizeof(T) == 4 ? e - rest : e);
}

// Sixteen raw products x of a lane -> the exponents' arguments w (log 2, before the log-sum-exp is taken off) and c, the factor of dS from
// P (dP - delta): the derivative of the cap.  dist(v): the distance of element v.
template <class T, int KIND, class Dist>
__device__ __forceinline__ void scores(const dof_f32x16& x, const DofScore& sc, bool bias, Dist dist, float* w, float* c) {
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    w[v] = x[v];
    c[v] = 1.0f;
  }
  if constexpr (KIND == 2) {
    dof_cap_tanh<16>(w, sc.mul);
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      c[v] *= fmaf(-w[v], w[v], 1.0f);
      w[v] *= sc.cap_l2;
    }
  } else {
#pragma unroll
    for (int v = 0; v < 16; ++v) w[v] *= sc.mul;
  }
  if (bias) {
#pragma unroll
    for (int v = 0; v < 16; ++v) w[v] -= sc.slope_l2 * fabsf(dist(v));
  }
}

// KIND: the score function (dof_attn_kind).  LONG: long sums are made of blocks (fp32; always in tall tiles)
template <class T, int DP, int NW, int KIND, bool LONG>
__global__ void __launch_bounds__(64 * NW, sizeof(T) == 4 && DP > 32 ? 1 : 2) k_attn_dq(DofAttnBwd B) {
  const DofAttnFwd& A = B.f;
  constexpr int kKeys = 32;  // per step: what leaves room for two wavefronts per SIMD
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
  float sum = 0.0f;  // of P dP: delta again, without the rounding of o
  DofLongNumber<T> pdp;
  const Lse lse = lse_of<T>(live ? A.lse[srow] : -INFINITY);
  const T* kp = static_cast<const T*>(A.k) + t.k0 * A.ks[0] + hk * A.ks[1];
  const T* vp = static_cast<const T*>(A.v) + t.k0 * A.vs[0] + hk * A.vs[1];

  dof_f32x16 dq[DT];
  DofLongSum<T, dof_f32x16, DT, LONG> ldq;
  Range<T> range;
  ldq.clear();
  Stage rk, rv;
  // Rows of few keys: delta from the rounded o is off by as much as rounding all of dq once more; they go through their keys twice, the
  // first time for the sum of P dP alone.
  for (int pass = sizeof(T) == 2 && kmax <= 2 * kKeys ? 0 : 1; pass < 2; ++pass) {
#pragma unroll
    for (int d = 0; d < DT; ++d) dq[d] = dof_zero16();
    if (kmax > 0) {
      rk.load(kp, A.ks[0], t.lk, A.dim, tid);
      rv.load(vp, A.vs[0], t.lk, A.dim, tid);
      rk.store(sk[0], tid);
      rv.store(sv[0], tid);
    }
    pdp = DofLongNumber<T>();
    for (int j0 = 0, buf = 0; j0 < kmax; j0 += kKeys, buf ^= 1) {
      __syncthreads();
      const int next = j0 + kKeys;
      if (next < kmax) {
        rk.load(kp + next * A.ks[0], A.ks[0], t.lk - next, A.dim, tid);
        rv.load(vp + next * A.vs[0], A.vs[0], t.lk - next, A.dim, tid);
      }
      if (j0 < wmax) {
        const bool partial = j0 + kKeys > wmin;
        dof_f32x16 x = dof_zero16(), y = dof_zero16();
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          x = dof_mma32<T>(sk[buf].rowfrag(col, 2 * s + half), q[s], x);
          y = dof_mma32<T>(sv[buf].rowfrag(col, 2 * s + half), g[s], y);
        }
        float ds[16], w[16], c[16];
        const float base = (float)(pos - j0 - 4 * half);
        const int left = kend - j0 - 4 * half;
        float part = 0.0f;
        if constexpr (KIND > 0) scores<T, KIND>(x, sc, A.slopes != nullptr, [&](int v) { return base - (float)(8 * (v / 4) + v % 4); }, w, c);
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const bool hidden = partial && 8 * (v / 4) + v % 4 >= left;  // not 0 x (what a hidden key holds)
          const float p = weight<T, KIND>(x[v], sc.mul, w[v], lse.value, lse.rest);
          ds[v] = hidden ? 0.0f : p * (KIND == 0 ? 1.0f : c[v]) * (y[v] - delta);
          part += hidden ? 0.0f : p * y[v];
        }
        pdp.add(part);
        if constexpr (Range<T>::kOn) {
          range.follow(Range<T>::top(ds), dq);
          range.apply(ds);
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const DofFrag<T> f = dof_frag_pack<T>(ds + 8 * s), rest = dof_frag_rest<T>(ds + 8 * s, f);
          const int r = 16 * s + 4 * half;
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            const DofFrag<T> k = sk[buf].colfrag(r, r + 8, 32 * d + col);
            dq[d] = dof_mma32<T>(k, f, dq[d]);
            if constexpr (sizeof(T) == 2) dq[d] = dof_mma32<T>(k, rest, dq[d]);
          }
        }
        ldq.count(dq, kKeys);
      }
      if (next < kmax) {
        rk.store(sk[buf ^ 1], tid);
        rv.store(sv[buf ^ 1], tid);
      }
    }
    sum = pdp.total();
    sum = (sum + dof_swap32(sum)) / Lift<T>::p;
    if (pass == 0) {
      delta = sum;
      __syncthreads();  // the second pass fills the images anew
    }
  }
  ldq.finish(dq);
  if (!live) return;
  if (half == 0) B.delta[srow] = sum;
  const float out = B.scale / Lift<T>::p / range.f;
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
// are computed once (five products), q, k, v and g are read once, and delta is the sum of P dP over the lanes.  dS turns from "lane = key"
// to "lane = query" through LDS for dq; dk and dv add up over the group's query heads in registers.
template <class T, int DP, int KIND>
__global__ void __launch_bounds__(64, DP <= 32 ? 2 : 1) k_attn_bwd_one(DofAttnBwd B) {
  const DofAttnFwd& A = B.f;
  constexpr int KS = DP / 16, DT = (DP + 31) / 32;
  using Tile = DofTile<T, 32, 32 * DT>;
  using Stage = DofStage<T, 32, 32 * DT, 64>;
  __shared__ Tile sq, sg, sk;
  __shared__ DofTile<T, 32, 32> sds[sizeof(T) == 2 ? 2 : 1];  // dS, [query][key], and what its rounding left
  alignas(16) __shared__ float sl[32];
  alignas(16) __shared__ float sr[32];
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
  Range<T> range;
  // the first row that sees the lane's key
  const int mine = !A.causal || col < t.prefix || col - off < 0 ? 0 : col - off;

  for (int h = hk * group; h < (hk + 1) * group; ++h) {
    rq.load(static_cast<const T*>(A.q) + t.q0 * A.qs[0] + h * A.qs[1], A.qs[0], t.lq, A.dim, lane);
    rg.load(static_cast<const T*>(B.g) + t.q0 * B.gs[0] + h * B.gs[1], B.gs[0], t.lq, A.dim, lane);
    const Lse lse = lse_of<T>(row ? A.lse[(t.q0 + col) * A.q_heads + h] : -INFINITY);
    __syncthreads();  // the previous head's reads are done
    rq.store(sq, lane);
    rg.store(sg, lane);
    if (half == 0) {
      sl[col] = lse.value;
      sr[col] = lse.rest;
    }
    __syncthreads();
    dof_f32x16 x = dof_zero16(), y = dof_zero16();
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      x = dof_mma32<T>(sq.rowfrag(col, 2 * s + half), sk.rowfrag(col, 2 * s + half), x);
      y = dof_mma32<T>(sg.rowfrag(col, 2 * s + half), vf[s], y);
    }
    float p[16], ds[16], w[16], c[16];
    const float base = (float)(off + 4 * half - col);
    const int left = live ? mine - 4 * half : 32;
    if constexpr (KIND > 0) {
      DofScore sc = A.score;
      if (A.slopes) sc.slope_l2 = A.slopes[h] * kLog2e;
      scores<T, KIND>(x, sc, A.slopes != nullptr, [&](int v) { return base + (float)(8 * (v / 4) + v % 4); }, w, c);
    }
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      const int r = 8 * (v / 4) + v % 4 + 4 * half;
      p[v] = weight<T, KIND>(x[v], A.score.mul, w[v], sl[r], sr[r]);
      const bool hidden = 8 * (v / 4) + v % 4 < left;
      p[v] = hidden ? 0.0f : p[v];
      // delta = the row's sum of P dP: over the 32 lanes that hold the row
      float d = hidden ? 0.0f : p[v] * y[v];
      d = dof_row16_sum(d);
      d += __shfl_xor(d, 16);
      ds[v] = hidden ? 0.0f : p[v] * (KIND == 0 ? 1.0f : c[v]) * (y[v] - d / Lift<T>::p);
    }
    // for dk the lanes' own factors; for dq, whose operand holds rows of all lanes, one for the document and head
    float dsk[16], whole = 1.0f;
#pragma unroll
    for (int v = 0; v < 16; ++v) dsk[v] = ds[v];
    if constexpr (Range<T>::kOn) {
      float mx = Range<T>::top(ds);
      range.follow(mx, dk);
      range.apply(dsk);
#pragma unroll
      for (int m = 1; m < 32; m <<= 1) mx = fmaxf(mx, __shfl_xor(mx, m));
      whole = Range<T>::fit(mx);
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const DofFrag<T> pf = dof_frag_pack<T>(p + 8 * s), df = dof_frag_pack<T>(dsk + 8 * s), rest = dof_frag_rest<T>(dsk + 8 * s, df);
      const int r = 16 * s + 4 * half;
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        dv[d] = dof_mma32<T>(sg.colfrag(r, r + 8, 32 * d + col), pf, dv[d]);
        const DofFrag<T> q = sq.colfrag(r, r + 8, 32 * d + col);
        dk[d] = dof_mma32<T>(q, df, dk[d]);
        if constexpr (sizeof(T) == 2) dk[d] = dof_mma32<T>(q, rest, dk[d]);
      }
    }
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      const int to = sds[0].offset(8 * (v / 4) + v % 4 + 4 * half, col / Tile::EPC);
      T* e = reinterpret_cast<T*>(sds[0].mem + to) + col % Tile::EPC;
      const float x = ds[v] * whole;
      DofElem<T>::put(e, x);
      if constexpr (sizeof(T) == 2) DofElem<T>::put(reinterpret_cast<T*>(sds[1].mem + to) + col % Tile::EPC, x - DofElem<T>::get(e));
    }
    __syncthreads();
    // dq (queries in registers, d over the lanes) = dS K
    dof_f32x16 dq[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) dq[d] = dof_zero16();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      // the eight keys of an operand are rows 16 s + 8 half .. of K, four and four
      const DofFrag<T> f = sds[0].rowfrag(col, 2 * s + half);
      const int r = 16 * s + 8 * half;
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const DofFrag<T> k = sk.colfrag(r, r + 4, 32 * d + col);
        dq[d] = dof_mma32<T>(f, k, dq[d]);
        if constexpr (sizeof(T) == 2) dq[d] = dof_mma32<T>(sds[1].rowfrag(col, 2 * s + half), k, dq[d]);
      }
    }
    const float out = B.scale / Lift<T>::p / whole;
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
  const float ok = B.scale / Lift<T>::p / range.f, ov = 1.0f / Lift<T>::p;
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
// registers only one wavefront fits a SIMD, and one alone does not hide its own latencies (16384 causal frames, 16 / 4
// heads of 128, before dS took its second product: 6.4 ms in one pass of 4 products, 3.3 in two of 5; with it, 2 + 4: 3.65 ms).
// A workgroup takes `heads_per` query heads of the group; several workgroups of one key tile leave fp32 parts for k_attn_join.
template <class T, int DP, int NW, int KIND, bool LONG, int WANT>
__global__ void __launch_bounds__(64 * NW, sizeof(T) == 4 && DP > 32 ? 1 : 2) k_attn_dkv(DofAttnBwd B) {
  const DofAttnFwd& A = B.f;
  constexpr bool DV = (WANT & 1) != 0, DK = (WANT & 2) != 0;
  constexpr int kRows = 32;  // query rows per step
  using Tile = DofTile<T, kRows, DP>;
  using Stage = DofStage<T, kRows, DP, 64 * NW>;
  __shared__ Tile sq[2], sg[2];
  alignas(16) __shared__ float sl[2][kRows];  // log-sum-exp, its rest
  alignas(16) __shared__ float sr[2][kRows];
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
  DofLongSum<T, dof_f32x16, DK ? DT : 1, LONG> ldk;
  DofLongSum<T, dof_f32x16, DV ? DT : 1, LONG> ldv;
  Range<T> range;  // of dS
  if constexpr (DK) ldk.clear();
  if constexpr (DV) ldv.clear();
#pragma unroll
  for (int d = 0; d < DT; ++d) {
    if constexpr (DK) dk[d] = dof_zero16();
    if constexpr (DV) dv[d] = dof_zero16();
  }

  Stage rq, rg;
  Lse rl = {0.0f, 0.0f};
  float rd = 0.0f;
  auto load = [&](int h, int i0) {
    rq.load(static_cast<const T*>(A.q) + (t.q0 + i0) * A.qs[0] + h * A.qs[1], A.qs[0], t.lq - i0, A.dim, tid);
    rg.load(static_cast<const T*>(B.g) + (t.q0 + i0) * B.gs[0] + h * B.gs[1], B.gs[0], t.lq - i0, A.dim, tid);
    if (tid < kRows) {
      rl = lse_of<T>(-INFINITY);
      rd = 0.0f;
      if (i0 + tid < t.lq) {
        const int64_t srow = (t.q0 + i0 + tid) * A.q_heads + h;
        rl = lse_of<T>(A.lse[srow]);
        rd = B.delta[srow];
      }
    }
  };
  auto store = [&](int buf) {
    rq.store(sq[buf], tid);
    rg.store(sg[buf], tid);
    if (tid < kRows) {
      sl[buf][tid] = rl.value;
      if (sizeof(T) == 4) sr[buf][tid] = rl.rest;
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
      float p[16], ds[16], w[16], c[16];
      const float base = (float)(i0 + off + 4 * half - key);
      const bool partial = i0 < w_full;
      const int left = mine - i0 - 4 * half;  // rows before this one do not see the lane's key
      if constexpr (KIND > 0) {
        DofScore sc = A.score;
        if (A.slopes) sc.slope_l2 = A.slopes[h] * kLog2e;
        scores<T, KIND>(x, sc, A.slopes != nullptr, [&](int v) { return base + (float)(8 * (v / 4) + v % 4); }, w, c);
      }
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const int r = 8 * (v / 4) + v % 4 + 4 * half;
        p[v] = weight<T, KIND>(x[v], A.score.mul, w[v], sl[buf][r], sizeof(T) == 4 ? sr[buf][r] : 0.0f);
        if constexpr (DK) ds[v] = p[v] * (KIND == 0 ? 1.0f : c[v]) * (y[v] - sd[buf][r]);
      }
      if (partial) {
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const bool hidden = 8 * (v / 4) + v % 4 < left;
          if constexpr (DV) p[v] = hidden ? 0.0f : p[v];
          if constexpr (DK) ds[v] = hidden ? 0.0f : ds[v];
        }
      }
      if constexpr (DK && Range<T>::kOn) {
        range.follow(Range<T>::top(ds), dk);
        range.apply(ds);
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
          const DofFrag<T> f = dof_frag_pack<T>(ds + 8 * s), rest = dof_frag_rest<T>(ds + 8 * s, f);
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            const DofFrag<T> q = sq[buf].colfrag(r, r + 8, 32 * d + col);
            dk[d] = dof_mma32<T>(q, f, dk[d]);
            if constexpr (sizeof(T) == 2) dk[d] = dof_mma32<T>(q, rest, dk[d]);
          }
        }
      }
      if constexpr (DK) ldk.count(dk, kRows);
      if constexpr (DV) ldv.count(dv, kRows);
    }
    if (next_h < h_lo + heads) store(buf ^ 1);
    h = next_h;
    i0 = next_i;
  }
  if constexpr (DK) ldk.finish(dk);
  if constexpr (DV) ldv.finish(dv);
  if (!live) return;
  const float ok = B.scale / Lift<T>::p / range.f, ov = 1.0f / Lift<T>::p;
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

// dk and dv (blockIdx.y) from the parts of several workgroups per key tile, added in order: a workgroup per `take` rows of a tile and key
// head (8, 16 or 32: about one group of four elements a thread), `pieces` of them per tile.  Rows of no tile have no parts and stay.
template <class T>
__global__ void __launch_bounds__(256) k_attn_join(DofAttnBwd B, int pieces, int take) {
  const DofAttnFwd& A = B.f;
  const int item = blockIdx.x / A.k_heads, hk = blockIdx.x - item * A.k_heads, tile = item / pieces;
  const DofAttnTile t = A.tiles[tile];
  const int first = t.row0 + (item - tile * pieces) * take, rows = t.lk - first < take ? t.lk - first : take;
  const int quads = A.dim / 4;
  const float* part = B.part + (blockIdx.y ? B.splits * B.k_rows * A.k_heads * A.dim : 0);
  const int64_t* st = blockIdx.y ? B.dvs : B.dks;
  for (int i = threadIdx.x; i < rows * quads; i += 256) {
    const int r = i / quads, e = 4 * (i - r * quads);
    const int64_t row = t.k0 + first + r;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k = 0; k < B.splits; ++k) {
      float v[4];
      dof_load_vec<float, 4>(part + ((k * B.k_rows + row) * A.k_heads + hk) * A.dim + e, v);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] += v[j];
    }
    dof_store_vec<T, 4>(static_cast<T*>(blockIdx.y ? B.dv : B.dk) + row * st[0] + hk * st[1] + e, s);
  }
}

template <class T, int DP>
void launch_dq(const DofAttnBwd& B, int flat, hipStream_t stream) {
  const unsigned blocks = (unsigned)((int64_t)B.f.n_tiles * B.f.q_heads);
  DOF_ATTN_KIND(B.f, KIND, {
    if (flat) DOF_ATTN_LONG(T, B.f.longest, LONG, DOF_LAUNCH((k_attn_dq<T, DP, 1, KIND, LONG>), (blocks, 1, 1), (64, 1, 1), stream, B));
    else DOF_LAUNCH((k_attn_dq<T, DP, 4, KIND, sizeof(T) == 4>), (blocks, 1, 1), (256, 1, 1), stream, B);
  });
}
template <class T, int DP, int WANT>
void launch_dkv_want(const DofAttnBwd& B, int flat, hipStream_t stream) {
  const unsigned blocks = (unsigned)((int64_t)B.f.n_tiles * B.f.k_heads * B.splits);
  DOF_ATTN_KIND(B.f, KIND, {
    if (flat)
      DOF_ATTN_LONG(T, (int64_t)B.f.longest * B.heads_per, LONG,
                    DOF_LAUNCH((k_attn_dkv<T, DP, 1, KIND, LONG, WANT>), (blocks, 1, 1), (64, 1, 1), stream, B));
    else DOF_LAUNCH((k_attn_dkv<T, DP, 4, KIND, sizeof(T) == 4, WANT>), (blocks, 1, 1), (256, 1, 1), stream, B);
  });
}
template <class T, int DP>
void launch_dkv(const DofAttnBwd& B, int flat, hipStream_t stream) {
  if constexpr (DP <= 64) {
    launch_dkv_want<T, DP, 3>(B, flat, stream);
  } else {
    launch_dkv_want<T, DP, 1>(B, flat, stream);
    launch_dkv_want<T, DP, 2>(B, flat, stream);
  }
}
template <class T, int DP>
void launch_one(const DofAttnBwd& B, hipStream_t stream) {
  const unsigned blocks = (unsigned)((int64_t)B.f.n_tiles * B.f.k_heads);
  DOF_ATTN_KIND(B.f, KIND, DOF_LAUNCH((k_attn_bwd_one<T, DP, KIND>), (blocks, 1, 1), (64, 1, 1), stream, B));
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
    if (B.splits > 1) {
      const int take = B.f.dim > 64 ? 8 : B.f.dim > 32 ? 16 : 32, pieces = (flat ? kAttnFlat : kAttnTall) / take;
      DOF_LAUNCH((k_attn_join<T>), ((unsigned)((int64_t)B.f.n_tiles * pieces * B.f.k_heads), 2, 1), (256, 1, 1), stream, B, pieces, take);
    }
  });
  return dof_check_launch("k_attn_dkv");
}

int dof_launch_attn_bwd_one(const DofAttnBwd& B, int dtype, hipStream_t stream) {
  DOF_SEQ_DISPATCH(dtype, T, {
    if (B.f.dim <= 16) launch_one<T, 16>(B, stream);
    else if (B.f.dim <= 32) launch_one<T, 32>(B, stream);
    else if (B.f.dim <= 64) launch_one<T, 64>(B, stream);
    else if constexpr (sizeof(T) == 2) {
      if (B.f.dim <= 96) launch_one<T, 96>(B, stream);
      else launch_one<T, 128>(B, stream);
    }
  });
  return dof_check_launch("k_attn_bwd_one");
}
