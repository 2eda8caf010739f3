// Attention over packed documents, forward.
//
//   s_ij = scale q_i.k_j ; s = cap tanh(s / cap) ; s -= slope |pos_i - j| ; softmax over the visible keys ; o_i = sum_j p_ij v_j
//
// A workgroup owns a tile of query rows of one document and head (32 rows per wavefront) and walks the document's visible keys, 32
// or 64 at a time, with a running maximum and sum; K and V pass through LDS (two images, the next one's loads in flight under the present
// one's products).  The products are transposed -- S^T = K Q^T, O^T = V^T P^T -- so that a lane owns one query: its maximum, sum and
// rescaling are lane-local but for one exchange with the other half-wavefront, and P^T leaves the first product in just the registers
// the second one wants it in (the key order inside a fragment is permuted, the same on both operands).  V^T is read from row-major
// LDS by the transposing LDS read.  Statistics and accumulators are fp32; P is rounded to the elements' type for its product (relative
// half a step per weight, as the inputs' own; fp16 weights are lifted out of their subnormals, see DofSoftmax), the sum l is taken of
// the unrounded weights.  As value and rest, two products, P would take o's error from 1.2 - 1.4 times that of rounding o once to 1.0:
// 24 ragged recordings with a bias 204 -> 250 us, 16384 frames, heads of 128, training 7.2 -> 7.9 ms (with dv's).  Not taken.
#include <cmath>

#include "deepof_hip.h"
#include "dof_rt.h"
#include "launchers.h"
#include "seq_attn.h"
#include "seq_attn_args.h"

namespace {

// Keys per step: 32, or 64 for heads over 64 (24 ragged recordings, heads of 64: 236 us with 64, 199 with 32, which leave room for four
// wavefronts per SIMD; 16384 frames, heads of 128: 1.40 ms with 64, 1.48 with 32: two wavefronts either way).  A single wavefront takes
// 32 and one LDS image: nobody else waits for it, and the smaller image lets more of them onto a CU.
// KIND: the score function (dof_attn_kind).  LONG: long sums are made of blocks (fp32; always in tall tiles)
template <class T, int DP, int NW, int KIND, bool LONG>
__global__ void __launch_bounds__(64 * NW, DP <= 32 ? (NW == 1 && sizeof(T) == 4 ? 3 : 4) : sizeof(T) == 4 && DP > 64 ? 1 : 2) k_attn_fwd(DofAttnFwd A) {
  constexpr int KU = NW == 1 || DP <= 64 ? 1 : 2, kKeys = 32 * KU, BUF = NW == 1 ? 1 : 2;
  constexpr int KS = DP / 16, DT = (DP + 31) / 32;  // DP = 16: half of the only 32-wide tile of d is padding
  using Tile = DofTile<T, kKeys, 32 * DT>;
  using Stage = DofStage<T, kKeys, 32 * DT, 64 * NW>;
  __shared__ Tile sk[BUF], sv[BUF];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, half = lane >> 5;
  int tile, h;
  dof_attn_item(blockIdx.x, A.n_tiles, A.q_heads, &tile, &h);
  const DofAttnTile t = A.tiles[tile];
  const int hk = h / (A.q_heads / A.k_heads);

  const int first = t.row0 + 32 * wave, row = first + col;
  const bool live = row < t.lq;
  const int last_wg = (t.row0 + 32 * NW < t.lq ? t.row0 + 32 * NW : t.lq) - 1;
  const int last = (first + 32 < t.lq ? first + 32 : t.lq) - 1;
  const int kmax = dof_attn_kend(t, A.causal, last_wg);                          // of the workgroup
  const int wmax = first < t.lq ? dof_attn_kend(t, A.causal, last) : 0;          // of the wavefront
  const int wmin = first < t.lq ? dof_attn_kend(t, A.causal, first) : 0;         // keys that all its rows see
  const int kend = live ? dof_attn_kend(t, A.causal, row) : 0;
  const int pos = row + t.lk - t.lq;
  DofScore sc = A.score;
  if (A.slopes) sc.slope_l2 = A.slopes[h] * kLog2e;

  DofFrag<T> q[KS];
  const T* qp = static_cast<const T*>(A.q) + (t.q0 + row) * A.qs[0] + h * A.qs[1];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int e = 16 * s + 8 * half;
    q[s] = dof_frag_zero<T>();
    if (live && e < A.dim) q[s] = dof_frag_load<T>(qp + e);
  }
  const T* kp = static_cast<const T*>(A.k) + t.k0 * A.ks[0] + hk * A.ks[1];
  const T* vp = static_cast<const T*>(A.v) + t.k0 * A.vs[0] + hk * A.vs[1];

  dof_f32x16 o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) o[d] = dof_zero16();
  DofLongSum<T, dof_f32x16, DT, LONG> lo;
  lo.clear();
  DofLongNumber<T> l;
  float m = -INFINITY;

  // In a step that some rows see only in part a hidden key's weight is zero, but zero times an infinity or NaN in V is not: such
  // values are left out of the products there (rare, and looked for in these steps only) and put where they are seen at the end.
  __shared__ int found;
  const int kmin = dof_attn_kend(t, A.causal, t.row0);
  if (tid == 0) found = 0;
  __syncthreads();
  Stage rk, rv;
  auto store_v = [&](int b, int j) {
    if ((j + kKeys < t.lk ? j + kKeys : t.lk) > kmin) rv.store_finite(sv[b], tid, &found);
    else rv.store(sv[b], tid);
  };
  if (kmax > 0) {
    rk.load(kp, A.ks[0], t.lk, A.dim, tid);
    rv.load(vp, A.vs[0], t.lk, A.dim, tid);
    rk.store(sk[0], tid);
    store_v(0, 0);
  }
  for (int j0 = 0, buf = 0; j0 < kmax; j0 += kKeys, buf ^= BUF - 1) {
    __syncthreads();
    const int next = j0 + kKeys;
    if (next < kmax) {
      rk.load(kp + next * A.ks[0], A.ks[0], t.lk - next, A.dim, tid);
      rv.load(vp + next * A.vs[0], A.vs[0], t.lk - next, A.dim, tid);
    }
    if (j0 < wmax) {
      dof_f32x16 x[KU];
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        x[u] = dof_zero16();
#pragma unroll
        for (int s = 0; s < KS; ++s) x[u] = dof_mma32<T>(sk[buf].rowfrag(32 * u + col, 2 * s + half), q[s], x[u]);
      }
      if constexpr (KIND > 0) {
        const float base = (float)(pos - j0 - 4 * half);
        if constexpr (KIND == 2) {
#pragma unroll
          for (int u = 0; u < KU; ++u) {
            float th[16];
#pragma unroll
            for (int v = 0; v < 16; ++v) th[v] = x[u][v];
            dof_cap_tanh<16>(th, sc.mul);
#pragma unroll
            for (int v = 0; v < 16; ++v) x[u][v] = sc.cap_l2 * th[v];
          }
          if (A.slopes) {
#pragma unroll
            for (int u = 0; u < KU; ++u)
#pragma unroll
              for (int v = 0; v < 16; ++v) x[u][v] -= sc.slope_l2 * fabsf(base - (float)(32 * u + 8 * (v / 4) + v % 4));
          }
        } else {
#pragma unroll
          for (int u = 0; u < KU; ++u)
#pragma unroll
            for (int v = 0; v < 16; ++v)
              x[u][v] = fmaf(x[u][v], sc.mul, -sc.slope_l2 * fabsf(base - (float)(32 * u + 8 * (v / 4) + v % 4)));
        }
      }
      const float unit = KIND == 0 ? sc.mul : 1.0f;  // of x, in log 2
      if (j0 + kKeys > wmin) {
        const int left = kend - j0 - 4 * half;
#pragma unroll
        for (int u = 0; u < KU; ++u)
#pragma unroll
          for (int v = 0; v < 16; ++v)
            if (32 * u + 8 * (v / 4) + v % 4 >= left) x[u][v] = -INFINITY;
      }
      float mt = -INFINITY;
#pragma unroll
      for (int u = 0; u < KU; ++u)
#pragma unroll
        for (int v = 0; v < 16; ++v) mt = fmaxf(mt, x[u][v]);
      mt = fmaxf(mt, dof_swap32(mt)) * unit;
      // The running maximum follows only when a tile's exceeds it by 2^kLag: until then the weights stay below that, which costs the
      // fp32 sums nothing, and the accumulators need no rescaling pass.
      if (dof_wave_any(mt > m + DofSoftmax<T>::kLag)) {
        // only of the rows that exceed theirs: a row's bits do not depend on the other rows of its wavefront
        const bool up = mt > m + DofSoftmax<T>::kLag;
        const float a = up ? dof_exp2(m - mt) : 1.0f;
        m = up ? mt : m;
        l.scale(a);
        lo.scale(a);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int v = 0; v < 16; ++v) o[d][v] *= a;
      }
      const float mm = m == -INFINITY ? 0.0f : m - DofSoftmax<T>::kUp;
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        float p[16];
        float part = 0.0f;  // one addition per step, not sixteen, to the long sum
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          p[v] = dof_exp2(fmaf(x[u][v], unit, -mm));
          part += p[v];
        }
        l.add(part);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const DofFrag<T> pf = dof_frag_pack<T>(p + 8 * s);
          const int r = 32 * u + 16 * s + 4 * half;
#pragma unroll
          for (int d = 0; d < DT; ++d) o[d] = dof_mma32<T>(sv[buf].colfrag(r, r + 8, 32 * d + col), pf, o[d]);
        }
      }
      lo.count(o, kKeys);
    }
    if (next < kmax) {
      if (BUF == 1) __syncthreads();
      rk.store(sk[buf ^ (BUF - 1)], tid);
      store_v(buf ^ (BUF - 1), next);
    }
  }

  lo.finish(o);
  float sum = l.total();
  sum += dof_swap32(sum);
  __syncthreads();
  if (!live) return;
  if (found) {
    for (int j = kmin / kKeys * kKeys; j < kend; ++j)
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int e = 32 * d + 8 * (v / 4) + 4 * half + v % 4;
          const float x = e < A.dim ? DofElem<T>::get(vp + j * A.vs[0] + e) : 0.0f;
          if (!(fabsf(x) < INFINITY)) o[d][v] += x;
        }
  }
  const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);  // no visible key: zeros; NaN stays NaN
  T* op = static_cast<T*>(A.o) + (t.q0 + row) * A.os[0] + h * A.os[1];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int v = 0; v < 16; v += 4) {
      const int e = 32 * d + 2 * v + 4 * half;
      if (e < A.dim) {
        const float r[4] = {o[d][v] * inv, o[d][v + 1] * inv, o[d][v + 2] * inv, o[d][v + 3] * inv};
        dof_store_vec<T, 4>(op + e, r);
      }
    }
  if (half == 0) A.lse[(t.q0 + row) * A.q_heads + h] = sum == 0.0f ? -INFINITY : (m + dof_log2(sum * DofSoftmax<T>::kDown)) * kLn2;
}

template <class T, int DP>
void launch(const DofAttnFwd& A, int flat, hipStream_t stream) {
  const unsigned blocks = (unsigned)((int64_t)A.n_tiles * A.q_heads);
  DOF_ATTN_KIND(A, KIND, {
    if (flat) DOF_ATTN_LONG(T, A.longest, LONG, DOF_LAUNCH((k_attn_fwd<T, DP, 1, KIND, LONG>), (blocks, 1, 1), (64, 1, 1), stream, A));
    else DOF_LAUNCH((k_attn_fwd<T, DP, 4, KIND, sizeof(T) == 4>), (blocks, 1, 1), (256, 1, 1), stream, A);
  });
}

}  // namespace

int dof_launch_attn_fwd(const DofAttnFwd& A, int dtype, int flat, hipStream_t stream) {
  DOF_SEQ_DISPATCH(dtype, T, {
    if (A.dim <= 16) launch<T, 16>(A, flat, stream);
    else if (A.dim <= 32) launch<T, 32>(A, flat, stream);
    else if (A.dim <= 64) launch<T, 64>(A, flat, stream);
    else if (A.dim <= 96) launch<T, 96>(A, flat, stream);
    else launch<T, 128>(A, flat, stream);
  });
  return dof_check_launch("k_attn_fwd");
}
