// RMS norm of every query / key head and rotation by its position, in one pass -- forward and backward.
//
//   forward    xhat = x / sqrt(mean(x^2) + eps);  y = xhat * w;  the pairs (a, b) of the first rot_dim elements become
//              (a cos t - b sin t, b cos t + a sin t), t = position * freqs[pair].  Pairs lie rot_dim / 2 apart (half layout) or
//              side by side (interleaved); the elements behind rot_dim pass unrotated.
//   backward   gy = the inverse rotation of g;  dw = sum over tokens and heads of gy * xhat;
//              dx = (w gy - xhat mean(w gy xhat)) / sqrt(mean(x^2) + eps).  xhat is recomputed from x: nothing is stored forward.
//
// Bound by memory: every element is read once and written once (backward: x and g read, dx written).  A row (one head of one
// token) is spread over just enough lanes that each holds VEC pairs -- 16-byte accesses where layout and alignment allow -- so the
// norm is a handful of lane exchanges and both members of a pair sit in one lane.  The angles of a token are shared by all its
// heads: a workgroup takes a few tokens, computes their sines and cosines once into LDS (the angle is reduced to half a turn in 64
// bits, so positions of any 32-bit size keep fp32 accuracy), then streams the rows.  Norm, rotation and sums are fp32, rounded
// once on the way out.  blockIdx.y: 0 = queries, 1 = keys.
#include <cmath>

#include "dof_rt.h"
#include "launchers.h"
#include "deepof_hip.h"
#include "seq_types.h"

namespace {

constexpr int kTable = 1024;     // (cos, sin) pairs of a workgroup's tokens
constexpr int kMaxDim = 256;
constexpr int kBwdBlocks = 1024; // workgroups per tensor in the backward pass = rows of the weight-gradient partials

struct Side {  // the query or the key tensor of a call
  const void* x;
  const void* g;   // backward: gradient at the output
  void* out;       // forward: y, backward: dx
  const float* w;  // NULL: no norm
  float* dw_part;  // backward with a norm: [kBwdBlocks][head_dim] partial weight gradients
  int64_t xt, xh, gt, gh, ot, oh;  // token and head strides, in elements
  int heads;
};

struct Args {
  Side side[2];
  const int32_t* pos;
  const double* freqs;
  int64_t tokens;
  int64_t chunks;
  float eps;
  int dim, half, interleaved;  // half = rot_dim / 2 pairs
  int tb;                      // tokens per chunk
  int lpr;                     // lanes per row, a power of two
};

// first element of the pairs p .. p + VEC - 1 and of their partners; the rest behind the rotated part is paired side by side
template <int VEC>
__device__ __forceinline__ void pair_at(const Args& A, int p, int* ia, int* ib, bool* adjacent) {
  if (p < A.half && !A.interleaved) {
    *ia = p;
    *ib = p + A.half;
    *adjacent = false;
  } else {
    *ia = 2 * p;   // interleaved, or rot_dim + 2 (p - half) = 2 p
    *ib = 2 * p + VEC;
    *adjacent = true;
  }
}

// the pairs as (a[i], b[i]) from the two runs of VEC elements
template <class T, int VEC>
__device__ __forceinline__ void load_pairs(const T* row, int ia, int ib, bool adjacent, float* a, float* b) {
  float u[VEC], v[VEC];
  dof_load_vec<T, VEC>(row + ia, u);
  dof_load_vec<T, VEC>(row + ib, v);
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const float fa = 2 * i < VEC ? u[(2 * i) % VEC] : v[(2 * i) % VEC];
    const float fb = 2 * i + 1 < VEC ? u[(2 * i + 1) % VEC] : v[(2 * i + 1) % VEC];
    a[i] = adjacent ? fa : u[i];
    b[i] = adjacent ? fb : v[i];
  }
}
template <class T, int VEC>
__device__ __forceinline__ void store_pairs(T* row, int ia, int ib, bool adjacent, const float* a, const float* b) {
  float u[VEC], v[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const float lo = (i & 1) ? b[i / 2] : a[i / 2];
    const float hi = ((i + VEC) & 1) ? b[(i + VEC) / 2] : a[(i + VEC) / 2];
    u[i] = adjacent ? lo : a[i];
    v[i] = adjacent ? hi : b[i];
  }
  dof_store_vec<T, VEC>(row + ia, u);
  dof_store_vec<T, VEC>(row + ib, v);
}

__device__ __forceinline__ float row_sum(float v, int lpr) {
  for (int m = lpr >> 1; m > 0; m >>= 1) v += __shfl_xor(v, m);
  return v;
}

// T = element type, VEC = pairs per lane; NI = rounds of lpr lanes over a row's pairs (2 only for VEC = 1 and heads over 128)
template <class T, int VEC, int NI, bool BWD>
__global__ void __launch_bounds__(256) k_norm_rope(Args A) {
  __shared__ float tab[2 * kTable];
  const Side& S = A.side[blockIdx.y];
  const int tid = threadIdx.x;
  const int lane = tid & (A.lpr - 1);
  const int rpp = 256 / A.lpr;  // rows per pass
  const int row0 = tid / A.lpr;
  const float inv_dim = 1.0f / (float)A.dim;
  const bool normed = S.w != nullptr;

  int ia[NI], ib[NI];
  bool adj[NI], live[NI];
  float wa[NI][VEC], wb[NI][VEC], da[NI][VEC], db[NI][VEC];
#pragma unroll
  for (int n = 0; n < NI; ++n) {
    const int p = (lane + n * A.lpr) * VEC;
    live[n] = 2 * p < A.dim;
    pair_at<VEC>(A, p, &ia[n], &ib[n], &adj[n]);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      wa[n][i] = wb[n][i] = 1.0f;
      da[n][i] = db[n][i] = 0.0f;
    }
    if (live[n] && normed) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        wa[n][i] = S.w[adj[n] ? ia[n] + 2 * i : ia[n] + i];
        wb[n][i] = S.w[adj[n] ? ia[n] + 2 * i + 1 : ib[n] + i];
      }
    }
  }

  for (int64_t chunk = blockIdx.x; chunk < A.chunks; chunk += gridDim.x) {
    const int64_t t0 = chunk * A.tb;
    const int nt = (int)(A.tokens - t0 < A.tb ? A.tokens - t0 : A.tb);
    __syncthreads();
    for (int e = tid; e < nt * A.half; e += 256) {
      const int t = e / A.half, p = e - t * A.half;
      float s, c;
      dof_sincos_turns((double)A.pos[t0 + t] * (A.freqs[p] * 0.15915494309189533577), &s, &c);
      tab[2 * e] = c;
      tab[2 * e + 1] = s;
    }
    __syncthreads();
    const int rows = nt * S.heads;
    for (int r = row0; r < (rows + rpp - 1) / rpp * rpp; r += rpp) {
      const bool inside = r < rows;
      const int t = inside ? r / S.heads : 0;
      const int h = inside ? r - t * S.heads : 0;
      const T* xr = static_cast<const T*>(S.x) + (t0 + t) * S.xt + h * S.xh;
      float a[NI][VEC], b[NI][VEC], ga[NI][VEC], gb[NI][VEC];
      float ss = 0.0f;
#pragma unroll
      for (int n = 0; n < NI; ++n) {
        if (inside && live[n]) {
          if (!BWD || normed) load_pairs<T, VEC>(xr, ia[n], ib[n], adj[n], a[n], b[n]);
          if (BWD) load_pairs<T, VEC>(static_cast<const T*>(S.g) + (t0 + t) * S.gt + h * S.gh, ia[n], ib[n], adj[n], ga[n], gb[n]);
        }
        if (!(inside && live[n])) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) a[n][i] = b[n][i] = ga[n][i] = gb[n][i] = 0.0f;
        } else if (BWD && !normed) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) a[n][i] = b[n][i] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) ss = fmaf(a[n][i], a[n][i], fmaf(b[n][i], b[n][i], ss));
      }
      float rn = 1.0f;
      if (normed) rn = 1.0f / sqrtf(row_sum(ss, A.lpr) * inv_dim + A.eps);
      float dot = 0.0f;
#pragma unroll
      for (int n = 0; n < NI; ++n) {
        const int p = (lane + n * A.lpr) * VEC;
        const bool rot = p < A.half;  // VEC divides half: the pairs of a lane are all rotated or none
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float c = rot ? tab[2 * (t * A.half + p + i)] : 1.0f;
          const float s = rot ? tab[2 * (t * A.half + p + i) + 1] : 0.0f;
          if (!BWD) {
            const float ya = a[n][i] * rn * wa[n][i], yb = b[n][i] * rn * wb[n][i];
            a[n][i] = ya * c - yb * s;
            b[n][i] = yb * c + ya * s;
          } else {
            const float ya = ga[n][i] * c + gb[n][i] * s, yb = gb[n][i] * c - ga[n][i] * s;
            if (normed) {
              a[n][i] *= rn;
              b[n][i] *= rn;
              da[n][i] = fmaf(ya, a[n][i], da[n][i]);
              db[n][i] = fmaf(yb, b[n][i], db[n][i]);
            }
            ga[n][i] = ya * wa[n][i];
            gb[n][i] = yb * wb[n][i];
            dot = fmaf(ga[n][i], a[n][i], fmaf(gb[n][i], b[n][i], dot));
          }
        }
      }
      if (BWD && normed) {
        const float mean = row_sum(dot, A.lpr) * inv_dim;
#pragma unroll
        for (int n = 0; n < NI; ++n)
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            ga[n][i] = rn * (ga[n][i] - a[n][i] * mean);
            gb[n][i] = rn * (gb[n][i] - b[n][i] * mean);
          }
      }
      T* orow = static_cast<T*>(S.out) + (t0 + t) * S.ot + h * S.oh;
#pragma unroll
      for (int n = 0; n < NI; ++n)
        if (inside && live[n]) store_pairs<T, VEC>(orow, ia[n], ib[n], adj[n], BWD ? ga[n] : a[n], BWD ? gb[n] : b[n]);
    }
  }

  if constexpr (BWD) {
    if (!normed) return;
    // the row groups of the workgroup meet in LDS in a fixed order (kMaxDim floats fit the table)
    for (int turn = 0; turn < rpp; ++turn) {
      __syncthreads();
      if (row0 == turn) {
#pragma unroll
        for (int n = 0; n < NI; ++n)
          if (live[n]) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              const int ea = adj[n] ? ia[n] + 2 * i : ia[n] + i, eb = adj[n] ? ia[n] + 2 * i + 1 : ib[n] + i;
              tab[ea] = turn ? tab[ea] + da[n][i] : da[n][i];
              tab[eb] = turn ? tab[eb] + db[n][i] : db[n][i];
            }
          }
      }
    }
    __syncthreads();
    for (int e = tid; e < A.dim; e += 256) S.dw_part[(int64_t)blockIdx.x * A.dim + e] = tab[e];
  }
}

// dw[e] = sum over the partial rows, in row order per thread and thread order in LDS: the same sum every run.
// One workgroup per 16 elements and side; 16 threads share an element.
__global__ void __launch_bounds__(256) k_norm_rope_dw(const float* part_q, const float* part_k, float* dwq, float* dwk, int rows, int dim) {
  __shared__ float sm[256];
  const float* part = blockIdx.y ? part_k : part_q;
  float* dw = blockIdx.y ? dwk : dwq;
  if (!dw) return;  // uniform over the workgroup
  const int e = blockIdx.x * 16 + (threadIdx.x & 15), seg = threadIdx.x >> 4;
  float s = 0.0f;
  if (e < dim)
    for (int r = seg; r < rows; r += 16) s += part[(int64_t)r * dim + e];
  sm[threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.x < 16 && e < dim) {
    float t = 0.0f;
    for (int i = 0; i < 16; ++i) t += sm[16 * i + threadIdx.x];
    dw[e] = t;
  }
}

int pow2_at_least(int n) {
  int p = 1;
  while (p < n) p *= 2;
  return p;
}

bool is_aligned(const void* p, int64_t st, int64_t sh, int elems, int size) {
  return (reinterpret_cast<uintptr_t>(p) % (uintptr_t)(elems * size)) == 0 && st % elems == 0 && sh % elems == 0;
}

int check(const DofNormRope* d, const char* who) {
  if (!d) { dof_set_error("%s: null descriptor", who); return DOF_ERR_ARG; }
  if (d->dtype < DOF_DTYPE_F32 || d->dtype > DOF_DTYPE_F16) { dof_set_error("%s: unknown dtype %d", who, (int)d->dtype); return DOF_ERR_ARG; }
  if (d->head_dim < 2 || d->head_dim > kMaxDim || d->head_dim % 2) {
    dof_set_error("%s: head_dim %d (an even number from 2 to %d is supported)", who, (int)d->head_dim, kMaxDim);
    return DOF_ERR_UNSUPPORTED;
  }
  if (d->rot_dim < 0 || d->rot_dim > d->head_dim || d->rot_dim % 2) {
    dof_set_error("%s: rot_dim %d must be even and at most head_dim %d", who, (int)d->rot_dim, (int)d->head_dim);
    return DOF_ERR_ARG;
  }
  if (d->q_heads < 1 || d->k_heads < 1 || d->q_heads > 65535 || d->k_heads > 65535 || d->tokens < 0) {
    dof_set_error("%s: bad sizes (tokens %lld, heads %d / %d)", who, (long long)d->tokens, (int)d->q_heads, (int)d->k_heads);
    return DOF_ERR_ARG;
  }
  return DOF_OK;
}

template <class T, int VEC, bool BWD>
void launch_vec(const Args& A, dim3 grid, hipStream_t stream) {
  if (VEC == 1 && A.dim > 128) DOF_LAUNCH((k_norm_rope<T, VEC, VEC == 1 ? 2 : 1, BWD>), (grid.x, grid.y, 1), (256, 1, 1), stream, A);
  else DOF_LAUNCH((k_norm_rope<T, VEC, 1, BWD>), (grid.x, grid.y, 1), (256, 1, 1), stream, A);
}

// The widest run that divides the rotated pairs, the row and every address and stride.
template <class T, bool BWD>
int launch(Args A, hipStream_t stream) {
  constexpr int most = 16 / (int)sizeof(T);
  int vec = most;
  auto fits = [&](int v) {
    if (A.half % v || (A.dim / 2) % v) return false;
    for (const Side& s : A.side) {
      if (!is_aligned(s.x, s.xt, s.xh, v, sizeof(T)) || !is_aligned(s.out, s.ot, s.oh, v, sizeof(T))) return false;
      if (BWD && !is_aligned(s.g, s.gt, s.gh, v, sizeof(T))) return false;
    }
    return true;
  };
  while (vec > 1 && !fits(vec)) vec /= 2;
  A.lpr = pow2_at_least((A.dim / 2 + vec - 1) / vec);
  if (A.lpr > 64) A.lpr = 64;
  // Tokens per workgroup: enough rows to pay for the angles, but no fewer than ~2048 workgroups while there are tokens for them
  // (65536 tokens: 16 per workgroup; a single token: one workgroup per tensor).
  int64_t tb = A.tokens / 2048;
  const int64_t top = A.half ? kTable / A.half : 64;
  if (tb > top) tb = top;
  if (tb > 64) tb = 64;
  if (tb < 1) tb = 1;
  A.tb = (int)tb;
  A.chunks = (A.tokens + tb - 1) / tb;
  int64_t blocks = A.chunks;
  if (BWD && blocks > kBwdBlocks) blocks = kBwdBlocks;
  if (blocks > 1 << 30) blocks = 1 << 30;
  const dim3 grid((unsigned)blocks, 2, 1);
  if constexpr (sizeof(T) == 2) {
    if (vec == 8) { launch_vec<T, 8, BWD>(A, grid, stream); return (int)blocks; }
  }
  if (vec == 4) launch_vec<T, 4, BWD>(A, grid, stream);
  else if (vec == 2) launch_vec<T, 2, BWD>(A, grid, stream);
  else launch_vec<T, 1, BWD>(A, grid, stream);
  return (int)blocks;
}

Args common(const DofNormRope* d, const int32_t* positions, const double* freqs) {
  Args A;
  A.pos = positions;
  A.freqs = freqs;
  A.tokens = d->tokens;
  A.eps = d->eps;
  A.dim = d->head_dim;
  A.half = d->rot_dim / 2;
  A.interleaved = d->interleaved != 0;
  A.tb = A.lpr = 1;
  A.chunks = 0;
  return A;
}

}  // namespace

extern "C" int dof_norm_rope_forward(const DofNormRope* d, const void* q, const void* k, const int32_t* positions, const double* freqs,
                                     const float* q_weight, const float* k_weight, void* q_out, void* k_out, void* stream) {
  const int rc = check(d, "dof_norm_rope_forward");
  if (rc != DOF_OK) return rc;
  if (d->tokens == 0) return DOF_OK;
  if (!q || !k || !q_out || !k_out || (d->rot_dim && (!positions || !freqs))) {
    dof_set_error("dof_norm_rope_forward: null tensor");
    return DOF_ERR_ARG;
  }
  Args A = common(d, positions, freqs);
  A.side[0] = {q, nullptr, q_out, q_weight, nullptr, d->q_stride[0], d->q_stride[1], 0, 0, d->q_out_stride[0], d->q_out_stride[1], d->q_heads};
  A.side[1] = {k, nullptr, k_out, k_weight, nullptr, d->k_stride[0], d->k_stride[1], 0, 0, d->k_out_stride[0], d->k_out_stride[1], d->k_heads};
  DOF_SEQ_DISPATCH(d->dtype, T, (launch<T, false>(A, (hipStream_t)stream)));
  return dof_check_launch("k_norm_rope");
}

extern "C" int64_t dof_norm_rope_workspace_bytes(const DofNormRope* d) {
  if (check(d, "dof_norm_rope_workspace_bytes") != DOF_OK) return -1;
  return 2LL * kBwdBlocks * d->head_dim * 4;
}

extern "C" int dof_norm_rope_backward(const DofNormRope* d, const void* gq, const void* gk, const void* q, const void* k,
                                      const int32_t* positions, const double* freqs, const float* q_weight, const float* k_weight,
                                      void* dq, void* dk, float* dq_weight, float* dk_weight, void* workspace, void* stream) {
  const int rc = check(d, "dof_norm_rope_backward");
  if (rc != DOF_OK) return rc;
  if (!q_weight != !dq_weight || !k_weight != !dk_weight) {
    dof_set_error("dof_norm_rope_backward: a weight and its gradient go together");
    return DOF_ERR_ARG;
  }
  const bool empty = d->tokens == 0;
  if (!empty && (!gq || !gk || !q || !k || !dq || !dk || (d->rot_dim && (!positions || !freqs)))) {
    dof_set_error("dof_norm_rope_backward: null tensor");
    return DOF_ERR_ARG;
  }
  if ((q_weight || k_weight) && !workspace) {
    dof_set_error("dof_norm_rope_backward: null workspace");
    return DOF_ERR_ARG;
  }
  int rows = 0;
  float* part = static_cast<float*>(workspace);
  if (!empty) {
    Args A = common(d, positions, freqs);
    A.side[0] = {q, gq, dq, q_weight, part, d->q_stride[0], d->q_stride[1], d->gq_stride[0], d->gq_stride[1],
                 d->q_out_stride[0], d->q_out_stride[1], d->q_heads};
    A.side[1] = {k, gk, dk, k_weight, part ? part + (int64_t)kBwdBlocks * d->head_dim : nullptr, d->k_stride[0], d->k_stride[1],
                 d->gk_stride[0], d->gk_stride[1], d->k_out_stride[0], d->k_out_stride[1], d->k_heads};
    DOF_SEQ_DISPATCH(d->dtype, T, (rows = launch<T, true>(A, (hipStream_t)stream)));
  }
  if (q_weight || k_weight)
    DOF_LAUNCH(k_norm_rope_dw, (dof_cdiv(d->head_dim, 16), 2, 1), (256, 1, 1), (hipStream_t)stream, part,
               part + (int64_t)kBwdBlocks * d->head_dim, dq_weight, dk_weight, rows, (int)d->head_dim);
  return dof_check_launch("k_norm_rope (backward)");
}
