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
  int one_run;                 // a lane's pairs are one aligned run
};

// Where a lane's pairs p .. p + VEC - 1 lie in a row: two runs of VEC elements, first members and second members (apart: the rotated part
// of the half layout), or one run of 2 VEC elements, pair by pair (interleaved, and the elements behind the rotated part: they start at
// rot_dim, so pair p starts at 2 p there too).
struct Place { int a, b; bool apart; };
__device__ __forceinline__ Place place_of(const Args& A, int p, int vec) {
  if (p < A.half && !A.interleaved) return {p, p + A.half, true};
  return {2 * p, 2 * p + vec, false};
}

// the runs as loaded, so that the next row's loads run under the present row's arithmetic
template <class T, int VEC, bool INTER> struct Raw {
  static constexpr int kBytes = (int)sizeof(T) * VEC;
  static constexpr bool kOne = INTER && 2 * kBytes <= 16;  // both runs are one access
  static constexpr int N = kOne ? (2 * kBytes + 3) / 4 : (kBytes + 3) / 4;
  DofWords<N> u, v;
  __device__ __forceinline__ void load(const T* row, const Place& at) {
    if constexpr (kOne) {
      u = *reinterpret_cast<const DofWords<N>*>(row + at.a);
    } else if constexpr (kBytes >= 4) {
      u = *reinterpret_cast<const DofWords<N>*>(row + at.a);
      v = *reinterpret_cast<const DofWords<N>*>(row + at.b);
    } else {
      u.w[0] = *reinterpret_cast<const uint16_t*>(row + at.a);
      v.w[0] = *reinterpret_cast<const uint16_t*>(row + at.b);
    }
  }
  __device__ __forceinline__ void pairs(const Place& at, float* a, float* b) const {
    float x[2 * VEC < 2 ? 2 : 2 * VEC + 2];  // the runs one behind the other
    if constexpr (kOne) {
      DofElem<T>::unpack(u, x);
    } else {
      DofElem<T>::unpack(u, x);
      float y[VEC + 1];
      DofElem<T>::unpack(v, y);
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[VEC + i] = y[i];
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      a[i] = !INTER && at.apart ? x[i] : x[2 * i];
      b[i] = !INTER && at.apart ? x[VEC + i] : x[2 * i + 1];
    }
  }
};
template <class T, int VEC, bool INTER>
__device__ __forceinline__ void store_pairs(T* row, const Place& at, const float* a, const float* b) {
  float x[2 * VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const bool apart = !INTER && at.apart;
    x[i] = apart ? a[i] : (i & 1) ? b[i / 2] : a[i / 2];
    x[VEC + i] = apart ? b[i] : ((i + VEC) & 1) ? b[(i + VEC) / 2] : a[(i + VEC) / 2];
  }
  if constexpr (Raw<T, VEC, INTER>::kOne) {
    dof_store_vec<T, 2 * VEC>(row + at.a, x);
  } else {
    dof_store_vec<T, VEC>(row + at.a, x);
    dof_store_vec<T, VEC>(row + at.b, x + VEC);
  }
}

// sum over the lpr lanes of a row (a uniform choice of lane permutations; every lane ends with the same bits)
__device__ __forceinline__ float row_sum(float v, int lpr) {
  if (lpr >= 2) v += dof_dpp_perm<0xB1>(v);
  if (lpr >= 4) v += dof_dpp_perm<0x4E>(v);
  if (lpr >= 8) v += dof_dpp_perm<0x141>(v);
  if (lpr >= 16) v += dof_dpp_perm<0x140>(v);
  if (lpr >= 32) v += __shfl_xor(v, 16);
  if (lpr >= 64) v += dof_swap32(v);
  return v;
}

// T = element type, VEC = pairs per lane; NI = rounds of lpr lanes over a row's pairs (2 only for VEC = 1 and heads over 128); INTER: no
// pair lies apart
template <class T, int VEC, int NI, bool INTER, bool BWD>
__global__ void __launch_bounds__(256) k_norm_rope(Args A) {
  __shared__ float tab[2 * kTable];
  const Side& S = A.side[blockIdx.y];
  const int tid = threadIdx.x;
  const int lane = tid & (A.lpr - 1);
  const int rpp = 256 / A.lpr;  // rows per pass
  const int row0 = tid / A.lpr;
  const float inv_dim = 1.0f / (float)A.dim;
  const bool normed = S.w != nullptr;

  Place at[NI];
  bool live[NI];
  float wa[NI][VEC], wb[NI][VEC], da[NI][VEC], db[NI][VEC];
  float ta[NI][VEC], tb[NI][VEC];  // weight gradients of whole chunks: two short chains of additions in place of a long one
#pragma unroll
  for (int n = 0; n < NI; ++n) {
    const int p = (lane + n * A.lpr) * VEC;
    live[n] = 2 * p < A.dim;
    at[n] = place_of(A, p, VEC);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      wa[n][i] = wb[n][i] = 1.0f;
      da[n][i] = db[n][i] = ta[n][i] = tb[n][i] = 0.0f;
      if (live[n] && normed) {
        wa[n][i] = S.w[at[n].apart ? at[n].a + i : at[n].a + 2 * i];
        wb[n][i] = S.w[at[n].apart ? at[n].b + i : at[n].a + 2 * i + 1];
      }
    }
  }

  Raw<T, VEC, INTER> rx[NI], rg[NI];
  const int t_step = rpp / S.heads, h_step = rpp - t_step * S.heads;
  for (int64_t chunk = blockIdx.x; chunk < A.chunks; chunk += gridDim.x) {
    const int64_t t0 = chunk * A.tb;
    const int nt = (int)(A.tokens - t0 < A.tb ? A.tokens - t0 : A.tb), rows = nt * S.heads;
    // row r = head h of token t0 + t; the next row of this thread is rpp further (one division per chunk)
    int t_next = row0 / S.heads, h_next = row0 - t_next * S.heads;
    auto load = [&](int r) {
      if (r >= rows) return;
      const T* xr = static_cast<const T*>(S.x) + (t0 + t_next) * S.xt + h_next * S.xh;
      const T* gr = static_cast<const T*>(S.g) + (t0 + t_next) * S.gt + h_next * S.gh;
#pragma unroll
      for (int n = 0; n < NI; ++n) {
        if (!live[n]) continue;
        if (!BWD || normed) rx[n].load(xr, at[n]);
        if (BWD) rg[n].load(gr, at[n]);
      }
    };
    load(row0);  // in flight while the angles are computed
    __syncthreads();
    for (int e = tid; e < nt * A.half; e += 256) {
      const int t = e / A.half, p = e - t * A.half;
      float s, c;
      dof_sincos_turns((double)A.pos[t0 + t] * (A.freqs[p] * 0.15915494309189533577), &s, &c);
      tab[2 * e] = c;
      tab[2 * e + 1] = s;
    }
    __syncthreads();
    for (int r = row0; r < (rows + rpp - 1) / rpp * rpp; r += rpp) {
      const bool inside = r < rows;
      const int t = inside ? t_next : 0, h = inside ? h_next : 0;
      t_next += t_step;
      h_next += h_step;
      if (h_next >= S.heads) {
        h_next -= S.heads;
        ++t_next;
      }
      float a[NI][VEC], b[NI][VEC], ga[NI][VEC], gb[NI][VEC];
      float ss = 0.0f;
#pragma unroll
      for (int n = 0; n < NI; ++n) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) a[n][i] = b[n][i] = ga[n][i] = gb[n][i] = 0.0f;
        if (inside && live[n]) {
          if (!BWD || normed) rx[n].pairs(at[n], a[n], b[n]);
          if (BWD) rg[n].pairs(at[n], ga[n], gb[n]);
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) ss = fmaf(a[n][i], a[n][i], fmaf(b[n][i], b[n][i], ss));
      }
      load(r + rpp);
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
        if (inside && live[n]) store_pairs<T, VEC, INTER>(orow, at[n], BWD ? ga[n] : a[n], BWD ? gb[n] : b[n]);
    }
    if (BWD && normed) {
#pragma unroll
      for (int n = 0; n < NI; ++n)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          ta[n][i] += da[n][i];
          tb[n][i] += db[n][i];
          da[n][i] = db[n][i] = 0.0f;
        }
    }
  }

  if constexpr (BWD) {
    if (!normed) return;
    // the row groups of a wavefront meet by lane exchanges, the four wavefronts in LDS, always in the same order
#pragma unroll
    for (int n = 0; n < NI; ++n)
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        for (int m = A.lpr; m < 64; m <<= 1) {
          ta[n][i] += __shfl_xor(ta[n][i], m);
          tb[n][i] += __shfl_xor(tb[n][i], m);
        }
    __syncthreads();
    if ((tid & 63) < A.lpr) {
#pragma unroll
      for (int n = 0; n < NI; ++n)
        if (live[n]) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            tab[(tid >> 6) * kMaxDim + (at[n].apart ? at[n].a + i : at[n].a + 2 * i)] = ta[n][i];
            tab[(tid >> 6) * kMaxDim + (at[n].apart ? at[n].b + i : at[n].a + 2 * i + 1)] = tb[n][i];
          }
        }
    }
    __syncthreads();
    for (int e = tid; e < A.dim; e += 256)
      S.dw_part[(int64_t)blockIdx.x * A.dim + e] = (tab[e] + tab[kMaxDim + e]) + (tab[2 * kMaxDim + e] + tab[3 * kMaxDim + e]);
  }
}

// dw[e] = sum over the partial rows, each thread's in row order, the threads' in thread order: the same sum every run.
// One workgroup per 8 elements and side; 32 threads share an element, eight loads in flight each.
__global__ void __launch_bounds__(256) k_norm_rope_dw(const float* part_q, const float* part_k, float* dwq, float* dwk, int rows, int dim) {
  __shared__ float sm[256];
  const float* part = blockIdx.y ? part_k : part_q;
  float* dw = blockIdx.y ? dwk : dwq;
  if (!dw) return;  // uniform over the workgroup
  const int e = blockIdx.x * 8 + (threadIdx.x & 7), seg = threadIdx.x >> 3;
  float s = 0.0f;
  if (e < dim)
    for (int r = seg; r < rows; r += 256) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = r + 32 * k < rows ? part[(int64_t)(r + 32 * k) * dim + e] : 0.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k) s += v[k];
    }
  sm[threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.x < 8 && e < dim) {
    float t = 0.0f;
    for (int i = 0; i < 32; ++i) t += sm[8 * i + threadIdx.x];
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
  if (VEC == 1 && A.dim > 128) DOF_LAUNCH((k_norm_rope<T, VEC, VEC == 1 ? 2 : 1, false, BWD>), (grid.x, grid.y, 1), (256, 1, 1), stream, A);
  else if (A.one_run) DOF_LAUNCH((k_norm_rope<T, VEC, 1, true, BWD>), (grid.x, grid.y, 1), (256, 1, 1), stream, A);
  else DOF_LAUNCH((k_norm_rope<T, VEC, 1, false, BWD>), (grid.x, grid.y, 1), (256, 1, 1), stream, A);
}

// The widest run that divides the rotated pairs, the row and every address and stride.
template <class T, bool BWD>
int launch(Args A, hipStream_t stream) {
  constexpr int most = 16 / (int)sizeof(T);
  int vec = most;
  auto fits = [&](int v) {
    if (A.half % v || (A.dim / 2) % v) return false;
    const bool one = (A.interleaved || A.half == 0) && 2 * v * (int)sizeof(T) <= 16;  // both runs in one access
    const int w = one ? 2 * v : v;
    for (const Side& s : A.side) {
      if (!is_aligned(s.x, s.xt, s.xh, w, sizeof(T)) || !is_aligned(s.out, s.ot, s.oh, w, sizeof(T))) return false;
      if (BWD && !is_aligned(s.g, s.gt, s.gh, w, sizeof(T))) return false;
    }
    return true;
  };
  while (vec > 1 && !fits(vec)) vec /= 2;
  A.one_run = (A.interleaved || A.half == 0) && fits(vec);
  A.lpr = pow2_at_least((A.dim / 2 + vec - 1) / vec);
  if (A.lpr > 64) A.lpr = 64;
  // Tokens per workgroup: enough rows to pay for the angles and the weights, but no fewer than 1024 workgroups per tensor while there are
  // tokens for them (20011 tokens of 16 heads of 80, fp16, forward + backward: 70 us with 1024, 76 with 2048, 82 with 512).
  int64_t tb = A.tokens / 1024;
  const int64_t top = A.half ? kTable / A.half : 64;
  if (tb > top) tb = top;
  if (tb > 64) tb = 64;
  if (tb < 1) tb = 1;
  A.tb = (int)tb;
  A.chunks = (A.tokens + tb - 1) / tb;
  int64_t blocks = A.chunks;
  if (BWD && blocks > kBwdBlocks) blocks = kBwdBlocks;
  if (blocks > 1 << 20) blocks = 1 << 20;  // a launch holds less than 2^32 threads; the kernel goes through the chunks in strides
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
  A.one_run = 0;
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
    DOF_LAUNCH(k_norm_rope_dw, (dof_cdiv(d->head_dim, 8), 2, 1), (256, 1, 1), (hipStream_t)stream, part,
               part + (int64_t)kBwdBlocks * d->head_dim, dq_weight, dk_weight, rows, (int)d->head_dim);
  return dof_check_launch("k_norm_rope (backward)");
}
