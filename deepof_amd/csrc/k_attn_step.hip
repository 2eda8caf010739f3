// The new frames of live streams against a paged key / value cache.
//
//   o_t = sum_j softmax_j(score(q_t, k_j)) v_j over the stream's cached frames and its new ones up to t
//
// Bound by memory: every cached key and value is read once (all query heads of a key head, times the new frames, share the read: they
// are the rows of one 16-row product, v_mfma_*_16x16x32).  The length of a stream is split over workgroups, and a workgroup's part
// over its four wavefronts, 32 frames at a time; each keeps its own running maximum and sum.  The wavefronts meet in LDS, the
// workgroups' partial results in the workspace, joined by k_attn_step_join.
//
// Inside a wavefront the products are transposed as in the forward pass (S^T = K Q^T, O^T = V^T P^T): keys go from memory straight
// into the operand registers (a lane's 16 bytes are eight elements of one key), values through a wavefront-private LDS tile for the
// transposing read, and the next tile's loads and page lookups are in flight under the present one's products.
// New frames are read from k and v, not from the cache, so storing them (by the first workgroup of a stream's head) races with nobody.
#include <cmath>
#include <cstring>

#include "deepof_hip.h"
#include "dof_rt.h"
#include "launchers.h"
#include "seq_attn.h"

namespace {

constexpr int kStepKeys = 32;   // frames per wavefront and round
constexpr int kMinTiles = 8;    // rounds worth a workgroup of their own: two per wavefront
constexpr int kMaxSplits = 512;

struct Step {
  DofAttnStep d;
  DofScore score;
  const void *q, *k, *v;
  void *kc, *vc;
  const int32_t *table, *lengths;
  const float* slopes;
  void* o;
  float* part;    // [stream][key head][split][row][dim] unnormalised sums, then [..][row][2] maximum and sum
  float* stat;
  int32_t splits, rows, row_blocks;
};

// Where a frame lives: page >= 0 and its slot there, a new frame (kFresh, its number), or nowhere.
constexpr int kNowhere = -1, kFresh = -2;
struct Slot { int page, at; };
__device__ __forceinline__ Slot find_slot(const Step& A, const int32_t* table, int len, int total, int key) {
  Slot s = {kNowhere, 0};
  if (key >= total) return s;
  const int p = key / A.d.page_size, page = table[p];
  if (page < 0 || page >= A.d.n_pages) return s;
  s.page = key < len ? page : kFresh;
  s.at = key < len ? key - p * A.d.page_size : key - len;
  return s;
}

struct Rows {  // one of the two cached tensors and its new frames, of one stream and head
  const char *cache, *fresh;
  int64_t page, slot, step;  // strides in bytes
};
template <class T> __device__ __forceinline__ const T* row_at(const Rows& r, int page, int at) {
  return reinterpret_cast<const T*>(page >= 0 ? r.cache + page * r.page + at * r.slot : r.fresh + at * r.step);
}

// RT: tiles of 16 rows.  MULTI: more than one new frame.
template <class T, int DP, int RT, bool MULTI>
__global__ void __launch_bounds__(256) k_attn_step(Step A) {
  using Tile = DofTile<T, kStepKeys, DP>;
  __shared__ Tile sv[4];
  __shared__ float sm[4][16 * RT], sl[4][16 * RT];
  constexpr int KS = DP / 32, DT = DP / 16, NV = (kStepKeys * Tile::CH + 63) / 64, EPC = Tile::EPC;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, quad = lane >> 4;
  const int dim = A.d.head_dim, nnew = A.d.new_frames, group = A.d.q_heads / A.d.k_heads;
  int64_t item = blockIdx.x;
  const int rb = (int)(item % A.row_blocks);
  item /= A.row_blocks;
  const int split = (int)(item % A.splits);
  item /= A.splits;
  const int hk = (int)(item % A.d.k_heads), b = (int)(item / A.d.k_heads);

  int len = A.lengths[b];
  if (len < 0) return;  // uniform: an idle stream
  const int64_t capacity = (int64_t)A.d.max_pages * A.d.page_size;
  if (len > capacity) len = (int)capacity;
  const int total = (int)(len + nnew < capacity ? len + nnew : capacity);
  const int tiles = (total + kStepKeys - 1) / kStepKeys;
  int per = (tiles + A.splits - 1) / A.splits;
  if (per < kMinTiles) per = kMinTiles;
  const int32_t* table = A.table + (int64_t)b * A.d.max_pages;

  if (split == 0 && rb == 0) {  // the new frames into the cache
    const int chunks = dim / EPC;
    for (int e = tid; e < nnew * chunks; e += 256) {
      const int t = e / chunks, c = e - t * chunks, at = len + t;
      if (at >= total) continue;
      const int p = at / A.d.page_size, page = table[p];
      if (page < 0 || page >= A.d.n_pages) continue;
      const int s = at - p * A.d.page_size;
      const T* kn = static_cast<const T*>(A.k) + b * A.d.k_stride[0] + t * A.d.k_stride[1] + hk * A.d.k_stride[2];
      const T* vn = static_cast<const T*>(A.v) + b * A.d.v_stride[0] + t * A.d.v_stride[1] + hk * A.d.v_stride[2];
      T* kd = static_cast<T*>(A.kc) + page * A.d.kc_stride[0] + s * A.d.kc_stride[1] + hk * A.d.kc_stride[2];
      T* vd = static_cast<T*>(A.vc) + page * A.d.vc_stride[0] + s * A.d.vc_stride[1] + hk * A.d.vc_stride[2];
      reinterpret_cast<DofWords<4>*>(kd)[c] = reinterpret_cast<const DofWords<4>*>(kn)[c];
      reinterpret_cast<DofWords<4>*>(vd)[c] = reinterpret_cast<const DofWords<4>*>(vn)[c];
    }
  }
  const int tile0 = split * per, tile1 = tile0 + per < tiles ? tile0 + per : tiles;
  if (A.splits > 1 && tile0 >= tile1 && split > 0) return;  // uniform; the join knows which parts exist

  // rows of this block: row r = new frame r / group, head r % group of the key head's group
  int kend[RT];
  float slope[RT];
  int pos[RT];
  DofFrag<T> q[RT][KS];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int r = rb * 16 * RT + 16 * i + col;
    const bool live = r < A.rows;
    const int t = live ? r / group : 0, g = live ? r - t * group : 0;
    pos[i] = len + t;
    kend[i] = live ? pos[i] + 1 : 0;
    slope[i] = A.slopes && live ? A.slopes[hk * group + g] * kLog2e : 0.0f;
    const T* qp = static_cast<const T*>(A.q) + b * A.d.q_stride[0] + t * A.d.q_stride[1] + (hk * group + g) * A.d.q_stride[2];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int e = 32 * s + 8 * quad;
      q[i][s] = dof_frag_zero<T>();
      if (live && e < dim) q[i][s] = dof_frag_load<T>(qp + e);
    }
  }
  Rows kr, vr;
  {
    const T* kc = static_cast<const T*>(A.kc) + hk * A.d.kc_stride[2];
    const T* vc = static_cast<const T*>(A.vc) + hk * A.d.vc_stride[2];
    const T* kn = static_cast<const T*>(A.k) + b * A.d.k_stride[0] + hk * A.d.k_stride[2];
    const T* vn = static_cast<const T*>(A.v) + b * A.d.v_stride[0] + hk * A.d.v_stride[2];
    const int64_t es = sizeof(T);
    kr = {(const char*)kc, (const char*)kn, A.d.kc_stride[0] * es, A.d.kc_stride[1] * es, A.d.k_stride[1] * es};
    vr = {(const char*)vc, (const char*)vn, A.d.vc_stride[0] * es, A.d.vc_stride[1] * es, A.d.v_stride[1] * es};
  }

  dof_f32x4 o[RT][DT];
  float m[RT], l[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.0f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[i][d] = dof_zero4();
  }

  DofFrag<T> kf[2][KS];
  DofWords<4> vreg[NV];
  auto slot_of = [&](int tile) { return find_slot(A, table, len, tile < tile1 ? total : 0, tile * kStepKeys + (lane & 31)); };
  auto load = [&](Slot slot) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int page = dof_shfl_int(slot.page, 16 * u + col), at = dof_shfl_int(slot.at, 16 * u + col);
      const T* p = row_at<T>(kr, page, at);
#pragma unroll
      for (int c = 0; c < KS; ++c) {
        const int e = 32 * c + 8 * quad;
        kf[u][c] = dof_frag_zero<T>();
        if (page != kNowhere && e < dim) kf[u][c] = dof_frag_load<T>(p + e);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = lane + 64 * i, r = e / Tile::CH, c = e - r * Tile::CH;
      const int page = dof_shfl_int(slot.page, r & 31), at = dof_shfl_int(slot.at, r & 31);
#pragma unroll
      for (int w = 0; w < 4; ++w) vreg[i].w[w] = 0u;
      if (r < kStepKeys && page != kNowhere && c * EPC < dim) vreg[i] = *reinterpret_cast<const DofWords<4>*>(row_at<T>(vr, page, at) + c * EPC);
    }
  };

  int tile = tile0 + wave;
  Slot slot = slot_of(tile), ahead = slot_of(tile + 4);
  load(slot);
  for (; tile < tile1; tile += 4) {
    const int j0 = tile * kStepKeys;
    const uint32_t there = (uint32_t)dof_ballot(slot.page != kNowhere && lane < 32);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = lane + 64 * i, r = e / Tile::CH, c = e - r * Tile::CH;
      if ((kStepKeys * Tile::CH) % 64 == 0 || r < kStepKeys) sv[wave].put(r, c, vreg[i]);
    }
    dof_f32x4 x[RT][2];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        x[i][u] = dof_zero4();
#pragma unroll
        for (int c = 0; c < KS; ++c) x[i][u] = dof_mma16<T>(kf[u][c], q[i][c], x[i][u]);
      }
    slot = ahead;
    if (tile + 4 < tile1) {  // uniform over the wavefront
      load(slot);
      ahead = slot_of(tile + 8);
    }
    DOF_WAVE_LDS_ORDER();
    // keys 16 u + 4 quad + e of the tile, e = 0 .. 3, sit in this lane's registers
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      float mt = -INFINITY;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int kk = 16 * u + 4 * quad + e;
          float w = x[i][u][e] * A.score.mul;
          if (A.score.cap_l2 != 0.0f) w = A.score.cap_l2 * dof_cap_tanh<T>(w);
          w -= slope[i] * fabsf((float)(pos[i] - j0 - kk));
          if (j0 + kk >= kend[i] || !((there >> kk) & 1u)) w = -INFINITY;
          x[i][u][e] = w;
          mt = fmaxf(mt, w);
        }
      mt = fmaxf(mt, __shfl_xor(mt, 16));
      mt = fmaxf(mt, dof_swap32(mt));
      if (dof_wave_any(mt > m[i] + 8.0f)) {  // as in the forward pass: the maximum follows in steps of 2^8
        const float mn = fmaxf(m[i], mt);
        const float a = mn == -INFINITY ? 1.0f : dof_exp2(m[i] - mn);
        m[i] = mn;
        l[i] *= a;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][d][e] *= a;
      }
      const float mm = m[i] == -INFINITY ? 0.0f : m[i];
      float p[8];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[4 * u + e] = dof_exp2(x[i][u][e] - mm);
          l[i] += p[4 * u + e];
        }
      const DofFrag<T> pf = dof_frag_pack<T>(p);
      // several new frames: a later one's value is hidden from the earlier rows, whose zero weight must not meet an infinity or NaN
      bool careful = false;
      if (MULTI && j0 + kStepKeys > len + 1) {
        bool bad = false;
#pragma unroll
        for (int d = 0; d < DT; ++d) bad |= dof_frag_nonfinite<T>(sv[wave].colfrag(4 * quad, 16 + 4 * quad, 16 * d + col));
        careful = dof_wave_any(bad);
      }
      if (!careful) {
#pragma unroll
        for (int d = 0; d < DT; ++d) o[i][d] = dof_mma16<T>(sv[wave].colfrag(4 * quad, 16 + 4 * quad, 16 * d + col), pf, o[i][d]);
      } else {
        float seen[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int kk = 16 * (e / 4) + 4 * quad + e % 4;
          seen[e] = j0 + kk < kend[i] && ((there >> kk) & 1u) ? 1.0f : 0.0f;
        }
        const DofFrag<T> sf = dof_frag_pack<T>(seen);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          DofFrag<T> f = sv[wave].colfrag(4 * quad, 16 + 4 * quad, 16 * d + col), pos_f, neg_f;
          dof_frag_split<T>(f, pos_f, neg_f);
          o[i][d] = dof_mma16<T>(f, pf, o[i][d]);
          const dof_f32x4 up = dof_mma16<T>(pos_f, sf, dof_zero4()), down = dof_mma16<T>(neg_f, sf, dof_zero4());
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (up[e] > 0.0f) o[i][d][e] += INFINITY;
            if (down[e] > 0.0f) o[i][d][e] -= INFINITY;
          }
        }
      }
    }
    DOF_WAVE_LDS_ORDER();
  }

  // the four wavefronts meet: a common maximum, then their sums one after the other
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    l[i] += __shfl_xor(l[i], 16);
    l[i] += dof_swap32(l[i]);
    if (quad == 0) {
      sm[wave][16 * i + col] = m[i];
      sl[wave][16 * i + col] = l[i];
    }
  }
  __syncthreads();  // also: every wavefront is done with its value tile
  float lt[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    float mn = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) mn = fmaxf(mn, sm[w][16 * i + col]);
    lt[i] = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float mw = sm[w][16 * i + col];
      lt[i] += mw == -INFINITY ? sl[w][16 * i + col] : sl[w][16 * i + col] * dof_exp2(mw - mn);
    }
    const float a = m[i] == -INFINITY ? 1.0f : dof_exp2(m[i] - mn);  // -inf: nothing seen, the sums are zeros (or NaN)
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][d][e] *= a;
    m[i] = mn;
  }
  float* meet = reinterpret_cast<float*>(sv);  // [16 RT rows][DP]
  static_assert(sizeof(sv) >= 16 * RT * DP * sizeof(float), "the value tiles hold the meeting place");
  for (int w = 1; w < 4; ++w) {
    if (wave == w) {
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) meet[(16 * i + col) * DP + 16 * d + 4 * quad + e] = o[i][d][e];
    }
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][d][e] += meet[(16 * i + col) * DP + 16 * d + 4 * quad + e];
    }
    __syncthreads();
  }
  if (wave != 0) return;
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int r = rb * 16 * RT + 16 * i + col;
    if (r >= A.rows) continue;
    if (A.splits == 1) {
      const int t = r / group, g = r - t * group;
      const float inv = lt[i] > 0.0f ? 1.0f / lt[i] : (lt[i] == 0.0f ? 0.0f : lt[i]);
      T* op = static_cast<T*>(A.o) + b * A.d.o_stride[0] + t * A.d.o_stride[1] + (hk * group + g) * A.d.o_stride[2];
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const int e = 16 * d + 4 * quad;
        if (e < dim) {
          const float v[4] = {o[i][d][0] * inv, o[i][d][1] * inv, o[i][d][2] * inv, o[i][d][3] * inv};
          dof_store_vec<T, 4>(op + e, v);
        }
      }
    } else {
      const int64_t at = (((int64_t)b * A.d.k_heads + hk) * A.splits + split) * A.rows + r;
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const int e = 16 * d + 4 * quad;
        if (e < dim) {
          const float v[4] = {o[i][d][0], o[i][d][1], o[i][d][2], o[i][d][3]};
          dof_store_vec<float, 4>(A.part + at * dim + e, v);
        }
      }
      if (quad == 0) {
        A.stat[at * 2] = m[i];
        A.stat[at * 2 + 1] = lt[i];
      }
    }
  }
}

// o of one row from its parts: a workgroup per row, eight groups of 32 lanes (four elements each) share the parts.
template <class T>
__global__ void __launch_bounds__(256) k_attn_step_join(Step A) {
  __shared__ float so[8][128];
  __shared__ float sw[kMaxSplits];
  __shared__ float red[4][2];
  const int tid = threadIdx.x, dim = A.d.head_dim, group = A.d.q_heads / A.d.k_heads;
  int64_t item = blockIdx.x;
  const int r = (int)(item % A.rows);
  item /= A.rows;
  const int hk = (int)(item % A.d.k_heads), b = (int)(item / A.d.k_heads);
  int len = A.lengths[b];
  if (len < 0) return;
  const int64_t capacity = (int64_t)A.d.max_pages * A.d.page_size;
  if (len > capacity) len = (int)capacity;
  const int total = (int)(len + A.d.new_frames < capacity ? len + A.d.new_frames : capacity);
  const int tiles = (total + kStepKeys - 1) / kStepKeys;
  int per = (tiles + A.splits - 1) / A.splits;
  if (per < kMinTiles) per = kMinTiles;
  int parts = (tiles + per - 1) / per;
  if (parts < 1) parts = 1;
  const int64_t base = ((int64_t)b * A.d.k_heads + hk) * A.splits;

  float mx = -INFINITY;
  for (int s = tid; s < parts; s += 256) mx = fmaxf(mx, A.stat[((base + s) * A.rows + r) * 2]);
  for (int k = 32; k > 0; k >>= 1) mx = fmaxf(mx, __shfl_xor(mx, k));
  if ((tid & 63) == 0) red[tid >> 6][0] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(red[0][0], red[1][0]), fmaxf(red[2][0], red[3][0]));
  float sum = 0.0f;
  for (int s = tid; s < parts; s += 256) {
    const float* st = A.stat + ((base + s) * A.rows + r) * 2;
    const float w = st[0] == -INFINITY ? 1.0f : dof_exp2(st[0] - mx);
    sw[s] = w;
    sum += w * st[1];
  }
  for (int k = 32; k > 0; k >>= 1) sum += __shfl_xor(sum, k);
  if ((tid & 63) == 0) red[tid >> 6][1] = sum;
  __syncthreads();
  sum = (red[0][1] + red[1][1]) + (red[2][1] + red[3][1]);
  const int e = 4 * (tid & 31), grp = tid >> 5;
  float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (e < dim)
    for (int s = grp; s < parts; s += 8) {
      float v[4];
      dof_load_vec<float, 4>(A.part + ((base + s) * A.rows + r) * dim + e, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = fmaf(sw[s], v[i], acc[i]);
    }
#pragma unroll
  for (int i = 0; i < 4; ++i) so[grp][e + i] = acc[i];
  __syncthreads();
  if (tid < 32 && e < dim) {
    const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int g = 0; g < 8; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += so[g][e + i];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] *= inv;
    const int t = r / group, g = r - t * group;
    dof_store_vec<T, 4>(static_cast<T*>(A.o) + b * A.d.o_stride[0] + t * A.d.o_stride[1] + (hk * group + g) * A.d.o_stride[2] + e, v);
  }
}

int check(const DofAttnStep* d, const char* who) {
  if (!d) { dof_set_error("%s: null descriptor", who); return DOF_ERR_ARG; }
  if (d->dtype < DOF_DTYPE_F32 || d->dtype > DOF_DTYPE_F16) { dof_set_error("%s: unknown dtype %d", who, (int)d->dtype); return DOF_ERR_ARG; }
  if (d->head_dim < 8 || d->head_dim > 128 || d->head_dim % 8) {
    dof_set_error("%s: head_dim %d (multiples of 8 from 8 to 128 are supported)", who, (int)d->head_dim);
    return DOF_ERR_UNSUPPORTED;
  }
  if (d->k_heads < 1 || d->q_heads < d->k_heads || d->q_heads % d->k_heads || d->streams < 0) {
    dof_set_error("%s: %d query heads are not a multiple of %d key heads, or bad streams", who, (int)d->q_heads, (int)d->k_heads);
    return DOF_ERR_ARG;
  }
  if (d->new_frames < 1 || d->new_frames > 16) {
    dof_set_error("%s: %d new frames (1 to 16 are supported; longer runs are dof_attention_forward's)", who, (int)d->new_frames);
    return DOF_ERR_UNSUPPORTED;
  }
  if (d->n_pages < 1 || d->page_size < 1 || d->max_pages < 1 || (int64_t)d->n_pages * d->page_size > 0x7FFFFFFF ||
      (int64_t)d->max_pages * d->page_size > 1 << 30) {
    dof_set_error("%s: bad cache (%d pages of %d frames, %d in a table)", who, (int)d->n_pages, (int)d->page_size, (int)d->max_pages);
    return DOF_ERR_ARG;
  }
  if (!std::isfinite(d->scale) || !std::isfinite(d->cap) || d->cap < 0.0f) {
    dof_set_error("%s: scale and cap must be finite, cap not negative", who);
    return DOF_ERR_ARG;
  }
  return DOF_OK;
}

// Row tiles of 16 per workgroup (1 or 2), blocks of them, and parts of a stream's length: enough workgroups to fill the chip and to
// even out streams of different length, none smaller than two rounds per wavefront.  From the table's width: the lengths themselves
// are device data (a workgroup whose part is empty ends at once).
struct Shape { int rows, rt, row_blocks, splits; };
Shape shape_of(const DofAttnStep* d) {
  Shape s;
  s.rows = d->q_heads / d->k_heads * d->new_frames;
  s.rt = s.rows > 16 ? 2 : 1;
  s.row_blocks = (s.rows + 16 * s.rt - 1) / (16 * s.rt);
  const int64_t base = (int64_t)d->streams * d->k_heads * s.row_blocks;
  const int64_t tiles = ((int64_t)d->max_pages * d->page_size + kStepKeys - 1) / kStepKeys;
  int64_t want = base > 0 ? (4096 + base - 1) / base : 1;
  const int64_t most = (tiles + kMinTiles - 1) / kMinTiles;
  if (want > most) want = most;
  if (want > kMaxSplits) want = kMaxSplits;
  s.splits = (int)(want < 1 ? 1 : want);
  return s;
}

bool aligned(const void* p, const int64_t* s, int size) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s[0] * size % 16 == 0 && s[1] * size % 16 == 0 && s[2] * size % 16 == 0;
}

template <class T, int DP>
void launch_rt(const Step& A, int rt, unsigned blocks, hipStream_t stream) {
  const bool multi = A.d.new_frames > 1;
  if (rt == 1 && !multi) DOF_LAUNCH((k_attn_step<T, DP, 1, false>), (blocks, 1, 1), (256, 1, 1), stream, A);
  else if (rt == 1) DOF_LAUNCH((k_attn_step<T, DP, 1, true>), (blocks, 1, 1), (256, 1, 1), stream, A);
  else if (!multi) DOF_LAUNCH((k_attn_step<T, DP, 2, false>), (blocks, 1, 1), (256, 1, 1), stream, A);
  else DOF_LAUNCH((k_attn_step<T, DP, 2, true>), (blocks, 1, 1), (256, 1, 1), stream, A);
}

}  // namespace

extern "C" int64_t dof_attention_step_workspace_bytes(const DofAttnStep* d) {
  if (check(d, "dof_attention_step_workspace_bytes") != DOF_OK) return -1;
  const Shape s = shape_of(d);
  if (s.splits == 1) return 0;
  return (int64_t)d->streams * d->k_heads * s.splits * s.rows * (d->head_dim + 2) * 4;
}

extern "C" int dof_attention_step(const DofAttnStep* d, const void* q, const void* k, const void* v, void* k_cache, void* v_cache,
                                  const int32_t* page_table, const int32_t* lengths, const float* slopes, void* o, void* workspace,
                                  void* stream) {
  const int rc = check(d, "dof_attention_step");
  if (rc != DOF_OK) return rc;
  if (d->streams == 0) return DOF_OK;
  const Shape s = shape_of(d);
  if (!q || !k || !v || !k_cache || !v_cache || !page_table || !lengths || !o || (s.splits > 1 && !workspace)) {
    dof_set_error("dof_attention_step: null tensor");
    return DOF_ERR_ARG;
  }
  const int size = d->dtype == DOF_DTYPE_F32 ? 4 : 2;
  if (!aligned(q, d->q_stride, size) || !aligned(k, d->k_stride, size) || !aligned(v, d->v_stride, size) || !aligned(o, d->o_stride, size) ||
      !aligned(k_cache, d->kc_stride, size) || !aligned(v_cache, d->vc_stride, size)) {
    dof_set_error("dof_attention_step: tensors and strides must be multiples of 16 bytes");
    return DOF_ERR_UNSUPPORTED;
  }
  const int64_t blocks = (int64_t)d->streams * d->k_heads * s.splits * s.row_blocks;
  const int64_t joins = (int64_t)d->streams * d->k_heads * s.rows;
  if (blocks > 0x7FFFFFFF || joins > 0x7FFFFFFF) {
    dof_set_error("dof_attention_step: too many streams and heads for one launch");
    return DOF_ERR_UNSUPPORTED;
  }
  Step A;
  memset(&A, 0, sizeof(A));
  A.d = *d;
  if (d->cap > 0.0f) {
    A.score.mul = d->scale / d->cap;
    A.score.cap_l2 = d->cap * kLog2e;
  } else {
    A.score.mul = d->scale * kLog2e;
  }
  A.q = q;
  A.k = k;
  A.v = v;
  A.kc = k_cache;
  A.vc = v_cache;
  A.table = page_table;
  A.lengths = lengths;
  A.slopes = slopes;
  A.o = o;
  A.part = static_cast<float*>(workspace);
  A.stat = A.part ? A.part + (int64_t)d->streams * d->k_heads * s.splits * s.rows * d->head_dim : nullptr;
  A.splits = s.splits;
  A.rows = s.rows;
  A.row_blocks = s.row_blocks;
  DOF_SEQ_DISPATCH(d->dtype, T, {
    if (d->head_dim <= 32) launch_rt<T, 32>(A, s.rt, (unsigned)blocks, (hipStream_t)stream);
    else if (d->head_dim <= 64) launch_rt<T, 64>(A, s.rt, (unsigned)blocks, (hipStream_t)stream);
    else if (d->head_dim <= 96) launch_rt<T, 96>(A, s.rt, (unsigned)blocks, (hipStream_t)stream);
    else launch_rt<T, 128>(A, s.rt, (unsigned)blocks, (hipStream_t)stream);
    if (s.splits > 1) DOF_LAUNCH((k_attn_step_join<T>), ((unsigned)joins, 1, 1), (256, 1, 1), (hipStream_t)stream, A);
  });
  return dof_check_launch("k_attn_step");
}
