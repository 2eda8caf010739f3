// The new frames of live streams against a paged key / value cache.
//
//   o_t = sum_j softmax_j(score(q_t, k_j)) v_j over the stream's cached frames and its new ones up to t
//
// Bound by memory: every cached key and value is read once (all query heads of a key head, times the new frames, share the read: they
// are the rows of one 16-row product, v_mfma_*_16x16x32).  The length of a stream is split over workgroups, and a workgroup's part
// over its four wavefronts, 32 frames at a time; each keeps its own running maximum and sum.  The wavefronts meet in LDS, the
// workgroups' partial results in the workspace, joined by k_attn_step_join.
//
// The lengths are device data, so the split is made on the device: every workgroup adds up the streams' lengths, takes the part size
// that yields about kTarget parts in all and finds the stream its own part lies in.  All parts are then about equally long, whatever the
// mix of streams, and few workgroups are left without one (a split made on the host for the longest possible stream left most of
// them empty or the longest stream's for the end: 64 streams of up to 5000 frames 81 us).  Work that every workgroup does for every
// stream grows with their square: more than kFind streams have a kernel of one workgroup that lists the parts first, and streams
// that all stay whole need no split.
//
// Inside a wavefront the products are transposed as in the forward pass (S^T = K Q^T, O^T = V^T P^T): keys go from memory straight
// into the operand registers (a lane's 16 bytes are eight elements of one key), values through a wavefront-private LDS tile for the
// transposing read, and the next tile's loads and page lookups are in flight under the present one's products.  A lane looks up one
// frame of a round and loads half of that frame's value itself, so that a round's loads are one address and fixed offsets per lane
// (with an address per load the address arithmetic took longer than the loads: 64 streams of up to 5000 frames 201 us).
// New frames are read from k and v, not from the cache, so storing them (by the first workgroup of a stream's head) races with nobody.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "deepof_hip.h"
#include "dof_rt.h"
#include "launchers.h"
#include "seq_attn.h"

namespace {

constexpr int kStepKeys = 32;   // frames per wavefront and round
constexpr int kMinTiles = 16;   // rounds of a part at least: four per wavefront
// Streams whose table holds no more rounds stay whole, which saves the second kernel for the join.  Replayed from a graph (eager calls
// hide their kernels behind the host), 8 / 2 heads of 64, one stream, whole against parts: 768 frames 11 / 15 us, 1024 13.6 / 14.7,
// 1536 18.6 / 14.7, 2048 24 / 15; 128 streams: 14 / 20, 17 / 22, 24 / 27, 30 / 37.
constexpr int kWhole = 32;
constexpr int kTarget = 1024;   // parts of a call in all: two rounds of two workgroups per CU

constexpr int kFind = 256;      // streams up to which every workgroup finds its part itself: one length per thread

struct Step {
  DofAttnStep d;
  DofScore score;
  const void *q, *k, *v;
  void *kc, *vc;
  const int32_t *table, *lengths;
  const float* slopes;
  void* o;
  float* part;    // [part][key head][row][dim] unnormalised sums
  float* stat;    // [part][key head][row][2] maximum and sum
  int32_t* sched; // [stream][2] first part and their number
  int32_t* units; // more than kFind streams in parts: [part] its stream (-1: none), then the part size in tiles
  int32_t parts;  // workgroups per key head and row block: parts at most; `whole`: streams
  int32_t whole;  // every stream is one part
  int32_t rows, row_blocks, min_tiles, join_lanes, page_shift;  // page_shift: log2 of the page size, -1 if it is no power of two
};

// the page of frame `key` and its slot there; page -1: nowhere
__device__ __forceinline__ int find_page(const Step& A, const int32_t* table, int total, int key, int* slot) {
  if (key >= total) return -1;
  const int p = A.page_shift >= 0 ? key >> A.page_shift : key / A.d.page_size, page = table[p];
  *slot = key - p * A.d.page_size;
  return page >= 0 && page < A.d.n_pages ? page : -1;
}

// frames of stream b after the call (0: idle)
__device__ __forceinline__ int frames_of(const Step& A, int b, int* len) {
  *len = A.lengths[b];
  if (*len < 0) return 0;
  const int64_t capacity = (int64_t)A.d.max_pages * A.d.page_size;
  if (*len > capacity) *len = (int)capacity;
  return (int)(*len + A.d.new_frames < capacity ? *len + A.d.new_frames : capacity);
}
__device__ __forceinline__ int tiles_of(const Step& A, int b) {
  int len;
  return (frames_of(A, b, &len) + kStepKeys - 1) / kStepKeys;
}

// tiles of a part, of `all` tiles of the streams
__device__ __forceinline__ int part_size(const Step& A, int64_t all) {
  const int64_t share = (all * A.d.k_heads * A.row_blocks + kTarget - 1) / kTarget, most = 1 << 30;  // more than the tiles of any stream
  return share > most ? (int)most : share > A.min_tiles ? (int)share : A.min_tiles;
}

// The stream and the part of it that is number `unit` of all parts, and the part size in tiles; by all 256 threads, for kFind streams.
struct Part { int stream, index, count, per; };
__device__ __forceinline__ Part find_part(const Step& A, int unit) {
  __shared__ int low[4], high[4], upto_wave[4], found[3];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int tiles = tid < A.d.streams ? tiles_of(A, tid) : 0;
  auto wave_sum = [&](int v) {
    for (int k = 32; k > 0; k >>= 1) v += dof_shfl_int(v, lane ^ k);
    return v;
  };
  const int lo = wave_sum(tiles & 0xFFFF), hi = wave_sum(tiles >> 16);  // in two halves of 16 bits: the sum itself may pass 32
  if (tid == 0) found[0] = -1;
  if (lane == 0) {
    low[wave] = lo;
    high[wave] = hi;
  }
  __syncthreads();
  Part p;
  p.per = part_size(A, (int64_t)(low[0] + low[1] + low[2] + low[3]) + ((int64_t)(high[0] + high[1] + high[2] + high[3]) << 16));
  const int n = (tiles + p.per - 1) / p.per;
  int upto = n;  // inclusive sum over the wavefront
  for (int k = 1; k < 64; k <<= 1) {
    const int below = dof_shfl_int(upto, lane >= k ? lane - k : lane);
    if (lane >= k) upto += below;
  }
  if (lane == 63) upto_wave[wave] = upto;
  __syncthreads();
  int first = upto - n;
  for (int w = 0; w < wave; ++w) first += upto_wave[w];
  if (n > 0 && unit >= first && unit < first + n) {
    found[0] = tid;
    found[1] = unit - first;
    found[2] = n;
  }
  __syncthreads();
  p.stream = found[0];
  p.index = found[1];
  p.count = found[2];
  return p;
}

// The parts of all streams, by one workgroup: sched and units.
__global__ void __launch_bounds__(1024) k_attn_step_plan(Step A) {
  __shared__ int64_t sums[1024];
  __shared__ int upto_wave[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int64_t all = 0;
  for (int b = tid; b < A.d.streams; b += 1024) all += tiles_of(A, b);
  sums[tid] = all;
  for (int k = 512; k > 0; k >>= 1) {
    __syncthreads();
    if (tid < k) sums[tid] += sums[tid + k];
  }
  __syncthreads();
  const int per = part_size(A, sums[0]);
  int before = 0;
  for (int b0 = 0; b0 < A.d.streams; b0 += 1024) {
    const int b = b0 + tid, n = b < A.d.streams ? (tiles_of(A, b) + per - 1) / per : 0;
    int upto = n;  // inclusive sum over the wavefront
    for (int k = 1; k < 64; k <<= 1) {
      const int below = dof_shfl_int(upto, lane >= k ? lane - k : lane);
      if (lane >= k) upto += below;
    }
    if (lane == 63) upto_wave[wave] = upto;
    __syncthreads();
    int first = before + upto - n;
    for (int w = 0; w < wave; ++w) first += upto_wave[w];
    for (int w = 0; w < 16; ++w) before += upto_wave[w];
    if (n > 0) {
      A.sched[2 * b] = first;
      A.sched[2 * b + 1] = n;
      for (int k = 0; k < n; ++k) A.units[first + k] = b;
    }
    __syncthreads();  // the next round writes upto_wave
  }
  for (int u = before + tid; u < A.parts; u += 1024) A.units[u] = -1;
  if (tid == 0) A.units[A.parts] = per;
}

// Four elements of a row's output: the sums divided by the weights' sum, and with several new frames the infinities and NaN among the
// values that the row sees of them (left out of the products).
template <class T>
__device__ __forceinline__ void finish(const Step& A, const int32_t* table, int b, int hk, int r, int e, int len, int total, float l, float* v) {
  const int group = A.d.q_heads / A.d.k_heads, t = r / group, g = r - t * group;
  const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);  // nothing seen: zeros; NaN stays NaN
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] *= inv;
  if (A.d.new_frames > 1)
    for (int i = 0; i <= t; ++i) {
      int slot;
      if (find_page(A, table, total, len + i, &slot) < 0) continue;
      const T* vn = static_cast<const T*>(A.v) + b * A.d.v_stride[0] + i * A.d.v_stride[1] + hk * A.d.v_stride[2] + e;
      float x[4];
      dof_load_vec<T, 4>(vn, x);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (!(fabsf(x[k]) < INFINITY)) v[k] += x[k];
    }
  dof_store_vec<T, 4>(static_cast<T*>(A.o) + b * A.d.o_stride[0] + t * A.d.o_stride[1] + (hk * group + g) * A.d.o_stride[2] + e, v);
}

// RT: tiles of 16 rows.  MULTI: more than one new frame.  LONG: a wavefront's sums may grow long and are made of blocks (fp32)
template <class T, int DP, int RT, bool MULTI, bool LONG>
__global__ void __launch_bounds__(256, sizeof(T) == 4 && DP > 32 * (3 - RT) + 32 ? 1 : 2) k_attn_step(Step A) {
  using Tile = DofTile<T, kStepKeys, DP>;
  __shared__ Tile sv[4];
  __shared__ float sm[4][16 * RT], sl[4][16 * RT];
  constexpr int KS = DP / 32, DT = DP / 16, NV = Tile::CH / 2, EPC = Tile::EPC;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, quad = lane >> 4;
  const int dim = A.d.head_dim, nnew = A.d.new_frames, group = A.d.q_heads / A.d.k_heads;
  int item = blockIdx.x;  // row block, then key head, then part
  const int rb = item % A.row_blocks;
  item /= A.row_blocks;
  const int unit = item / A.d.k_heads, hk = item - unit * A.d.k_heads;
  Part part;
  if (A.whole) {
    part = {unit, 0, 1, 1 << 30};
  } else if (A.units) {
    part.stream = A.units[unit];
    part.per = A.units[A.parts];
    part.index = part.stream < 0 ? 0 : unit - A.sched[2 * part.stream];
    part.count = part.stream < 0 ? 0 : A.sched[2 * part.stream + 1];
  } else {
    part = find_part(A, unit);
  }
  if (part.stream < 0) return;  // uniform: fewer parts than workgroups
  const int b = part.stream;
  int len;
  const int total = frames_of(A, b, &len);
  if (total == 0) return;  // uniform: idle
  const int tiles = (total + kStepKeys - 1) / kStepKeys;
  const int32_t* table = A.table + (int64_t)b * A.d.max_pages;
  if (A.sched && !A.units && part.index == 0 && hk == 0 && rb == 0 && tid == 0) {
    A.sched[2 * b] = unit;
    A.sched[2 * b + 1] = part.count;
  }

  if (part.index == 0 && rb == 0) {  // the new frames into the cache
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
  const int tile0 = part.index * part.per, tile1 = tile0 + part.per < tiles ? tile0 + part.per : tiles;

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
  // byte offsets of a frame from the first element of this head in the caches; a new frame's lead to k and v themselves
  const char* const kbase = reinterpret_cast<const char*>(static_cast<const T*>(A.kc) + hk * A.d.kc_stride[2]);
  const char* const vbase = reinterpret_cast<const char*>(static_cast<const T*>(A.vc) + hk * A.d.vc_stride[2]);
  const int64_t kfresh = reinterpret_cast<const char*>(static_cast<const T*>(A.k) + b * A.d.k_stride[0] + hk * A.d.k_stride[2]) - kbase;
  const int64_t vfresh = reinterpret_cast<const char*>(static_cast<const T*>(A.v) + b * A.d.v_stride[0] + hk * A.d.v_stride[2]) - vbase;

  dof_f32x4 o[RT][DT];
  DofLongSum<T, dof_f32x4, DT, LONG> lo[RT];
  DofLongNumber<T> l[RT];
  float m[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    m[i] = -INFINITY;
    lo[i].clear();
#pragma unroll
    for (int d = 0; d < DT; ++d) o[i][d] = dof_zero4();
  }

  DofFrag<T> kf[2][KS];
  DofWords<4> vreg[NV];
  struct Where { int page, slot; };
  // the lane's frame of a tile (lanes l and l + 32: the same one)
  auto look_up = [&](int tile) {
    Where w = {-1, 0};
    w.page = find_page(A, table, tile < tile1 ? total : 0, tile * kStepKeys + (lane & 31), &w.slot);
    return w;
  };
  // Loads of a tile.  A frame that is nowhere reads the head's first one instead: its score is masked, its value made zero.  Elements
  // behind the head size read its start: those of keys are made zero before the product (an infinity there would meet q's zeros),
  // those of values are columns of the result that are not written.
  auto load = [&](int tile, Where w) {
    const int key = tile * kStepKeys + (lane & 31);
    int64_t ko = w.page * A.d.kc_stride[0] + w.slot * A.d.kc_stride[1], vo = w.page * A.d.vc_stride[0] + w.slot * A.d.vc_stride[1];
    ko = w.page < 0 ? 0 : ko * (int64_t)sizeof(T);
    vo = w.page < 0 ? 0 : vo * (int64_t)sizeof(T);
    if (w.page >= 0 && key >= len) {
      ko = kfresh + (key - len) * A.d.k_stride[1] * (int64_t)sizeof(T);
      vo = vfresh + (key - len) * A.d.v_stride[1] * (int64_t)sizeof(T);
    }
    const int lo = (int)(uint32_t)ko, hi = (int)(ko >> 32);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t l32 = (uint32_t)dof_shfl_int(lo, 16 * u + col);
      const int64_t off = ((int64_t)dof_shfl_int(hi, 16 * u + col) << 32) | l32;
      const T* p = reinterpret_cast<const T*>(kbase + off);
#pragma unroll
      for (int c = 0; c < KS; ++c) {
        const int e = 32 * c + 8 * quad;
        kf[u][c] = dof_frag_load<T>(p + (e < dim ? e : 0));
      }
    }
    const T* p = reinterpret_cast<const T*>(vbase + vo);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = ((lane >> 5) + 2 * i) * EPC;
      vreg[i] = *reinterpret_cast<const DofWords<4>*>(p + (e < dim ? e : 0));
    }
  };

  int tile = tile0 + wave;
  Where here = look_up(tile), ahead = look_up(tile + 4);
  load(tile, here);
  for (; tile < tile1; tile += 4) {
    const int j0 = tile * kStepKeys;
    const uint32_t there = (uint32_t)dof_ballot(here.page >= 0);
    const bool inner = there == 0xFFFFFFFFu && j0 + kStepKeys <= len + 1;  // uniform: every row sees every frame of the tile
    if (!inner) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int k = 0; k < 4; ++k) vreg[i].w[k] = here.page >= 0 ? vreg[i].w[k] : 0u;
        // several new frames: a later one's value is hidden from the earlier rows, whose zero weight must not meet an infinity or
        // NaN; finish() puts such values where they are seen
        if (MULTI && j0 + (lane & 31) >= len) dof_make_finite<T>(vreg[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) sv[wave].put(lane & 31, (lane >> 5) + 2 * i, vreg[i]);
    if (32 * (KS - 1) + 8 * quad >= dim) kf[0][KS - 1] = kf[1][KS - 1] = dof_frag_zero<T>();
    dof_f32x4 x[RT][2];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        x[i][u] = dof_zero4();
#pragma unroll
        for (int c = 0; c < KS; ++c) x[i][u] = dof_mma16<T>(kf[u][c], q[i][c], x[i][u]);
      }
    if (tile + 4 < tile1) {  // uniform over the wavefront
      here = ahead;
      load(tile + 4, here);
      ahead = look_up(tile + 8);
    }
    DOF_WAVE_LDS_ORDER();
    // keys 16 u + 4 quad + e of the tile, e = 0 .. 3, sit in this lane's registers
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      if (A.score.cap_l2 != 0.0f) {
        float th[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) th[k] = x[i][k / 4][k % 4];
        dof_cap_tanh<8>(th, A.score.mul);
#pragma unroll
        for (int k = 0; k < 8; ++k) x[i][k / 4][k % 4] = A.score.cap_l2 * th[k];
      } else {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[i][u][e] *= A.score.mul;
      }
      if (A.slopes) {
        const float base = (float)(pos[i] - j0 - 4 * quad);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[i][u][e] -= slope[i] * fabsf(base - (float)(16 * u + e));
      }
      if (!inner) {
        const uint32_t mine = there >> (4 * quad);
        const int left = kend[i] - j0 - 4 * quad;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool seen = (16 * u + e < left) & (((mine >> (16 * u + e)) & 1u) != 0u);
            x[i][u][e] = seen ? x[i][u][e] : -INFINITY;
          }
      }
      float mt = -INFINITY;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) mt = fmaxf(mt, x[i][u][e]);
      mt = fmaxf(mt, __shfl_xor(mt, 16));
      mt = fmaxf(mt, dof_swap32(mt));
      if (dof_wave_any(mt > m[i] + DofSoftmax<T>::kLag)) {  // as in the forward pass: the maximum follows in steps, row by row
        const bool up = mt > m[i] + DofSoftmax<T>::kLag;
        const float a = up ? dof_exp2(m[i] - mt) : 1.0f;
        m[i] = up ? mt : m[i];
        l[i].scale(a);
        lo[i].scale(a);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][d][e] *= a;
      }
      const float mm = m[i] == -INFINITY ? 0.0f : m[i] - DofSoftmax<T>::kUp;  // a factor of the sums as of the weights
      float p[8], part = 0.0f;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[4 * u + e] = dof_exp2(x[i][u][e] - mm);
          part += p[4 * u + e];
        }
      l[i].add(part);
      // 16-bit weights as value and rest: rounded once they made o's error 1.4 times that of rounding it; the second product runs under
      // the loads (64 streams of up to 5000 frames 56.7 -> 57.9 us, two streams of 200000 frames 94.4 -> 95.5)
      const DofFrag<T> pf = dof_frag_pack<T>(p), rest = dof_frag_rest<T>(p, pf);
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const DofFrag<T> vf = sv[wave].colfrag(4 * quad, 16 + 4 * quad, 16 * d + col);
        o[i][d] = dof_mma16<T>(vf, pf, o[i][d]);
        if constexpr (sizeof(T) == 2) o[i][d] = dof_mma16<T>(vf, rest, o[i][d]);
      }
      lo[i].count(o[i], kStepKeys / 2);  // terms: kLongTerms allows for two per addition, a 16x16x4 product adds four
    }
    DOF_WAVE_LDS_ORDER();
  }

  // The four wavefronts meet in LDS: each leaves its sums in its own value tile, then every thread adds up the four of its elements,
  // weighted to the rows' common maximum.
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    lo[i].finish(o[i]);
    float sum = l[i].total();
    sum += __shfl_xor(sum, 16);
    sum += dof_swap32(sum);
    if (quad == 0) {
      sm[wave][16 * i + col] = m[i];
      sl[wave][16 * i + col] = sum;
    }
  }
  static_assert(sizeof(Tile) >= 16 * DP * sizeof(float), "a value tile holds sixteen rows of sums");
  auto meet = [&](int w, int row, int c) { return reinterpret_cast<DofWords<4>*>(sv[w].mem) + row * (DP / 4) + (c ^ (row & 7)); };
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    if (i > 0) __syncthreads();
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      const float v[4] = {o[i][d][0], o[i][d][1], o[i][d][2], o[i][d][3]};
      DofElem<float>::pack(v, *meet(wave, col, 4 * d + quad));
    }
    __syncthreads();
    for (int e4 = tid; e4 < 4 * DP; e4 += 256) {
      const int row = e4 / (DP / 4), c = e4 - row * (DP / 4), r = rb * 16 * RT + 16 * i + row, at = 16 * i + row;
      if (r >= A.rows || 4 * c >= dim) continue;
      float mn = -INFINITY;
#pragma unroll
      for (int w = 0; w < 4; ++w) mn = fmaxf(mn, sm[w][at]);
      float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f}, lt = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = sm[w][at] == -INFINITY ? 1.0f : dof_exp2(sm[w][at] - mn);  // -inf: nothing seen, zeros (or NaN)
        float v[4];
        DofElem<float>::unpack(*meet(w, row, c), v);
        lt = fmaf(f, sl[w][at], lt);
#pragma unroll
        for (int k = 0; k < 4; ++k) sum[k] = fmaf(f, v[k], sum[k]);
      }
      if (part.count == 1) {
        finish<T>(A, table, b, hk, r, 4 * c, len, total, lt, sum);
      } else {
        const int64_t to = ((int64_t)unit * A.d.k_heads + hk) * A.rows + r;
        dof_store_vec<float, 4>(A.part + to * dim + 4 * c, sum);
        if (c == 0) {
          A.stat[to * 2] = mn;
          A.stat[to * 2 + 1] = lt;
        }
      }
    }
  }
}

// o of the streams in several parts: a workgroup per row, groups of 32 lanes (four elements each) share the parts, four loads in flight
// each.  Few rows (of long streams, in many parts): a workgroup per row and 32 elements, groups of 8 lanes.
template <class T>
__global__ void __launch_bounds__(256) k_attn_step_join(Step A) {
  __shared__ float so[1152];  // [groups][4 lanes + 4]: 32 x 36 or 8 x 132
  __shared__ float red[4][2];
  const int tid = threadIdx.x, dim = A.d.head_dim, lanes = A.join_lanes, groups = 256 / lanes, pitch = 4 * lanes + 4;
  int item = blockIdx.x;
  const int r = item % A.rows;
  item /= A.rows;
  const int b = item / A.d.k_heads, hk = item - b * A.d.k_heads;
  int len;
  const int total = frames_of(A, b, &len);
  if (total == 0) return;
  const int first = A.sched[2 * b], parts = A.sched[2 * b + 1];
  if (parts == 1) return;  // written by its only workgroup
  auto at = [&](int s) { return ((int64_t)(first + s) * A.d.k_heads + hk) * A.rows + r; };

  float mx = -INFINITY;
  for (int s = tid; s < parts; s += 256) mx = fmaxf(mx, A.stat[at(s) * 2]);
  for (int k = 32; k > 0; k >>= 1) mx = fmaxf(mx, __shfl_xor(mx, k));
  if ((tid & 63) == 0) red[tid >> 6][0] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(red[0][0], red[1][0]), fmaxf(red[2][0], red[3][0]));
  auto weight = [&](float m) { return m == -INFINITY ? 1.0f : dof_exp2(m - mx); };  // -inf: nothing seen, zeros (or NaN)
  float sum = 0.0f;
  for (int s = tid; s < parts; s += 256) sum = fmaf(weight(A.stat[at(s) * 2]), A.stat[at(s) * 2 + 1], sum);
  for (int k = 32; k > 0; k >>= 1) sum += __shfl_xor(sum, k);
  if ((tid & 63) == 0) red[tid >> 6][1] = sum;
  const int l = tid & (lanes - 1), e = 4 * (lanes * (int)blockIdx.y + l), grp = tid / lanes;
  float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (e < dim) {
    for (int s0 = grp; s0 < parts; s0 += 4 * groups) {
      float v[4][4], w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const bool in = s0 + groups * k < parts;
        const int64_t from = at(in ? s0 + groups * k : s0);
        dof_load_vec<float, 4>(A.part + from * dim + e, v[k]);
        w[k] = A.stat[from * 2];
        if (!in) v[k][0] = v[k][1] = v[k][2] = v[k][3] = 0.0f;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float f = weight(w[k]);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = fmaf(f, v[k][i], acc[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) so[grp * pitch + 4 * l + i] = acc[i];
  __syncthreads();
  sum = (red[0][1] + red[1][1]) + (red[2][1] + red[3][1]);
  if (tid < lanes && e < dim) {
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int g = 0; g < groups; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += so[g * pitch + 4 * l + i];
    finish<T>(A, A.table + (int64_t)b * A.d.max_pages, b, hk, r, e, len, total, sum, v);
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

// Row tiles of 16 per workgroup (1 or 2), blocks of them, and the most parts that find_part can make of the streams: each at most
// one more than its share, and no more than its table holds.
struct Shape { int rows, rt, row_blocks, min_tiles; int64_t parts; };
Shape shape_of(const DofAttnStep* d) {
  Shape s;
  s.rows = d->q_heads / d->k_heads * d->new_frames;
  s.rt = s.rows > 16 ? 2 : 1;
  s.row_blocks = (s.rows + 16 * s.rt - 1) / (16 * s.rt);
  const int64_t tiles = ((int64_t)d->max_pages * d->page_size + kStepKeys - 1) / kStepKeys;
  s.min_tiles = tiles <= kWhole ? kWhole : kMinTiles;
  s.parts = d->streams + kTarget / ((int64_t)d->k_heads * s.row_blocks);
  const int64_t most = (tiles + s.min_tiles - 1) / s.min_tiles * d->streams;
  if (s.parts > most) s.parts = most;
  return s;
}
bool joins(const DofAttnStep* d, const Shape& s) { return s.parts > d->streams; }
int64_t part_floats(const DofAttnStep* d, const Shape& s) { return s.parts * d->k_heads * s.rows * d->head_dim; }

bool aligned(const void* p, const int64_t* s, int size) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s[0] * size % 16 == 0 && s[1] * size % 16 == 0 && s[2] * size % 16 == 0;
}

template <class T, int DP, int RT>
void launch_rt(const Step& A, bool grows, unsigned blocks, hipStream_t stream) {
  const bool multi = A.d.new_frames > 1;
  if constexpr (sizeof(T) == 4) {
    if (grows) {
      if (multi) DOF_LAUNCH((k_attn_step<T, DP, RT, true, true>), (blocks, 1, 1), (256, 1, 1), stream, A);
      else DOF_LAUNCH((k_attn_step<T, DP, RT, false, true>), (blocks, 1, 1), (256, 1, 1), stream, A);
      return;
    }
  }
  if (multi) DOF_LAUNCH((k_attn_step<T, DP, RT, true, false>), (blocks, 1, 1), (256, 1, 1), stream, A);
  else DOF_LAUNCH((k_attn_step<T, DP, RT, false, false>), (blocks, 1, 1), (256, 1, 1), stream, A);
}
template <class T, int DP>
void launch(const Step& A, int rt, bool grows, unsigned blocks, hipStream_t stream) {
  if (rt == 1) launch_rt<T, DP, 1>(A, grows, blocks, stream);
  else launch_rt<T, DP, 2>(A, grows, blocks, stream);
}

}  // namespace

extern "C" int64_t dof_attention_step_workspace_bytes(const DofAttnStep* d) {
  if (check(d, "dof_attention_step_workspace_bytes") != DOF_OK) return -1;
  const Shape s = shape_of(d);
  if (!joins(d, s)) return 0;
  return (part_floats(d, s) + s.parts * d->k_heads * s.rows * 2 + 2 * (int64_t)d->streams + (d->streams > kFind ? s.parts + 1 : 0)) * 4;
}

extern "C" int dof_attention_step(const DofAttnStep* d, const void* q, const void* k, const void* v, void* k_cache, void* v_cache,
                                  const int32_t* page_table, const int32_t* lengths, const float* slopes, void* o, void* workspace,
                                  void* stream) {
  const int rc = check(d, "dof_attention_step");
  if (rc != DOF_OK) return rc;
  if (d->streams == 0) return DOF_OK;
  const Shape s = shape_of(d);
  if (!q || !k || !v || !k_cache || !v_cache || !page_table || !lengths || !o || (joins(d, s) && !workspace)) {
    dof_set_error("dof_attention_step: null tensor");
    return DOF_ERR_ARG;
  }
  const int size = d->dtype == DOF_DTYPE_F32 ? 4 : 2;
  if (!aligned(q, d->q_stride, size) || !aligned(k, d->k_stride, size) || !aligned(v, d->v_stride, size) || !aligned(o, d->o_stride, size) ||
      !aligned(k_cache, d->kc_stride, size) || !aligned(v_cache, d->vc_stride, size)) {
    dof_set_error("dof_attention_step: tensors and strides must be multiples of 16 bytes");
    return DOF_ERR_UNSUPPORTED;
  }
  const int64_t blocks = s.parts * d->k_heads * s.row_blocks;
  const int64_t rows = (int64_t)d->streams * d->k_heads * s.rows;
  if (blocks >= 1 << 24 || rows >= 1 << 24) {  // of 256 threads: a launch holds less than 2^32
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
  if (joins(d, s)) {
    A.part = static_cast<float*>(workspace);
    A.stat = A.part + part_floats(d, s);
    A.sched = reinterpret_cast<int32_t*>(A.stat + s.parts * d->k_heads * s.rows * 2);
    if (d->streams > kFind) A.units = A.sched + 2 * (int64_t)d->streams;
  }
  A.parts = (int32_t)s.parts;
  A.whole = !joins(d, s);
  A.rows = s.rows;
  A.row_blocks = s.row_blocks;
  A.min_tiles = s.min_tiles;
  A.join_lanes = rows < 512 ? 8 : 32;
  A.page_shift = -1;
  if ((d->page_size & (d->page_size - 1)) == 0)
    while ((int64_t)1 << (A.page_shift + 1) <= d->page_size) ++A.page_shift;
  // the most tiles that the streams' tables let a part have, four wavefronts to share them, kStepKeys / 4 additions each
  const int64_t tiles = ((int64_t)d->max_pages * d->page_size + kStepKeys - 1) / kStepKeys, share = d->streams * tiles * d->k_heads * s.row_blocks / kTarget;
  const bool grows = std::max<int64_t>(s.min_tiles, share) / 4 * (kStepKeys / 2) > kLongTerms;
  if (A.units) DOF_LAUNCH(k_attn_step_plan, (1, 1, 1), (1024, 1, 1), (hipStream_t)stream, A);
  DOF_SEQ_DISPATCH(d->dtype, T, {
    if (d->head_dim <= 32) launch<T, 32>(A, s.rt, grows, (unsigned)blocks, (hipStream_t)stream);
    else if (d->head_dim <= 64) launch<T, 64>(A, s.rt, grows, (unsigned)blocks, (hipStream_t)stream);
    else if (d->head_dim <= 96) launch<T, 96>(A, s.rt, grows, (unsigned)blocks, (hipStream_t)stream);
    else launch<T, 128>(A, s.rt, grows, (unsigned)blocks, (hipStream_t)stream);
    if (joins(d, s)) DOF_LAUNCH((k_attn_step_join<T>), ((unsigned)rows, dof_cdiv(d->head_dim, 4 * A.join_lanes), 1), (256, 1, 1), (hipStream_t)stream, A);
  });
  return dof_check_launch("k_attn_step");
}
