// The packed documents of an attention call and what its kernels share: the plan's tiles, the mask, the score function.
#pragma once
#include "seq_tiles.h"

// One tile of a document: rows row0 .. of its query (or key) rows.  The plan's table is four lists of these: query tiles of 128 and of
// 32 rows, key tiles of 128 and of 32 rows, each sorted by falling work so that the longest run first.
struct DofAttnTile {
  int64_t q0, k0;       // first query / key row of the document
  int32_t lq, lk;       // its rows
  int32_t prefix;       // causal: keys below this one are visible to every row
  int32_t row0;
};
constexpr int kAttnTall = 128, kAttnFlat = 32;

// keys visible to row i of a document: 0 .. kend - 1.  Row i stands at key position i + lk - lq.  Non-decreasing in i.
__device__ __forceinline__ int dof_attn_kend(const DofAttnTile& t, int causal, int i) {
  if (!causal) return t.lk;
  int e = i + (t.lk - t.lq) + 1;
  e = e > t.prefix ? e : t.prefix;
  e = e < t.lk ? e : t.lk;
  return e > 0 ? e : 0;
}

// Scores in units of log 2, from the raw product q.k:  x = scale log2(e) q.k, or with a cap  cap log2(e) tanh(scale q.k / cap);
// minus slope log2(e) |distance|.
struct DofScore {
  float mul;       // scale log2(e)                 cap: scale / cap
  float cap_l2;    // cap log2(e), 0 without a cap
  float slope_l2;  // slope log2(e) of the head
};
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// The running maximum of a softmax follows a new tile's only when that exceeds it by 2^kLag; weights are kept as 2^kUp times themselves
// (products and sum alike, so that the factor leaves with the division).  fp16 has 5 exponent bits: without a factor a weight
// below 2^-25 of the maximum is zero in the products while the sum counts it, and many such weights are a recording's tail.  With
// 2^11 what a weight loses is at most 2^-36 of the largest, and the largest, 2^(4 + 11), stays below 65504.
template <class T> struct DofSoftmax {
  static constexpr float kLag = 8.0f, kUp = 0.0f, kDown = 1.0f;
};
template <> struct DofSoftmax<DofF16> {
  static constexpr float kLag = 4.0f, kUp = 11.0f, kDown = 1.0f / 2048.0f;  // kDown: 2^-kUp, for the logarithm of a sum
};

// t[i] = tanh(t[i] mul) of N scores of a lane.  Below 0.6 of the cap, where capped scores mostly lie, an odd polynomial (fitted to
// tanh(x) / x on [0, 0.6], relative error 1.5e-8) takes 8 instructions, none of them transcendental; from there on
// 1 - 2 / (1 + 2^(2 log2(e) x)), whose quotient is below 0.47: off by 3 roundings of that and one of the result.  Which of them a
// score takes depends on it alone: what other rows and hidden keys hold only decides whether the wavefront computes the second at all.
__device__ __forceinline__ float dof_tanh_near(float x) {
  const float y = x * x;
  float c = fmaf(y, -0.006276387721300125f, 0.021116213873028755f);
  c = fmaf(y, c, -0.053875137120485306f);
  c = fmaf(y, c, 0.13332924246788025f);
  c = fmaf(y, c, -0.3333333134651184f);
  return fmaf(x * y, c, x);
}
template <int N> __device__ __forceinline__ void dof_cap_tanh(float* t, float mul) {
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    t[i] *= mul;
    top = fmaxf(top, fabsf(t[i]));
  }
  if (dof_wave_any(!(top < 0.6f))) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float x = dof_opaque(t[i]);  // the squares of both branches, computed before them, took 16 registers
      const float far = fmaf(-2.0f, dof_rcp(1.0f + dof_exp2(x * (2.0f * kLog2e))), 1.0f);
      t[i] = fabsf(x) < 0.6f ? dof_tanh_near(x) : far;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = dof_tanh_near(t[i]);
  }
}

// Blocks are dealt to the eight XCDs in turn, each with an L2 of its own.  Where the heads divide over the XCDs (or the XCDs over the
// heads), a head's tiles go to as few XCDs as that allows -- its keys and values, and those of its group's neighbours, then come from
// that L2 -- and in every case the tiles keep their order, longest first, on each XCD.
__device__ __forceinline__ void dof_attn_item(int block, int n_tiles, int heads, int* tile, int* head) {
  const int c = block & 7, n = block >> 3;
  if (heads % 8 == 0) {
    const int per = heads >> 3;
    *tile = n / per;
    *head = c * per + n - *tile * per;
  } else if (8 % heads == 0 && n_tiles % (8 / heads) == 0) {
    const int share = 8 / heads;
    *head = c / share;
    *tile = n * share + c % share;
  } else {
    *tile = block / heads;
    *head = block - *tile * heads;
  }
}
