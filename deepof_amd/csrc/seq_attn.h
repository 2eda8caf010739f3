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

// tanh(raw mul) for the cap: fp32 inputs take the library's; 16-bit ones 1 - 2 / (1 + 2^(2 log2(e) mul raw)), whose absolute error of 2^-22
// is far below half a step of the inputs the score is made of
template <class T> __device__ __forceinline__ float dof_cap_tanh(float raw, float mul) {
  if constexpr (sizeof(T) == 4) return tanhf(raw * mul);
  else return fmaf(-2.0f, dof_rcp(1.0f + dof_exp2(raw * (mul * (2.0f * kLog2e)))), 1.0f);
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
