// Arguments of the attention kernels' launchers (k_attn_fwd.hip, k_attn_bwd.hip), filled by attention.hip.
#pragma once
#include "seq_attn.h"

struct DofAttnFwd {
  const DofAttnTile* tiles;
  int32_t n_tiles, q_heads, k_heads, dim, causal;
  int32_t longest;      // most rows or keys of a document
  DofScore score;
  const float* slopes;  // per query head, NULL: no bias
  const void *q, *k, *v;
  void* o;
  float* lse;           // (query rows, q_heads)
  int64_t qs[2], ks[2], vs[2], os[2];  // row and head strides
};

struct DofAttnBwd {
  DofAttnFwd f;          // f.tiles: query tiles (dq kernel) or key tiles (dk / dv kernel); f.o and f.lse are read
  const void* g;         // gradient at o
  float* delta;          // (query rows, q_heads): sum of g o over a row, written by the dq kernel, read by the dk / dv kernel
  float scale;           // d(score) / d(q.k) without the cap
  void *dq, *dk, *dv;
  int64_t gs[2], dqs[2], dks[2], dvs[2];
  // dk / dv: a group's query heads in `splits` workgroups of `heads_per` each; more than one leave fp32 parts
  // [dk, dv][split][key row][key head][dim] in `part`
  int32_t splits, heads_per;
  int64_t k_rows;
  float* part;
};

// The kernels' score function: 0 plain (scale > 0; its multiplication is part of the exponent's), 1 with a distance bias (or another
// scale), 2 capped, with or without a bias.
static inline int dof_attn_kind(const DofAttnFwd& A) {
  if (A.score.cap_l2 != 0.0f) return 2;
  return A.slopes || !(A.score.mul > 0.0f) ? 1 : 0;
}
// DOF_ATTN_KIND(A, KIND, expr): expr with KIND = that number
#define DOF_ATTN_KIND(A, KIND, ...)                                       \
  do {                                                                    \
    const int _kind = dof_attn_kind(A);                                   \
    if (_kind == 0) { constexpr int KIND = 0; __VA_ARGS__; }              \
    else if (_kind == 1) { constexpr int KIND = 1; __VA_ARGS__; }         \
    else { constexpr int KIND = 2; __VA_ARGS__; }                         \
  } while (0)

// DOF_ATTN_LONG(T, terms, LONG, expr): expr with LONG = whether sums of so many terms are made of blocks (fp32 elements)
#define DOF_ATTN_LONG(T, terms, LONG, ...)                                                     \
  do {                                                                                         \
    if constexpr (sizeof(T) == 4) {                                                            \
      if ((terms) > kLongTerms) { constexpr bool LONG = true; __VA_ARGS__; break; }            \
    }                                                                                          \
    { constexpr bool LONG = false; __VA_ARGS__; }                                              \
  } while (0)

int dof_launch_attn_fwd(const DofAttnFwd& A, int dtype, int flat, hipStream_t stream);
int dof_launch_attn_dq(const DofAttnBwd& A, int dtype, int flat, hipStream_t stream);
int dof_launch_attn_dkv(const DofAttnBwd& A, int dtype, int flat, hipStream_t stream);
int dof_launch_attn_bwd_one(const DofAttnBwd& B, int dtype, hipStream_t stream);  // heads of at most 64 (fp32) or 128
