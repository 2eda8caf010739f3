// Host side of the attention operators: the plan of a packed batch and the C-ABI entry points of the forward and backward passes.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <exception>
#include <vector>

#include "deepof_hip.h"
#include "dof_rt.h"
#include "launchers.h"
#include "seq_attn_args.h"

namespace {

constexpr int64_t kMaxRows = 1 << 30;           // of one document

int check_plan_args(int32_t n_docs, const int64_t* q_off, const int64_t* k_off, const void* out) {
  if (n_docs < 0 || (n_docs > 0 && (!q_off || !k_off)) || !out) {
    dof_set_error("dof_attn_plan: bad argument (n_docs %d)", (int)n_docs);
    return DOF_ERR_ARG;
  }
  for (int32_t i = 0; i < n_docs; ++i) {
    const int64_t lq = q_off[i + 1] - q_off[i], lk = k_off[i + 1] - k_off[i];
    if (q_off[i] < 0 || k_off[i] < 0 || lq < 0 || lk < 0 || lq > kMaxRows || lk > kMaxRows) {
      dof_set_error("dof_attn_plan: the offsets of document %d do not rise (or it has more than 2^30 rows)", (int)i);
      return DOF_ERR_ARG;
    }
  }
  return DOF_OK;
}

// keys visible to row i, as dof_attn_kend
int64_t kend(int64_t lq, int64_t lk, int64_t prefix, int causal, int64_t i) {
  if (!causal) return lk;
  return std::max<int64_t>(0, std::min(lk, std::max(prefix, i + lk - lq + 1)));
}

// The tiles of one list, longest first (documents and rows in order among equals).
void list_tiles(const DofAttnPlan* p, const int64_t* q_off, const int64_t* k_off, const int32_t* prefix, bool keys, int rows, int64_t n,
                DofAttnTile* out) {
  std::vector<int64_t> work((size_t)n);
  bool falling = true;
  int64_t at = 0;
  for (int32_t d = 0; d < p->n_docs; ++d) {
    const int64_t lq = q_off[d + 1] - q_off[d], lk = k_off[d + 1] - k_off[d];
    const int64_t pre = prefix ? std::max(0, prefix[d]) : 0;
    for (int64_t r = 0; r < (keys ? lk : lq); r += rows, ++at) {
      out[at] = {q_off[d], k_off[d], (int32_t)lq, (int32_t)lk, (int32_t)std::min(pre, lk), (int32_t)r};
      if (keys) work[at] = !p->causal || r < pre ? lq : lq - std::min(lq, std::max<int64_t>(0, r - (lk - lq)));
      else work[at] = kend(lq, lk, pre, p->causal, std::min(r + rows, lq) - 1);
      falling = falling && (at == 0 || work[at] <= work[at - 1]);
    }
  }
  if (falling) return;
  std::vector<int64_t> order((size_t)n);
  for (int64_t i = 0; i < n; ++i) order[i] = i;
  std::stable_sort(order.begin(), order.end(), [&](int64_t a, int64_t b) { return work[a] > work[b]; });
  std::vector<DofAttnTile> sorted((size_t)n);
  for (int64_t i = 0; i < n; ++i) sorted[i] = out[order[i]];
  std::copy(sorted.begin(), sorted.end(), out);
}

int64_t count_tiles(int32_t n_docs, const int64_t* off, int rows) {
  int64_t n = 0;
  for (int32_t i = 0; i < n_docs; ++i) n += (off[i + 1] - off[i] + rows - 1) / rows;
  return n;
}

bool aligned(const void* p, const int64_t* s, int size) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s[0] * size % 16 == 0 && s[1] * size % 16 == 0;
}

int check(const DofAttnPlan* p, const void* table, const DofAttention* d, const char* who) {
  if (!p || !d || (!table && p->table_bytes > 0)) {
    dof_set_error("%s: null plan, table or descriptor", who);
    return DOF_ERR_ARG;
  }
  if (d->dtype < DOF_DTYPE_F32 || d->dtype > DOF_DTYPE_F16) {
    dof_set_error("%s: unknown dtype %d", who, (int)d->dtype);
    return DOF_ERR_ARG;
  }
  if (d->head_dim < 8 || d->head_dim > 128 || d->head_dim % 8) {
    dof_set_error("%s: head_dim %d (multiples of 8 from 8 to 128 are supported)", who, (int)d->head_dim);
    return DOF_ERR_UNSUPPORTED;
  }
  if (d->k_heads < 1 || d->q_heads < d->k_heads || d->q_heads % d->k_heads) {
    dof_set_error("%s: %d query heads are not a multiple of %d key heads", who, (int)d->q_heads, (int)d->k_heads);
    return DOF_ERR_ARG;
  }
  if (!std::isfinite(d->scale) || !std::isfinite(d->cap) || d->cap < 0.0f) {
    dof_set_error("%s: scale and cap must be finite, cap not negative", who);
    return DOF_ERR_ARG;
  }
  for (int i = 0; i < 4; ++i)
    if (p->n_tiles[i] < 0) {
      dof_set_error("%s: bad plan", who);
      return DOF_ERR_ARG;
    }
  return DOF_OK;
}

// a launch holds less than 2^32 threads: a wavefront per flat tile and head, four per tall one
int check_launch(int64_t tiles, int64_t heads, int flat, const char* who) {
  if (tiles > ((1LL << 32) - 1) / (flat ? 64 : 256) / heads) {
    dof_set_error("%s: too many tiles for one launch (%lld tiles, %lld heads)", who, (long long)tiles, (long long)heads);
    return DOF_ERR_UNSUPPORTED;
  }
  return DOF_OK;
}

// list 0: query tiles of 128 rows, 1: of 32; 2: key tiles of 128, 3: of 32
const DofAttnTile* list_at(const DofAttnPlan* p, const void* table, int list) {
  return static_cast<const DofAttnTile*>(table) + p->first[list];
}

// Tiles of 128 rows (four wavefronts share what is staged) unless the documents are so short that most of such a tile is empty
// (fewer than 2.5 flat tiles of 32 rows per tall one).  Few tiles are no reason for flat ones: a lone wavefront that
// stages for itself is slower than the CUs left empty cost (one recording of 5000 frames, 2 / 1 heads of 128, training: 0.83 ms tall,
// 2.16 flat; of 300 frames, 4 heads of 64: 49 and 53 us).
int flat_tiles(const DofAttnPlan* p, int which) { return p->n_tiles[which + 1] * 2 < p->n_tiles[which] * 5; }

// dk / dv: a workgroup per key tile and key head goes through all query heads of the group.  Where those are too few to fill the chip
// evenly (a causal tile's work ranges from nothing to all rows), the group's heads are shared out; the fp32 parts cost a write and a
// read of the key rows per share.
struct Shares { int flat, splits, heads_per; };
Shares shares_of(const DofAttnPlan* p, const DofAttention* d) {
  const int group = d->q_heads / d->k_heads;
  Shares s;
  s.flat = flat_tiles(p, 2);
  const int64_t items = p->n_tiles[2 + s.flat] * d->k_heads;
  int64_t want = items > 0 ? (2048 + items - 1) / items : 1;
  if (want > group) want = group;
  s.heads_per = (int)((group + want - 1) / want);
  s.splits = (group + s.heads_per - 1) / s.heads_per;
  return s;
}

// Small documents: one kernel for all three gradients (4096 windows of 25 frames, 4 heads of 16, fp32: 84 us, dq and dk / dv kernels 138).
// fp32 heads over 64 would not fit its registers, nor the blocks that fp32 sums over more rows and query heads than kLongTerms want.
bool one_pass(const DofAttnPlan* p, const DofAttention* d) {
  if (!p->small) return false;
  if (d->dtype != DOF_DTYPE_F32) return true;
  return d->head_dim <= 64 && (int64_t)p->longest * (d->q_heads / d->k_heads) <= kLongTerms;
}

int64_t delta_bytes(const DofAttnPlan* p, const DofAttention* d) { return (p->q_rows * d->q_heads * 4 + 15) / 16 * 16; }
int64_t workspace_bytes(const DofAttnPlan* p, const DofAttention* d) {  // 0: none (one kernel, or keys without any query row)
  if (one_pass(p, d)) return 0;
  const Shares s = shares_of(p, d);
  return delta_bytes(p, d) + (s.splits > 1 ? 2 * s.splits * p->k_rows * d->k_heads * d->head_dim * 4 : 0);
}

DofAttnFwd forward_args(const DofAttention* d, const void* q, const void* k, const void* v, const float* slopes, void* o, float* lse) {
  DofAttnFwd A;
  memset(&A, 0, sizeof(A));
  A.q_heads = d->q_heads;
  A.k_heads = d->k_heads;
  A.dim = d->head_dim;
  A.slopes = slopes;
  if (d->cap > 0.0f) {
    A.score.mul = d->scale / d->cap;
    A.score.cap_l2 = d->cap * kLog2e;
  } else {
    A.score.mul = d->scale * kLog2e;
  }
  A.q = q;
  A.k = k;
  A.v = v;
  A.o = o;
  A.lse = lse;
  for (int i = 0; i < 2; ++i) {
    A.qs[i] = d->q_stride[i];
    A.ks[i] = d->k_stride[i];
    A.vs[i] = d->v_stride[i];
    A.os[i] = d->o_stride[i];
  }
  return A;
}

int set_tiles(DofAttnFwd* A, const DofAttnPlan* p, const void* table, int which, int flat) {
  A->causal = p->causal;
  A->longest = p->longest;
  A->n_tiles = (int32_t)p->n_tiles[which + flat];
  A->tiles = list_at(p, table, which + flat);
  return A->n_tiles;
}

}  // namespace

extern "C" int dof_attn_plan_size(int32_t n_docs, const int64_t* q_off, const int64_t* k_off, int32_t causal, DofAttnPlan* plan) {
  const int rc = check_plan_args(n_docs, q_off, k_off, plan);
  if (rc != DOF_OK) return rc;
  plan->n_docs = n_docs;
  plan->causal = causal != 0;
  plan->small = 1;
  plan->longest = 0;
  for (int32_t i = 0; i < n_docs; ++i) {
    const int64_t lq = q_off[i + 1] - q_off[i], lk = k_off[i + 1] - k_off[i];
    plan->longest = (int32_t)std::max<int64_t>(plan->longest, std::max(lq, lk));
    if (lq > kAttnFlat || lk > kAttnFlat || (lq > 0 && lk == 0)) plan->small = 0;
  }
  plan->q_rows = n_docs ? q_off[n_docs] : 0;
  plan->k_rows = n_docs ? k_off[n_docs] : 0;
  plan->n_tiles[0] = count_tiles(n_docs, q_off, kAttnTall);
  plan->n_tiles[1] = count_tiles(n_docs, q_off, kAttnFlat);
  plan->n_tiles[2] = count_tiles(n_docs, k_off, kAttnTall);
  plan->n_tiles[3] = count_tiles(n_docs, k_off, kAttnFlat);
  // Equal lists are kept once: documents of one tile each (tall and flat), and queries and keys of the same rows whose work is the same
  bool self = true;
  int64_t with_rows = 0;
  for (int32_t i = 0; i < n_docs; ++i) {
    self = self && q_off[i + 1] - q_off[i] == k_off[i + 1] - k_off[i];
    with_rows += q_off[i + 1] > q_off[i];
  }
  int64_t entries = 0;
  for (int i = 0; i < 4; ++i) {
    int same = -1;
    if (i % 2 == 1 && plan->n_tiles[i] == plan->n_tiles[i - 1]) same = i - 1;
    else if (i >= 2 && self && (!causal || plan->n_tiles[i] == with_rows)) same = i - 2;
    plan->first[i] = same >= 0 ? plan->first[same] : entries;
    if (same < 0) entries += plan->n_tiles[i];
  }
  plan->table_bytes = entries * (int64_t)sizeof(DofAttnTile);
  return DOF_OK;
}

extern "C" int dof_attn_plan_table(const DofAttnPlan* plan, const int64_t* q_off, const int64_t* k_off, const int32_t* prefix,
                                   void* table) {
  if (!plan) {
    dof_set_error("dof_attn_plan_table: null plan");
    return DOF_ERR_ARG;
  }
  DofAttnPlan again;
  const int rc = dof_attn_plan_size(plan->n_docs, q_off, k_off, plan->causal, &again);
  if (rc != DOF_OK) return rc;
  if (memcmp(again.n_tiles, plan->n_tiles, sizeof(again.n_tiles)) || memcmp(again.first, plan->first, sizeof(again.first)) || again.table_bytes != plan->table_bytes) {
    dof_set_error("dof_attn_plan_table: the offsets are not those the plan was sized for");
    return DOF_ERR_ARG;
  }
  if (plan->table_bytes == 0) return DOF_OK;
  if (!table) {
    dof_set_error("dof_attn_plan_table: null table");
    return DOF_ERR_ARG;
  }
  try {
    int64_t done = 0;
    for (int i = 0; i < 4; ++i) {
      if (plan->first[i] < done || plan->n_tiles[i] == 0) continue;  // kept as an earlier list
      list_tiles(plan, q_off, k_off, prefix, i >= 2, i % 2 ? kAttnFlat : kAttnTall, plan->n_tiles[i],
                 static_cast<DofAttnTile*>(table) + plan->first[i]);
      done = plan->first[i] + plan->n_tiles[i];
    }
  } catch (const std::exception& e) {
    dof_set_error("dof_attn_plan_table: %s", e.what());
    return DOF_ERR_STATE;
  }
  return DOF_OK;
}

extern "C" int dof_attention_forward(const DofAttnPlan* plan, const void* table, const DofAttention* d, const void* q, const void* k,
                                     const void* v, const float* slopes, void* o, float* lse, void* stream) {
  int rc = check(plan, table, d, "dof_attention_forward");
  if (rc != DOF_OK) return rc;
  if (plan->n_tiles[0] == 0) return DOF_OK;
  const bool keys = plan->n_tiles[2] > 0;  // documents without any key need no k and v
  if (!q || !o || !lse || (keys && (!k || !v))) {
    dof_set_error("dof_attention_forward: null tensor");
    return DOF_ERR_ARG;
  }
  const int size = d->dtype == DOF_DTYPE_F32 ? 4 : 2;
  if (!aligned(q, d->q_stride, size) || !aligned(k, d->k_stride, size) || !aligned(v, d->v_stride, size) || !aligned(o, d->o_stride, size)) {
    dof_set_error("dof_attention_forward: tensors and strides must be multiples of 16 bytes");
    return DOF_ERR_UNSUPPORTED;
  }
  DofAttnFwd A = forward_args(d, q, k, v, slopes, o, lse);
  const int flat = flat_tiles(plan, 0);
  rc = check_launch(plan->n_tiles[flat], d->q_heads, flat, "dof_attention_forward");
  if (rc != DOF_OK) return rc;
  set_tiles(&A, plan, table, 0, flat);
  return dof_launch_attn_fwd(A, d->dtype, flat, (hipStream_t)stream);
}

extern "C" int64_t dof_attention_workspace_bytes(const DofAttnPlan* plan, const DofAttention* d) {
  static const char none = 0;
  if (check(plan, &none, d, "dof_attention_workspace_bytes") != DOF_OK) return -1;
  return workspace_bytes(plan, d);
}

extern "C" int dof_attention_backward(const DofAttnPlan* plan, const void* table, const DofAttention* d, const void* g, const void* q,
                                      const void* k, const void* v, const float* slopes, const void* o, const float* lse, void* dq,
                                      void* dk, void* dv, void* workspace, void* stream) {
  int rc = check(plan, table, d, "dof_attention_backward");
  if (rc != DOF_OK) return rc;
  const bool rows = plan->n_tiles[0] > 0, keys = plan->n_tiles[2] > 0;
  if (!rows && !keys) return DOF_OK;
  const bool one = one_pass(plan, d);
  if ((!workspace && workspace_bytes(plan, d) > 0) || (rows && (!g || !q || !o || !lse || !dq)) || (keys && (!k || !v || !dk || !dv))) {
    dof_set_error("dof_attention_backward: null tensor");
    return DOF_ERR_ARG;
  }
  const int size = d->dtype == DOF_DTYPE_F32 ? 4 : 2;
  if (!aligned(q, d->q_stride, size) || !aligned(k, d->k_stride, size) || !aligned(v, d->v_stride, size) || !aligned(o, d->o_stride, size) ||
      !aligned(g, d->g_stride, size) || !aligned(dq, d->dq_stride, size) || !aligned(dk, d->dk_stride, size) ||
      !aligned(dv, d->dv_stride, size)) {
    dof_set_error("dof_attention_backward: tensors and strides must be multiples of 16 bytes");
    return DOF_ERR_UNSUPPORTED;
  }
  DofAttnBwd B;
  memset(&B, 0, sizeof(B));
  B.f = forward_args(d, q, k, v, slopes, const_cast<void*>(o), const_cast<float*>(lse));
  B.g = g;
  B.delta = static_cast<float*>(workspace);
  B.scale = d->scale;
  B.dq = dq;
  B.dk = dk;
  B.dv = dv;
  for (int i = 0; i < 2; ++i) {
    B.gs[i] = d->g_stride[i];
    B.dqs[i] = d->dq_stride[i];
    B.dks[i] = d->dk_stride[i];
    B.dvs[i] = d->dv_stride[i];
  }
  static const char who[] = "dof_attention_backward";
  if (one) {
    rc = check_launch(plan->n_tiles[3], d->k_heads, 1, who);
    if (rc != DOF_OK) return rc;
    set_tiles(&B.f, plan, table, 2, 1);
    return dof_launch_attn_bwd_one(B, d->dtype, (hipStream_t)stream);
  }
  const int flat = flat_tiles(plan, 0);
  const Shares s = shares_of(plan, d);
  rc = check_launch(plan->n_tiles[flat], d->q_heads, flat, who);
  if (rc == DOF_OK) rc = check_launch(plan->n_tiles[2 + s.flat], (int64_t)d->k_heads * s.splits, s.flat, who);
  if (rc != DOF_OK) return rc;
  if (rows) {
    set_tiles(&B.f, plan, table, 0, flat);
    rc = dof_launch_attn_dq(B, d->dtype, flat, (hipStream_t)stream);
    if (rc != DOF_OK) return rc;
  }
  if (keys) {
    B.splits = s.splits;
    B.heads_per = s.heads_per;
    B.k_rows = plan->k_rows;
    B.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + delta_bytes(plan, d));
    set_tiles(&B.f, plan, table, 2, s.flat);
    rc = dof_launch_attn_dkv(B, d->dtype, s.flat, (hipStream_t)stream);
  }
  return rc;
}
