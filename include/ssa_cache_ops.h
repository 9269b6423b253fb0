/*
 * Operators on a KV cache for generation with drafted tokens and a bounded
 * cache (gfx950), next to ssa_decode (ssa_mi355x.h), whose rules they follow:
 * the caller owns every buffer, a call checks its arguments on the host,
 * returns an SSA_* status before any launch when one is invalid, only enqueues
 * on `stream` (a hipStream_t, NULL = default stream), never allocates and never
 * synchronises.  Caches are [B, Hkv, capacity, D] in bf16 or fp16, D in
 * {32, 64, 128}, in the layout of ssa_decode; cache_seqlens is a device int32
 * array, clamped to [0, capacity] on the device.  Nothing here has a reference
 * counterpart: the reference's generation loop re-runs the whole prefix for
 * every token (training/train/train_ssa_triton/generate_triton.py:315-331).
 */
#ifndef SSA_CACHE_OPS_H
#define SSA_CACHE_OPS_H

#include <stdint.h>

#include "ssa_mi355x.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Most drafted tokens of one tree. */
#define SSA_TREE_MAX_NODES 1024

/*
 * Attention of a tree of drafted tokens over a cache.  The keys and values of
 * the `nodes` drafted tokens of sequence b are its last cached rows, node j at
 * row L_b - nodes + j (L_b = cache_seqlens[b]).  Node i attends every row
 * before L_b - nodes and node j's row where tree_mask[i][j] is not 0 (for a
 * tree: j = i or an ancestor of i).  A sequence shorter than `nodes` holds its
 * last L_b nodes only.  A node that sees no row gets out = 0, m = -inf.  What
 * the rows that a node does not see hold, NaN and infinities included, does
 * not reach its result.
 */
typedef struct ssa_tree_args {
  ssa_tensor4 q;        /* [B, Hq, nodes, D] */
  ssa_tensor4 k_cache;  /* [B, Hkv, capacity, D] */
  ssa_tensor4 v_cache;  /* [B, Hkv, capacity, D] */
  ssa_tensor4 out;      /* [B, Hq, nodes, D], written */
  float* m;             /* optional (NULL: not written) [B, Hq, nodes] contiguous fp32,
                           log2 of the sum of exp(t), as ssa_fwd's */
  const int32_t* cache_seqlens;
  const uint8_t* tree_mask; /* device, [nodes][nodes] bytes, one such matrix every
                               mask_stride_b bytes (0: one for all sequences) */
  int64_t mask_stride_b;
  const float* ssa_n;
  const float* ssa_b;
  int32_t batch, heads_q, heads_kv, capacity, head_dim;
  int32_t dtype;
  int32_t nodes;        /* 1 .. SSA_TREE_MAX_NODES */
  int32_t num_splits;   /* ranges that the keys are split into; 0 = library choice */
  float softmax_scale;
  void* workspace;      /* ssa_tree_workspace_bytes() bytes, 16-byte aligned; may be
                           NULL when that is 0 (one split) */
} ssa_tree_args;

/* Key splits of ssa_tree_attention for num_splits = `requested`; 0 on invalid arguments. */
int32_t ssa_tree_num_splits(int32_t batch, int32_t heads_q, int32_t heads_kv, int32_t capacity, int32_t nodes,
                            int32_t requested);
/* Workspace bytes: about (head_dim + 2) fp32 per (batch, q-head, node, split)
   with more than one split, else 0; 0 on invalid arguments. */
int64_t ssa_tree_workspace_bytes(int32_t batch, int32_t heads_q, int32_t heads_kv, int32_t capacity,
                                 int32_t head_dim, int32_t nodes, int32_t requested);
int32_t ssa_tree_attention(const ssa_tree_args* args, void* stream);

/*
 * The attention that `queries` query rows paid to every cached key, added to
 * the keys' weights: query t of sequence b stands at row L_b - queries + t and
 * sees the rows up to its own, and
 *   weights[b][hk][j] += sum over the q-heads of group hk and the queries t
 *                        that see row j of exp2(log2(e) t_tj - m_t),
 * m the normalisers that ssa_fwd, ssa_decode or ssa_tree_attention wrote.  A
 * query whose m is -inf adds nothing.  Weights at rows >= L_b are left as they
 * are.  No atomics: the sums have a fixed order.
 */
typedef struct ssa_key_weights_args {
  ssa_tensor4 q;        /* [B, Hq, queries, D] */
  ssa_tensor4 k_cache;  /* [B, Hkv, capacity, D] */
  const float* m;       /* [B, Hq, queries] contiguous fp32 */
  float* weights;       /* [B, Hkv, capacity] fp32, the last dimension contiguous, updated */
  int64_t weights_stride_b, weights_stride_h;
  const int32_t* cache_seqlens;
  const float* ssa_n;
  const float* ssa_b;
  int32_t batch, heads_q, heads_kv, capacity, head_dim;
  int32_t dtype;
  int32_t queries;      /* 1 .. capacity */
  float softmax_scale;
  void* workspace;      /* ssa_key_weights_workspace_bytes() bytes, 16-byte aligned; may
                           be NULL when that is 0 */
} ssa_key_weights_args;

/* Workspace bytes: a float per cached row and chunk of the queries where these
   are split over workgroups (many queries of few heads), else 0; 0 on invalid
   arguments. */
int64_t ssa_key_weights_workspace_bytes(int32_t batch, int32_t heads_q, int32_t heads_kv, int32_t capacity,
                                        int32_t queries);
int32_t ssa_key_weights(const ssa_key_weights_args* args, void* stream);

/*
 * Cuts every cache that holds more than `keep` rows to `keep` of them, in
 * place and in their order: the first `sinks` and the last `recent` rows
 * (sinks + recent <= keep) and, of the others, those of largest weight; of
 * equal weights the lower row stays, and NaN counts as the lowest weight.
 * Every (sequence, kv-head) keeps rows of its own.  Rows at and behind the new
 * length are left as they are.
 */
typedef struct ssa_cache_evict_args {
  ssa_tensor4 k_cache, v_cache; /* updated; no two elements at one address,
                                   in one of them or in both */
  const float* weights;         /* [B, Hkv, capacity] fp32, the last dimension contiguous */
  int64_t weights_stride_b, weights_stride_h;
  const int32_t* cache_seqlens;
  int32_t* seqlens_out;         /* [B], written: min(L_b, keep); not cache_seqlens itself */
  float* weights_out;           /* [B, Hkv, capacity] contiguous, written: the kept rows'
                                   weights, then zeros; not overlapping `weights` */
  int32_t* kept;                /* [B, Hkv, keep] contiguous, written: the rows that stayed,
                                   ascending, then -1 */
  int32_t batch, heads_kv, capacity, head_dim;
  int32_t dtype;
  int32_t keep, sinks, recent;
} ssa_cache_evict_args;

int32_t ssa_cache_evict(const ssa_cache_evict_args* args, void* stream);

/*
 * Accepts a path of a drafted tree: with first = L_b - nodes, row
 * first + path[b][i] moves to row first + i for i < accepted[b], and the new
 * length is first + accepted[b].  accepted is clamped to [0, depth] and every
 * path entry to [0, nodes) on the device; a path may name its nodes in any
 * order.  A sequence shorter than `nodes` is left as it is.  Rows at and
 * behind the new length that no accepted node moved to are left as they are.
 */
typedef struct ssa_cache_accept_args {
  ssa_tensor4 k_cache, v_cache; /* updated; no two elements at one address,
                                   in one of them or in both */
  const int32_t* cache_seqlens;
  const int32_t* path;          /* device, [B][depth] contiguous */
  const int32_t* accepted;      /* device, [B] */
  int32_t* seqlens_out;         /* [B], written; not cache_seqlens itself */
  int32_t batch, heads_kv, capacity, head_dim;
  int32_t dtype;
  int32_t nodes, depth;         /* 1 <= depth <= nodes <= SSA_TREE_MAX_NODES */
} ssa_cache_accept_args;

int32_t ssa_cache_accept(const ssa_cache_accept_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* SSA_CACHE_OPS_H */
