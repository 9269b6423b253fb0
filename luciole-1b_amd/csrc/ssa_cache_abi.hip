// C ABI of the cache operators (include/ssa_cache_ops.h): host-side validation
// and dispatch.  Nothing is launched unless every check passes.
#include <stdint.h>

#include <algorithm>

#include "../../include/ssa_cache_ops.h"
#include "ssa_cache_ops.hpp"

namespace {

using ssa::Tensor4;

#define SSA_TRY(expr)              \
  do {                             \
    const int32_t st_ = (expr);    \
    if (st_ != SSA_OK) return st_; \
  } while (0)

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

int32_t check_tensor(const ssa_tensor4& t) {
  if (t.ptr == nullptr) return SSA_ERR_NULL_POINTER;
  if (!aligned16(t.ptr)) return SSA_ERR_ALIGNMENT;
  if ((t.stride_b % 8) != 0 || (t.stride_h % 8) != 0 || (t.stride_s % 8) != 0) return SSA_ERR_ALIGNMENT;
  if (t.stride_b < 0 || t.stride_h < 0 || t.stride_s < 0) return SSA_ERR_ALIGNMENT;
  // tile loads address rows with 32-bit byte offsets from a per-tile base
  if (t.stride_s >= (1ll << 24)) return SSA_ERR_ALIGNMENT;
  return SSA_OK;
}

// The dimensions of a [B, H, S, D] view that have more than one step, by ascending stride.
struct Steps {
  struct Dim {
    int64_t stride, size;
  } d[3];
  int n = 0;
  Steps(const ssa_tensor4& t, int32_t B, int32_t H, int32_t S) {
    for (const Dim& x : {Dim{t.stride_b, B}, Dim{t.stride_h, H}, Dim{t.stride_s, S}})
      if (x.size > 1) d[n++] = x;
    std::sort(d, d + n, [](const Dim& x, const Dim& y) { return x.stride < y.stride; });
  }
  // elements from the first to the last, both counted
  __int128 span(int32_t D) const {
    __int128 e = D;
    for (int i = 0; i < n; ++i) e += static_cast<__int128>(d[i].stride) * (d[i].size - 1);
    return e;
  }
  // every element at an address of its own: each stride steps over everything below it
  bool disjoint(int32_t D) const {
    __int128 extent = D;
    for (int i = 0; i < n; ++i) {
      if (d[i].stride < extent) return false;
      extent += static_cast<__int128>(d[i].stride) * (d[i].size - 1);
    }
    return true;
  }
  // Of a disjoint view and its copy `apart` elements on: some element at one address.
  // What the steps below the i-th add up to is less than its stride, so only the
  // two numbers of steps next to apart / stride come into question.
  bool meets(__int128 apart, int32_t D, int i) const {
    if (i < 0) return apart < D && apart > -D;
    const __int128 s = d[i].stride, low = apart / s - (apart % s < 0 ? 1 : 0);
    for (__int128 k = low; k <= low + 1; ++k)
      if (k < d[i].size && k > -d[i].size && meets(apart - k * s, D, i - 1)) return true;
    return false;
  }
};

// Keys and values that are both written: no address twice, in either or in both.
// Where one reaches between the other's rows (one buffer of both) they have one layout.
bool disjoint_caches(const ssa_tensor4& k, const ssa_tensor4& v, int32_t B, int32_t H, int32_t S, int32_t D) {
  const Steps ks(k, B, H, S), vs(v, B, H, S);
  if (!ks.disjoint(D) || !vs.disjoint(D)) return false;
  const __int128 ka = reinterpret_cast<uintptr_t>(k.ptr), va = reinterpret_cast<uintptr_t>(v.ptr);
  if (ka + 2 * ks.span(D) <= va || va + 2 * vs.span(D) <= ka) return true;
  if ((B > 1 && k.stride_b != v.stride_b) || (H > 1 && k.stride_h != v.stride_h) || (S > 1 && k.stride_s != v.stride_s))
    return false;
  return !ks.meets((va - ka) / 2, D, ks.n - 1);
}

int32_t check_types(int32_t D, int32_t dtype) {
  if (D != 32 && D != 64 && D != 128) return SSA_ERR_HEAD_DIM;
  if (dtype != SSA_DTYPE_BF16 && dtype != SSA_DTYPE_FP16) return SSA_ERR_DTYPE;
  return SSA_OK;
}

// Caches that every kernel here indexes with int32 rows and blocks: capacities
// up to 2^30, at most 2^24 kv-heads over all sequences and 2^28 (sequence,
// kv-head, 128 rows) units.
bool cache_ok(int32_t B, int32_t Hkv, int32_t cap) {
  if (B <= 0 || Hkv <= 0 || cap <= 0 || cap > (1 << 30)) return false;
  const int64_t bh = static_cast<int64_t>(B) * Hkv;
  return bh <= (1ll << 24) && bh * ((static_cast<int64_t>(cap) + 127) / 128) <= (1ll << 28);
}

// ... and query rows [B, Hq, T] counted with int32.
bool rows_ok(int32_t B, int32_t Hq, int32_t Hkv, int32_t T) {
  if (Hq <= 0 || Hkv <= 0 || T <= 0 || Hq % Hkv != 0) return false;
  const int64_t bh = static_cast<int64_t>(B) * Hq;
  return bh < (1ll << 30) && bh * T < (1ll << 30);
}

bool tree_ok(int32_t B, int32_t Hq, int32_t Hkv, int32_t cap, int32_t T, int32_t requested, ssa::TreePlan& plan) {
  if (!cache_ok(B, Hkv, cap) || !rows_ok(B, Hq, Hkv, T) || T > SSA_TREE_MAX_NODES || requested < 0) return false;
  // workgroups over all splits, and the merge's threads, stay below 2^30
  plan = ssa::tree_plan(B, Hq, Hkv, cap, T, requested);
  return plan.units * plan.splits < (1ll << 30);
}

bool weights_ok(int32_t B, int32_t Hq, int32_t Hkv, int32_t cap, int32_t T) {
  // a tile of 128 keys may end up to 127 behind the last query, and the first row
  // that would see its last key is counted with int32 too
  return cache_ok(B, Hkv, cap) && rows_ok(B, Hq, Hkv, T) && T <= cap &&
         static_cast<int64_t>(Hq / Hkv) * (static_cast<int64_t>(T) + 128) < (1ll << 31);
}

int64_t tree_ml_floats(int64_t recs) { return (2 * recs + 3) & ~static_cast<int64_t>(3); }

Tensor4 to_t4(const ssa_tensor4& t) { return Tensor4{t.ptr, t.stride_b, t.stride_h, t.stride_s}; }

int32_t launch_status(hipError_t e) { return e == hipSuccess ? SSA_OK : SSA_ERR_LAUNCH; }

}  // namespace

extern "C" {

int32_t ssa_tree_num_splits(int32_t batch, int32_t heads_q, int32_t heads_kv, int32_t capacity, int32_t nodes,
                            int32_t requested) {
  ssa::TreePlan plan;
  return tree_ok(batch, heads_q, heads_kv, capacity, nodes, requested, plan) ? plan.splits : 0;
}

int64_t ssa_tree_workspace_bytes(int32_t batch, int32_t heads_q, int32_t heads_kv, int32_t capacity,
                                 int32_t head_dim, int32_t nodes, int32_t requested) {
  ssa::TreePlan plan;
  if (!tree_ok(batch, heads_q, heads_kv, capacity, nodes, requested, plan)) return 0;
  if (head_dim != 32 && head_dim != 64 && head_dim != 128) return 0;
  if (plan.splits <= 1) return 0;
  const int64_t recs = static_cast<int64_t>(batch) * heads_q * nodes * plan.splits;
  return (tree_ml_floats(recs) + recs * head_dim) * 4;
}

int32_t ssa_tree_attention(const ssa_tree_args* a, void* stream) {
  if (a == nullptr) return SSA_ERR_NULL_POINTER;
  ssa::TreePlan plan;
  if (!tree_ok(a->batch, a->heads_q, a->heads_kv, a->capacity, a->nodes, a->num_splits, plan)) return SSA_ERR_SHAPE;
  SSA_TRY(check_types(a->head_dim, a->dtype));
  SSA_TRY(check_tensor(a->q));
  SSA_TRY(check_tensor(a->k_cache));
  SSA_TRY(check_tensor(a->v_cache));
  SSA_TRY(check_tensor(a->out));
  if (a->cache_seqlens == nullptr || a->tree_mask == nullptr || a->ssa_n == nullptr || a->ssa_b == nullptr)
    return SSA_ERR_NULL_POINTER;
  if (a->mask_stride_b < 0) return SSA_ERR_ALIGNMENT;
  ssa::TreeParams p{};
  p.splits = plan.splits;
  p.split_keys = plan.split_keys;
  p.rows = plan.rows;
  if (p.splits > 1) {
    if (a->workspace == nullptr) return SSA_ERR_NULL_POINTER;
    if (!aligned16(a->workspace)) return SSA_ERR_ALIGNMENT;
    const int64_t recs = static_cast<int64_t>(a->batch) * a->heads_q * a->nodes * p.splits;
    p.ws_ml = static_cast<float*>(a->workspace);
    p.ws_acc = p.ws_ml + tree_ml_floats(recs);
  }
  p.q = to_t4(a->q);
  p.k = to_t4(a->k_cache);
  p.v = to_t4(a->v_cache);
  p.o = to_t4(a->out);
  p.m = a->m;
  p.seqlens = a->cache_seqlens;
  p.mask = a->tree_mask;
  p.mask_sb = a->mask_stride_b;
  p.n_ptr = a->ssa_n;
  p.b_ptr = a->ssa_b;
  p.B = a->batch;
  p.Hq = a->heads_q;
  p.Hkv = a->heads_kv;
  p.cap = a->capacity;
  p.T = a->nodes;
  p.scale = a->softmax_scale;
  return launch_status(ssa::launch_tree(p, a->dtype, a->head_dim, static_cast<hipStream_t>(stream)));
}

int64_t ssa_key_weights_workspace_bytes(int32_t batch, int32_t heads_q, int32_t heads_kv, int32_t capacity,
                                        int32_t queries) {
  if (!weights_ok(batch, heads_q, heads_kv, capacity, queries)) return 0;
  const int64_t chunks = ssa::weights_chunks(batch, heads_q, heads_kv, capacity, queries);
  return chunks > 1 ? chunks * batch * heads_kv * capacity * 4 : 0;
}

int32_t ssa_key_weights(const ssa_key_weights_args* a, void* stream) {
  if (a == nullptr) return SSA_ERR_NULL_POINTER;
  if (!weights_ok(a->batch, a->heads_q, a->heads_kv, a->capacity, a->queries)) return SSA_ERR_SHAPE;
  SSA_TRY(check_types(a->head_dim, a->dtype));
  SSA_TRY(check_tensor(a->q));
  SSA_TRY(check_tensor(a->k_cache));
  if (a->m == nullptr || a->weights == nullptr || a->cache_seqlens == nullptr || a->ssa_n == nullptr ||
      a->ssa_b == nullptr)
    return SSA_ERR_NULL_POINTER;
  if (!aligned4(a->m) || !aligned4(a->weights)) return SSA_ERR_ALIGNMENT;
  // every weight is written: rows of capacity floats, none over another
  if (!Steps({nullptr, a->weights_stride_b, a->weights_stride_h, 0}, a->batch, a->heads_kv, 1).disjoint(a->capacity))
    return SSA_ERR_ALIGNMENT;
  ssa::KeyWeightsParams p{};
  p.chunks = ssa::weights_chunks(a->batch, a->heads_q, a->heads_kv, a->capacity, a->queries);
  p.chunk_rows = ssa::weights_chunk_rows(a->batch, a->heads_q, a->heads_kv, a->capacity, a->queries);
  if (p.chunks > 1) {
    if (a->workspace == nullptr) return SSA_ERR_NULL_POINTER;
    if (!aligned16(a->workspace)) return SSA_ERR_ALIGNMENT;
    p.ws = static_cast<float*>(a->workspace);
  }
  p.q = to_t4(a->q);
  p.k = to_t4(a->k_cache);
  p.m = a->m;
  p.w = a->weights;
  p.w_sb = a->weights_stride_b;
  p.w_sh = a->weights_stride_h;
  p.seqlens = a->cache_seqlens;
  p.n_ptr = a->ssa_n;
  p.b_ptr = a->ssa_b;
  p.B = a->batch;
  p.Hq = a->heads_q;
  p.Hkv = a->heads_kv;
  p.cap = a->capacity;
  p.T = a->queries;
  p.scale = a->softmax_scale;
  return launch_status(ssa::launch_key_weights(p, a->dtype, a->head_dim, static_cast<hipStream_t>(stream)));
}

int32_t ssa_cache_evict(const ssa_cache_evict_args* a, void* stream) {
  if (a == nullptr) return SSA_ERR_NULL_POINTER;
  if (!cache_ok(a->batch, a->heads_kv, a->capacity) || a->keep <= 0 || a->keep > a->capacity || a->sinks < 0 ||
      a->recent < 0 || static_cast<int64_t>(a->sinks) + a->recent > a->keep)
    return SSA_ERR_SHAPE;
  SSA_TRY(check_types(a->head_dim, a->dtype));
  SSA_TRY(check_tensor(a->k_cache));
  SSA_TRY(check_tensor(a->v_cache));
  if (a->weights == nullptr || a->cache_seqlens == nullptr || a->seqlens_out == nullptr || a->weights_out == nullptr ||
      a->kept == nullptr)
    return SSA_ERR_NULL_POINTER;
  if (!aligned4(a->weights) || !aligned4(a->weights_out) || !aligned4(a->kept)) return SSA_ERR_ALIGNMENT;
  if (a->weights_stride_b < 0 || a->weights_stride_h < 0 || a->seqlens_out == a->cache_seqlens ||
      a->weights_out == a->weights ||
      !disjoint_caches(a->k_cache, a->v_cache, a->batch, a->heads_kv, a->capacity, a->head_dim))
    return SSA_ERR_ALIGNMENT;
  ssa::EvictParams p{};
  p.k = to_t4(a->k_cache);
  p.v = to_t4(a->v_cache);
  p.w = a->weights;
  p.w_sb = a->weights_stride_b;
  p.w_sh = a->weights_stride_h;
  p.seqlens = a->cache_seqlens;
  p.lens_out = a->seqlens_out;
  p.w_out = a->weights_out;
  p.kept = a->kept;
  p.B = a->batch;
  p.Hkv = a->heads_kv;
  p.cap = a->capacity;
  p.D = a->head_dim;
  p.keep = a->keep;
  p.sinks = a->sinks;
  p.recent = a->recent;
  return launch_status(ssa::launch_evict(p, static_cast<hipStream_t>(stream)));
}

int32_t ssa_cache_accept(const ssa_cache_accept_args* a, void* stream) {
  if (a == nullptr) return SSA_ERR_NULL_POINTER;
  if (!cache_ok(a->batch, a->heads_kv, a->capacity) || a->nodes <= 0 || a->nodes > SSA_TREE_MAX_NODES ||
      a->depth <= 0 || a->depth > a->nodes)
    return SSA_ERR_SHAPE;
  SSA_TRY(check_types(a->head_dim, a->dtype));
  SSA_TRY(check_tensor(a->k_cache));
  SSA_TRY(check_tensor(a->v_cache));
  if (a->cache_seqlens == nullptr || a->path == nullptr || a->accepted == nullptr || a->seqlens_out == nullptr)
    return SSA_ERR_NULL_POINTER;
  if (a->seqlens_out == a->cache_seqlens ||
      !disjoint_caches(a->k_cache, a->v_cache, a->batch, a->heads_kv, a->capacity, a->head_dim))
    return SSA_ERR_ALIGNMENT;
  ssa::AcceptParams p{};
  p.k = to_t4(a->k_cache);
  p.v = to_t4(a->v_cache);
  p.seqlens = a->cache_seqlens;
  p.path = a->path;
  p.accepted = a->accepted;
  p.lens_out = a->seqlens_out;
  p.B = a->batch;
  p.Hkv = a->heads_kv;
  p.cap = a->capacity;
  p.D = a->head_dim;
  p.T = a->nodes;
  p.depth = a->depth;
  return launch_status(ssa::launch_accept(p, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
