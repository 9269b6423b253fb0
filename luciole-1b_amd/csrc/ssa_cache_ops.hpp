// Parameters and launchers of the cache operators (include/ssa_cache_ops.h).
#pragma once

#include <hip/hip_runtime.h>

#include "ssa_common.hpp"

namespace ssa {

// A q-head group's rows: row r = node * G + g (g the head within the group),
// so that 32 consecutive rows share their nodes' masks.
struct TreeParams {
  Tensor4 q, k, v, o;
  float* m;  // optional [B, Hq, T]
  const int* seqlens;
  const uint8_t* mask;  // [T][T] bytes, mask_sb bytes from one sequence's to the next
  int64_t mask_sb;
  const float* n_ptr;
  const float* b_ptr;
  float* ws_ml;   // [B * Hq * T * splits][2]
  float* ws_acc;  // [B * Hq * T * splits][D]
  int B, Hq, Hkv, cap, T;
  int splits, split_keys;  // split s: keys s * split_keys ..
  float scale;
};

struct KeyWeightsParams {
  Tensor4 q, k;
  const float* m;
  float* w;
  int64_t w_sb, w_sh;
  const int* seqlens;
  const float* n_ptr;
  const float* b_ptr;
  float* ws;  // chunks > 1: [chunks][B * Hkv][cap]
  int B, Hq, Hkv, cap, T;
  int chunks, chunk_rows;  // the rows (queries of all heads of a group) of one chunk
  float scale;
};

struct EvictParams {
  Tensor4 k, v;
  const float* w;
  int64_t w_sb, w_sh;
  const int* seqlens;
  int* lens_out;
  float* w_out;
  int* kept;
  int B, Hkv, cap, D, keep, sinks, recent;
};

struct AcceptParams {
  Tensor4 k, v;
  const int* seqlens;
  const int* path;
  const int* accepted;
  int* lens_out;
  int B, Hkv, cap, D, T, depth;
};

// q rows that one workgroup of the tree kernels covers.
inline int tree_rows_per_block(int64_t rows) { return rows <= 32 ? 32 : rows <= 64 ? 64 : rows <= 128 ? 128 : 256; }

// Workgroups of a tree launch per split, or -1 beyond 2^30.
inline int64_t tree_units(int B, int Hq, int Hkv, int T) {
  const int64_t rows = static_cast<int64_t>(Hq / Hkv) * T;
  const int per = tree_rows_per_block(rows);
  return static_cast<int64_t>(B) * Hkv * ((rows + per - 1) / per);
}

// Keys of a split (a multiple of 256, the steps of every kernel) for a wanted
// number of splits.  The default takes the number that makes
//   rounds of one workgroup a CU * (keys of a split + what one costs beside them)
// least: a workgroup's start, end and share of the merge take as long as about
// 400 keys (measured: 8 to 12 us, 16 to 32 ns a key).
constexpr int kTreeStep = 256, kTreeOverhead = 400, kCUs = 256;
inline int tree_split_keys(int B, int Hq, int Hkv, int cap, int T, int requested) {
  const auto keys_of = [cap](int64_t splits) {
    const int64_t keys = (cap + splits - 1) / splits;
    return (keys + kTreeStep - 1) / kTreeStep * kTreeStep;
  };
  if (requested > 0) return static_cast<int>(keys_of(requested));
  const int64_t units = tree_units(B, Hq, Hkv, T);
  int64_t most = 2 * kCUs / units;
  if (most < 4) most = 4;
  if (most > (cap + kTreeStep - 1) / kTreeStep) most = (cap + kTreeStep - 1) / kTreeStep;
  int64_t best = keys_of(1), least = (units + kCUs - 1) / kCUs * (best + kTreeOverhead);
  for (int64_t s = 2; s <= most; ++s) {
    const int64_t keys = keys_of(s), n = (cap + keys - 1) / keys;
    const int64_t cost = (units * n + kCUs - 1) / kCUs * (keys + kTreeOverhead);
    if (cost < least) {
      least = cost;
      best = keys;
    }
  }
  return static_cast<int>(best);
}
inline int tree_splits(int B, int Hq, int Hkv, int cap, int T, int requested) {
  const int keys = tree_split_keys(B, Hq, Hkv, cap, T, requested);
  return static_cast<int>((static_cast<int64_t>(cap) + keys - 1) / keys);
}

// Key weights of more than 32 rows: rows of a stage and keys of a workgroup.
constexpr int kWeightsStage = 128;
constexpr int kWeightsKeys = 128;
// Rows of a chunk (whole stages): about 2048 workgroups in all, so that those of
// many rows and of few even out, of 1024 rows at least.
inline int weights_chunk_rows(int B, int Hq, int Hkv, int cap, int T) {
  const int64_t rows = static_cast<int64_t>(Hq / Hkv) * T;
  const int64_t blocks = static_cast<int64_t>(B) * Hkv * ((cap + kWeightsKeys - 1) / kWeightsKeys);
  const int64_t want = 2048 / blocks, most = rows / 1024;
  int64_t n = want < most ? want : most;
  if (n < 1 || rows <= 32) n = 1;
  const int64_t per = (rows + n - 1) / n;
  return static_cast<int>((per + kWeightsStage - 1) / kWeightsStage * kWeightsStage);
}
// ... and the chunks that hold rows: every one is written, every one is read.
inline int weights_chunks(int B, int Hq, int Hkv, int cap, int T) {
  const int64_t rows = static_cast<int64_t>(Hq / Hkv) * T, per = weights_chunk_rows(B, Hq, Hkv, cap, T);
  return static_cast<int>((rows + per - 1) / per);
}

hipError_t launch_tree(const TreeParams& p, int dtype, int D, hipStream_t stream);
hipError_t launch_key_weights(const KeyWeightsParams& p, int dtype, int D, hipStream_t stream);
hipError_t launch_evict(const EvictParams& p, hipStream_t stream);
hipError_t launch_accept(const AcceptParams& p, hipStream_t stream);

}  // namespace ssa
