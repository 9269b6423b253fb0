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
  int B, Hq, Hkv, cap, T, splits;
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
  int B, Hq, Hkv, cap, T;
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

inline int tree_splits(int B, int Hq, int Hkv, int cap, int T, int requested) {
  const int64_t most = (cap + 127ll) / 128;
  int64_t want = requested;
  if (want <= 0) {
    const int64_t units = tree_units(B, Hq, Hkv, T);
    want = (256 + units - 1) / units;
    const int64_t longest = (cap + 255ll) / 256;
    if (want > longest) want = longest;
  }
  if (want > most) want = most;
  return static_cast<int>(want < 1 ? 1 : want);
}

hipError_t launch_tree(const TreeParams& p, int dtype, int D, hipStream_t stream);
hipError_t launch_key_weights(const KeyWeightsParams& p, int dtype, int D, hipStream_t stream);
hipError_t launch_evict(const EvictParams& p, hipStream_t stream);
hipError_t launch_accept(const AcceptParams& p, hipStream_t stream);

}  // namespace ssa
