// Parameters and launchers of the cache operators (include/ssa_cache_ops.h).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

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
  int rows;                // rows of a workgroup (TreePlan)
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

// How a tree launch is cut: rows of a group per workgroup, row blocks x kv-heads x
// sequences, keys of a split (a multiple of 256, the steps of every kernel).
struct TreePlan {
  int rows;
  int64_t units;
  int split_keys, splits;
};

// The plan of least estimated time, ns:
//   rounds of one workgroup a CU * (start and end + keys of a split * time of one)
//   + the merge's launch, if any, and its splits + the masked keys of the last split
// The constants were fitted to 2300 measured calls on caches read from HBM: 28
// shapes (1 to 64 sequences, 8 to 8192 rows of a group, 1000 to 65536 keys) at all
// head dims, in every form and with 1 to 64 splits.  The plans chosen take 2 %
// longer than each shape's best, 12 % at most; workgroups of as many rows as there are
// take 10 and 136 %.  So few keys or workgroups go to 32 rows (2 x 24/8 heads x
// 1000 x 32, 61 nodes: 9.9 us a call, 17.6 with 256 rows), most others to 64 (1 x 8 x
// 16384 x 64, 1024 nodes: 106, 32 rows 116, 128 rows 138, 256 rows 207, whose last
// split holds all masked keys), long caches of many rows to 256 (1 x 32/8 x 65536 x
// 64, 64 nodes: 73.8, 128 rows 77.5; head dim 128: 120, 128 rows 128, 64 rows 141).
// A split's share of the merge counts where one head has a long cache (1 x 16/1 x
// 65536 x 64, 2 nodes: 128 splits 16.9 us, 256 19.7, 64 18.5).
constexpr int kTreeStep = 256, kCUs = 256;
inline TreePlan tree_plan(int B, int Hq, int Hkv, int cap, int T, int requested) {
  struct Form {
    int rows;
    int64_t start, key;  // ns; tenths of ns
  };
  constexpr Form kForms[] = {{32, 7000, 80}, {64, 9000, 110}, {128, 12000, 195}, {256, 12000, 350}};
  constexpr int64_t kMerge = 4500, kMergeSplit = 20;
  const int64_t rows = static_cast<int64_t>(Hq / Hkv) * T;
  const int64_t steps = (static_cast<int64_t>(cap) + kTreeStep - 1) / kTreeStep;
  TreePlan best{};
  int64_t least = INT64_MAX;
  for (const Form& f : kForms) {
    const int64_t units = static_cast<int64_t>(B) * Hkv * ((rows + f.rows - 1) / f.rows);
    int64_t most = 2 * kCUs / units;
    if (most < 4) most = 4;
    if (requested > 0) most = requested;
    if (most > steps) most = steps;
    int64_t per;  // steps of a split
    // numbers of splits of one length of their own: the next is the least that shortens them
    for (int64_t s = requested > 0 ? most : 1; s <= most; s = per > 1 ? (steps + per - 2) / (per - 1) : most + 1) {
      per = (steps + s - 1) / s;
      const int64_t keys = per * kTreeStep, n = (cap + keys - 1) / keys;
      const int64_t masked = T < keys ? T : keys;
      const int64_t cost = (units * n + kCUs - 1) / kCUs * (f.start + keys * f.key / 10) +
                           (n > 1 ? kMerge + kMergeSplit * n : 0) + 3 * masked * f.rows / 10;
      if (cost < least) {
        least = cost;
        best = TreePlan{f.rows, units, static_cast<int>(keys), static_cast<int>(n)};
      }
    }
  }
  return best;
}

// Key weights: keys of a workgroup, and rows of a stage (whole stages make a chunk).
constexpr int kWeightsStage = 64;
constexpr int kWeightsKeys = 128;
inline int64_t weights_blocks(int B, int Hkv, int cap) {
  return static_cast<int64_t>(B) * Hkv * ((static_cast<int64_t>(cap) + kWeightsKeys - 1) / kWeightsKeys);
}
// One wave of rows (32 a stage) or two (64).  One, whose workgroups are small and many to
// a CU, up to 64 rows (4 x 16 x 8192 x 128, 48 rows: 31.6 us, two 47.6) and, where
// there are 8 workgroups a CU, up to 512 (192 rows 55 and 72, head dim 64 40 and
// 44); two beyond (768 rows at head dim 64: 117, one 121) and where few
// workgroups are to hide a row's latency (1 x 32/8 x 4096 x 64, 192 rows: 6.5, one
// 8.4; 768 rows 15.4 and 25.2).
inline bool weights_one_wave(int64_t rows, int64_t blocks) { return rows <= 64 || (rows <= 512 && blocks >= 8 * 256); }
// Rows of a chunk (whole stages): about 2048 workgroups in all, so that those of
// many rows and of few even out (1 x 32/8 x 4096 x 64, 4096 queries: 155 us in
// one chunk, 107 in 8), of 512 rows at least (1 x 8 x 2048 x 64, 1200 rows: 21.9 in
// one, 16.0 in two, the join's launch included; 256 rows a chunk cost 1 x 32/8 x
// 4096 x 128, 1536 rows, 37.8 for 33.2).
inline int weights_chunk_rows(int B, int Hq, int Hkv, int cap, int T) {
  const int64_t rows = static_cast<int64_t>(Hq / Hkv) * T;
  const int64_t want = 2048 / weights_blocks(B, Hkv, cap), most = rows / 512;
  int64_t n = want < most ? want : most;
  if (n < 1) n = 1;
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
