// Global-memory plans of the cache operators' kernels that stream tiles
// (ssa_tree.hip, ssa_key_weights.hip): for one workgroup, wave and lane, what it
// works on, which rows every direct-to-LDS load fetches, which partial results it
// writes and which of them the joining kernel reads.  __host__ __device__, as
// ssa_plan.hpp: tests/host_addr/cache_replay.cpp runs the same code for every workgroup,
// wave and lane of a problem on host memory.
#pragma once

#include "ssa_cache_ops.hpp"
#include "ssa_row_tile.hpp"

namespace ssa {

__host__ __device__ __forceinline__ int clamped_length(int held, int cap) {
  return held < 0 ? 0 : (held > cap ? cap : held);
}

// ----------------------------------------------------------------------------
// Tree attention
constexpr int kMaxNodes = 1024;
constexpr int kMaskWords = kMaxNodes / 32 + 1;  // words of a packed mask row, one of padding

// What a workgroup works on.
struct TreeUnit {
  int b, hk, row0, nrows, split;  // rows row0 .. row0 + nrows - 1 of the group's R
  int G, base, kbeg, kend, ntile;
  const char* kg;
  const char* vg;
  float n, c;  // t = n sign(s) log2(1 + c |s|)
  __host__ __device__ __forceinline__ TreeUnit(const TreeParams& p, int block, int per, int nqb) {
    int u = block;
    // the splits' first ranges of all sequences, then the second ones ...: the
    // short last ranges come late
    const int nbh = p.B * p.Hkv, whole = nbh * nqb;
    split = u / whole;
    u -= split * whole;
    const int qb = u / nbh;
    u -= qb * nbh;
    b = u / p.Hkv;
    hk = u - b * p.Hkv;
    // the three scalars a workgroup waits for, on their way together
    const int held = load_table_entry(p.seqlens, b);
    n = __builtin_bit_cast(float, load_table_entry(reinterpret_cast<const int*>(p.n_ptr), 0));
    c = p.scale * __builtin_bit_cast(float, load_table_entry(reinterpret_cast<const int*>(p.b_ptr), 0));
    G = p.Hq / p.Hkv;
    row0 = qb * per;
    nrows = per < G * p.T - row0 ? per : G * p.T - row0;
    const int L = clamped_length(held, p.cap);
    base = L - p.T;
    const int64_t beg = static_cast<int64_t>(split) * p.split_keys;
    kbeg = beg < L ? static_cast<int>(beg) : L;
    kend = beg + p.split_keys < L ? static_cast<int>(beg + p.split_keys) : L;
    ntile = (kend - kbeg + 31) / 32;
    kg = static_cast<const char*>(p.k.ptr) + (b * p.k.sb + hk * p.k.sh) * 2;
    vg = static_cast<const char*>(p.v.ptr) + (b * p.v.sb + hk * p.v.sh) * 2;
  }
  // a tile's keys that some rows may not see: the tree's
  __host__ __device__ __forceinline__ bool masked(int key0) const { return key0 + 32 > base; }
};

__host__ __device__ __forceinline__ int mask_stride(int T) { return 2 * ((T + 63) / 64) + 1; }

// Splits that hold keys of sequence b.
__host__ __device__ __forceinline__ int tree_own_splits(const TreeParams& p, int b) {
  const int64_t L = clamped_length(load_table_entry(p.seqlens, b), p.cap);
  return static_cast<int>((L + p.split_keys - 1) / p.split_keys);
}

// Two stages of 32 KW U keys, a K tile and a V tile each; wave (qw, kw) takes
// the stage's key tiles kw, kw + KW, ...
template <int D, int QW, int KW>
struct TreeCfg {
  static constexpr int NW = QW * KW;
  // tiles of a wave and stage: two where a stage's K and V then take 40 KB at
  // most (a longer first stage costs a short range of keys more than its barriers)
  static constexpr int U = 2 * KW * 2 * RowTile<D>::BLOCK <= 40 * 1024 ? 2 : 1;
  static constexpr int BLOCKS = KW * U;
  static constexpr int KEYS = 32 * BLOCKS;
  static constexpr int TILE = BLOCKS * RowTile<D>::BLOCK;
  // the key waves' exchange: each hands the others their shares of its acc
  static constexpr int J = D / 8;                    // float4 of a lane's acc
  static constexpr int JB = J > KW ? J / KW : 1;     // of a wave's share
  static constexpr int MERGE = KW == 1 ? 0 : QW * J * (KW - 1) * 1024;
  static constexpr int SMEM = 4 * TILE > MERGE ? 4 * TILE : MERGE;
  static constexpr int WORDS = 32 * QW * kMaskWords > 128 * NW ? 32 * QW * kMaskWords : 128 * NW;
};

// Stage i of the workgroup's keys to its buffer i & 1, K tiles and then V tiles.
template <int D, int QW, int KW, typename Mem = DeviceMem>
__host__ __device__ __forceinline__ void tree_load_stage(const TreeParams& p, const TreeUnit& u, int i, uint32_t lds0,
                                                         int wave, int lane, const RowLoad<D, true>& lk,
                                                         const RowLoad<D, false>& lv, const Mem& mem = Mem()) {
  using C = TreeCfg<D, QW, KW>;
  const uint32_t dst = lds0 + (i & 1) * 2 * C::TILE;
  const int row0 = u.kbeg + C::KEYS * i;
  row_tile_load<D, C::BLOCKS, C::NW, true>(u.kg, p.k.ss, row0, u.kend, dst, wave, lane, lk, mem);
  row_tile_load<D, C::BLOCKS, C::NW, false>(u.vg, p.v.ss, row0, u.kend, dst + C::TILE, wave, lane, lv, mem);
}

// Element (row, d) of the result, or of the split's partial.
struct RowOut {
  int64_t rec;  // (global row) * splits + split
  int64_t mrow;  // index into m [B, Hq, T]
  int64_t off;   // element offset of the row in out
  __host__ __device__ __forceinline__ RowOut(const TreeParams& p, const TreeUnit& u, int row) {
    const int r = u.row0 + row, node = r / u.G, h = u.hk * u.G + r - node * u.G;
    rec = ((static_cast<int64_t>(u.b) * p.Hkv + u.hk) * (u.G * p.T) + r) * p.splits + u.split;
    mrow = (static_cast<int64_t>(u.b) * p.Hq + h) * p.T + node;
    off = u.b * p.o.sb + h * p.o.sh + node * p.o.ss;
  }
};

// ----------------------------------------------------------------------------
// Key weights
template <int D, int KW, int RW>
struct WeightsCfg {
  static constexpr int NW = KW * RW;
  static constexpr int KEYS = 32 * KW;
  static constexpr int ROWS = 32 * RW;              // rows of a stage
  static constexpr int QB = ROWS * D * 2;           // bytes of its Q rows
  static constexpr int PIECES = BlockLayout<D>::IPB;  // 1 KB pieces of a 32-row block
};

// The first row whose query stands at `key` or behind it.
__host__ __device__ __forceinline__ int first_row(int key, int first, int G) {
  return key > first ? (key - first) * G : 0;
}

// What a workgroup of KEYS keys and stages of ROWS rows works on.
struct WeightsUnit {
  int chunk, bh, b, hk, L, key0;
  int G, first;   // first: position of query 0
  int rstart, R;  // rows from the stage of the first query that sees key0 on; those of the chunk
  __host__ __device__ __forceinline__ WeightsUnit(const KeyWeightsParams& p, int block, int ntiles, int KEYS, int ROWS) {
    // all (sequence, head) pairs of a key tile together: the tiles of most rows come first
    const int nbh = p.B * p.Hkv;
    chunk = block / (nbh * ntiles);
    const int tile = (block - chunk * nbh * ntiles) / nbh;
    bh = block % nbh;
    b = bh / p.Hkv;
    hk = bh - b * p.Hkv;
    L = clamped_length(load_table_entry(p.seqlens, b), p.cap);
    key0 = tile * KEYS;
    G = p.Hq / p.Hkv;
    first = L - p.T;
    const int64_t chunk0 = static_cast<int64_t>(chunk) * p.chunk_rows;
    const int64_t rows = static_cast<int64_t>(G) * p.T, end = chunk0 + p.chunk_rows;
    R = static_cast<int>(rows < end ? rows : end);
    const int sees = first_row(key0, first, G) / ROWS * ROWS, from = static_cast<int>(chunk0);
    rstart = sees > from ? sees : from;
  }
  __host__ __device__ __forceinline__ bool behind() const { return key0 >= L; }    // the sequence
  __host__ __device__ __forceinline__ bool unseen() const { return rstart >= R; }  // its keys, by the chunk's rows
};

// The row of its 32-row block that a lane of wave (kw, rw) fetches, as (query,
// head), moved on by one stage at a time.
template <int D, int KW, int RW>
struct WeightsRows {
  using C = WeightsCfg<D, KW, RW>;
  LoadLane ll;
  int t, g, dt, dg;
  __host__ __device__ __forceinline__ WeightsRows(const KeyWeightsParams& p, const WeightsUnit& u, int lane, int kw,
                                                  int rw)
      : ll(lane, kw, p.q.ss) {
    const int r = u.rstart + 32 * rw + ll.r;
    t = r / u.G;
    g = r - t * u.G;
    dt = C::ROWS / u.G;
    dg = C::ROWS - dt * u.G;
  }
  // the row as a query and a head of the group; past the last the last head's last query
  struct Row {
    bool in;
    int t, g;
  };
  __host__ __device__ __forceinline__ Row row(const KeyWeightsParams& p, const WeightsUnit& u) const {
    const bool in = t < p.T;
    return Row{in, in ? t : p.T - 1, in ? g : u.G - 1};
  }
  // the wave's pieces of stage i's Q rows to buffer i & 1; qbase: the group's first head
  template <typename Mem = DeviceMem>
  __host__ __device__ __forceinline__ void load(const KeyWeightsParams& p, const Row& r, const char* qbase, int i,
                                                uint32_t lds0, int kw, int rw, const Mem& mem = Mem()) const {
    const char* src = qbase + (r.g * p.q.sh + r.t * p.q.ss) * 2 + ll.hoff;
    const uint32_t dst = lds0 + (i & 1) * C::QB + rw * BlockLayout<D>::BLOCK;
#pragma unroll
    for (int cp = 0; cp < C::PIECES / KW; ++cp)
      mem.load16_global(dst + (kw + KW * cp) * 1024, src + (kw + KW * cp) * 32);
    if (C::PIECES < KW) {
      if (kw < C::PIECES) mem.load16_global(dst + kw * 1024, src + kw * 32);
    }
  }
  __host__ __device__ __forceinline__ void next(const WeightsUnit& u) {
    t += dt;
    g += dg;
    if (g >= u.G) {
      g -= u.G;
      ++t;
    }
  }
};
__host__ __device__ __forceinline__ const char* weights_queries(const KeyWeightsParams& p, const WeightsUnit& u) {
  return static_cast<const char*>(p.q.ptr) + (u.b * p.q.sb + static_cast<int64_t>(u.hk) * u.G * p.q.sh) * 2;
}

// The first chunk whose sums of `key` were written (the rows before see none of its tile).
__host__ __device__ __forceinline__ int weights_first_chunk(const KeyWeightsParams& p, int L, int key) {
  const int sees = first_row(key / kWeightsKeys * kWeightsKeys, L - p.T, p.Hq / p.Hkv) / kWeightsStage * kWeightsStage;
  return sees / p.chunk_rows;
}
// A key's place in a chunk's sums.
__host__ __device__ __forceinline__ int64_t weights_slot(const KeyWeightsParams& p, int64_t chunk, int64_t bh, int key) {
  return (chunk * p.B * p.Hkv + bh) * p.cap + key;
}

}  // namespace ssa
