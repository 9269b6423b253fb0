// LDS tiles of whole rows for kernels that stream a KV cache once.
//
// A tile is a stack of 32-row blocks, a block PIECES pieces of 1 KB, each
// written by one direct-to-LDS load whose lanes read whole rows: every four
// lanes fetch 64 contiguous bytes in lane order, so an instruction touches 8 to
// 16 cache lines where the chunk-major blocks of ssa_tile.hpp touch 32 to 64.
// Two things keep the reads off each other's banks without breaking that
// order: the 64-byte quarters of a piece's rows are permuted by the row's slot,
// and each piece starts 16 bytes later, modulo 256, than the one before.
//
//   K (read row by row, 16 lanes one chunk of 16 rows): rows 0-15 of a block,
//     and 16-31, fall into 16 different 16-byte columns of the banks (two to
//     a column at D = 32);
//   V (transpose reads, 16 lanes 32 bytes of 4 consecutive rows): the 4 rows
//     lie in 4 different 64-byte columns.
#pragma once

#include "ssa_tile.hpp"

namespace ssa {

template <int D>
struct RowTile {
  static constexpr int ROWB = 2 * D;            // bytes of a row
  static constexpr int LPR = ROWB / 16;         // lanes that load one
  static constexpr int RPP = 1024 / ROWB;       // rows of a piece
  static constexpr int PIECES = 32 / RPP;       // pieces of a block
  // piece p's first byte
  __host__ __device__ static constexpr int off(int p) { return p * 1024 + (p & 3) * 16 + (p >> 2) * 256; }
  static constexpr int BLOCK = (off(PIECES - 1) + 1024 + 255) / 256 * 256;
  // quarter permutation of slot s of a piece
  __host__ __device__ static constexpr int swz(int s) { return D == 128 ? s & 3 : D == 64 ? (s >> 1) & 1 : 0; }
  // row of (piece, slot): a part by the slot and a part by the piece
  __host__ __device__ static constexpr int k_slot_row(int s) { return D == 64 ? 4 * s : D == 32 ? (s & 3) + 8 * (s >> 2) : s; }
  __host__ __device__ static constexpr int k_piece_row(int p) { return D == 64 ? p : 4 * p; }
  __host__ __device__ static constexpr int v_piece_row(int p) { return RPP * p; }
};

// What a lane loads of every piece of a matrix [*, D] (row stride ss elements,
// below 2^24): byte voff from the piece's first row.
template <int D, bool K>
struct RowLoad {
  uint32_t voff;
  __host__ __device__ __forceinline__ static int row(int lane) {
    using R = RowTile<D>;
    const int s = lane / R::LPR;
    return K ? R::k_slot_row(s) : s;
  }
  __host__ __device__ __forceinline__ static int chunk(int lane) {
    using R = RowTile<D>;
    return (lane % R::LPR) ^ (4 * R::swz(lane / R::LPR));
  }
  __host__ __device__ __forceinline__ RowLoad(int lane, int64_t ss)
      : voff(static_cast<uint32_t>(row(lane) * ss * 2 + chunk(lane) * 16)) {}
};

// BLOCKS blocks of rows row0 .. of g to LDS byte address lds, piece j from wave
// j % NW; rows at and past nrows repeat the last.  Whole tiles whose rows span
// less than 2^31 bytes go through one descriptor with 32-bit offsets.
template <int D, int BLOCKS, int NW, bool K, typename Mem = DeviceMem>
__host__ __device__ __forceinline__ void row_tile_load(const char* g, int64_t ss, int row0, int nrows, uint32_t lds,
                                                       int wave, int lane, const RowLoad<D, K>& rl,
                                                       const Mem& mem = Mem()) {
  using R = RowTile<D>;
  constexpr int N = BLOCKS * R::PIECES, PER = (N + NW - 1) / NW;
  if (row0 + 32 * BLOCKS <= nrows && ss * 2 * 32 * BLOCKS < (1ll << 31)) {
    const i32x4_t rs = raw_rsrc(g + static_cast<int64_t>(row0) * ss * 2);
    const int ss2 = static_cast<int>(ss * 2);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int j = wave + NW * i;
      if (N % NW != 0 && j >= N) break;
      const int blk = j / R::PIECES, p = j % R::PIECES;
      mem.load16(lds + blk * R::BLOCK + R::off(p), rs, rl.voff,
                 (32 * blk + (K ? R::k_piece_row(p) : R::v_piece_row(p))) * ss2);
    }
  } else {
    const char* gc = g + RowLoad<D, K>::chunk(lane) * 16;
#pragma unroll 1
    for (int j = wave; j < N; j += NW) {
      const int blk = j / R::PIECES, p = j % R::PIECES;
      int row = row0 + 32 * blk + (K ? R::k_piece_row(p) : R::v_piece_row(p)) + RowLoad<D, K>::row(lane);
      row = row < nrows ? row : nrows - 1;
      mem.load16_global(lds + blk * R::BLOCK + R::off(p), gc + row * ss * 2);
    }
  }
}

// K: chunk 2 ds + hh of row l32 of a block.
template <int D>
struct RowTileK {
  static constexpr int Q = D / 32;  // 64-byte quarters of a row
  uint32_t b[Q];
  __host__ __device__ __forceinline__ RowTileK(int l32, int hh) {
    using R = RowTile<D>;
    const int p = D == 128 ? l32 >> 2 : D == 64 ? l32 & 3 : (l32 >> 2) & 1;
    const int s = D == 128 ? l32 & 3 : D == 64 ? l32 >> 2 : (l32 & 3) + 4 * (l32 >> 3);
#pragma unroll
    for (int q = 0; q < Q; ++q)
      b[q] = static_cast<uint32_t>(R::off(p) + s * R::ROWB + (q ^ R::swz(s)) * 64 + hh * 16);
  }
  // at: byte address of a block
  __host__ __device__ __forceinline__ uint32_t address(uint32_t at, int ds) const {
    return b[ds >> 1] + at + (ds & 1) * 32;
  }
  template <typename V>
  __device__ __forceinline__ V read(uint32_t at, int ds) const {
    return *(const __attribute__((address_space(3))) V*)(uintptr_t)address(at, ds);
  }
};

// V: column 32 db + l32 of rows 16 ks + 8 hi + 4 hh + (0..3) of a block, four
// elements (the k-slots 4 hi .. of an MFMA operand), as tile_read_tr.
template <int D>
struct RowTileV {
  static constexpr int Q = D / 32;
  uint32_t b[Q];
  __host__ __device__ __forceinline__ explicit RowTileV(int lane) {
    using R = RowTile<D>;
    const int g = lane >> 4, i = lane & 15, hh = lane >> 5;
    // (piece, slot) of row 4 hh + i / 4; the rest of the row is an immediate
    const int p = D == 128 ? hh : 0;
    const int s = D == 128 ? i >> 2 : 4 * hh + (i >> 2);
#pragma unroll
    for (int db = 0; db < Q; ++db)
      b[db] = static_cast<uint32_t>(R::off(p) + s * R::ROWB + (db ^ R::swz(s)) * 64 + (g & 1) * 32 + (i & 3) * 8);
  }
  // the lane's 8 bytes: row 16 ks + 8 hi + 4 hh + i / 4, columns 32 db + 16 (g & 1) + 4 (i & 3)
  // .., for lane i of the wave's 16 lanes g
  __host__ __device__ __forceinline__ uint32_t address(uint32_t at, int ks, int hi, int db) const {
    using R = RowTile<D>;
    const int imm = D == 128 ? R::off(4 * ks + 2 * hi) : D == 64 ? R::off(2 * ks + hi) : R::off(ks) + hi * 8 * R::ROWB;
    return b[db] + at + imm;
  }
  template <typename V4>
  __device__ __forceinline__ V4 read(uint32_t at, int ks, int hi, int db) const {
    typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
    const bf16x4_t v = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
        (__attribute__((address_space(3))) bf16x4_t*)(uintptr_t)address(at, ks, hi, db));
    return __builtin_bit_cast(V4, v);
  }
};

}  // namespace ssa
