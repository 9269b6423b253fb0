// SSA attention of a tree of drafted tokens over a KV cache, for gfx950.
//
// Node i of T drafted tokens attends every cached row before the tree's and the
// rows of its own branch:
//   out_i = sum_j p_ij v_j,  p_i = softmax over visible j of n sign(s) ln(1 + b |s|),  s = scale q_i . k_j
// in base 2: t = n sign(s) log2(1 + scale b |q.k|), p = 2^(t - m), with the
// running maximum and sum of the online softmax in fp32 and p rounded to the
// input type for the product with V (the rounding errors of the keys are
// independent, and together stay below the output's own rounding).
//
// The G q-heads of a group and their T nodes are R = G T rows over one stream
// of keys, row r = node * G + head.  As in the decode step the rows are the
// matrix cores' columns:
//   S^T = K Q^T (A = 32 keys from LDS, B = 32 rows of Q in registers)
//   O^T += V^T P^T (A = V^T by LDS transpose reads, B = P^T from S^T)
// so a lane pair (l, l + 32) holds one row.  Two forms:
//   * up to 64 rows (tree_stream_kernel): the cache's stream is the bound; each
//     wave streams its own tiles of 32 keys through a private LDS ring, for one
//     or two groups of 32 rows at once, and the waves merge at the end;
//   * more (tree_wide_kernel): the transform (one log2 and one exp2 a pair) is
//     the bound; QW groups of 32 rows by KW key waves share each stage of keys,
//     and the key waves merge at the end.
// The keys are split over workgroups in ranges of one length for all sequences
// (a ragged batch is then a number of equal pieces of work, and a sequence's
// result does not depend on the others); partials (m, l, acc) meet in split
// order in tree_merge_kernel.
//
// The running maximum is moved only when a lane's sum of a tile passes a bound
// with the old one (kTreeSum): the rescaling of acc and the tile's maximum are
// then rare, a quarter of the vector work.
//
// The mask is packed to one bit per node when a workgroup's keys reach the
// tree's rows; tiles before them do no mask work.
#include "ssa_cache_ops.hpp"
#include "ssa_common.hpp"
#include "ssa_launch.hpp"
#include "ssa_plan.hpp"
#include "ssa_tile.hpp"

namespace ssa {

namespace {

constexpr int kMaxNodes = 1024;
constexpr int kMaskWords = kMaxNodes / 32 + 1;  // words of a packed mask row, one of padding
// A lane's sum of 16 p with the old maximum: below it no p overflows fp16, and
// sums of 2^30 keys stay far from fp32's range.
constexpr float kTreeSum = 16384.f;

__device__ __forceinline__ int clamped_length(const TreeParams& p, int b) {
  const int L = load_table_entry(p.seqlens, b);
  return L < 0 ? 0 : (L > p.cap ? p.cap : L);
}

// What a workgroup works on.
struct TreeUnit {
  int b, hk, row0, nrows, split;  // rows row0 .. row0 + nrows - 1 of the group's R
  int G, base, kbeg, kend, ntile;
  const char* kg;
  const char* vg;
  __device__ __forceinline__ TreeUnit(const TreeParams& p, int block, int per, int nqb) {
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
    G = p.Hq / p.Hkv;
    row0 = qb * per;
    nrows = min(per, G * p.T - row0);
    const int L = clamped_length(p, b);
    base = L - p.T;
    const int64_t beg = static_cast<int64_t>(split) * p.split_keys;
    kbeg = beg < L ? static_cast<int>(beg) : L;
    kend = beg + p.split_keys < L ? static_cast<int>(beg + p.split_keys) : L;
    ntile = (kend - kbeg + 31) / 32;
    kg = static_cast<const char*>(p.k.ptr) + (b * p.k.sb + hk * p.k.sh) * 2;
    vg = static_cast<const char*>(p.v.ptr) + (b * p.v.sb + hk * p.v.sh) * 2;
  }
  // a tile's keys that some rows may not see: the tree's
  __device__ __forceinline__ bool masked(int key0) const { return key0 + 32 > base; }
};

__device__ __forceinline__ int mask_stride(int T) { return 2 * ((T + 63) / 64) + 1; }

// Mask rows of the nodes of rows row0 .. row0 + nrows - 1, one bit a node, 64
// nodes by one ballot; the word behind the last is 0.
__device__ __forceinline__ void pack_mask(const TreeParams& p, const TreeUnit& u, uint32_t* words, int tid,
                                          int nthreads) {
  const int lane = tid & 63, W = mask_stride(p.T), chunks = (p.T + 63) / 64;
  const int n0 = u.row0 / u.G, nn = (u.row0 + u.nrows - 1) / u.G - n0 + 1;
  const uint8_t* mask = p.mask + u.b * p.mask_sb + static_cast<int64_t>(n0) * p.T;
  for (int i = tid >> 6; i < nn * chunks; i += nthreads >> 6) {
    const int n = i / chunks, c = i - n * chunks, col = 64 * c + lane;
    const uint64_t bits = __ballot(col < p.T && mask[n * p.T + col] != 0);
    if (lane == 0) {
      words[n * W + 2 * c] = static_cast<uint32_t>(bits);
      words[n * W + 2 * c + 1] = static_cast<uint32_t>(bits >> 32);
      if (c == chunks - 1) words[n * W + 2 * chunks] = 0;
    }
  }
}

// Keys key0 .. key0 + 31 that a node sees, as bits; j0 = key0 - base < T.
__device__ __forceinline__ uint32_t mask_window(const uint32_t* row, int j0) {
  if (j0 < 0) return (row[0] << -j0) | ((1u << -j0) - 1u);
  return __builtin_amdgcn_alignbit(row[(j0 >> 5) + 1], row[j0 >> 5], j0 & 31);
}

// 32 rows of a wave: Q, the running maximum and sum, the unnormalised output.
template <typename T, int D>
struct RowGroup {
  typename Vec8<T>::type q[D / 16];
  f32x16 acc[D / 32];
  float m, l;
  // the lane's row `row` of the group (a row past the end reads zeros)
  __device__ __forceinline__ void init(const TreeParams& p, const TreeUnit& u, int row, int hh) {
    typedef typename Vec8<T>::type v8;
    const bool in = row < u.nrows;
    const int r = u.row0 + (in ? row : 0), node = r / u.G, h = u.hk * u.G + r - node * u.G;
    const T* src = static_cast<const T*>(p.q.ptr) + u.b * p.q.sb + h * p.q.sh + node * p.q.ss;
#pragma unroll
    for (int ds = 0; ds < D / 16; ++ds) q[ds] = in ? load16<v8>(src + ds * 16 + 8 * hh) : zero8<v8>();
#pragma unroll
    for (int d = 0; d < D / 32; ++d) acc[d] = f32x16{};
    m = -INFINITY;
    l = 0.f;
  }
};

template <typename T>
__device__ __forceinline__ bool not_finite(uint32_t two) {
  constexpr uint32_t E = __is_same(T, __bf16) ? 0x7f80u : 0x7c00u;
  return (two & E) == E || (two & (E << 16)) == (E << 16);
}

// All ones where bit `i` of win is set, else 0.
__device__ __forceinline__ uint32_t seen_mask(uint32_t win, int i) {
  return static_cast<uint32_t>(static_cast<int32_t>(win << (31 - i)) >> 31);
}
// Bit of accumulator entry r in a window shifted by 4 hh (crow()).
__device__ __forceinline__ constexpr int bit_of(int r) { return 8 * (r >> 2) + (r & 3); }

// What the infinities and NaN of a tile of V add to the rows that see them:
// kind 0 / 1 / 2 counts the +inf / -inf / NaN that each row sees in each
// column, by a product with the rows' 0 / 1 masks.
template <typename T, int D, int NQ>
__device__ void add_not_finite(const TrBase<D>& vt, int blk, RowGroup<T, D> (&st)[NQ], const uint32_t (&win)[NQ]) {
  typedef typename Vec8<T>::type v8;
  typedef T v4 __attribute__((ext_vector_type(4)));
#pragma unroll 1
  for (int kind = 0; kind < 3; ++kind) {
    const float add = kind == 0 ? INFINITY : kind == 1 ? -INFINITY : __builtin_nanf("");
#pragma unroll
    for (int db = 0; db < D / 32; ++db) {
      v8 hit[2];
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const v4 lo = tile_read_tr<D, v4>(vt, blk, ks, 0, db), hi = tile_read_tr<D, v4>(vt, blk, ks, 1, db);
        const v8 vf = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = static_cast<float>(vf[e]);
          const bool is = kind == 0 ? v == INFINITY : kind == 1 ? v == -INFINITY : v != v;
          hit[ks][e] = static_cast<T>(is ? 1.f : 0.f);
        }
      }
#pragma unroll
      for (int g = 0; g < NQ; ++g) {
        v8 seen[2];
#pragma unroll
        for (int r = 0; r < 16; ++r)
          seen[r >> 3][r & 7] = static_cast<T>(__uint_as_float(seen_mask(win[g], bit_of(r)) & 0x3f800000u));
        f32x16 count = f32x16{};
        count = mfma32(hit[0], seen[0], count);
        count = mfma32(hit[1], seen[1], count);
#pragma unroll
        for (int r = 0; r < 16; ++r) st[g].acc[db][r] += count[r] > 0.f ? add : 0.f;
      }
    }
  }
}

// One tile of 32 keys for NQ groups of 32 rows: scores, transform, softmax
// update and the product with V.  win[g]: the keys that the lane's row of group
// g sees, shifted by 4 hh (MASKED).
template <typename T, int D, bool NPOS, bool MASKED, int NQ>
__device__ __forceinline__ void tree_tile(const RowBase<D>& kr, const TrBase<D>& vt, int blk, RowGroup<T, D> (&st)[NQ],
                                          const uint32_t (&win)[NQ], float c, float n) {
  typedef typename Vec8<T>::type v8;
  typedef T v4 __attribute__((ext_vector_type(4)));
  constexpr int ND16 = D / 16, ND32 = D / 32;
  constexpr uint32_t kOut = NPOS ? 0xff800000u : 0x7f800000u;  // the score of the lowest t: -inf or +inf
  f32x16 s[NQ];
#pragma unroll
  for (int g = 0; g < NQ; ++g) s[g] = f32x16{};
#pragma unroll
  for (int ds = 0; ds < ND16; ++ds) {
    const v8 kf = tile_read_row<D, v8>(kr, blk, ds);
#pragma unroll
    for (int g = 0; g < NQ; ++g) s[g] = mfma32(kf, st[g].q[ds], s[g]);
  }
  v8 pb[NQ][2];
#pragma unroll
  for (int g = 0; g < NQ; ++g) {
    if constexpr (!MASKED) {
      float sum = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float x = s[g][r];
        const float pv = fast_exp2(fmaf(n, copysignf(fast_log2(fmaf(c, fabsf(x), 1.f)), x), -st[g].m));
        sum += pv;
        pb[g][r >> 3][r & 7] = static_cast<T>(pv);
      }
      // m = -inf (nothing seen yet) gives an infinite or NaN sum
      if (__builtin_expect(__all(sum <= kTreeSum), 1)) {
        st[g].l += sum;
        continue;
      }
    }
    float z = -INFINITY;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      if constexpr (MASKED) {
        const uint32_t in = seen_mask(win[g], bit_of(r));
        s[g][r] = __uint_as_float((__float_as_uint(s[g][r]) & in) | (kOut & ~in));
      }
      z = fmaxf(z, NPOS ? s[g][r] : -s[g][r]);
    }
    z = pair_max(z);
    const float top = NPOS ? z : -z;
    const float tmax = z == -INFINITY ? -INFINITY : n * copysignf(fast_log2(fmaf(c, fabsf(top), 1.f)), top);
    const float mnew = fmaxf(st[g].m, tmax);
    const float alpha = fast_exp2(mnew == -INFINITY ? 0.f : st[g].m - mnew);
    st[g].m = mnew;
#pragma unroll
    for (int d = 0; d < ND32; ++d) st[g].acc[d] *= alpha;
    float l = st[g].l * alpha;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float x = s[g][r];
      float pv = fast_exp2(fmaf(n, copysignf(fast_log2(fmaf(c, fabsf(x), 1.f)), x), -mnew));
      if constexpr (MASKED) pv = __uint_as_float(__float_as_uint(pv) & seen_mask(win[g], bit_of(r)));
      l += pv;
      pb[g][r >> 3][r & 7] = static_cast<T>(pv);
    }
    st[g].l = l;
  }
  bool bad = false;
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
    for (int db = 0; db < ND32; ++db) {
      const v4 lo = tile_read_tr<D, v4>(vt, blk, ks, 0, db), hi = tile_read_tr<D, v4>(vt, blk, ks, 1, db);
      v8 vf = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      if constexpr (MASKED) {
        // a masked row's p is 0, and 0 times an infinity or NaN is not: such
        // values leave the product here and join below where they are seen
        const u32x4 w = __builtin_bit_cast(u32x4, vf);
        const int b = int(not_finite<T>(w[0])) | int(not_finite<T>(w[1])) | int(not_finite<T>(w[2])) | int(not_finite<T>(w[3]));
        if (__builtin_expect(__any(b), 0)) {
          bad = true;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float v = static_cast<float>(vf[e]);
            if (!(fabsf(v) < INFINITY)) vf[e] = static_cast<T>(0.f);
          }
        }
      }
#pragma unroll
      for (int g = 0; g < NQ; ++g) st[g].acc[db] = mfma32(vf, pb[g][ks], st[g].acc[db]);
    }
  }
  if constexpr (MASKED) {
    if (__builtin_expect(bad, 0)) add_not_finite<T, D, NQ>(vt, blk, st, win);
  }
}

// Element (row, d) of the result, or of the split's partial.
struct RowOut {
  int64_t rec;  // (global row) * splits + split
  int64_t mrow;  // index into m [B, Hq, T]
  int64_t off;   // element offset of the row in out
  __device__ __forceinline__ RowOut(const TreeParams& p, const TreeUnit& u, int row) {
    const int r = u.row0 + row, node = r / u.G, h = u.hk * u.G + r - node * u.G;
    rec = ((static_cast<int64_t>(u.b) * p.Hkv + u.hk) * (u.G * p.T) + r) * p.splits + u.split;
    mrow = (static_cast<int64_t>(u.b) * p.Hq + h) * p.T + node;
    off = u.b * p.o.sb + h * p.o.sh + node * p.o.ss;
  }
};

// ------------------------------------------------------------ up to 64 rows
template <int D, int NQ>
struct StreamCfg : DecodeCfg<D> {
  using C = DecodeCfg<D>;
  static constexpr int MASK_BYTES = 32 * NQ * kMaskWords * 4;
};

template <typename T, int D, bool NPOS, int NQ>
__device__ __forceinline__ void tree_stream_body(const TreeParams& p, char* smem, uint32_t* words, const TreeUnit& u) {
  using C = DecodeCfg<D>;
  constexpr int NW = C::NW, NB = C::NB, ND32 = D / 32;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hh = lane >> 5;
  const float n = *p.n_ptr;
  const float c = p.scale * *p.b_ptr;
  const int ntw = u.ntile > wave ? (u.ntile - wave + NW - 1) / NW : 0;  // tiles of this wave

  const LoadLane lk0(lane, 0, p.k.ss), lk1(lane, 1, p.k.ss), lv0(lane, 0, p.v.ss), lv1(lane, 1, p.v.ss);
  const uint32_t ring = lds_addr(smem) + wave * NB * C::TB;
  const RowBase<D> rb(l32, hh);
  const TrBase<D> tb(lane);
  // past the wave's last tile the rows clamp to kend - 1 (loads into a free
  // buffer, never read), so that one wait count fits every iteration
  auto issue = [&](int i) {
    const int row0 = u.kbeg + 32 * (wave + NW * i);
    const uint32_t dst = ring + (i % NB) * C::TB;
    block_load_wave<D>(u.kg, p.k.ss, row0, u.kend, dst, lk0, lk1);
    block_load_wave<D>(u.vg, p.v.ss, row0, u.kend, dst + C::BLOCK, lv0, lv1);
  };
  if (ntw > 0) {
#pragma unroll
    for (int i = 0; i < NB - 1; ++i) issue(i);
  }
  RowGroup<T, D> st[NQ];
#pragma unroll
  for (int g = 0; g < NQ; ++g) st[g].init(p, u, 32 * g + l32, hh);
  const bool reaches = u.kend > u.kbeg && u.kend > u.base;
  if (reaches) pack_mask(p, u, words, tid, NW * 64);
  __syncthreads();
  if (ntw > 0) {
    const int W = mask_stride(p.T), n0 = u.row0 / u.G;
    const uint32_t* mrow[NQ];
#pragma unroll
    for (int g = 0; g < NQ; ++g) mrow[g] = words + ((u.row0 + min(32 * g + l32, u.nrows - 1)) / u.G - n0) * W;
    for (int i = 0; i < ntw; ++i) {
      wait_lgkm<0>();  // reads of tile i - 1, whose buffer the next issue overwrites
      issue(i + NB - 1);
      wait_vm<(NB - 1) * C::LPT>();  // tile i has landed
      const uint32_t buf = ring + (i % NB) * C::TB;
      const RowBase<D> kr = at_tile(rb, buf);
      const TrBase<D> vt = at_tile(tb, buf + C::BLOCK);
      const int key0 = u.kbeg + 32 * (wave + NW * i);
      uint32_t win[NQ] = {};
      if (u.masked(key0)) {
#pragma unroll
        for (int g = 0; g < NQ; ++g) win[g] = mask_window(mrow[g], key0 - u.base) >> (4 * hh);
        tree_tile<T, D, NPOS, true, NQ>(kr, vt, 0, st, win, c, n);
      } else {
        tree_tile<T, D, NPOS, false, NQ>(kr, vt, 0, st, win, c, n);
      }
    }
    wait_vm<0>();  // the trailing prefetches land before the ring is reused
  }

  // Merge the waves: (m, l) per row and acc[row][d] through LDS, then one
  // thread per (row, d) combines them in wave order.
  float* ml = reinterpret_cast<float*>(smem);                  // [NW][2][32]
  float* accs = reinterpret_cast<float*>(smem + C::ML_BYTES);  // [NW][32][ACC_LD]
#pragma unroll
  for (int g = 0; g < NQ; ++g) {
    const float l_tot = pair_sum(st[g].l);
    __syncthreads();
    if (hh == 0) {
      ml[(wave * 2 + 0) * 32 + l32] = st[g].m;
      ml[(wave * 2 + 1) * 32 + l32] = l_tot;
    }
#pragma unroll
    for (int db = 0; db < ND32; ++db) {
#pragma unroll
      for (int r = 0; r < 16; ++r) accs[(wave * 32 + l32) * C::ACC_LD + db * 32 + crow(r, hh)] = st[g].acc[db][r];
    }
    __syncthreads();
    const int rows = min(32, u.nrows - 32 * g);
    for (int e = tid; e < rows * D; e += NW * 64) {
      const int q = e / D, d = e - q * D;
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < NW; ++w) M = fmaxf(M, ml[(w * 2) * 32 + q]);
      float Ls = 0.f, O = 0.f;
      if (M != -INFINITY) {
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          const float sc = fast_exp2(ml[(w * 2) * 32 + q] - M);
          // a wave that saw no key of this row has m = -inf, l = 0, acc = 0
          Ls += ml[(w * 2 + 1) * 32 + q] * sc;
          O += accs[(w * 32 + q) * C::ACC_LD + d] * sc;
        }
      }
      const RowOut o(p, u, 32 * g + q);
      if (p.splits == 1) {
        const float l_safe = Ls == 0.f ? 1.f : Ls;
        static_cast<T*>(const_cast<void*>(p.o.ptr))[o.off + d] = static_cast<T>(O * (1.f / l_safe));
        if (d == 0 && p.m != nullptr) p.m[o.mrow] = M + log2f(l_safe);
      } else {
        p.ws_acc[o.rec * D + d] = O;
        if (d == 0) {
          p.ws_ml[2 * o.rec] = M;
          p.ws_ml[2 * o.rec + 1] = Ls;
        }
      }
    }
  }
}

// ------------------------------------------------------------ more than 64 rows
// Two stages of 32 KW U keys, a K tile and a V tile each; wave (qw, kw) takes
// the stage's key tiles kw, kw + KW, ...
template <int D, int QW, int KW>
struct WideCfg {
  static constexpr int NW = QW * KW;
  static constexpr int U = D == 128 ? 2 / KW : 4 / KW;  // tiles of a wave and stage
  static constexpr int KEYS = 32 * KW * U;
  static constexpr int TILE = KEYS * D * 2;
  static constexpr int SMEM = 4 * TILE;
  static_assert(U >= 1 && (KW == 1 || KW / 2 * QW * 64 * (D / 32) * 64 <= SMEM), "the key waves' merge");
};

template <typename T, int D, bool NPOS, int QW, int KW>
__device__ __forceinline__ void tree_wide_body(const TreeParams& p, char* smem, uint32_t* words, const TreeUnit& u) {
  using C = WideCfg<D, QW, KW>;
  typedef T v4 __attribute__((ext_vector_type(4)));
  constexpr int ND32 = D / 32, NW = C::NW;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int qw = wave / KW, kw = wave - qw * KW;
  const int l32 = lane & 31, hh = lane >> 5;
  const LoadLane lk(lane, wave, p.k.ss), lv(lane, wave, p.v.ss);
  const uint32_t lds0 = lds_addr(smem);
  const RowBase<D> rb(l32, hh);
  const TrBase<D> tb(lane);
  const int nst = (u.kend - u.kbeg + C::KEYS - 1) / C::KEYS;
  auto issue = [&](int i) {
    const uint32_t dst = lds0 + (i & 1) * 2 * C::TILE;
    tile_load_async<D, C::KEYS, NW>(u.kg, p.k.ss, u.kbeg + C::KEYS * i, u.kend, dst, wave, lk);
    tile_load_async<D, C::KEYS, NW>(u.vg, p.v.ss, u.kbeg + C::KEYS * i, u.kend, dst + C::TILE, wave, lv);
  };
  if (nst > 0) issue(0);
  const float n = *p.n_ptr;
  const float c = p.scale * *p.b_ptr;
  RowGroup<T, D> st[1];
  const int row = 32 * qw + l32;
  st[0].init(p, u, row, hh);
  const bool reaches = nst > 0 && u.kend > u.base;
  if (reaches) pack_mask(p, u, words, tid, NW * 64);
  const uint32_t* mrow =
      words + ((u.row0 + min(row, u.nrows - 1)) / u.G - u.row0 / u.G) * mask_stride(p.T);
  const bool works = 32 * qw < u.nrows;
  for (int i = 0; i < nst; ++i) {
    wait_vm<0>();     // this wave's share of stage i has landed
    __syncthreads();  // and everyone's; everyone is done with the other buffer
    if (i + 1 < nst) issue(i + 1);
    if (!works) continue;
    const uint32_t buf = lds0 + (i & 1) * 2 * C::TILE + kw * BlockLayout<D>::BLOCK;
    const RowBase<D> kr = at_tile(rb, buf);
    const TrBase<D> vt = at_tile(tb, buf + C::TILE);
#pragma unroll
    for (int t = 0; t < C::U; ++t) {
      const int key0 = u.kbeg + C::KEYS * i + 32 * (kw + KW * t);
      if (key0 >= u.kend) break;
      uint32_t win[1] = {0};
      if (u.masked(key0)) {
        win[0] = mask_window(mrow, key0 - u.base) >> (4 * hh);
        tree_tile<T, D, NPOS, true, 1>(kr, vt, KW * t, st, win, c, n);
      } else {
        tree_tile<T, D, NPOS, false, 1>(kr, vt, KW * t, st, win, c, n);
      }
    }
  }
  float m = st[0].m, l = st[0].l;
  // the upper half of the key waves hands its (m, l, acc) to the lower, lane by
  // lane through LDS, until one is left
  if constexpr (KW > 1) {
    f32x4_t* accs = reinterpret_cast<f32x4_t*>(smem);
    float* ml = reinterpret_cast<float*>(words);
#pragma unroll
    for (int half = KW / 2; half >= 1; half /= 2) {
      __syncthreads();  // the stages, or the last exchange, have been read
      const int slot = qw * half + (kw - half);
      if (works && kw >= half && kw < 2 * half) {
        ml[(2 * slot) * 64 + lane] = m;
        ml[(2 * slot + 1) * 64 + lane] = l;
#pragma unroll
        for (int j = 0; j < 4 * ND32; ++j) {
          f32x4_t x;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = st[0].acc[j / 4][4 * (j % 4) + e];
          accs[(slot * 4 * ND32 + j) * 64 + lane] = x;
        }
      }
      __syncthreads();
      if (works && kw < half) {
        const int from = qw * half + kw;
        const float m2 = ml[(2 * from) * 64 + lane], l2 = ml[(2 * from + 1) * 64 + lane];
        const float M = fmaxf(m, m2), ref = M == -INFINITY ? 0.f : M;
        const float f1 = fast_exp2(m - ref), f2 = fast_exp2(m2 - ref);
        m = M;
        l = l * f1 + l2 * f2;
#pragma unroll
        for (int j = 0; j < 4 * ND32; ++j) {
          const f32x4_t x = accs[(from * 4 * ND32 + j) * 64 + lane];
#pragma unroll
          for (int e = 0; e < 4; ++e) st[0].acc[j / 4][4 * (j % 4) + e] = st[0].acc[j / 4][4 * (j % 4) + e] * f1 + x[e] * f2;
        }
      }
    }
    if (kw > 0) return;
  }
  l = pair_sum(l);
  if (row >= u.nrows) return;
  const RowOut o(p, u, row);
  if (p.splits == 1) {
    const float l_safe = l == 0.f ? 1.f : l;
    const float inv = 1.f / l_safe;
    T* dst = static_cast<T*>(const_cast<void*>(p.o.ptr)) + o.off;
#pragma unroll
    for (int db = 0; db < ND32; ++db) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        v4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = static_cast<T>(st[0].acc[db][4 * g + e] * inv);
        *reinterpret_cast<v4*>(dst + 32 * db + 8 * g + 4 * hh) = x;
      }
    }
    if (hh == 0 && p.m != nullptr) p.m[o.mrow] = m + log2f(l_safe);
  } else {
    float* dst = p.ws_acc + o.rec * D;
#pragma unroll
    for (int db = 0; db < ND32; ++db) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f32x4_t x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = st[0].acc[db][4 * g + e];
        *reinterpret_cast<f32x4_t*>(dst + 32 * db + 8 * g + 4 * hh) = x;
      }
    }
    if (hh == 0) {
      p.ws_ml[2 * o.rec] = m;
      p.ws_ml[2 * o.rec + 1] = l;
    }
  }
}

}  // namespace

template <typename T, int D, int NQ>
__global__ __launch_bounds__(DecodeCfg<D>::NW * 64) void tree_stream_kernel(TreeParams p, int nunits) {
  __shared__ __attribute__((aligned(1024))) char smem[DecodeCfg<D>::SMEM];
  __shared__ uint32_t words[32 * NQ * kMaskWords];
  const int block = folded_block();
  if (block >= nunits) return;
  const TreeUnit u(p, block, 32 * NQ, 1);
  if (p.splits > 1 && u.kend <= u.kbeg) return;  // a shorter sequence: nothing to merge
  if (*p.n_ptr >= 0.f)
    tree_stream_body<T, D, true, NQ>(p, smem, words, u);
  else
    tree_stream_body<T, D, false, NQ>(p, smem, words, u);
}

template <typename T, int D, int QW, int KW>
__global__ __launch_bounds__(QW* KW * 64) void tree_wide_kernel(TreeParams p, int nunits, int nqb) {
  __shared__ __attribute__((aligned(1024))) char smem[WideCfg<D, QW, KW>::SMEM];
  __shared__ uint32_t words[32 * QW * kMaskWords];
  const int block = folded_block();
  if (block >= nunits) return;
  const TreeUnit u(p, block, 32 * QW, nqb);
  if (p.splits > 1 && u.kend <= u.kbeg) return;  // a shorter sequence: nothing to merge
  if (*p.n_ptr >= 0.f)
    tree_wide_body<T, D, true, QW, KW>(p, smem, words, u);
  else
    tree_wide_body<T, D, false, QW, KW>(p, smem, words, u);
}

// The splits' partials of a row in split order: out = sum_s acc_s 2^(m_s - M) /
// sum_s l_s 2^(m_s - M).  D / 4 threads a row, four columns each, and SW such
// groups that take every SW-th split and meet in LDS; every load is independent
// of the running state.
template <typename T, int D, int SW>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeParams p, int nrows) {
  typedef T v4 __attribute__((ext_vector_type(4)));
  constexpr int TPR = D / 4, RPB = 256 / (TPR * SW);
  static_assert(RPB >= 1, "a row's threads in one workgroup");
  __shared__ f32x4_t part[SW > 1 ? 256 : 1];
  const int tid = threadIdx.x, col = tid % TPR * 4, sw = tid / TPR % SW, in = tid / (TPR * SW);
  const int row = min(folded_block() * RPB + in, nrows - 1);  // a row past the end repeats the last
  const int G = p.Hq / p.Hkv, R = G * p.T;
  const int bh = row / R, r = row - bh * R, node = r / G;
  const int b = bh / p.Hkv, h = (bh - b * p.Hkv) * G + r - node * G;
  const int64_t L = clamped_length(p, b);
  const int ns = static_cast<int>((L + p.split_keys - 1) / p.split_keys);  // the sequence's own splits
  const int64_t rec0 = static_cast<int64_t>(row) * p.splits;
  const float* ml = p.ws_ml + 2 * rec0;
  float M = -INFINITY;
#pragma unroll 4
  for (int s = 0; s < ns; ++s) M = fmaxf(M, ml[2 * s]);
  const float ref = M == -INFINITY ? 0.f : M;
  float Ls = 0.f;
#pragma unroll 4
  for (int s = 0; s < ns; ++s) Ls += ml[2 * s + 1] * fast_exp2(ml[2 * s] - ref);
  f32x4_t O = f32x4_t{};
#pragma unroll 4
  for (int s = sw; s < ns; s += SW)
    O += *reinterpret_cast<const f32x4_t*>(p.ws_acc + (rec0 + s) * D + col) * fast_exp2(ml[2 * s] - ref);
  if constexpr (SW > 1) {
    part[tid] = O;
    __syncthreads();
    if (sw > 0) return;
#pragma unroll
    for (int w = 1; w < SW; ++w) O += part[tid + w * TPR];
  }
  const float l_safe = Ls == 0.f ? 1.f : Ls;
  const float inv = 1.f / l_safe;
  v4 x;
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = static_cast<T>(O[e] * inv);
  *reinterpret_cast<v4*>(static_cast<T*>(const_cast<void*>(p.o.ptr)) + b * p.o.sb + h * p.o.sh + node * p.o.ss + col) =
      x;
  if (col == 0 && p.m != nullptr) p.m[(static_cast<int64_t>(b) * p.Hq + h) * p.T + node] = M + log2f(l_safe);
}

namespace {

template <typename T, int D, int SW>
void launch_merge(const TreeParams& p, hipStream_t s) {
  const int n = p.B * p.Hq * p.T, rpb = 1024 / (D * SW);
  hipLaunchKernelGGL((tree_merge_kernel<T, D, SW>), folded_grid((n + rpb - 1) / rpb, 256), dim3(256), 0, s, p, n);
}

template <typename T, int D>
hipError_t launch_tree_t(const TreeParams& p, hipStream_t s) {
  const int64_t rows = static_cast<int64_t>(p.Hq / p.Hkv) * p.T;
  const int per = tree_rows_per_block(rows);
  const int nqb = static_cast<int>((rows + per - 1) / per);
  const int units = static_cast<int>(tree_units(p.B, p.Hq, p.Hkv, p.T) * p.splits);
  constexpr int ST = DecodeCfg<D>::NW * 64;
  constexpr int WT = D == 128 ? 512 : 1024, KW = D == 128 ? 1 : 2;  // threads; key waves of 8 row groups
  if (per == 32)
    hipLaunchKernelGGL((tree_stream_kernel<T, D, 1>), folded_grid(units, ST), dim3(ST), 0, s, p, units);
  else if (per == 64)
    hipLaunchKernelGGL((tree_stream_kernel<T, D, 2>), folded_grid(units, ST), dim3(ST), 0, s, p, units);
  else if (per == 128)
    hipLaunchKernelGGL((tree_wide_kernel<T, D, 4, 2 * KW>), folded_grid(units, WT), dim3(WT), 0, s, p, units, nqb);
  else
    hipLaunchKernelGGL((tree_wide_kernel<T, D, 8, KW>), folded_grid(units, WT), dim3(WT), 0, s, p, units, nqb);
  if (p.splits > 8)
    launch_merge<T, D, 4>(p, s);
  else if (p.splits > 1)
    launch_merge<T, D, 1>(p, s);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_tree_dt(const TreeParams& p, int D, hipStream_t s) {
  switch (D) {
    case 32: return launch_tree_t<T, 32>(p, s);
    case 64: return launch_tree_t<T, 64>(p, s);
    case 128: return launch_tree_t<T, 128>(p, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

hipError_t launch_tree(const TreeParams& p, int dtype, int D, hipStream_t stream) {
  if (dtype == 0) return launch_tree_dt<__bf16>(p, D, stream);
  return launch_tree_dt<_Float16>(p, D, stream);
}

}  // namespace ssa
