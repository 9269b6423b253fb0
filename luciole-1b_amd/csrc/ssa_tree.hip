// SSA attention of a tree of drafted tokens over a KV cache, for gfx950.
//
// Node i of T drafted tokens attends every cached row before the tree's and the
// rows of its own branch:
//   out_i = sum_j p_ij v_j,  p_i = softmax over visible j of n sign(s) ln(1 + b |s|),  s = scale q_i . k_j
// in base 2: t = n sign(s) log2(1 + scale b |q.k|), p = 2^(t - m), with the
// running maximum and sum of the online softmax in fp32 and p rounded to the
// input type for the product with V, the type that the matrix cores take at full
// rate: half a step of each key's share, independent from key to key.  With 61
// nodes over 1000 keys that makes the error of the output 0.0020 of its norm in
// bf16, where its own rounding is 0.0017 (over 65536 keys 0.0017 with it, in fp16
// 0.00025 and 0.00021).  In fp16 the step would grow for small p; kTreeLift keeps them off that.
//
// The G q-heads of a group and their T nodes are R = G T rows over one stream
// of keys, row r = node * G + head.  As in the decode step the rows are the
// matrix cores' columns:
//   S^T = K Q^T (A = 32 keys from LDS, B = 32 rows of Q in registers)
//   O^T += V^T P^T (A = V^T by LDS transpose reads, B = P^T from S^T)
// so a lane pair (l, l + 32) holds one row.  A workgroup is QW groups of 32 rows by
// KW key waves: each stage of keys goes to LDS once, by direct-to-LDS loads two
// stages deep, for all groups; every wave takes its own tiles of 32 keys, and the
// key waves of a group meet at the end.  What bounds it:
//   * the stream of the cache where the rows are few: 16 x 16 heads x 4096 x 128
//     in fp16, 64 nodes, 2048 to 4096 rows a sequence, takes 93 us for 411 MB, 4.4 TB/s (the
//     first form, each wave with tiles of its own and 32 rows, took 132, tiles that are not
//     whole rows 106);
//   * the transform where they are many, and the products that stand alone: 73 VALU
//     and 32 transcendental instructions for 32 x 32 scores, 804 cycles of one SIMD, and
//     256 of products at D = 64, of which the counters have 56 % beside vector
//     instructions.  Every stage's barrier lets the waves of a SIMD start their products
//     together.  1 x 32/8 x 65536 x 64, 64 nodes, has 49 us of transforms and
//     16 of products at the 2.1 GHz that the GPU holds then, and takes 73, merge
//     included; 8 x 32/8 x 4096 x 64, 32 nodes, has 12 and 4 on its longest
//     workgroups (2048 keys, 64 rows) and takes 29;
//   * a workgroup's start and end where both are few: 8 to 12 us, of which the load of
//     the length, the first stage's latency, the exchange and the stores are 3 to 5
//     each: 1 x 16 x 2048 x 128, 8 nodes, takes 14 us.  At head dims 64 and 128
//     LDS holds one workgroup a CU, so no other one fills that time.
// How many rows a workgroup has, and how many splits the keys, is in tree_plan().
//
// The keys are split over workgroups in ranges of one length for all sequences
// (a ragged batch is then a number of equal pieces of work, and a sequence's
// result does not depend on the others); partials (m, l, acc) meet in split
// order in tree_merge_kernel.
//
// The reference m of a row's exponents is its running maximum only loosely (and
// kTreeLift below it): it starts at an exponent of 0 where that suits the first scores and
// moves on when a lane's sum of a tile passes a bound (kTreeSum), so that the
// rescaling of acc and the tile's maximum, a quarter of the vector work, are rare.
//
// The mask is packed to one bit per node when a workgroup's keys reach the
// tree's rows; stages before them run in a loop of its own without any mask work.
// Packing takes a workgroup 4000 cycles and the masked tiles as long again, in
// the last split only; fetching the mask's bytes before the first stage's loads
// put its registers into both loops and made 1 x 32/8 x 65536 x 64 80 us for 74.
//
// The compiler keeps 5 (bf16) and 6 (fp16) registers of the 256-row form at D = 64 in scratch in
// the body for n < 0 (8 bytes reloaded a stage), none in the one for n >= 0.
#include "ssa_cache_plan.hpp"
#include "ssa_common.hpp"
#include "ssa_launch.hpp"

namespace ssa {

namespace {

// The reference of a row's exponents lies this far below its largest one.  p in
// fp16 has its full bits down to 2^-14 only, and below 2^-25 p would be nothing in
// the product with V but not in the sum l: with p up to 2^10 (or a lane's sum of
// at least that) a key counts within 2^-25 of 2^10, 2^-35 of its row's sum.  Keys of
// 2^-25.06 beside a few of 1 were lost before (their share of the result, all of it
// where the few have values of 0).  bf16 has fp32's range.
template <typename T>
constexpr float kTreeLift = __is_same(T, __bf16) ? 0.f : 10.f;
// A lane's sum of 16 p with the old reference: up to it no p overflows fp16, and
// sums of 2^30 keys stay far from fp32's range.
template <typename T>
constexpr float kTreeSum = __is_same(T, __bf16) ? 16384.f : 65504.f;
// ... and the least one of a row that has seen nothing yet: 2^kTreeLift
template <typename T>
constexpr float kTreeFirst = __is_same(T, __bf16) ? 1.f : 1024.f;

// Mask rows of the nodes of rows row0 .. row0 + nrows - 1, one bit a node, 64
// nodes by one ballot; the word behind the last is 0.
__device__ __forceinline__ void pack_mask(const TreeParams& p, const TreeUnit& u, uint32_t* words, int tid,
                                          int nthreads) {
  const int lane = tid & 63, W = mask_stride(p.T), chunks = (p.T + 63) / 64;
  const int n0 = u.row0 / u.G, nn = (u.row0 + u.nrows - 1) / u.G - n0 + 1;
  const uint8_t* mask = p.mask + u.b * p.mask_sb + static_cast<int64_t>(n0) * p.T;
  const int waves = nthreads >> 6;
  for (int i0 = tid >> 6; i0 < nn * chunks; i0 += 4 * waves) {
    uint8_t byte[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {  // four loads on their way at a time
      const int i = i0 + x * waves, n = i / chunks, col = 64 * (i - n * chunks) + lane;
      byte[x] = i < nn * chunks && col < p.T ? mask[n * p.T + col] : 0;
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int i = i0 + x * waves, n = i / chunks, c = i - n * chunks;
      const uint64_t bits = __ballot(byte[x] != 0);
      if (lane == 0 && i < nn * chunks) {
        words[n * W + 2 * c] = static_cast<uint32_t>(bits);
        words[n * W + 2 * c + 1] = static_cast<uint32_t>(bits >> 32);
        if (c == chunks - 1) words[n * W + 2 * chunks] = 0;
      }
    }
  }
}

// Keys key0 .. key0 + 31 that a node sees, as bits; j0 = key0 - base < T.
__device__ __forceinline__ uint32_t mask_window(const uint32_t* row, int j0) {
  if (j0 <= -32) return 0xffffffffu;
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

// All ones where bit `i` of win is set, else 0.
__device__ __forceinline__ uint32_t seen_mask(uint32_t win, int i) {
  return static_cast<uint32_t>(static_cast<int32_t>(win << (31 - i)) >> 31);
}
// Bit of accumulator entry r in a window shifted by 4 hh (crow()).
__device__ __forceinline__ constexpr int bit_of(int r) { return 8 * (r >> 2) + (r & 3); }

// The sign bit of each half of a word that holds an infinity or NaN: adding one
// to an exponent of all ones carries into it.
template <typename T>
__device__ __forceinline__ uint32_t not_finite(uint32_t two) {
  constexpr uint32_t E = __is_same(T, __bf16) ? 0x7f807f80u : 0x7c007c00u;
  constexpr uint32_t ONE = __is_same(T, __bf16) ? 0x00800080u : 0x04000400u;
  return ((two & E) + ONE) & 0x80008000u;
}

// A masked row's p is 0, and 0 times an infinity or NaN is not: such values of a
// block of V (32 rows at vat) become 0 in LDS, and `bad` there tells
// add_not_finite() to add them where they are seen.  Waves that share the block
// write the same.
template <typename T, int D>
__device__ __forceinline__ void clear_not_finite(uint32_t vat, int lane, int* bad) {
#pragma unroll 1
  for (int i = 0; i < RowTile<D>::PIECES; ++i) {
    auto at = (__attribute__((address_space(3))) u32x4*)(uintptr_t)(vat + RowTile<D>::off(i) + lane * 16);
    u32x4 w = *at;
    uint32_t any = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t f = not_finite<T>(w[e]);
      any |= f;
      w[e] &= ~(f | (f - (f >> 15)));
    }
    if (any) {
      *at = w;
      *bad = 1;
    }
  }
}

// q.k of the wave's 32 rows and a block of 32 keys at kat.
template <typename T, int D>
__device__ __forceinline__ f32x16 tree_scores(const RowTileK<D>& rk, uint32_t kat, const RowGroup<T, D>& st) {
  f32x16 s = f32x16{};
#pragma unroll
  for (int ds = 0; ds < D / 16; ++ds) s = mfma32(rk.template read<typename Vec8<T>::type>(kat, ds), st.q[ds], s);
  return s;
}

// One tile of 32 keys for the wave's 32 rows: transform of its scores, softmax
// update and the product with its block of V at vat.  MASKED: win holds the keys
// that the lane's row sees, shifted by 4 hh.
template <typename T, int D, bool NPOS, bool MASKED>
__device__ __forceinline__ void tree_tile(f32x16 s, const RowTileV<D>& rv, uint32_t vat, RowGroup<T, D>& st,
                                          uint32_t win, float c, float n) {
  typedef typename Vec8<T>::type v8;
  typedef T v4 __attribute__((ext_vector_type(4)));
  constexpr int ND32 = D / 32;
  constexpr uint32_t kOut = NPOS ? 0xff800000u : 0x7f800000u;  // the score of the lowest t: -inf or +inf
  v8 pb[2];
  bool done = false;
  if constexpr (!MASKED) {
    // a row that has seen nothing yet starts from an exponent of 0: then its sum
    // has to be large enough as well
    const bool fresh = st.m == -INFINITY;
    const float ref = fresh ? -kTreeLift<T> : st.m;
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float x = s[r];
      const float pv = fast_exp2(fmaf(n, copysignf(fast_log2(fmaf(c, fabsf(x), 1.f)), x), -ref));
      sum += pv;
      pb[r >> 3][r & 7] = static_cast<T>(pv);
    }
    done = __all(sum <= kTreeSum<T> && (!fresh || sum >= kTreeFirst<T>));
    if (done) {
      st.m = ref;
      st.l += sum;
    }
  }
  if (__builtin_expect(!done, MASKED)) {
    float z = -INFINITY;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float x = s[r];
      pin(x);  // nothing of this branch is computed before it
      if constexpr (MASKED) {
        const uint32_t in = seen_mask(win, bit_of(r));
        x = __uint_as_float((__float_as_uint(x) & in) | (kOut & ~in));
      }
      s[r] = x;
      z = fmaxf(z, NPOS ? x : -x);
    }
    z = pair_max(z);
    const float top = NPOS ? z : -z;
    const float tmax = z == -INFINITY ? -INFINITY : n * copysignf(fast_log2(fmaf(c, fabsf(top), 1.f)), top);
    const float mnew = fmaxf(st.m, tmax - kTreeLift<T>);
    const float alpha = fast_exp2(mnew == -INFINITY ? 0.f : st.m - mnew);
    st.m = mnew;
#pragma unroll
    for (int d = 0; d < ND32; ++d) st.acc[d] *= alpha;
    float l = st.l * alpha;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float x = s[r];
      float pv = fast_exp2(fmaf(n, copysignf(fast_log2(fmaf(c, fabsf(x), 1.f)), x), -mnew));
      if constexpr (MASKED) pv = __uint_as_float(__float_as_uint(pv) & seen_mask(win, bit_of(r)));
      l += pv;
      pb[r >> 3][r & 7] = static_cast<T>(pv);
    }
    st.l = l;
  }
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
    for (int db = 0; db < ND32; ++db) {
      const v4 lo = rv.template read<v4>(vat, ks, 0, db), hi = rv.template read<v4>(vat, ks, 1, db);
      st.acc[db] = mfma32(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7), pb[ks], st.acc[db]);
    }
  }
}

// The infinities and NaN that clear_not_finite() took out of the tree's rows of V, added
// to the rows that see them: the wave's tiles from key0 on, every `step` keys.
template <typename T, int D>
__device__ __forceinline__ void add_not_finite(const TreeParams& p, const TreeUnit& u, const uint32_t* mrow, int key0,
                                               int step, int hh, f32x16* acc) {
  typedef T v4 __attribute__((ext_vector_type(4)));
#pragma unroll 1
  for (int k0 = key0; k0 < u.kend; k0 += step) {
    if (!u.masked(k0)) continue;
    const uint32_t win = mask_window(mrow, k0 - u.base);
#pragma unroll 1
    for (int k = 0; k < 32; ++k) {
      if (k0 + k >= u.kend) break;
      const bool seen = win >> k & 1;
      const T* row = reinterpret_cast<const T*>(u.vg) + (k0 + k) * p.v.ss + 4 * hh;
#pragma unroll
      for (int j = 0; j < D / 8; ++j) {
        const v4 x = *reinterpret_cast<const v4*>(row + 8 * j);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v = static_cast<float>(x[e]);
          acc[j / 4][4 * (j % 4) + e] += seen && !(fabsf(v) < INFINITY) ? v : 0.f;
        }
      }
    }
  }
}

template <typename T, int D, bool NPOS, int QW, int KW>
__device__ __forceinline__ void tree_body(const TreeParams& p, char* smem, uint32_t* words, int* bad,
                                          const TreeUnit& u) {
  using C = TreeCfg<D, QW, KW>;
  typedef T v4 __attribute__((ext_vector_type(4)));
  constexpr int NW = C::NW;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int qw = wave / KW, kw = wave - qw * KW;
  const int l32 = lane & 31, hh = lane >> 5;
  const RowLoad<D, true> lk(lane, p.k.ss);
  const RowLoad<D, false> lv(lane, p.v.ss);
  const uint32_t lds0 = lds_addr(smem);
  const int nst = (u.kend - u.kbeg + C::KEYS - 1) / C::KEYS;
  auto issue = [&](int i) {
    tree_load_stage<D, QW, KW>(p, u, i, lds0, wave, lane, lk, lv);
  };
  if (nst > 0) issue(0);
  const float n = u.n, c = u.c;
  RowGroup<T, D> st;
  const int row = 32 * qw + l32;
  st.init(p, u, row, hh);
  const bool reaches = nst > 0 && u.kend > u.base;
  if (reaches) pack_mask(p, u, words, tid, NW * 64);
  if (tid == 0) *bad = 0;
  const uint32_t* mrow =
      words + ((u.row0 + min(row, u.nrows - 1)) / u.G - u.row0 / u.G) * mask_stride(p.T);
  const bool works = 32 * qw < u.nrows;
  const RowTileK<D> rk(l32, hh);
  const RowTileV<D> rv(lane);
  // stages of keys that every row sees, then the rest in a loop of its own (what
  // only that needs stays out of the first one's registers)
  const int open = min(u.base, u.kend) - u.kbeg;
  const int plain = open > 0 ? open / C::KEYS : 0;
  auto arrive = [&](int i) {
    wait_vm<0>();     // this wave's share of stage i has landed
    __syncthreads();  // and everyone's; everyone is done with the other buffer
    if (i + 1 < nst) issue(i + 1);
  };
  int i = 0;
  for (; i < plain; ++i) {
    arrive(i);
    if (!works) continue;
    const uint32_t kat = lds0 + (i & 1) * 2 * C::TILE + kw * RowTile<D>::BLOCK;
    const auto scores = [&](int t) { return tree_scores(rk, kat + KW * t * RowTile<D>::BLOCK, st); };
    const auto rest = [&](const f32x16& s, int t) {
      tree_tile<T, D, NPOS, false>(s, rv, kat + C::TILE + KW * t * RowTile<D>::BLOCK, st, 0, c, n);
    };
    if constexpr (C::U == 2 && D != 64) {
      // the second tile's scores are on the matrix cores while the first's go
      // through the transform (at D = 64 that would not fit 128 registers)
      const f32x16 s0 = scores(0), s1 = scores(1);
      rest(s0, 0);
      rest(s1, 1);
    } else {
#pragma unroll
      for (int t = 0; t < C::U; ++t) rest(scores(t), t);
    }
  }
#pragma unroll 1
  for (; i < nst; ++i) {
    arrive(i);
    if (!works) continue;
#pragma unroll 1
    for (int t = 0; t < C::U; ++t) {
      const int key0 = u.kbeg + C::KEYS * i + 32 * (kw + KW * t);
      if (key0 >= u.kend) break;
      const uint32_t kat = lds0 + (i & 1) * 2 * C::TILE + (kw + KW * t) * RowTile<D>::BLOCK, vat = kat + C::TILE;
      uint32_t win = 0xffffffffu;
      if (u.masked(key0)) {
        win = mask_window(mrow, key0 - u.base);
        clear_not_finite<T, D>(vat, lane, bad);
      }
      tree_tile<T, D, NPOS, true>(tree_scores(rk, kat, st), rv, vat, st, win >> (4 * hh), c, n);
    }
  }
  if (reaches) {
    __syncthreads();  // every wave's tiles have been looked at
    if (__builtin_expect(*bad != 0, 0))
      add_not_finite<T, D>(p, u, mrow, u.kbeg + 32 * kw, 32 * KW, hh, st.acc);
  }
  float m = st.m, l = st.l;
  // Each key wave takes a share of the columns: it scales its acc to the common
  // maximum, hands the others theirs through LDS and adds up its own, the key
  // waves in order.
  constexpr int J = C::J, JB = C::JB;
  f32x4_t mine[JB];
  const int j0 = kw * JB;  // its float4s of a lane's acc; none where there are more waves than float4s
  if constexpr (KW > 1) {
    f32x4_t* accs = reinterpret_cast<f32x4_t*>(smem);
    float* ml = reinterpret_cast<float*>(words);
    __syncthreads();  // the stages and masks have been read
    ml[(2 * wave) * 64 + lane] = m;
    ml[(2 * wave + 1) * 64 + lane] = l;
    __syncthreads();
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < KW; ++w) M = fmaxf(M, ml[(2 * (qw * KW + w)) * 64 + lane]);
    const float ref = M == -INFINITY ? 0.f : M;
    l = 0.f;
#pragma unroll
    for (int w = 0; w < KW; ++w)
      l += ml[(2 * (qw * KW + w) + 1) * 64 + lane] * fast_exp2(ml[(2 * (qw * KW + w)) * 64 + lane] - ref);
    const float f = fast_exp2(m - ref);
    m = M;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int owner = j / JB;
      f32x4_t x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = st.acc[j / 4][4 * (j % 4) + e] * f;
      if (kw != owner)
        accs[((qw * J + j) * (KW - 1) + kw - (kw > owner ? 1 : 0)) * 64 + lane] = x;
      else
        mine[j % JB] = x;
    }
    __syncthreads();
    if (j0 >= J) return;
#pragma unroll
    for (int j = 0; j < JB; ++j) {
      f32x4_t sum = f32x4_t{};
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        if (w == kw)
          sum += mine[j];
        else
          sum += accs[((qw * J + j0 + j) * (KW - 1) + w - (w > kw ? 1 : 0)) * 64 + lane];
      }
      mine[j] = sum;
    }
  } else {
#pragma unroll
    for (int j = 0; j < JB; ++j) {
#pragma unroll
      for (int e = 0; e < 4; ++e) mine[j][e] = st.acc[j / 4][4 * (j % 4) + e];
    }
  }
  l = pair_sum(l);
  if (row >= u.nrows) return;
  const RowOut o(p, u, row);
  if (p.splits == 1) {
    const float l_safe = l == 0.f ? 1.f : l;
    const float inv = 1.f / l_safe;
    T* dst = static_cast<T*>(const_cast<void*>(p.o.ptr)) + o.off + 8 * j0 + 4 * hh;
#pragma unroll
    for (int j = 0; j < JB; ++j) {
      v4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = static_cast<T>(mine[j][e] * inv);
      *reinterpret_cast<v4*>(dst + 8 * j) = x;
    }
    if (kw == 0 && hh == 0 && p.m != nullptr) p.m[o.mrow] = m + log2f(l_safe);
  } else {
    float* dst = p.ws_acc + o.rec * D + 8 * j0 + 4 * hh;
#pragma unroll
    for (int j = 0; j < JB; ++j) *reinterpret_cast<f32x4_t*>(dst + 8 * j) = mine[j];
    if (kw == 0 && hh == 0) {
      p.ws_ml[2 * o.rec] = m;
      p.ws_ml[2 * o.rec + 1] = l;
    }
  }
}

}  // namespace

template <typename T, int D, int QW, int KW>
__global__ __launch_bounds__(QW* KW * 64) void tree_kernel(TreeParams p, int nunits, int nqb) {
  __shared__ __attribute__((aligned(1024))) char smem[TreeCfg<D, QW, KW>::SMEM];
  __shared__ uint32_t words[TreeCfg<D, QW, KW>::WORDS];  // packed masks; later the key waves' m and l
  __shared__ int bad;  // the tree's rows of V held an infinity or NaN
  const int block = folded_block();
  if (block >= nunits) return;
  const TreeUnit u(p, block, 32 * QW, nqb);
  if (p.splits > 1 && u.kend <= u.kbeg) return;  // a shorter sequence: nothing to merge
  if (u.n >= 0.f)
    tree_body<T, D, true, QW, KW>(p, smem, words, &bad, u);
  else
    tree_body<T, D, false, QW, KW>(p, smem, words, &bad, u);
}

// The splits' partials of a row in split order: out = sum_s acc_s 2^(m_s - M) /
// sum_s l_s 2^(m_s - M).  D / 4 threads a row, four columns each, and SW such
// groups that take every SW-th split and meet in LDS; every load is independent
// of the running state.  A launch and two dependent loads: 3.8 us for 128 rows of 8
// splits, 5.9 for 2048 of 32 (17 MB).  SW = 4 pays from more than 8 splits on (32
// splits of 128 rows x 64, the whole call: 14.7 us, SW = 1 16.2; 8 splits: 13.5 and
// 12.6).
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
  const int ns = tree_own_splits(p, b);
  const int64_t rec0 = static_cast<int64_t>(row) * p.splits;
  const float* ml = p.ws_ml + 2 * rec0;
  // the row's lanes of a wave take a split each for the maximum and the sum
  constexpr int LANES = TPR * SW < 64 ? TPR * SW : 64;
  const int at = tid % LANES;
  float M = -INFINITY;
  for (int s = at; s < ns; s += LANES) M = fmaxf(M, ml[2 * s]);
#pragma unroll
  for (int off = LANES / 2; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor(M, off, 64));
  const float ref = M == -INFINITY ? 0.f : M;
  float Ls = 0.f;
  for (int s = at; s < ns; s += LANES) Ls += ml[2 * s + 1] * fast_exp2(ml[2 * s] - ref);
#pragma unroll
  for (int off = LANES / 2; off > 0; off >>= 1) Ls += __shfl_xor(Ls, off, 64);
  f32x4_t O = f32x4_t{};
#pragma unroll 8
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
  const int nqb = static_cast<int>((rows + p.rows - 1) / p.rows);
  const int units = static_cast<int>(static_cast<int64_t>(p.B) * p.Hkv * nqb * p.splits);
  const auto go = [&](auto kernel, int threads) {
    hipLaunchKernelGGL(kernel, folded_grid(units, threads), dim3(threads), 0, s, p, units, nqb);
  };
  constexpr int W = D == 128 ? 8 : 16;  // waves of a workgroup: 128 KB of LDS, 128 or 256 registers
  if (p.rows == 32)
    go(tree_kernel<T, D, 1, W / 2>, W / 2 * 64);
  else if (p.rows == 64)
    go(tree_kernel<T, D, 2, W / 2>, W * 64);
  else if (p.rows == 128)
    go(tree_kernel<T, D, 4, W / 4>, W * 64);
  else if (p.rows == 256)
    go(tree_kernel<T, D, 8, W / 8>, W * 64);
  else
    return hipErrorInvalidValue;
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
