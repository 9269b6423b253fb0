// The attention that query rows paid to cached keys, added to the keys'
// weights, for gfx950:
//   w_j += sum over rows r that see key j of p_rj,  p_rj = 2^(t_rj - m_r),
//   t_rj = n sign(s) log2(1 + scale b |s|),  s = q_r . k_j
// with the rows' normalisers m given, so one pass over the rows suffices and
// nothing but the scores' products is needed: S = Q K^T (A = 32 rows of Q from
// LDS, B = 32 keys in registers), whose result holds one key per lane pair and
// 16 rows in each lane's registers.  A key's sum over the rows stays in its
// lanes from the first row to the last (fp32, fixed order, no atomics).
//
// The G heads of a group and their T queries are rows r = t * G + head, so the
// causal mask only bounds the first row of a workgroup's keys and the rows
// near it.  A workgroup is KW key waves of 32 keys by RW row waves of 32 rows; Q
// rows pass through LDS in stages of 32 RW rows, two in flight.  Many rows are
// split over workgroups in chunks, whose sums a second kernel adds up in their
// order.
//
// With few rows the stream of K is the bound: 16 x 32/8 heads x 4096 x 64, 2048 to
// 4096 rows a sequence, with one query takes 15.7 us for 53.5 MB (K, the weights in and out;
// 3.4 TB/s, a copy 4.8), 4 x 16 x 8192 x 128 with 32 queries 23.5 for 104 MB (4.4).
// K goes straight to registers, 32 keys a wave and once, so the waves of a CU
// (20 at D = 64) are what keeps loads on their way; a wave that has its scores has none
// in flight.  With many it is the transform, one log2 and one exp2 a pair, 768 cycles
// for 32 x 32 pairs on one SIMD, and the part of the product (128 cycles at D = 64) that is
// not beside it, half by the counters: 1 x 32/8 x 4096 x 64 with 4096 queries takes
// 108.5 us, 4 of them the join, and the transforms alone 93 to 96 at the 2.1 GHz
// that the GPU holds then.  Two groups of 32 keys a wave, so that an operand read
// from LDS serves two products, took as long there (106 and 107 us) and 1.1 to 1.4
// times as long at D = 128, where their registers halve the waves of a SIMD.
#include "ssa_cache_plan.hpp"
#include "ssa_common.hpp"
#include "ssa_launch.hpp"

namespace ssa {

template <typename T, int D, int KW, int RW>
__global__ __launch_bounds__(KW* RW * 64) void key_weights_kernel(KeyWeightsParams p, int ntiles, int nblocks) {
  using C = WeightsCfg<D, KW, RW>;
  typedef typename Vec8<T>::type v8;
  constexpr int ND16 = D / 16;
  static_assert(KW % 2 == 0, "one piece parity per wave");
  __shared__ __attribute__((aligned(1024))) char qs[2 * C::QB];
  __shared__ __attribute__((aligned(16))) float ms[2][C::ROWS];  // m of the stage's rows
  __shared__ __attribute__((aligned(16))) int ps[2][C::ROWS];    // and their positions; -1: adds nothing
  __shared__ int odd[2][RW];  // a row of the block adds nothing
  __shared__ float part[C::NW][32];

  const int block = folded_block();
  if (block >= nblocks) return;
  const WeightsUnit u(p, block, ntiles, C::KEYS, C::ROWS);
  if (u.behind() || u.unseen()) return;
  const int b = u.b, hk = u.hk, L = u.L, key0 = u.key0, G = u.G, first = u.first, rstart = u.rstart, R = u.R;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kw = wave / RW, rw = wave - kw * RW;
  const int l32 = lane & 31, hh = lane >> 5;
  const float n = *p.n_ptr, c = p.scale * *p.b_ptr;
  const int kbase = key0 + 32 * kw;  // this wave's keys

  const int nst = (R - rstart + C::ROWS - 1) / C::ROWS;
  // rows of whole blocks that see every key of the wave
  const int rall = first_row(kbase + 31, first, G);

  WeightsRows<D, KW, RW> rows(p, u, lane, kw, rw);
  const char* qbase = weights_queries(p, u);
  const float* mbase = p.m + (static_cast<int64_t>(b) * p.Hq + hk * G) * p.T;
  const uint32_t lds0 = lds_addr(qs);
  float mv = 0.f;
  int pv = -1;
  auto issue = [&](int i) {
    const auto r = rows.row(p, u);
    rows.load(p, r, qbase, i, lds0, kw, rw);
    if (kw == 0 && hh == 0) {
      mv = mbase[static_cast<int64_t>(r.g) * p.T + r.t];
      // chunks end with a stage, so a row past R is past the last query
      pv = r.in && mv != -INFINITY ? first + r.t : -1;
    }
    rows.next(u);
  };
  issue(0);

  v8 kf[ND16];
  const int key = kbase + l32;  // this lane's
  {
    const T* src = static_cast<const T*>(p.k.ptr) + b * p.k.sb + hk * p.k.sh + min(key, L - 1) * p.k.ss + 8 * hh;
#pragma unroll
    for (int ds = 0; ds < ND16; ++ds) kf[ds] = load16<v8>(src + ds * 16);
  }
  float sum = 0.f;
  const RowBase<D> rb(l32, hh);

  for (int i = 0; i < nst; ++i) {
    if (kw == 0) {
      if (hh == 0) {
        ms[i & 1][32 * rw + rows.ll.r] = mv;
        ps[i & 1][32 * rw + rows.ll.r] = pv;
      }
      const bool any = __any(hh == 0 && pv < 0);
      if (lane == 0) odd[i & 1][rw] = any;
    }
    wait_vm<0>();     // this wave's share of the stage has landed
    __syncthreads();  // and everyone's; everyone is done with the other buffers
    if (i + 1 < nst) issue(i + 1);
    const int row0 = rstart + i * C::ROWS + 32 * rw;
    if (row0 >= R) continue;
    const RowBase<D> qr = at_tile(rb, lds0 + (i & 1) * C::QB + rw * BlockLayout<D>::BLOCK);
    f32x16 s = f32x16{};
#pragma unroll
    for (int ds = 0; ds < ND16; ++ds) s = mfma32(tile_read_row<D, v8>(qr, 0, ds), kf[ds], s);
    // every row of the block sees every key of the wave, but near the diagonal
    const bool all = row0 >= rall && !odd[i & 1][rw];
    if (all) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x4_t m4 = *reinterpret_cast<const f32x4_t*>(&ms[i & 1][32 * rw + 8 * j + 4 * hh]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = s[4 * j + e];
          sum += fast_exp2(fmaf(n, copysignf(fast_log2(fmaf(c, fabsf(x), 1.f)), x), -m4[e]));
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float m = ms[i & 1][32 * rw + 8 * j + 4 * hh + e];
          const int pos = ps[i & 1][32 * rw + 8 * j + 4 * hh + e];
          const float x = s[4 * j + e];
          const float pr = fast_exp2(fmaf(n, copysignf(fast_log2(fmaf(c, fabsf(x), 1.f)), x), -m));
          sum += pos >= key ? pr : 0.f;
        }
      }
    }
  }
  const float both = pair_sum(sum);
  if (hh == 0) part[wave][l32] = both;
  __syncthreads();
  float* w = p.chunks == 1 ? p.w + b * p.w_sb + hk * p.w_sh
                           : p.ws + weights_slot(p, u.chunk, u.bh, 0);
  for (int e = tid; e < C::KEYS; e += C::NW * 64) {
    const int at = key0 + e;
    if (at >= L) break;
    float total = 0.f;
#pragma unroll
    for (int r = 0; r < RW; ++r) total += part[e / 32 * RW + r][e % 32];
    w[at] = p.chunks == 1 ? w[at] + total : total;
  }
}

// The chunks' sums of each key, in order: a stream of [chunks][keys] floats, 4.2 us
// for 8 chunks of 32768 keys, as long as a launch takes.
__global__ __launch_bounds__(256) void key_weights_join_kernel(KeyWeightsParams p, int blocks_per_head, int nblocks) {
  const int block = folded_block();
  if (block >= nblocks) return;
  const int bh = block / blocks_per_head, key = (block - bh * blocks_per_head) * 256 + threadIdx.x;
  const int b = bh / p.Hkv, hk = bh - b * p.Hkv;
  const int L = clamped_length(load_table_entry(p.seqlens, b), p.cap);
  if (key >= L) return;
  float total = 0.f;
  for (int c = weights_first_chunk(p, L, key); c < p.chunks; ++c) total += p.ws[weights_slot(p, c, bh, key)];
  p.w[b * p.w_sb + hk * p.w_sh + key] += total;
}

namespace {

template <typename T, int D, int KW, int RW>
hipError_t launch_weights(const KeyWeightsParams& p, hipStream_t s) {
  using C = WeightsCfg<D, KW, RW>;
  const int ntiles = (p.cap + C::KEYS - 1) / C::KEYS;
  const int heads = p.B * p.Hkv;
  const int blocks = heads * ntiles * p.chunks;
  hipLaunchKernelGGL((key_weights_kernel<T, D, KW, RW>), folded_grid(blocks, C::NW * 64), dim3(C::NW * 64), 0, s,
                     p, ntiles, blocks);
  if (p.chunks > 1) {
    if (C::KEYS != kWeightsKeys || C::ROWS != kWeightsStage) return hipErrorInvalidValue;  // as the join counts them
    const int per = (p.cap + 255) / 256;
    hipLaunchKernelGGL(key_weights_join_kernel, folded_grid(heads * per, 256), dim3(256), 0, s, p, per, heads * per);
  }
  return hipGetLastError();
}

template <typename T, int D>
hipError_t launch_weights_t(const KeyWeightsParams& p, hipStream_t s) {
  const int64_t rows = static_cast<int64_t>(p.Hq / p.Hkv) * p.T;
  constexpr int KW = kWeightsKeys / 32;
  if (weights_one_wave(rows, weights_blocks(p.B, p.Hkv, p.cap))) return launch_weights<T, D, KW, 1>(p, s);
  return launch_weights<T, D, KW, kWeightsStage / 32>(p, s);
}

template <typename T>
hipError_t launch_weights_dt(const KeyWeightsParams& p, int D, hipStream_t s) {
  switch (D) {
    case 32: return launch_weights_t<T, 32>(p, s);
    case 64: return launch_weights_t<T, 64>(p, s);
    case 128: return launch_weights_t<T, 128>(p, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

hipError_t launch_key_weights(const KeyWeightsParams& p, int dtype, int D, hipStream_t stream) {
  if (dtype == 0) return launch_weights_dt<__bf16>(p, D, stream);
  return launch_weights_dt<_Float16>(p, D, stream);
}

}  // namespace ssa
