// Rows of a KV cache moved in place: eviction by weight and the acceptance of a
// drafted path, for gfx950.
//
// Eviction keeps `keep` rows of each (sequence, kv-head).  evict_select_kernel
// finds the weight of the last row that stays by a radix selection over the
// weights' bits in an order-preserving form (three histograms of 12, 10 and 10
// bits), then writes the kept rows' indices and weights in ascending order: a
// row's place is the number of rows before it that stay, that is of rows above
// the threshold plus the smaller of the rows at it and the number of those that
// stay, so one scan of two counts places everything.  evict_move_kernel moves
// the rows.  In place and in order: place i's row comes from kept[i] >= i, and
// chunk by chunk every source is read before the chunk's places are written;
// a later chunk's sources lie behind every place written so far.
//
// What they take (bf16, the kernels alone): 8 x 8 heads x 4096 x 64 cut to 2048 rows,
// selection 6 to 7 us and moves 10 to 11 (67 MB read and written, 6 to 6.5 TB/s);
// 1 x 16 x 32768 x 128 cut to 4096, 24 and 16.  The selection is bound by the latency of its steps (three
// passes over registers, each with two scans and five barriers) on one CU a head, and by
// the scalar registers that its unrolled loops over the keys keep in vector registers (65
// of the 16-key form, 169 of the 32-key one, 202 with a second stretch, none of the 4-key one), the
// moves by their bytes where they fill the GPU and by the dependent chunks of a
// slice where they do not.
#include "ssa_cache_ops.hpp"
#include "ssa_common.hpp"
#include "ssa_launch.hpp"

namespace ssa {

namespace {

constexpr int kSelect = 1024;  // threads of a selection
constexpr int kBins = 4096;

typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));

// Unsigned order of weights: NaN below everything, -0 equal to +0.
__device__ __forceinline__ uint32_t order_bits(float w) {
  if (w != w) return 0;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u >> 31) ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int clamped_len(const int* lens, int b, int cap) {
  const int L = load_table_entry(lens, b);
  return L < 0 ? 0 : (L > cap ? cap : L);
}

// Inclusive sum over the wave's lanes.
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
  // within rows of 16 lanes, then each row's last lane into the next row(s)
#define SSA_DPP(ctrl, rows) x += __builtin_amdgcn_update_dpp(0u, x, ctrl, rows, 0xf, false)
  SSA_DPP(0x111, 0xf);  // row_shr:1
  SSA_DPP(0x112, 0xf);  // row_shr:2
  SSA_DPP(0x114, 0xf);  // row_shr:4
  SSA_DPP(0x118, 0xf);  // row_shr:8
  SSA_DPP(0x142, 0xa);  // row_bcast:15
  SSA_DPP(0x143, 0xc);  // row_bcast:31
#undef SSA_DPP
  return x;
}

// Inclusive sum over the workgroup's threads (kSelect of them); `waves` holds
// one value per wave.  Two barriers.
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t* waves, int tid, uint32_t& total) {
  const int lane = tid & 63, wave = tid >> 6;
  x = wave_scan(x);
  __syncthreads();  // the last scan's values have been read
  if (lane == 63) waves[wave] = x;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSelect / 64; ++w) {
    const uint32_t v = waves[w];
    before += w < wave ? v : 0;
    all += v;
  }
  total = all;
  return x + before;
}

}  // namespace

// A wave takes 64 E consecutive rows, four consecutive ones a lane at a time, a
// workgroup a stretch of 1024 E.  The first stretch's keys stay in registers for
// every pass, with kFar the second's in LDS; a cache longer than that (65536 rows
// at E = 32) is read by every pass from there on.  Rows that stay in any case rank
// above every weight, rows past the length with the lowest, where the lower row
// wins.
//
// E is the least that holds the capacity in registers, up to 32: more lengthens
// every step, less reads the weights again in every pass (whole calls: 8 x 8 x
// 1024 x 64, E = 4 10.4 us, 16 15.0, 32 18.7; 16384 rows, E = 16 26.9, 4 30.1, 32
// 31.5; 1 x 16 x 32768, E = 32 35, 16 40, 4 44; at 8192 rows E = 4 would be 7 %
// faster than 16).  E = 64 was slower than 32; the
// second stretch in LDS takes 65536 rows from 63 to 55 us.  Rows that stay in any case are
// left out of the histograms, and 256 rows past the length at once: their lanes
// would add to one bin, 78 us for 28 with 6451 such rows of 32972.
template <int E, bool kFar = false>
__global__ __launch_bounds__(kSelect) void evict_select_kernel(EvictParams p, int nblocks) {
  constexpr int STRETCH = kSelect * E;
  constexpr uint32_t kMust = 0xffffffffu;
  __shared__ __attribute__((aligned(16))) uint32_t far[kFar ? STRETCH : 4];
  __shared__ uint32_t hist[kBins];
  __shared__ uint32_t waves[kSelect / 64];
  __shared__ uint32_t found[2];  // digit, rows above it
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, block = folded_block();
  if (block >= nblocks) return;
  const int b = block / p.Hkv, h = block - b * p.Hkv;
  const int L = clamped_len(p.seqlens, b, p.cap);
  const float* w = p.w + b * p.w_sb + h * p.w_sh;
  const int64_t bh = block;
  float* w_out = p.w_out + bh * p.cap;
  int* kept = p.kept + bh * p.keep;
  if (h == 0 && tid == 0) p.lens_out[b] = min(L, p.keep);
  if (L <= p.keep) {
    for (int i = tid; i < p.cap; i += kSelect) w_out[i] = i < L ? w[i] : 0.f;
    for (int i = tid; i < p.keep; i += kSelect) kept[i] = i < L ? i : -1;
    return;
  }
  const int mine = wave * 64 * E + 4 * lane;  // the lane's first row of a stretch; then every 256th
  const int lo = p.sinks, hi = L - p.recent;  // rows [lo, hi) are chosen from
  const int stretches = (L - 1) / STRETCH + 1;
  auto load = [&](int i, uint32_t* k) {  // the keys of rows i .. i + 3
    f32x4_u x = {0.f, 0.f, 0.f, 0.f};
    if (i + 3 < L) {
      x = *reinterpret_cast<const f32x4_u*>(w + i);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < L) x[e] = w[i + e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) k[e] = i + e >= L ? 0u : (i + e < lo || i + e >= hi) ? kMust : order_bits(x[e]);
  };
  uint32_t key[E];
#pragma unroll
  for (int j = 0; j < E / 4; ++j) load(mine + 256 * j, key + 4 * j);
  u32x4* far4 = reinterpret_cast<u32x4*>(far);
  if (kFar && stretches > 1) {
#pragma unroll 4
    for (int j = 0; j < E / 4; ++j) {
      uint32_t k[4];
      load(STRETCH + mine + 256 * j, k);
      far4[kSelect * j + tid] = u32x4{k[0], k[1], k[2], k[3]};  // read by this thread only
    }
  }
  // f(first of four rows, their keys) for the lane's rows of stretch s, in order;
  // not for 256 rows past the length (a histogram's lowest bin would take them
  // one by one)
  const int wave0 = __builtin_amdgcn_readfirstlane(wave * 64 * E);
  auto each = [&](int s, auto&& f) {
    if (s == 0) {
#pragma unroll
      for (int j = 0; j < E / 4; ++j)
        if (wave0 + 256 * j < L) f(mine + 256 * j, key + 4 * j);
    } else {
      const int r0 = s * STRETCH + mine;  // below 2^30 + 2^15
#pragma unroll 2
      for (int j = 0; j < E / 4; ++j) {
        if (s * STRETCH + wave0 + 256 * j >= L) break;
        uint32_t k[4];
        if (kFar && s == 1) {
          const u32x4 v = far4[kSelect * j + tid];
#pragma unroll
          for (int e = 0; e < 4; ++e) k[e] = v[e];
        } else {
          load(r0 + 256 * j, k);
        }
        f(r0 + 256 * j, k);
      }
    }
  };
  uint32_t need = p.keep - p.sinks - p.recent;  // rows that stay, of those that share the prefix
  uint32_t prefix = 0;
  if (need == 0) {
    prefix = kMust;
    need = p.keep;
  } else {
    constexpr int kShift[3] = {20, 10, 0}, kWidth[3] = {12, 10, 10};
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      const int bins = 1 << kWidth[pass];
      for (int i = tid; i < bins; i += kSelect) hist[i] = 0;
      __syncthreads();
      for (int s = 0; s < stretches; ++s)
        each(s, [&](int, const uint32_t* k) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (k[e] != kMust && (pass == 0 || (k[e] >> (kShift[pass] + kWidth[pass])) == prefix))
              atomicAdd(&hist[(k[e] >> kShift[pass]) & (bins - 1)], 1u);
        });
      __syncthreads();
      // bins from the top: thread i takes `per` bins downwards from the i-th group
      const int per = bins / kSelect;
      uint32_t sum = 0;
      for (int x = 0; x < per; ++x) sum += hist[bins - 1 - per * tid - x];
      uint32_t total;
      const uint32_t upto = block_scan(sum, waves, tid, total);
      uint32_t above = upto - sum;
      if (above < need && upto >= need) {
        int bin = bins - 1 - per * tid;
        while (above + hist[bin] < need) above += hist[bin--];
        found[0] = bin;
        found[1] = above;
      }
      __syncthreads();
      prefix = (prefix << kWidth[pass]) | found[0];
      need -= found[1];
    }
  }
  const uint32_t ties = need;  // rows at the threshold that stay, the lowest first
  uint32_t above0 = 0, at0 = 0;  // rows before this stretch above the threshold; at it
  for (int s = 0; s < stretches; ++s) {
    // the wave's counts: above in the low half, at the threshold in the high
    uint32_t both = 0;
    each(s, [&](int, const uint32_t* k) {
#pragma unroll
      for (int e = 0; e < 4; ++e) both += (k[e] > prefix) + ((k[e] == prefix) << 16);
    });
    // a wave's 64 E rows are at most 2^11, a workgroup's at most 2^15: no carry
    uint32_t total = 0, before_waves = 0;
    const uint32_t sum = wave_scan(both);
    __syncthreads();
    if (lane == 63) waves[wave] = sum;
    __syncthreads();
#pragma unroll
    for (int x = 0; x < kSelect / 64; ++x) {
      before_waves += x < wave ? waves[x] : 0;
      total += waves[x];
    }
    each(s, [&](int i, const uint32_t* k) {
      uint32_t count = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) count += (k[e] > prefix) + ((k[e] == prefix) << 16);
      const uint32_t upto = wave_scan(count);
      uint32_t before = before_waves + upto - count;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool over = k[e] > prefix, even = k[e] == prefix;
        const uint32_t at = at0 + (before >> 16), place = above0 + (before & 0xffffu) + (at < ties ? at : ties);
        if (over || (even && at < ties)) kept[place] = i + e;
        before += over + (even << 16);
      }
      before_waves += __builtin_amdgcn_readlane(upto, 63);
    });
    above0 += total & 0xffffu;
    at0 += total >> 16;
  }
  // behind the kept rows' weights, which evict_move_kernel gathers
  const int n4 = (p.cap - p.keep) / 4;
  for (int i = tid; i < n4; i += kSelect)
    *reinterpret_cast<f32x4_u*>(w_out + p.keep + 4 * static_cast<int64_t>(i)) = f32x4_u{0.f, 0.f, 0.f, 0.f};
  if (tid < (p.cap - p.keep) % 4) w_out[p.keep + 4 * static_cast<int64_t>(n4) + tid] = 0.f;
}

// One workgroup per (sequence, kv-head) that gathers the kept rows' weights, then
// one per (tensor, sequence, kv-head, slice of SP 16-byte pieces of a row), the
// slices of a head on one XCD.  The next chunk's rows are on their way while
// this one's are written.  16 waves a slice, since a chunk is one round trip to
// memory: 1024 rows of 64 bytes a chunk.
template <int SP, int U>
__global__ __launch_bounds__(1024) void evict_move_kernel(EvictParams p, int slices, int nblocks) {
  constexpr int ROWS = 1024 / SP, CHUNK = U * ROWS;  // rows of one step, U steps a chunk
  const int heads = p.B * p.Hkv, tid = threadIdx.x;
  int block = folded_block();
  if (block >= nblocks) return;
  const bool weighs = block < heads;
  block -= heads;
  const int units = 2 * heads, slice = weighs ? 0 : block / units;
  int u = weighs ? block + heads : block - slice * units;
  const bool is_v = u & 1;
  if (!weighs) u >>= 1;
  const int h = u % p.Hkv, b = u / p.Hkv;
  if (clamped_len(p.seqlens, b, p.cap) <= p.keep) return;
  const int* kept = p.kept + static_cast<int64_t>(u) * p.keep;
  if (weighs) {
    const float* w = p.w + b * p.w_sb + h * p.w_sh;
    float* w_out = p.w_out + static_cast<int64_t>(u) * p.cap;
    for (int64_t r0 = tid; r0 < p.keep; r0 += 8 * 1024) {
      int src[8];
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) src[j] = kept[r0 + 1024 * j < p.keep ? r0 + 1024 * j : p.keep - 1];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = w[src[j]];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (r0 + 1024 * j < p.keep) w_out[r0 + 1024 * j] = x[j];
    }
    return;
  }
  const Tensor4& t = is_v ? p.v : p.k;
  const int piece = slice * SP + tid % SP, row = tid / SP;
  char* base = static_cast<char*>(const_cast<void*>(t.ptr)) + (b * t.sb + h * t.sh) * 2 + piece * 16;
  const int64_t step = t.ss * 2;
  // kept[r] - r never falls: a chunk whose last row stays in place stays whole
  int r0 = 0;
  while (r0 < p.keep) {
    const int last = (p.keep - r0 < CHUNK ? p.keep : r0 + CHUNK) - 1;
    if (load_table_entry(kept, last) != last) break;
    r0 = last + 1;
  }
  u32x4 v[U], next[U];
  int src[U];
  auto index = [&](int at) {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int r = at + j * ROWS + row;
      src[j] = r < p.keep ? kept[r] : r;
    }
  };
  auto fetch = [&](u32x4 (&to)[U], int at) {
#pragma unroll
    for (int j = 0; j < U; ++j)
      if (src[j] != at + j * ROWS + row) to[j] = *reinterpret_cast<const u32x4*>(base + src[j] * step);
  };
  if (r0 >= p.keep) return;
  index(r0);
  fetch(v, r0);
  for (; r0 < p.keep; r0 += CHUNK) {  // below 2^30 + CHUNK
    bool moves[U];
#pragma unroll
    for (int j = 0; j < U; ++j) moves[j] = src[j] != r0 + j * ROWS + row;
    const bool more = p.keep - r0 > CHUNK;
    if (more) index(r0 + CHUNK);
    __builtin_amdgcn_s_waitcnt(0);  // the chunk's rows are in registers ...
    __syncthreads();                // ... everywhere
    if (more) fetch(next, r0 + CHUNK);
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int r = r0 + j * ROWS + row;
      if (moves[j]) *reinterpret_cast<u32x4*>(base + r * step) = v[j];
      v[j] = next[j];
    }
  }
}

// One workgroup per (tensor, sequence, kv-head, slice of `sp` pieces): all
// depth * sp <= 1024 pieces are read before the first is written, so the path
// may be in any order.  2.8 us for 1 x 16 x 128, 4 rows, and 3.7 for 64 x 8 x 64, 16
// rows (4 MB): a launch and three dependent loads, of which the shortest launch
// takes 2.4.
__global__ __launch_bounds__(256) void accept_kernel(AcceptParams p, int sp, int slices, int nblocks) {
  const int block = folded_block();
  if (block >= nblocks) return;
  int u = block;
  const int slice = u % slices;
  u /= slices;
  const bool is_v = u & 1;
  const Tensor4& t = is_v ? p.v : p.k;
  u >>= 1;
  const int h = u % p.Hkv, b = u / p.Hkv;
  const int L = clamped_len(p.seqlens, b, p.cap);
  const int first = L - p.T;
  int n = load_table_entry(p.accepted, b);
  n = first < 0 ? 0 : (n < 0 ? 0 : (n > p.depth ? p.depth : n));
  if (threadIdx.x == 0 && slice == 0 && !is_v && h == 0) p.lens_out[b] = first < 0 ? L : first + n;
  if (n == 0) return;
  const int pieces = p.D / 8;
  char* base = static_cast<char*>(const_cast<void*>(t.ptr)) + (b * t.sb + h * t.sh) * 2;
  u32x4 v[4];
  int64_t to[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int e = threadIdx.x + 256 * j, i = e / sp, piece = slice * sp + e - i * sp;
    to[j] = -1;
    if (i < n && piece < pieces) {
      int node = p.path[static_cast<int64_t>(b) * p.depth + i];
      node = node < 0 ? 0 : (node >= p.T ? p.T - 1 : node);
      if (node != i) {
        to[j] = (first + i) * t.ss * 2 + piece * 16;
        v[j] = *reinterpret_cast<const u32x4*>(base + (first + node) * t.ss * 2 + piece * 16);
      }
    }
  }
  __builtin_amdgcn_s_waitcnt(0);  // the rows are in registers ...
  __syncthreads();                // ... everywhere
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (to[j] >= 0) *reinterpret_cast<u32x4*>(base + to[j]) = v[j];
}

hipError_t launch_evict(const EvictParams& p, hipStream_t s) {
  const int heads = p.B * p.Hkv;
  const dim3 grid = folded_grid(heads, kSelect);
  if (p.cap <= 4 * kSelect)
    hipLaunchKernelGGL(evict_select_kernel<4>, grid, dim3(kSelect), 0, s, p, heads);
  else if (p.cap <= 16 * kSelect)
    hipLaunchKernelGGL(evict_select_kernel<16>, grid, dim3(kSelect), 0, s, p, heads);
  else if (p.cap <= 32 * kSelect)
    hipLaunchKernelGGL(evict_select_kernel<32>, grid, dim3(kSelect), 0, s, p, heads);
  else
    hipLaunchKernelGGL((evict_select_kernel<32, true>), grid, dim3(kSelect), 0, s, p, heads);
  // 64-byte slices move at the rate of a copy where they fill the GPU (512 and 1152
  // workgroups; slices of 32 bytes take 1.7 times as long); up to 128 workgroups
  // half the slice on twice as many is 20 to 25 % shorter
  const auto move = [&](auto kernel, int sp) {
    const int slices = p.D / 8 / sp, blocks = heads * (1 + 2 * slices);
    hipLaunchKernelGGL(kernel, folded_grid(blocks, 1024), dim3(1024), 0, s, p, slices, blocks);
  };
  if (heads * 2 * (p.D / 32) <= 128)
    move(evict_move_kernel<2, 8>, 2);
  else
    move(evict_move_kernel<4, 4>, 4);
  return hipGetLastError();
}

hipError_t launch_accept(const AcceptParams& p, hipStream_t s) {
  const int pieces = p.D / 8;
  const int most = 1024 / p.depth;  // >= 1: depth <= 1024
  const int sp = pieces < most ? pieces : most;
  const int slices = (pieces + sp - 1) / sp;
  const int blocks = p.B * p.Hkv * 2 * slices;
  hipLaunchKernelGGL(accept_kernel, folded_grid(blocks, 256), dim3(256), 0, s, p, sp, slices, blocks);
  return hipGetLastError();
}

}  // namespace ssa
