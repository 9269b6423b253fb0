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
// workgroup 1024 E: a cache of up to that many rows is read once and its keys
// stay in registers for every pass, a longer one is read by each.  Rows that
// stay in any case rank above every weight and rows past the length below or
// with the lowest, where the lower row wins.
template <int E>
__global__ __launch_bounds__(kSelect) void evict_select_kernel(EvictParams p, int nblocks) {
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
  constexpr int STRETCH = kSelect * E;
  const int mine = wave * 64 * E + 4 * lane;  // the lane's first row of a stretch; then every 256th
  const int lo = p.sinks, hi = L - p.recent;  // rows [lo, hi) are chosen from
  uint32_t key[E];
  auto load = [&](int r0) {
#pragma unroll
    for (int j = 0; j < E / 4; ++j) {
      const int i = r0 + mine + 256 * j;
      f32x4_u x = {0.f, 0.f, 0.f, 0.f};
      if (i + 3 < L) {
        x = *reinterpret_cast<const f32x4_u*>(w + i);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (i + e < L) x[e] = w[i + e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t k = order_bits(x[e]);
        key[4 * j + e] = i + e >= L ? 0u : (i + e < lo || i + e >= hi) ? 0xffffffffu : k;
      }
    }
  };
  const bool once = L <= STRETCH;
  if (once) load(0);
  for (int i = p.keep + tid; i < p.cap; i += kSelect) w_out[i] = 0.f;
  uint32_t need = p.keep;  // rows that stay, of those that share the prefix
  uint32_t prefix = 0;
  constexpr int kShift[3] = {20, 10, 0}, kWidth[3] = {12, 10, 10};
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int bins = 1 << kWidth[pass];
    for (int i = tid; i < bins; i += kSelect) hist[i] = 0;
    __syncthreads();
    for (int r0 = 0; r0 < L; r0 += STRETCH) {
      if (!once) load(r0);
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (pass == 0 || (key[j] >> (kShift[pass] + kWidth[pass])) == prefix)
          atomicAdd(&hist[(key[j] >> kShift[pass]) & (bins - 1)], 1u);
    }
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
  const uint32_t ties = need;  // rows at the threshold that stay, the lowest first
  uint32_t above0 = 0, at0 = 0;  // rows before this stretch above the threshold; at it
  for (int r0 = 0; r0 < L; r0 += STRETCH) {
    if (!once) load(r0);
    // the wave's counts: above in the low half, at the threshold in the high
    uint32_t up = 0, eq = 0;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      up += key[j] > prefix;
      eq += key[j] == prefix;
    }
    // a wave's 64 E rows are at most 2^11, a workgroup's at most 2^15: no carry
    uint32_t total, before_waves = 0;
    {
      const uint32_t sum = wave_scan(up | (eq << 16));
      __syncthreads();
      if (lane == 63) waves[wave] = sum;
      __syncthreads();
      total = 0;
#pragma unroll
      for (int x = 0; x < kSelect / 64; ++x) {
        before_waves += x < wave ? waves[x] : 0;
        total += waves[x];
      }
    }
#pragma unroll
    for (int j = 0; j < E / 4; ++j) {
      uint32_t count = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) count += (key[4 * j + e] > prefix) + ((key[4 * j + e] == prefix) << 16);
      const uint32_t upto = wave_scan(count);
      uint32_t before = before_waves + upto - count;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool over = key[4 * j + e] > prefix, even = key[4 * j + e] == prefix;
        const uint32_t at = at0 + (before >> 16), place = above0 + (before & 0xffffu) + (at < ties ? at : ties);
        if (over || (even && at < ties)) {
          const int i = r0 + mine + 256 * j + e;
          kept[place] = i;
          w_out[place] = w[i];
        }
        before += over + (even << 16);
      }
      before_waves += __builtin_amdgcn_readlane(upto, 63);
    }
    above0 += total & 0xffffu;
    at0 += total >> 16;
  }
}

// One workgroup per (tensor, sequence, kv-head, slice of SP 16-byte pieces of a
// row), the slices of a head on one XCD.  The next chunk's rows are on their way
// while this one's are written.
template <int SP>
__global__ __launch_bounds__(1024) void evict_move_kernel(EvictParams p, int slices, int nblocks) {
  constexpr int U = 4, ROWS = 1024 / SP;  // rows of one step, U steps a chunk
  const int block = folded_block();
  if (block >= nblocks) return;
  const int units = nblocks / slices;
  const int slice = block / units;
  int u = block - slice * units;
  const Tensor4& t = (u & 1) ? p.v : p.k;
  u >>= 1;
  const int h = u % p.Hkv, b = u / p.Hkv;
  const int L = clamped_len(p.seqlens, b, p.cap);
  if (L <= p.keep) return;
  const int* kept = p.kept + static_cast<int64_t>(u) * p.keep;
  const int tid = threadIdx.x, piece = slice * SP + tid % SP, row = tid / SP;
  char* base = static_cast<char*>(const_cast<void*>(t.ptr)) + (b * t.sb + h * t.sh) * 2 + piece * 16;
  const int64_t step = t.ss * 2;
  u32x4 v[U], next[U];
  int src[U];
  auto index = [&](int r0) {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int r = r0 + j * ROWS + row;
      src[j] = r < p.keep ? kept[r] : r;
    }
  };
  auto fetch = [&](u32x4 (&to)[U], int r0) {
#pragma unroll
    for (int j = 0; j < U; ++j)
      if (src[j] != r0 + j * ROWS + row) to[j] = *reinterpret_cast<const u32x4*>(base + src[j] * step);
  };
  index(0);
  fetch(v, 0);
  for (int r0 = 0; r0 < p.keep; r0 += U * ROWS) {
    bool moves[U];
#pragma unroll
    for (int j = 0; j < U; ++j) moves[j] = src[j] != r0 + j * ROWS + row;
    const bool more = r0 + U * ROWS < p.keep;
    if (more) index(r0 + U * ROWS);
    __builtin_amdgcn_s_waitcnt(0);  // the chunk's rows are in registers ...
    __syncthreads();                // ... everywhere
    if (more) fetch(next, r0 + U * ROWS);
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
// may be in any order.
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
  else
    hipLaunchKernelGGL(evict_select_kernel<32>, grid, dim3(kSelect), 0, s, p, heads);
  const auto move = [&](auto kernel, int sp) {
    const int slices = p.D / 8 / sp;
    const int blocks = heads * 2 * slices;
    hipLaunchKernelGGL(kernel, folded_grid(blocks, 1024), dim3(1024), 0, s, p, slices, blocks);
  };
  if (heads * 2 * (p.D / 32) < 256)
    move(evict_move_kernel<2>, 2);
  else
    move(evict_move_kernel<4>, 4);
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
