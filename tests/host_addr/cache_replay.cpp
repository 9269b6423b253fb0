// Replays, on the CPU, the global-memory plans of the cache operators' streaming
// kernels (csrc/ssa_cache_plan.hpp, with the tiles of ssa_row_tile.hpp and
// ssa_tile.hpp) for every workgroup, wave and lane of a problem, in every form the
// kernels are built in.  Each direct-to-LDS load is performed on exact-size
// host buffers (AddressSanitizer sees any stray byte, UndefinedBehaviorSanitizer any
// overflow of the offset arithmetic); every 8 bytes of a cache hold a tag of their
// own (tensor, sequence, head, row, columns).  Checked:
//
//  * the grid's workgroups cover every (sequence, kv-head, rows, split), or
//    (sequence, kv-head, keys, chunk of rows), exactly once;
//  * after a stage's loads every operand address that the kernel's lanes read
//    holds the row and columns the lane means, rows past the end the last one, and
//    no LDS byte outside the stage's buffer was written;
//  * buffer-descriptor offsets stay inside the descriptor's range;
//  * what the joining kernel reads of the workspace was written once, inside the
//    size the plan reports: the splits of a sequence's own rows, the chunks of
//    rows that see a key.
#include <cinttypes>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <memory>
#include <set>
#include <string>
#include <tuple>
#include <vector>

#include "ssa_cache_plan.hpp"

using namespace ssa;

namespace {

long g_checks = 0, g_fail = 0;
std::string g_ctx;

void failf(const char* fmt, ...) {
  if (g_fail++ < 25) {
    va_list ap;
    va_start(ap, fmt);
    fprintf(stderr, "FAIL [%s] ", g_ctx.c_str());
    vfprintf(stderr, fmt, ap);
    fputc('\n', stderr);
    va_end(ap);
  }
}
#define CHECK(cond, ...)             \
  do {                               \
    ++g_checks;                      \
    if (!(cond)) failf(__VA_ARGS__); \
  } while (0)

std::string fmt(const char* f, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, f);
  vsnprintf(buf, sizeof buf, f, ap);
  va_end(ap);
  return buf;
}

uint64_t tag(int which, int b, int h, int row, int col) {
  return (static_cast<uint64_t>(which) << 60) | (static_cast<uint64_t>(b) << 48) | (static_cast<uint64_t>(h) << 36) |
         (static_cast<uint64_t>(row) << 12) | static_cast<uint64_t>(col);
}

// A [B, H, N, D] tensor of 2-byte elements, contiguous or [B, N, H, D] in memory,
// tagged; its last byte is its buffer's last.
struct Tagged {
  int B, H, N, D;
  int64_t sb, sh, ss;
  std::unique_ptr<char[]> mem;
  Tagged(int which, int B_, int H_, int N_, int D_, bool rows_outside) : B(B_), H(H_), N(N_), D(D_) {
    if (rows_outside)
      sh = D, ss = static_cast<int64_t>(H) * D, sb = ss * N;
    else
      ss = D, sh = static_cast<int64_t>(N) * D, sb = sh * H;
    mem.reset(new char[static_cast<size_t>(B) * H * N * D * 2]);
    for (int b = 0; b < B; ++b)
      for (int h = 0; h < H; ++h)
        for (int r = 0; r < N; ++r)
          for (int c = 0; c < D; c += 4) {
            const uint64_t t = tag(which, b, h, r, c);
            memcpy(mem.get() + (b * sb + h * sh + r * ss + c) * 2, &t, 8);
          }
  }
  Tensor4 t4() const { return Tensor4{mem.get(), sb, sh, ss}; }
};

std::vector<uint8_t> g_lds, g_written;
int g_lane = 0;

void lds_store(uint32_t l, const char* p, size_t bytes) {
  CHECK(l + bytes <= g_lds.size(), "LDS byte %u + %zu past the allocation of %zu", l, bytes, g_lds.size());
  if (l + bytes > g_lds.size()) return;
  memcpy(g_lds.data() + l, p, bytes);
  for (size_t i = 0; i < bytes; ++i) {
    CHECK(!g_written[l + i], "LDS byte %zu written twice in one stage", l + i);
    g_written[l + i] = 1;
  }
}

struct HostMem {
  void load16(uint32_t lds, const i32x4_t& rs, uint32_t voff, int soff) const {
    CHECK(soff >= 0 && rs[2] == 0x7fffffff, "scalar offset %d", soff);
    const uint64_t off = static_cast<uint64_t>(voff) + static_cast<uint32_t>(soff);
    CHECK(off + 16 <= 0x7fffffffull, "buffer offset %" PRIu64 " past the descriptor's range", off);
    const uint64_t a = static_cast<uint32_t>(rs[0]) | (static_cast<uint64_t>(static_cast<uint32_t>(rs[1]) & 0xffffu) << 32);
    lds_store(lds + 16 * g_lane, reinterpret_cast<const char*>(a) + off, 16);
  }
  void load16_global(uint32_t lds, const void* src) const {
    lds_store(lds + 16 * g_lane, static_cast<const char*>(src), 16);
  }
};

void expect(uint32_t at, uint64_t want, const char* what, int row, int col) {
  uint64_t got = 0;
  CHECK(at + 8 <= g_lds.size(), "%s row %d column %d read at LDS byte %u", what, row, col, at);
  if (at + 8 > g_lds.size()) return;
  memcpy(&got, g_lds.data() + at, 8);
  CHECK(got == want && g_written[at] && g_written[at + 7], "%s row %d column %d at LDS byte %u: %016" PRIx64 ", want %016" PRIx64,
        what, row, col, at, got, want);
}

void fresh_stage() { std::fill(g_written.begin(), g_written.end(), 0); }

// Nothing outside [from, to) written.
void inside(uint32_t from, uint32_t to) {
  for (uint32_t i = 0; i < g_written.size(); ++i)
    if (g_written[i]) CHECK(i >= from && i < to, "LDS byte %u written outside the stage's buffer [%u, %u)", i, from, to);
}

// ---------------------------------------------------------------------------
struct TreeCase {
  int B, Hq, Hkv, cap, T, splits;
  std::vector<int> lens;
  bool rows_outside;
};

template <int D, int QW, int KW>
void run_tree(const TreeCase& c) {
  using C = TreeCfg<D, QW, KW>;
  const Tagged k(1, c.B, c.Hkv, c.cap, D, c.rows_outside), v(2, c.B, c.Hkv, c.cap, D, c.rows_outside);
  const float one = 1.f;
  TreeParams p{};
  p.k = k.t4(), p.v = v.t4();
  p.o = Tensor4{nullptr, static_cast<int64_t>(c.Hq) * c.T * D, static_cast<int64_t>(c.T) * D, D};
  p.seqlens = c.lens.data();
  p.n_ptr = p.b_ptr = &one;
  p.B = c.B, p.Hq = c.Hq, p.Hkv = c.Hkv, p.cap = c.cap, p.T = c.T;
  p.rows = 32 * QW;
  // as many splits as asked for, whole steps of keys each
  const int steps = (c.cap + kTreeStep - 1) / kTreeStep, per = (steps + c.splits - 1) / c.splits;
  p.split_keys = per * kTreeStep;
  p.splits = (c.cap + p.split_keys - 1) / p.split_keys;
  const int G = c.Hq / c.Hkv, nqb = (G * c.T + p.rows - 1) / p.rows;
  const int units = c.B * c.Hkv * nqb * p.splits;
  const int64_t recs = static_cast<int64_t>(c.B) * c.Hq * c.T * p.splits;
  std::vector<uint8_t> partial(recs, 0), result(static_cast<size_t>(c.B) * c.Hq * c.T, 0);
  std::set<std::tuple<int, int, int, int>> seen;
  g_lds.assign(C::SMEM, 0);
  g_written.assign(C::SMEM, 0);
  for (int block = 0; block < units; ++block) {
    const TreeUnit u(p, block, p.rows, nqb);
    g_ctx = fmt("tree D=%d QW=%d KW=%d B=%d Hq=%d Hkv=%d cap=%d T=%d block %d (b %d hk %d row0 %d split %d)", D, QW, KW,
                c.B, c.Hq, c.Hkv, c.cap, c.T, block, u.b, u.hk, u.row0, u.split);
    CHECK(seen.insert({u.b, u.hk, u.row0, u.split}).second, "unit dispatched twice");
    CHECK(u.b >= 0 && u.b < c.B && u.hk >= 0 && u.hk < c.Hkv && u.nrows > 0 && u.row0 + u.nrows <= G * c.T, "unit out of range");
    const int L = clamped_length(c.lens[u.b], c.cap);
    CHECK(u.kbeg >= 0 && u.kend <= L && u.kend - u.kbeg <= p.split_keys && u.kbeg <= u.kend, "keys %d .. %d of %d",
          u.kbeg, u.kend, L);
    CHECK(u.n == 1.f && u.base == L - c.T, "scalars");
    // the mask's rows of the unit fit the packed words
    const int nodes = (u.row0 + u.nrows - 1) / G - u.row0 / G + 1;
    CHECK(nodes * mask_stride(c.T) <= C::WORDS, "%d mask rows of %d words past %d", nodes, mask_stride(c.T), C::WORDS);
    if (u.kend > u.base && u.kend > u.kbeg)  // the last tile's window of the mask
      CHECK(((u.kend - 1 - u.base) >> 5) + 1 < mask_stride(c.T), "mask window past its row");
    const int nst = (u.kend - u.kbeg + C::KEYS - 1) / C::KEYS;
    for (int i = 0; i < nst; ++i) {
      fresh_stage();
      for (int w = 0; w < C::NW; ++w)
        for (g_lane = 0; g_lane < 64; ++g_lane) {
          const RowLoad<D, true> lk(g_lane, p.k.ss);
          const RowLoad<D, false> lv(g_lane, p.v.ss);
          tree_load_stage<D, QW, KW>(p, u, i, 0u, w, g_lane, lk, lv, HostMem());
        }
      const uint32_t buf = (i & 1) * 2 * C::TILE;
      inside(buf, buf + 2 * C::TILE);
      // every operand address of every lane
      for (int blk = 0; blk < C::BLOCKS; ++blk) {
        const int key0 = u.kbeg + C::KEYS * i + 32 * blk;
        const uint32_t kat = buf + blk * RowTile<D>::BLOCK, vat = kat + C::TILE;
        for (int lane = 0; lane < 64; ++lane) {
          const int l32 = lane & 31, hh = lane >> 5, g = lane >> 4, x = lane & 15;
          const RowTileK<D> rk(l32, hh);
          const RowTileV<D> rv(lane);
          const int krow = key0 + l32 < u.kend ? key0 + l32 : u.kend - 1;
          for (int ds = 0; ds < D / 16; ++ds)
            for (int half = 0; half < 2; ++half)
              expect(rk.address(kat, ds) + 8 * half, tag(1, u.b, u.hk, krow, 16 * ds + 8 * hh + 4 * half), "K", krow, ds);
          for (int ks = 0; ks < 2; ++ks)
            for (int hi = 0; hi < 2; ++hi)
              for (int db = 0; db < D / 32; ++db) {
                const int r = key0 + 16 * ks + 8 * hi + 4 * hh + x / 4, vrow = r < u.kend ? r : u.kend - 1;
                expect(rv.address(vat, ks, hi, db), tag(2, u.b, u.hk, vrow, 32 * db + 16 * (g & 1) + 4 * (x & 3)), "V", vrow,
                       db);
              }
        }
      }
    }
    if (p.splits > 1 && u.kend <= u.kbeg) continue;
    for (int row = 0; row < u.nrows; ++row) {
      const RowOut o(p, u, row);
      CHECK(o.rec >= 0 && o.rec < recs && o.mrow >= 0 && o.mrow < static_cast<int64_t>(result.size()), "row %d out of range", row);
      CHECK(o.off == o.mrow * D, "row %d: element %" PRId64 " of the result, row %" PRId64, row, o.off, o.mrow);
      if (o.rec < 0 || o.rec >= recs) continue;
      CHECK(!partial[o.rec], "partial %" PRId64 " written twice", o.rec);
      partial[o.rec] = 1;
      if (u.split == 0) result[o.mrow] = 1;
    }
  }
  CHECK(static_cast<int>(seen.size()) == units, "%zu units of %d", seen.size(), units);
  // the merge's rows in order, each with the splits of its sequence
  for (int b = 0; b < c.B; ++b) {
    const int ns = tree_own_splits(p, b);
    CHECK(ns <= p.splits, "%d splits of %d", ns, p.splits);
    for (int64_t row = static_cast<int64_t>(b) * c.Hq * c.T; row < static_cast<int64_t>(b + 1) * c.Hq * c.T; ++row)
      for (int s = 0; s < p.splits; ++s)
        CHECK(partial[row * p.splits + s] == (s < ns || p.splits == 1), "row %" PRId64 " split %d of %d", row, s, ns);
  }
}

template <int D>
void run_tree_forms(const TreeCase& c) {
  constexpr int W = D == 128 ? 8 : 16;
  run_tree<D, 1, W / 2>(c);
  run_tree<D, 2, W / 2>(c);
  run_tree<D, 4, W / 4>(c);
  run_tree<D, 8, W / 8>(c);
}

// ---------------------------------------------------------------------------
struct WeightsCase {
  int B, Hq, Hkv, cap, T;
  std::vector<int> lens;
  bool rows_outside;
};

template <int D, int RW>
void run_weights(const WeightsCase& c, bool chunks) {
  constexpr int KW = kWeightsKeys / 32;
  using C = WeightsCfg<D, KW, RW>;
  const Tagged q(3, c.B, c.Hq, c.T, D, c.rows_outside);
  KeyWeightsParams p{};
  p.q = q.t4();
  p.seqlens = c.lens.data();
  p.B = c.B, p.Hq = c.Hq, p.Hkv = c.Hkv, p.cap = c.cap, p.T = c.T;
  const int G = c.Hq / c.Hkv, rows = G * c.T, nbh = c.B * c.Hkv;
  p.chunks = chunks ? weights_chunks(c.B, c.Hq, c.Hkv, c.cap, c.T) : 1;
  p.chunk_rows = chunks ? weights_chunk_rows(c.B, c.Hq, c.Hkv, c.cap, c.T) : (rows + kWeightsStage - 1) / kWeightsStage * kWeightsStage;
  const int ntiles = (c.cap + C::KEYS - 1) / C::KEYS, blocks = nbh * ntiles * p.chunks;
  std::vector<uint8_t> written(static_cast<size_t>(p.chunks) * nbh * c.cap, 0);
  std::vector<int> seen(static_cast<size_t>(nbh) * ntiles, 0);  // rows of the unit's chunks
  g_lds.assign(2 * C::QB, 0);
  g_written.assign(2 * C::QB, 0);
  for (int block = 0; block < blocks; ++block) {
    const WeightsUnit u(p, block, ntiles, C::KEYS, C::ROWS);
    g_ctx = fmt("weights D=%d RW=%d B=%d Hq=%d Hkv=%d cap=%d T=%d chunks=%d block %d (b %d hk %d key0 %d chunk %d)", D, RW,
                c.B, c.Hq, c.Hkv, c.cap, c.T, p.chunks, block, u.b, u.hk, u.key0, u.chunk);
    CHECK(u.bh == u.b * c.Hkv + u.hk && u.b < c.B && u.chunk < p.chunks && u.key0 < c.cap, "unit out of range");
    if (u.behind() || u.unseen()) continue;
    CHECK(u.rstart % C::ROWS == 0 || u.rstart == u.chunk * p.chunk_rows, "first row %d", u.rstart);
    seen[static_cast<size_t>(u.bh) * ntiles + u.key0 / C::KEYS] += u.R - u.rstart;
    const int nst = (u.R - u.rstart + C::ROWS - 1) / C::ROWS;
    for (int i = 0; i < nst; ++i) {
      fresh_stage();
      for (int w = 0; w < C::NW; ++w) {
        const int kw = w / RW, rw = w - kw * RW;
        for (g_lane = 0; g_lane < 64; ++g_lane) {
          WeightsRows<D, KW, RW> lane(p, u, g_lane, kw, rw);
          for (int x = 0; x < i; ++x) lane.next(u);
          const int r = u.rstart + i * C::ROWS + 32 * rw + lane.ll.r;
          const auto as = lane.row(p, u);
          CHECK(as.in == (r < rows), "row %d of %d", r, rows);
          if (r < rows) CHECK(as.t == r / G && as.g == r % G, "row %d as query %d head %d", r, as.t, as.g);
          lane.load(p, as, weights_queries(p, u), i, 0u, kw, rw, HostMem());
        }
      }
      const uint32_t buf = (i & 1) * C::QB;
      inside(buf, buf + C::QB);
      for (int rw = 0; rw < RW; ++rw)
        for (int l32 = 0; l32 < 32; ++l32) {
          const int r0 = u.rstart + i * C::ROWS + 32 * rw + l32, r = r0 < rows ? r0 : rows - 1;
          for (int ch = 0; ch < D / 8; ++ch)
            for (int half = 0; half < 2; ++half)
              // chunk-major blocks of ssa_tile.hpp: chunk c of row r at position r ^ 4 (c & 3)
              expect(buf + rw * BlockLayout<D>::BLOCK + ch * 512 + ((l32 ^ (4 * (ch & 3))) << 4) + 8 * half,
                     tag(3, u.b, u.hk * G + r % G, r / G, 8 * ch + 4 * half), "Q", r, ch);
        }
    }
    for (int e = 0; e < C::KEYS && u.key0 + e < u.L; ++e) {
      const int64_t at = weights_slot(p, u.chunk, u.bh, u.key0 + e);
      CHECK(at >= 0 && at < static_cast<int64_t>(written.size()) && !written[at], "sum %" PRId64 " written twice or outside", at);
      if (at >= 0 && at < static_cast<int64_t>(written.size())) written[at] = 1;
    }
  }
  for (int bh = 0; bh < nbh; ++bh) {
    const int L = clamped_length(c.lens[bh / c.Hkv], c.cap), first = L - c.T;
    for (int key = 0; key < L; ++key) {
      // the rows that see the key are in the tile's chunks
      const int sees = first_row(key, first, G), got = seen[static_cast<size_t>(bh) * ntiles + key / C::KEYS];
      CHECK(got >= rows - sees, "key %d: %d rows of %d looked at", key, got, rows - sees);
      for (int ch = chunks ? weights_first_chunk(p, L, key) : 0; ch < p.chunks; ++ch)
        CHECK(written[weights_slot(p, ch, bh, key)] || (!chunks && sees >= rows), "head %d key %d: chunk %d was not written", bh, key, ch);
    }
  }
}

template <int D>
void run_weights_forms(const WeightsCase& c) {
  run_weights<D, 1>(c, false);
  run_weights<D, 2>(c, false);
  if (weights_chunks(c.B, c.Hq, c.Hkv, c.cap, c.T) > 1) run_weights<D, kWeightsStage / 32>(c, true);
}

}  // namespace

int main(int argc, char** argv) {
  const bool quick = argc > 1 && strcmp(argv[1], "--quick") == 0;
  const std::vector<TreeCase> trees = {
      {1, 4, 4, 64, 1, 1, {64}, false},
      {2, 8, 2, 700, 13, 3, {700, 45}, true},
      {4, 6, 2, 300, 61, 1, {0, 300, 61, 1000}, false},
      {3, 3, 1, 1030, 130, 2, {1030, -3, 129}, true},
      {2, 2, 1, 2304, 5, 9, {2304, 700}, false},
      {1, 2, 2, 1100, 1024, 2, {1100}, false},
  };
  const std::vector<WeightsCase> weights = {
      {2, 8, 2, 300, 1, {300, 130}, false},
      {1, 33, 1, 200, 1, {200}, true},
      {4, 6, 2, 128, 20, {0, 7, 20, 500}, false},
      {2, 4, 4, 260, 260, {260, 260}, true},
      {1, 24, 8, 390, 333, {390}, false},
      {1, 8, 1, 1280, 150, {1250}, false},    // chunks of rows
      {1, 32, 1, 640, 100, {640}, true},
      {2, 7, 1, 513, 500, {513, 499}, false},
  };
  for (size_t i = 0; i < trees.size(); ++i) {
    const long f0 = g_fail;
    run_tree_forms<64>(trees[i]);
    if (!quick || i < 4) run_tree_forms<32>(trees[i]), run_tree_forms<128>(trees[i]);
    printf("tree %zu %s\n", i, g_fail == f0 ? "ok" : "FAILED");
    fflush(stdout);
  }
  for (size_t i = 0; i < weights.size(); ++i) {
    const long f0 = g_fail;
    run_weights_forms<64>(weights[i]);
    if (!quick) run_weights_forms<32>(weights[i]), run_weights_forms<128>(weights[i]);
    printf("weights %zu %s\n", i, g_fail == f0 ? "ok" : "FAILED");
    fflush(stdout);
  }
  printf("%ld checks, %ld failures\n", g_checks, g_fail);
  return g_fail == 0 ? 0 : 1;
}
