/*
 * Host-side validation of include/ssa_cache_ops.h under AddressSanitizer and
 * UndefinedBehaviorSanitizer (tests/test_host_cache_sanitize.py builds and runs it; no
 * GPU is needed).  Every entry point is called with NULL, with each integer field
 * at 0, -1, INT32_MIN, INT32_MAX and large sizes, alone and in pairs, and with
 * each stride negative, unaligned and huge; the size queries get the same extremes.
 * Calls that pass validation reach a kernel launch, which fails without a device:
 * what is checked is that validation, the plans and the launches' arithmetic have
 * no undefined behaviour for any arguments, and the status codes of known-bad
 * ones.  The pointers are fake, so the program refuses to run where a GPU is
 * visible.
 */
#include <stddef.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include "../../include/ssa_cache_ops.h"

#define FAKE ((void*)(uintptr_t)0x100000)
#define FAR ((void*)((uintptr_t)1 << 46))

/* HIP runtime (libamdhip64): hipError_t is an int-sized enum, hipSuccess = 0 */
int hipGetDeviceCount(int* count);

static int failures = 0;
static long calls = 0;

static void expect(int got, int want, const char* what) {
  if (got != want) {
    fprintf(stderr, "FAIL %s: status %d, expected %d\n", what, got, want);
    ++failures;
  }
}

static const int32_t kInts[] = {0, -1, 1, 7, INT32_MIN, INT32_MAX, 1 << 30, (1 << 30) + 1, 1 << 24, 1024, 1025};
static const int64_t kStrides[] = {-8, 0, 4, 8, INT64_MIN, INT64_MAX & ~(int64_t)7, (int64_t)1 << 24, (int64_t)1 << 40,
                                   (int64_t)1 << 61};
#define NI ((int)(sizeof(kInts) / sizeof(kInts[0])))
#define NS ((int)(sizeof(kStrides) / sizeof(kStrides[0])))

static ssa_tensor4 t4(void* at, int64_t heads, int64_t rows) {
  ssa_tensor4 t = {at, heads * rows * 64, rows * 64, 64};
  return t;
}

static ssa_tree_args base_tree(void) {
  ssa_tree_args a;
  memset(&a, 0, sizeof a);
  a.q = a.out = t4(FAKE, 8, 16);
  a.k_cache = t4(FAKE, 2, 4096), a.v_cache = t4(FAR, 2, 4096);
  a.m = (float*)FAKE;
  a.cache_seqlens = (const int32_t*)FAKE;
  a.tree_mask = (const uint8_t*)FAKE;
  a.ssa_n = a.ssa_b = (const float*)FAKE;
  a.batch = 2, a.heads_q = 8, a.heads_kv = 2, a.capacity = 4096, a.head_dim = 64;
  a.dtype = SSA_DTYPE_BF16, a.nodes = 16, a.softmax_scale = 0.125f, a.workspace = FAKE;
  return a;
}

static ssa_key_weights_args base_weights(void) {
  ssa_key_weights_args a;
  memset(&a, 0, sizeof a);
  a.q = t4(FAKE, 8, 16);
  a.k_cache = t4(FAKE, 2, 4096);
  a.m = (const float*)FAKE;
  a.weights = (float*)FAR;
  a.weights_stride_b = 2 * 4096, a.weights_stride_h = 4096;
  a.cache_seqlens = (const int32_t*)FAKE;
  a.ssa_n = a.ssa_b = (const float*)FAKE;
  a.batch = 2, a.heads_q = 8, a.heads_kv = 2, a.capacity = 4096, a.head_dim = 64;
  a.dtype = SSA_DTYPE_FP16, a.queries = 16, a.softmax_scale = 0.125f, a.workspace = FAKE;
  return a;
}

static ssa_cache_evict_args base_evict(void) {
  ssa_cache_evict_args a;
  memset(&a, 0, sizeof a);
  a.k_cache = t4(FAKE, 2, 4096), a.v_cache = t4(FAR, 2, 4096);
  a.weights = (const float*)FAKE;
  a.weights_stride_b = 2 * 4096, a.weights_stride_h = 4096;
  a.cache_seqlens = (const int32_t*)FAKE;
  a.seqlens_out = (int32_t*)FAR, a.weights_out = (float*)FAR, a.kept = (int32_t*)FAR;
  a.batch = 2, a.heads_kv = 2, a.capacity = 4096, a.head_dim = 64, a.dtype = SSA_DTYPE_BF16;
  a.keep = 1000, a.sinks = 4, a.recent = 64;
  return a;
}

static ssa_cache_accept_args base_accept(void) {
  ssa_cache_accept_args a;
  memset(&a, 0, sizeof a);
  a.k_cache = t4(FAKE, 2, 4096), a.v_cache = t4(FAR, 2, 4096);
  a.cache_seqlens = a.path = a.accepted = (const int32_t*)FAKE;
  a.seqlens_out = (int32_t*)FAR;
  a.batch = 2, a.heads_kv = 2, a.capacity = 4096, a.head_dim = 64, a.dtype = SSA_DTYPE_FP16;
  a.nodes = 16, a.depth = 5;
  return a;
}

static int32_t run_tree(const void* a) { return ssa_tree_attention((const ssa_tree_args*)a, NULL); }
static int32_t run_weights(const void* a) { return ssa_key_weights((const ssa_key_weights_args*)a, NULL); }
static int32_t run_evict(const void* a) { return ssa_cache_evict((const ssa_cache_evict_args*)a, NULL); }
static int32_t run_accept(const void* a) { return ssa_cache_accept((const ssa_cache_accept_args*)a, NULL); }

/* Every integer field and every pair of them, every stride field, of one entry point's arguments. */
static void sweep(const char* what, int32_t (*run)(const void*), const void* base, size_t size, const size_t* ints, int n,
                  const size_t* strides, int m) {
  unsigned char a[512];
  if (size > sizeof a) {
    fprintf(stderr, "FAIL %s: arguments of %zu bytes\n", what, size);
    ++failures;
    return;
  }
  expect(run(NULL), SSA_ERR_NULL_POINTER, what);
  for (int i = 0; i < n; ++i)
    for (int x = 0; x < NI; ++x)
      for (int j = i; j < n; ++j)
        for (int y = 0; y < (j == i ? 1 : NI); ++y, ++calls) {
          memcpy(a, base, size);
          if (j != i) memcpy(a + ints[j], &kInts[y], 4);
          memcpy(a + ints[i], &kInts[x], 4);
          const int32_t s = run(a);
          if (strcmp(ssa_status_string(s), ssa_status_string(INT32_MAX)) == 0) expect(s, SSA_OK, what); /* no status */
        }
  for (int i = 0; i < m; ++i)
    for (int x = 0; x < NS; ++x)
      for (int j = i; j < m; ++j)
        for (int y = 0; y < (j == i ? 1 : NS); ++y)
          for (int z = 0; z < NI; ++z, ++calls) { /* with one integer field too: products of sizes and strides */
            memcpy(a, base, size);
            if (j != i) memcpy(a + strides[j], &kStrides[y], 8);
            memcpy(a + strides[i], &kStrides[x], 8);
            memcpy(a + ints[(x + y + z) % n], &kInts[z], 4);
            run(a);
          }
}

#define OFF(type, field) offsetof(type, field)
#define STRIDES(type, field) OFF(type, field.stride_b), OFF(type, field.stride_h), OFF(type, field.stride_s)
#define COUNT(x) ((int)(sizeof(x) / sizeof((x)[0])))

static void sweep_entries(void) {
  {
    typedef ssa_tree_args T;
    const T base = base_tree();
    const size_t ints[] = {OFF(T, batch),    OFF(T, heads_q), OFF(T, heads_kv), OFF(T, capacity),
                           OFF(T, head_dim), OFF(T, dtype),   OFF(T, nodes),    OFF(T, num_splits)};
    const size_t strides[] = {STRIDES(T, q), STRIDES(T, k_cache), STRIDES(T, v_cache), STRIDES(T, out), OFF(T, mask_stride_b)};
    sweep("ssa_tree_attention", run_tree, &base, sizeof base, ints, COUNT(ints), strides, COUNT(strides));
  }
  {
    typedef ssa_key_weights_args T;
    const T base = base_weights();
    const size_t ints[] = {OFF(T, batch),    OFF(T, heads_q), OFF(T, heads_kv), OFF(T, capacity),
                           OFF(T, head_dim), OFF(T, dtype),   OFF(T, queries)};
    const size_t strides[] = {STRIDES(T, q), STRIDES(T, k_cache), OFF(T, weights_stride_b), OFF(T, weights_stride_h)};
    sweep("ssa_key_weights", run_weights, &base, sizeof base, ints, COUNT(ints), strides, COUNT(strides));
  }
  {
    typedef ssa_cache_evict_args T;
    const T base = base_evict();
    const size_t ints[] = {OFF(T, batch), OFF(T, heads_kv), OFF(T, capacity), OFF(T, head_dim),
                           OFF(T, dtype), OFF(T, keep),     OFF(T, sinks),    OFF(T, recent)};
    const size_t strides[] = {STRIDES(T, k_cache), STRIDES(T, v_cache), OFF(T, weights_stride_b), OFF(T, weights_stride_h)};
    sweep("ssa_cache_evict", run_evict, &base, sizeof base, ints, COUNT(ints), strides, COUNT(strides));
    T a = base;
    a.v_cache.ptr = (char*)FAKE + 128; /* a row further */
    expect(ssa_cache_evict(&a, NULL), SSA_ERR_ALIGNMENT, "ssa_cache_evict of overlapping caches");
    a = base;
    a.sinks = a.recent = INT32_MAX;
    expect(ssa_cache_evict(&a, NULL), SSA_ERR_SHAPE, "ssa_cache_evict of more fixed rows than int32 holds");
  }
  {
    typedef ssa_cache_accept_args T;
    const T base = base_accept();
    const size_t ints[] = {OFF(T, batch), OFF(T, heads_kv), OFF(T, capacity), OFF(T, head_dim),
                           OFF(T, dtype), OFF(T, nodes),    OFF(T, depth)};
    const size_t strides[] = {STRIDES(T, k_cache), STRIDES(T, v_cache)};
    sweep("ssa_cache_accept", run_accept, &base, sizeof base, ints, COUNT(ints), strides, COUNT(strides));
  }
}

static void sweep_queries(void) {
  for (int a = 0; a < NI; ++a)
    for (int b = 0; b < NI; ++b)
      for (int c = 0; c < NI; ++c)
        for (int d = 0; d < NI; ++d) {
          const int32_t x = kInts[a], y = kInts[b], z = kInts[c], t = kInts[d];
          const int64_t r[] = {
              ssa_tree_num_splits(x, y, y, z, t, 0),
              ssa_tree_num_splits(x, y, 1, z, t, x),
              ssa_tree_workspace_bytes(x, y, y, z, 64, t, 0),
              ssa_tree_workspace_bytes(x, y, 1, z, 128, t, z),
              ssa_key_weights_workspace_bytes(x, y, y, z, t),
              ssa_key_weights_workspace_bytes(x, y, 1, z, t),
          };
          for (int i = 0; i < COUNT(r); ++i, ++calls)
            if (r[i] < 0) {
              fprintf(stderr, "FAIL size query %d negative for (%d, %d, %d, %d)\n", i, x, y, z, t);
              ++failures;
            }
        }
  expect(ssa_tree_workspace_bytes(1, 8, 8, 4096, 96, 4, 0) != 0, 0, "workspace of head dim 96");
}

int main(void) {
  int devices = 0;
  if (hipGetDeviceCount(&devices) == 0 && devices > 0) {
    printf("skipped: %d GPU(s) visible; this program passes fake device pointers\n", devices);
    return 0;
  }
  sweep_queries();
  sweep_entries();
  printf("host validation of the cache operators: %ld calls, %d failures\n", calls, failures);
  return failures != 0;
}
