// The library's plans of the cache operators (csrc/ssa_cache_ops.hpp) for calls
// read from stdin, one a line: "tree B Hq Hkv capacity T splits" gives the rows of a
// workgroup, the keys of a split and the splits.
#include <cstdio>

#include "ssa_cache_ops.hpp"

int main() {
  int B, Hq, Hkv, cap, T, splits;
  while (std::scanf(" tree %d %d %d %d %d %d", &B, &Hq, &Hkv, &cap, &T, &splits) == 6) {
    const ssa::TreePlan p = ssa::tree_plan(B, Hq, Hkv, cap, T, splits);
    std::printf("%d %d %d\n", p.rows, p.split_keys, p.splits);
  }
  return 0;
}
