// How calls over the paged KV cache are cut (csrc/paged_index.hpp), on the host, for
// every size that the calls take.
#include <cstdio>
#include <cstdlib>

#include "paged_index.hpp"

using namespace mh;

static void need(bool ok, const char *what) {
  if (ok) return;
  std::printf("%s\n", what);
  std::exit(1);
}

// The join's groups read their partners' shares in LDS: each read lies within the
// workgroup and finds the same row's next group at the same head values.
static void check_join() {
  for (int hd = 16; hd <= kPagedHeadMax; hd += 16)
    for (int splits = 2; splits <= 256; ++splits) {
      const JoinShape s = join_shape(hd, splits);
      need(s.per * s.groups * s.rows <= kJoinThreads && s.rows >= 1, "a join's rows fit a workgroup");
      for (int tid = 0; tid < kJoinThreads; ++tid) {
        const JoinUnit u = join_unit(tid, s.per, s.groups, s.rows);
        if (!u.on || u.group != 0) continue;
        for (int k = 1; k < s.groups; ++k) {
          need(tid + k * s.per < kJoinThreads, "a join's reads lie within the workgroup");
          const JoinUnit v = join_unit(tid + k * s.per, s.per, s.groups, s.rows);
          need(v.on && v.row == u.row && v.group == k && v.d == u.d, "a join's groups follow each other");
        }
      }
    }
}

int main() {
  check_join();
  std::puts("ok");
}
