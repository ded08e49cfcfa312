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

// Every cut fits a launch, whatever the bounds; as many tiles as the bounds ask
// for where they fit.
static void check_launches() {
  for (int B : {1, 2, 7, 256, 4096, 100000, kPagedMaxBlocks / 8})
    for (int kv : {1, 2, 8})
      for (int G : {1, 4, 64})
        for (int max_q : {0, 1, 2, 17, 300, 5000, 131072, 1 << 30 >> 6})
          for (int max_len : {0, 1, 100, 70000, 0x7fffffff})
            for (int window : {0, 1, 5000}) {
              const PagedShape s = paged_shape(B, kv * G, kv, max_q, max_len, window);
              const int64_t pairs = int64_t(B) * kv;
              need(pairs * s.tiles * s.splits <= kPagedMaxBlocks && s.tiles >= 1 && s.splits >= 1, "a call's workgroups fit a launch");
              const int64_t per = s.wide ? kPagedWideRows : 16, tiles = std::max<int64_t>(1, (int64_t(max_q) * G + per - 1) / per);
              need(s.tiles == tiles || pairs * s.splits * (s.tiles + 1) > kPagedMaxBlocks, "fewer tiles only where a launch ends");
            }
}

int main() {
  check_join();
  check_launches();
  std::puts("ok");
}
