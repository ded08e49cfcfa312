// Index rules of the paged 8-bit KV cache, shared by its kernels and, free of
// device code, run by the host up to sizes that no test can allocate
// (tests/cxx/paged_index_check.cpp).
//
// A page holds P tokens of every key/value head.  Keys lie [page][head][P][hd],
// values [page][head][hd][P]: a page's values are stored transposed, so that
// both products of attention read their operand in 16-byte runs along the
// contracted dimension.  A slot is page * P + place.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <algorithm>

namespace mh {

constexpr int kPageMin = 16, kPageMax = 256;  // tokens per page, powers of two
constexpr int kPagedHeadMax = 256;            // head size, a multiple of 16
constexpr int kKeyBlock = 64;                 // keys that a wave takes at once

__host__ __device__ __forceinline__ bool page_in_pool(int page, int n_pages) { return page >= 0 && page < n_pages; }

// Byte of a page's first key or value of a head.  64 bits: a pool passes 2^32
// bytes at a million pages of 16 tokens and a few heads.
__host__ __device__ __forceinline__ int64_t page_base(int page, int heads, int head, int tokens, int hd) {
  return (int64_t(page) * heads + head) * (int64_t(tokens) * hd);
}

// Keys [lo, hi) that queries i0..i1 (inclusive) of a sequence with n queries and
// len keys can see: query i stands at position len - n + i.
struct KeyRange {
  int lo, hi;
};
__host__ __device__ __forceinline__ KeyRange seen_keys(int len, int n, int i0, int i1, bool causal, int window) {
  KeyRange r;
  const int64_t p0 = int64_t(len) - n + i0, p1 = int64_t(len) - n + i1;
  const int64_t hi = causal ? (p1 + 1 < len ? p1 + 1 : len) : len;
  const int64_t lo = window > 0 ? p0 - window + 1 : 0;
  r.lo = int(lo < 0 ? 0 : lo);
  r.hi = int(hi < 0 ? 0 : hi);
  if (r.hi < r.lo) r.hi = r.lo;
  return r;
}

// Share s of `splits` of a key range: `chunk` keys (a multiple of kKeyBlock) from
// the range's start rounded down to a block; the last share takes what is left,
// so that the shares cover the range whatever length the chunk was chosen for.
__host__ __device__ __forceinline__ KeyRange key_share(KeyRange all, int s, int splits, int chunk) {
  const int first = all.lo & ~(kKeyBlock - 1);
  const int64_t a = int64_t(first) + int64_t(s) * chunk, b = s + 1 < splits ? a + chunk : int64_t(all.hi);
  KeyRange r;
  r.lo = int(a < all.hi ? a : all.hi);
  r.hi = int(b < all.hi ? b : all.hi);
  if (r.hi < r.lo) r.hi = r.lo;
  return r;
}

// What a request of `len` cached and `fresh` new tokens holds and needs, in
// pages, with room for `width` pages in its row of the block table.
struct PlanNeed {
  int len, fresh, have, need;
};
__host__ __device__ __forceinline__ PlanNeed plan_need(int len, int fresh, int page, int width) {
  PlanNeed n;
  n.len = len > 0 ? len : 0;
  n.fresh = fresh > 0 ? fresh : 0;
  if (n.fresh > 0x7fffffff - n.len) n.fresh = 0x7fffffff - n.len;
  const int have = n.len / page + (n.len % page != 0), all = n.len + n.fresh, need = all / page + (all % page != 0);
  n.have = have;
  n.need = need < width ? need : width;
  if (n.need < n.have) n.need = n.have;
  return n;
}
// Requests of a plan: its work grows with their square (2^18 take 46 ms).
constexpr int kPlanMaxRequests = 1 << 20;
// Workgroups per request of the plan, which go round its tokens: one for each
// 1024 tokens that there may be, at most 1024 in all (one prompt of 131072
// tokens 6 us, 302 with one workgroup; 12 of 2500 4.0 against 6.6).
inline int plan_groups(int B, int64_t cap) {
  return int(std::max<int64_t>(1, std::min<int64_t>(1024 / std::max(B, 1), (cap + 1023) / 1024)));
}

// Tokens per workgroup of the store: one while that leaves at most 4096
// workgroups (a decode step: every token starts a run), up to 64 for prompts,
// where one token in a page does (17k tokens, 8 heads of 128, pages of 64: 34 us;
// at most 2048 workgroups 37, 8192 38, 16384 39).
inline int store_tokens(int n, int heads) { return int(std::min<int64_t>(64, std::max<int64_t>(1, int64_t(n) * heads / 4096))); }

// Workgroup i of a launch over `pairs` (sequence, key/value head) pairs of `per`
// items each.  Workgroups go round the eight XCDs, each with an L2 of its own:
// eight pairs at a time, one to an XCD, so that the items that read the same
// keys find them there (6 chunks of prompts, 8 heads, when this was chosen: 816 us; a
// pair's items after another over all XCDs 820, all pairs' first items, then all
// second ones 1029).  The pairs left over go round all of them.
constexpr int kXcds = 8;
struct PairItem {
  int pair, item;
};
__host__ __device__ __forceinline__ PairItem pair_item(uint32_t i, int pairs, int per) {
  PairItem r;
  const uint32_t whole = uint32_t(pairs / kXcds) * kXcds * uint32_t(per);
  if (i < whole) {
    const uint32_t j = i / kXcds;
    r.pair = int(i % kXcds + kXcds * (j / uint32_t(per)));
    r.item = int(j % uint32_t(per));
  } else {
    r.pair = pairs / kXcds * kXcds + int((i - whole) / uint32_t(per));
    r.item = int((i - whole) % uint32_t(per));
  }
  return r;
}

// Tokens of a table row: the kernels look a few blocks past the last one in 32 bits.
constexpr int kPagedMaxKeys = 0x7fffffff - 4095;

// How a call is cut: rows of one (sequence, key/value head) in tiles, and each
// tile's keys in `splits` shares of `chunk`.
struct PagedShape {
  int wide, tiles, splits, chunk;
};
// Workgroups of a launch: kernels walk the tiles past those that it has.
constexpr int kPagedMaxBlocks = (1 << 23) - 1;
// Rows that a workgroup of the wide form takes: 32 to each of four waves.
constexpr int kPagedWideRows = 128;
inline PagedShape paged_shape(int B, int Hq, int Hkv, int max_q, int max_len, int window) {
  PagedShape s;
  const int64_t rows = int64_t(max_q) * (Hq / Hkv);
  s.wide = rows > 16;
  const int per = s.wide ? kPagedWideRows : 16;
  s.tiles = int(std::max<int64_t>(1, (rows + per - 1) / per));
  // Shares so that the workgroups, two to a CU, are all there at once or nearly
  // (64 requests of up to 8192 keys, 8 heads of 128: one share 121 us, two 133 +
  // join 5, four 145 + 6; 2 requests of which one has 131072: 32 shares 85 + 6,
  // 64 74 + 7, 128 83 + 12), none shorter than one block per wave.
  const int64_t whole = std::max<int64_t>(1, int64_t(B) * Hkv * s.tiles);
  const int64_t longest = std::min(max_len, kPagedMaxKeys);
  const int64_t keys = window > 0 ? std::min<int64_t>(longest, int64_t(window) + max_q + kKeyBlock) : longest;
  const int64_t least = 4 * kKeyBlock;
  int64_t n = std::min<int64_t>((keys + least - 1) / least, 1025 / (whole + 1));
  n = std::max<int64_t>(1, std::min<int64_t>(n, 256));
  s.chunk = int(((keys + n - 1) / n + least - 1) / least * least);
  if (s.chunk == 0) s.chunk = int(least);
  s.splits = int(std::max<int64_t>(1, (keys + s.chunk - 1) / s.chunk));
  s.tiles = int(std::min<int64_t>(s.tiles, std::max<int64_t>(1, kPagedMaxBlocks / std::max<int64_t>(1, int64_t(B) * Hkv * s.splits))));
  return s;
}
// Workspace: the shares' outputs, then their (maximum, sum) pairs.
inline size_t paged_part_bytes(int n_rows, int Hq, int hd, int splits) {
  return splits > 1 ? size_t(n_rows) * Hq * splits * hd * 4 : 0;
}
inline size_t paged_workspace_bytes(int n_rows, int Hq, int hd, int splits) {
  return splits > 1 ? paged_part_bytes(n_rows, Hq, hd, splits) + size_t(n_rows) * Hq * splits * 8 : 0;
}

// How a workgroup of the join is cut: hd / 4 threads take a share's values, `groups`
// of them a row, each every groups-th share (with one, a row of 64 shares took
// 31 us for 128 rows), and `rows` rows.  Where hd / 4 * groups does not divide
// the workgroup, its last threads have no row, and no partners to read from.
constexpr int kJoinThreads = 256;
struct JoinShape {
  int per, groups, rows;
};
constexpr int64_t kJoinMaxBlocks = (1 << 24) - 1;  // 2^32 threads
inline JoinShape join_shape(int hd, int splits) {
  JoinShape s;
  s.per = hd / 4;
  s.groups = std::max(1, std::min((splits + 3) / 4, kJoinThreads / s.per));
  s.rows = kJoinThreads / (s.per * s.groups);
  return s;
}
struct JoinUnit {
  int row, group, d;  // d: the first of its four head values
  bool on;
};
__host__ __device__ __forceinline__ JoinUnit join_unit(int tid, int per, int groups, int rows) {
  const int unit = tid / per;
  JoinUnit u;
  u.row = unit / groups;
  u.group = unit - u.row * groups;
  u.d = 4 * (tid - unit * per);
  u.on = u.row < rows;
  return u;
}

}  // namespace mh
