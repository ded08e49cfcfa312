// The index rules of the paged KV cache (csrc/paged_index.hpp) on the host: the
// shares of a key range hold every seen key once and no other, for lengths up to
// the largest; page bases pass 32 bits; plans never leave a table's width; cuts
// of calls stay within a launch.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "paged_index.hpp"

using namespace mh;

static void need(bool ok, const char *what) {
  if (ok) return;
  std::printf("%s\n", what);
  std::exit(1);
}

static void check_range(int len, int n, bool causal, int window) {
  for (int i = 0; i < n; i += 1 + n / 7) {
    const long p = long(len) - n + i;
    long lo = window > 0 ? p - window + 1 : 0, hi = causal ? p + 1 : len;
    if (lo < 0) lo = 0;
    if (hi > len) hi = len;
    if (hi < 0) hi = 0;
    if (hi < lo) hi = lo;
    const KeyRange r = seen_keys(len, n, i, i, causal, window);
    need(hi == lo ? r.lo == r.hi : (r.lo == lo && r.hi == hi), "seen_keys of one query");
  }
}

int main() {
  std::mt19937 rng(1);
  auto upto = [&](int n) { return int(rng() % unsigned(n)); };
  for (int t = 0; t < 20000; ++t) {
    const int big = t % 3 == 0 ? 0x7fffff00 : t % 3 == 1 ? 5000 : 70;
    const int len = upto(big), n = 1 + upto(t % 2 ? 5 : 300);
    check_range(len, n, t & 1, t % 5 ? 0 : 1 + upto(900));
  }
  // every key once: small ranges key by key, large ones by their ends
  for (int t = 0; t < 4000; ++t) {
    KeyRange all;
    all.lo = upto(700);
    all.hi = all.lo + upto(1500);
    const int chunk = kKeyBlock * (1 + upto(6)), splits = 1 + upto(9);
    std::vector<int> hits(2300, 0);
    for (int s = 0; s < splits; ++s) {
      const KeyRange r = key_share(all, s, splits, chunk);
      need(r.lo <= r.hi && r.hi <= all.hi, "share within the range");
      if (r.lo < r.hi) need(r.lo % kKeyBlock == 0, "share starts on a block");
      for (int k = r.lo; k < r.hi; ++k) ++hits[size_t(k)];
    }
    for (int k = all.lo; k < all.hi; ++k) need(hits[size_t(k)] == 1, "every key once");
    for (int k = all.hi; k < 2300; ++k) need(hits[size_t(k)] == 0, "no key past the range");
  }
  for (int t = 0; t < 20000; ++t) {
    KeyRange all;
    all.hi = 0x7fffffff - upto(1000000);
    all.lo = upto(2) ? all.hi - upto(100000) : upto(1000);
    const int splits = 1 + upto(256), chunk = kKeyBlock * (1 + upto(1 << 20));
    long at = all.lo & ~(kKeyBlock - 1);
    for (int s = 0; s < splits; ++s) {
      const KeyRange r = key_share(all, s, splits, chunk);
      if (r.lo == r.hi) continue;
      need(r.lo == at, "shares follow each other");
      at = r.hi;
    }
    need(at == all.hi || all.lo == all.hi, "the last share ends the range");
  }
  need(page_base(1 << 20, 8, 7, 64, 128) == ((int64_t(1) << 23) + 7) * 8192, "page_base in 64 bits");
  need(!page_in_pool(-1, 4) && page_in_pool(0, 4) && page_in_pool(3, 4) && !page_in_pool(4, 4), "page_in_pool");

  for (int page : {16, 32, 64, 128, 256})
    for (int t = 0; t < 20000; ++t) {
      const int width = upto(3) ? upto(50) : 0x7fffffff / page;
      const int len = upto(4) ? upto(4000) - 3 : 0x7fffffff - upto(300), fresh = upto(4) ? upto(4000) - 3 : 0x7fffffff - upto(300);
      const PlanNeed n = plan_need(len, fresh, page, width);
      need(n.len >= 0 && n.fresh >= 0 && long(n.len) + n.fresh <= 0x7fffffffL, "plan lengths");
      need(n.have == (long(n.len) + page - 1) / page, "pages held");
      need(n.need >= n.have && (n.need == n.have || n.need <= width), "pages needed within the table");
      if (n.need < width && n.need > n.have) need(n.need == (long(n.len) + n.fresh + page - 1) / page, "pages needed");
    }
  for (int n : {1, 5, 64, 1000, 16384, 100000, 0x7fffffff})
    for (int heads : {1, 8, 65535}) {
      const int per = store_tokens(n, heads);
      need(per >= 1 && per <= 64, "tokens per workgroup of the store");
    }
  for (int t = 0; t < 300; ++t) {  // every item of every pair once
    const int pairs = 1 + upto(40), per = 1 + upto(30);
    std::vector<int> hits(size_t(pairs * per), 0);
    for (int i = 0; i < pairs * per; ++i) {
      const PairItem r = pair_item(uint32_t(i), pairs, per);
      need(r.pair >= 0 && r.pair < pairs && r.item >= 0 && r.item < per, "pair and item");
      ++hits[size_t(r.pair * per + r.item)];
    }
    for (int h : hits) need(h == 1, "every item once");
  }
  for (int t = 0; t < 50000; ++t) {
    const int kv = 1 + upto(16), g = 1 + upto(16), hd = 16 * (1 + upto(16)), B = 1 + upto(t % 4 ? 300 : 100000);
    const int max_q = 1 + upto(t % 2 ? 4 : 5000), max_len = upto(t % 3 ? 0x7fffffff : 5000), window = t % 5 ? 0 : 1 + upto(5000);
    const PagedShape s = paged_shape(B, kv * g, kv, max_q, max_len, window);
    need(s.tiles >= 1 && s.splits >= 1 && s.splits <= 256 && s.chunk % kKeyBlock == 0, "cut of a call");
    const long keys = window ? std::min<long>(max_len, long(window) + max_q + kKeyBlock) : max_len;
    need(long(s.splits) * s.chunk >= keys, "the shares hold the longest request");
    need((s.splits > 1) == (paged_workspace_bytes(max_q, kv * g, hd, s.splits) > 0), "workspace where shares are joined");
  }
  need(paged_shape(0, 8, 8, 0, 0, 0).splits == 1, "empty call");
  std::puts("ok");
}
