// Host check of neurst_amd/csrc/paged_index.h: every tile of every ragged batch is found, by one workgroup only, and whatever
// the index arrays hold nothing leads out of range.  Prints "ok" or the first mistake.
#include <stdio.h>
#include <stdlib.h>
#include <vector>

#include "../../neurst_amd/csrc/paged_index.h"

static uint64_t g_state = 88172645463325252ull;
static uint32_t rnd(uint32_t n) {
  g_state ^= g_state << 13;
  g_state ^= g_state >> 7;
  g_state ^= g_state << 17;
  return (uint32_t)(g_state >> 11) % n;
}

static int find(const PagedIndex& x, int64_t tile, int64_t mult, int64_t per, int64_t extra) {
  return paged_search(x.batch, [&](int lo, int step, int width) {
    int n = 0, lanes = 0;
    for (int i = 0; i < 64 && i * step < width; ++i, ++lanes) {
      const int b = lo + i * step;
      if (b < 0 || b >= x.batch) { printf("candidate %d of %d\n", b, x.batch); exit(1); }
      n += paged_tile_start(x.cu[b], mult, per, extra, b) <= tile;
    }
    if (lanes * (int64_t)step < width) { printf("64 candidates do not reach %d\n", width); exit(1); }
    return n;
  });
}

int main() {
  for (int round = 0; round < 400; ++round) {
    const int B = 1 + rnd(round % 10 == 0 ? 9000 : 200), page_log2 = 4 + rnd(4), wide = 1 + rnd(20);
    const int most = 1 + rnd(round % 3 ? 40 : 300), bad = round % 4 == 3;
    std::vector<int32_t> cu(B + 1, 0), ctx(B), table((size_t)B * wide);
    cu[0] = rnd(5) == 0 ? (int)rnd(40) : 0;
    for (int b = 0; b < B; ++b) {
      const int n = rnd(3) ? (int)rnd(most) : 0, cap = wide << page_log2;
      cu[b + 1] = cu[b] + (n < cap ? n : cap);
      ctx[b] = cu[b + 1] - cu[b] + (int)rnd(cap - (cu[b + 1] - cu[b]) + 1);
    }
    PagedIndex x = {table.data(), cu.data(), ctx.data(), cu[B] + (int64_t)rnd(30), wide, B, wide, page_log2, 1 + (int)rnd(50), 1};
    for (auto& t : table) t = rnd(x.n_pages);
    if (bad)
      for (int k = 0; k < 12; ++k) {
        const int32_t wild[] = {-1, 0, INT32_MAX, INT32_MIN, (int32_t)rnd(100000), -(int32_t)rnd(100000)};
        cu[rnd(B + 1)] = wild[rnd(6)];
        ctx[rnd(B)] = wild[rnd(6)];
        table[rnd(B * wide)] = wild[rnd(6)];
      }
    const struct { int64_t mult, per, extra; } shapes[] = {{1, 64, 2}, {1 + rnd(12), 16, 1}, {1 + rnd(12), 128, 1}, {1 + rnd(12), 256, 1}};
    for (auto& t : shapes) {
      const int64_t tiles = paged_tiles(x.tokens, B, t.mult, t.per, t.extra);
      std::vector<int64_t> found(B, 0);
      for (int64_t i = 0; i < tiles; ++i) {
        const int b = find(x, i, t.mult, t.per, t.extra);
        if (b < -1 || b >= B) { printf("sequence %d of %d\n", b, B); return 1; }
        if (b < 0) continue;
        const PagedSeq s = paged_seq(x, b);
        if (s.new_tokens && (s.row0 < 0 || s.row0 + s.new_tokens > x.tokens)) { printf("rows out of range\n"); return 1; }
        if (s.ctx < 0 || s.ctx > wide << page_log2 || (s.ctx && s.ctx < s.new_tokens)) { printf("context out of range\n"); return 1; }
        if (s.ctx) {
          const int id = paged_page(x, b, rnd(s.ctx));
          if (id < -1 || id >= x.n_pages) { printf("page out of range\n"); return 1; }
        }
        if (bad) continue;
        if (s.bad) { printf("good lengths refused\n"); return 1; }
        const int64_t own = i - paged_tile_start(cu[b], t.mult, t.per, t.extra, b);
        // what the kernels make of tile `own`: the cache write has tiles aligned in the cache, attention tiles of rows
        const int64_t begin = t.extra == 2 ? (int64_t)((s.ctx - s.new_tokens) & ~63) + own * 64 : own * t.per;
        const int64_t end = t.extra == 2 ? s.ctx : s.new_tokens * t.mult;
        if (own < 0) { printf("tile before its sequence\n"); return 1; }
        if (begin < end && (t.extra != 2 || s.new_tokens)) ++found[b];
      }
      if (!bad)
        for (int b = 0; b < B; ++b) {
          const int64_t n = cu[b + 1] - cu[b], first = ctx[b] - n;
          const int64_t want = !n ? 0 : t.extra == 2 ? (ctx[b] - (first & ~63ll) + 63) / 64 : (n * t.mult + t.per - 1) / t.per;
          if (found[b] != want) { printf("sequence %d has %lld of %lld tiles\n", b, (long long)found[b], (long long)want); return 1; }
        }
    }
  }
  printf("ok\n");
  return 0;
}
