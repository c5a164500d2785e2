// Host check of what the kernels make of a tile (neurst_amd/csrc/paged_index.h): whatever cu_new holds - starts that fall, rows
// past the tensors, negative ones - the rows and positions of every tile of every sequence lie inside that sequence's own
// and inside the tensors.  Prints "ok" or the first mistake.
#include <stdio.h>
#include <vector>

#include "../../neurst_amd/csrc/paged_index.h"

static uint64_t g_state = 362436069362436069ull;
static uint32_t rnd(uint32_t n) {
  g_state ^= g_state << 13;
  g_state ^= g_state >> 7;
  g_state ^= g_state << 17;
  return (uint32_t)(g_state >> 11) % n;
}

struct Shape { int64_t mult; int per, extra; };

static int check(const std::vector<int32_t>& cu, const std::vector<int32_t>& ctx, int64_t tokens, int wide, int page_log2, int own, Shape t, int* seen_behind) {
  const int B = (int)ctx.size();
  PagedIndex x = {nullptr, cu.data(), ctx.data(), tokens, wide, B, wide, page_log2, 1, own};
  const int64_t tiles = paged_tiles(tokens, B, t.mult, t.per, t.extra);
  for (int64_t i = 0; i < tiles; ++i) {
    const int b = paged_search(B, [&](int lo, int step, int width) {
      int n = 0;
      for (int k = 0; k < 64 && k * step < width; ++k) n += paged_tile_start(cu[lo + k * step], t.mult, t.per, t.extra, lo + k * step) <= i;
      return n;
    });
    if (b < 0) continue;
    const PagedSeq s = paged_seq(x, b);
    const int64_t mine = i - paged_tile_start(s.cu, t.mult, t.per, t.extra, b);
    *seen_behind += mine < 0;
    int64_t r0, r1;      // packed rows that the tile reads and writes
    if (t.extra == 2) {
      int p0, p1;
      if (!paged_tile_positions(s, mine, t.per, p0, p1)) continue;
      if (p0 < 0 || p1 <= p0 || p1 - p0 > t.per || p1 > (int64_t)wide << page_log2) { printf("positions %d .. %d\n", p0, p1); return 1; }
      r0 = s.row0 + (p0 - (s.ctx - s.new_tokens));
      r1 = s.row0 + (p1 - 1 - (s.ctx - s.new_tokens));
    } else {
      int begin, count;
      if (!paged_tile_rows(s, mine, t.mult, t.per, begin, count)) continue;
      if (begin < 0 || count < 1 || count > t.per) { printf("rows %d + %d\n", begin, count); return 1; }
      r0 = s.row0 + begin / t.mult;
      r1 = s.row0 + (begin + count - 1) / t.mult;
    }
    if (r0 < cu[b] || r1 >= cu[b + 1] || r0 < 0 || r1 >= tokens) {
      printf("tile %lld: rows %lld .. %lld of sequence %d (%d .. %d), %lld tokens\n", (long long)i, (long long)r0, (long long)r1, b, cu[b], cu[b + 1],
             (long long)tokens);
      return 1;
    }
  }
  return 0;
}

int main() {
  int behind = 0;
  // a sequence that is told by counting starts and begins behind the tile
  if (check({0, 1000000, 2, 12}, {5, 5, 12}, 12, 4, 4, 1, {1, 16, 1}, &behind)) return 1;
  if (!behind) { printf("no tile before its sequence\n"); return 1; }
  for (int round = 0; round < 3000; ++round) {
    const int B = 1 + rnd(round % 50 == 0 ? 700 : 70), page_log2 = 4 + rnd(4), wide = 1 + rnd(20), cap = wide << page_log2;
    std::vector<int32_t> cu(B + 1, 0), ctx(B);
    for (int b = 0; b < B; ++b) {
      const int n = rnd(3) ? (int)rnd(cap < 200 ? cap : 200) : 0;
      cu[b + 1] = cu[b] + n;
      ctx[b] = n + (int)rnd(cap - n + 1);
    }
    const int64_t tokens = cu[B] + (int64_t)rnd(30);
    for (int k = 0; k < 1 + (int)rnd(8); ++k) {
      const int32_t wild[] = {-1, 0, INT32_MAX, INT32_MIN, (int32_t)rnd(1000000), -(int32_t)rnd(1000000), (int32_t)rnd((uint32_t)tokens + 2)};
      cu[rnd(B + 1)] = wild[rnd(7)];
      if (rnd(2)) ctx[rnd(B)] = wild[rnd(7)];
    }
    const Shape shapes[] = {{1, 64, 2}, {1 + rnd(12), 16, 1}, {1 + rnd(12), 128, 1}};
    for (const Shape& t : shapes)
      for (int own = 0; own < 2; ++own)
        if (check(cu, ctx, tokens, wide, page_log2, t.extra == 2 ? 1 : own, t, &behind)) return 1;
  }
  printf("ok\n");
  return 0;
}
