// Index arithmetic of the paged key/value cache, shared by the kernels of paged.hip / paged_attn.hip and a host test.
//
// A call brings N new tokens, packed by sequence: sequence b owns rows cu[b] .. cu[b + 1] - 1, and its cache holds ctx[b]
// tokens WITH them, so its row j stands at position ctx[b] - n_b + j.  Position p lives in page table[b][p >> page_log2],
// slot p & (page - 1).
//
// All of it is read from device memory, where the host cannot check it, so every use goes through the functions below:
// lengths that do not fit leave the sequence out, a page id outside the pool leaves its keys out, and both raise a bit of
// the caller's status word.  Nothing is read or written out of range whatever the four arrays hold.
#pragma once
#include <stdint.h>
#ifdef __HIPCC__
#define NEURST_HD __host__ __device__ __forceinline__
#else
#define NEURST_HD static inline
#endif

enum { PAGED_BAD_PAGE = 1, PAGED_BAD_LENGTH = 2 };

struct PagedIndex {
  const int32_t* table;     // [B][wide]
  const int32_t* cu;        // [B + 1]
  const int32_t* ctx;       // [B]
  int64_t tokens;           // N, rows of the packed tensors
  int64_t ld_table;
  int batch, wide, page_log2, n_pages;
  int own;                  // the new tokens are part of the cache: ctx >= their number
};

struct PagedSeq {
  int64_t row0;   // first packed row
  int new_tokens; // rows of this sequence (0: nothing to do)
  int ctx;        // tokens in the cache with them (0: nothing visible)
  int bad;
  int32_t cu;     // cu[b] as it is
};

// Lengths of sequence b.  Rows out of range: the sequence is left out.  A cache shorter than the rows it should hold (`own`),
// or longer than the page table: the rows exist but nothing is visible to them.
NEURST_HD PagedSeq paged_seq_of(const PagedIndex& x, int32_t begin, int32_t end, int32_t ctx) {
  PagedSeq s;
  s.row0 = begin;
  s.bad = 0;
  s.new_tokens = 0;
  s.ctx = 0;
  s.cu = begin;
  if (begin < 0 || end < begin || end > x.tokens) {
    s.bad = PAGED_BAD_LENGTH;
    return s;
  }
  s.new_tokens = end - begin;
  if (ctx < (x.own ? s.new_tokens : 0) || ctx > ((int64_t)x.wide << x.page_log2)) {
    s.bad = PAGED_BAD_LENGTH;
    return s;
  }
  s.ctx = ctx;
  return s;
}
NEURST_HD PagedSeq paged_seq(const PagedIndex& x, int b) { return paged_seq_of(x, x.cu[b], x.cu[b + 1], x.ctx[b]); }

// page of position p (0 <= p < wide << page_log2 is the caller's to hold), -1 for an id outside the pool
NEURST_HD int paged_page(const PagedIndex& x, int b, int p) {
  const int id = x.table[(int64_t)b * x.ld_table + (p >> x.page_log2)];
  return (unsigned)id < (unsigned)x.n_pages ? id : -1;
}

// Tiles of `per` rows without a host-side plan: sequence b's tiles start at floor(cu[b] * mult / per) + extra * b, which
// leaves room for ceil(rows_b * mult / per) (extra = 1) or one more (extra = 2) whatever the lengths are, so a grid of
// floor(N * mult / per) + extra * B tiles covers every ragged batch and a tile finds its sequence by that formula alone.
NEURST_HD int64_t paged_tile_start(int64_t cu_b, int64_t mult, int64_t per, int64_t extra, int64_t b) {
  return (cu_b < 0 ? 0 : cu_b) * mult / per + extra * b;
}
static inline int64_t paged_tiles(int64_t tokens, int64_t batch, int64_t mult, int64_t per, int64_t extra) {
  return tokens * mult / per + extra * batch;
}

// The sequence a tile belongs to: the last b with tile_start(b) <= tile, -1 for none.  count(lo, step, width) says how many of
// the at most 64 candidates lo, lo + step, .. below lo + width start at or before the tile.  cu that does not grow gives some
// sequence or none, never an index out of range; that sequence may begin behind the tile, so what the tile is of it goes
// through one of the two functions below.
template <typename Count> NEURST_HD int paged_search(int batch, Count count) {
  int lo = 0, width = batch;
  for (;;) {
    const int step = (width + 63) >> 6;
    const int n = count(lo, step, width);
    if (n == 0) return -1;
    const int last = lo + (n - 1) * step;
    if (step == 1) return last;
    width = lo + width - last < step ? lo + width - last : step;
    lo = last;
  }
}

// Rows begin .. begin + count - 1 of a sequence's new_tokens * mult that its tile `own` of `per` rows has; false: none
NEURST_HD bool paged_tile_rows(const PagedSeq& s, int64_t own, int64_t mult, int per, int& begin, int& count) {
  const int64_t rows = (int64_t)s.new_tokens * mult;
  if (own < 0 || own * per >= rows) return false;
  begin = (int)(own * per);
  count = (int)(rows - own * per < per ? rows - own * per : per);
  return true;
}
// Positions p0 .. p1 - 1 of a sequence's new tokens in its tile `own` of `per` (a power of two) positions aligned in the
// cache; false: none
NEURST_HD bool paged_tile_positions(const PagedSeq& s, int64_t own, int per, int& p0, int& p1) {
  if (own < 0 || s.ctx == 0 || s.new_tokens == 0) return false;
  const int first = s.ctx - s.new_tokens;
  const int64_t lo = (int64_t)(first & ~(per - 1)) + own * per;
  if (lo >= s.ctx) return false;
  p0 = lo < first ? first : (int)lo;
  p1 = lo + per < s.ctx ? (int)(lo + per) : s.ctx;
  return true;
}
