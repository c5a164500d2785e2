// Device helpers of the paged cache kernels.
#pragma once
#include "common.h"
#include "paged_index.h"

// paged_search with one wave counting 64 candidates at a time, and the lengths of the sequence found: the lanes of the last
// round load those of their candidates along with its start, so that one trip to memory serves both (batches up to 64)
__device__ __forceinline__ int paged_locate(const PagedIndex& x, int64_t tile, int64_t mult, int64_t per, int64_t extra, int lane, PagedSeq& s) {
  int first = 0;
  int32_t begin = 0, end = 0, ctx = 0;
  const int b = paged_search(x.batch, [&](int lo, int step, int width) {
    const int c = lo + lane * step;
    const bool in = lane * step < width;
    first = lo;
    if (in) {
      begin = x.cu[c];
      end = x.cu[c + 1];
      ctx = x.ctx[c];
    }
    return (int)__popcll(__ballot(in && paged_tile_start(begin, mult, per, extra, c) <= tile));
  });
  const int at = b < 0 ? 0 : (b - first) & 63;      // the last round steps by one
  s = paged_seq_of(x, __builtin_amdgcn_readlane(begin, at), __builtin_amdgcn_readlane(end, at), __builtin_amdgcn_readlane(ctx, at));
  return b;
}

__device__ __forceinline__ void paged_report(int32_t* status, int bits) {
  if (status && bits) atomicOr(status, bits);
}

// The last workgroup of a launch looks over every sequence's lengths and does nothing else: tiles alone would not do, since
// none leads to a sequence behind a start that is out of range.  It runs beside the others (8 sequences of one token over 500
// keys: attention 6.9 us, 7.2 with the tiles reporting; the append of 64 tokens 5.3 either way).
__device__ __forceinline__ void paged_look_over(const PagedIndex& x, int32_t* status) {
  int bad = 0;
  for (int b = threadIdx.x; b < x.batch; b += blockDim.x) bad |= paged_seq(x, b).bad;
  paged_report(status, bad);
}

#define PAGED_CHECK_INDEX(name)                                                                                            \
  NEURST_CHECK_ARG(page_table && cu_new && ctx_len, name ": null index pointer");                                           \
  NEURST_CHECK_ARG(tokens >= 0 && tokens <= INT32_MAX && batch >= 0 && batch <= (1 << 20), name ": bad token or sequence count"); \
  NEURST_CHECK_ARG(n_pages > 0 && n_pages <= INT32_MAX && wide > 0 && wide <= INT32_MAX && (ld_table >= wide || ld_table == 0), name ": bad page counts");          \
  NEURST_CHECK_ARG(page_size >= 16 && page_size <= 4096 && (page_size & (page_size - 1)) == 0,                              \
                   name ": page_size must be a power of two in 16..4096");                                                  \
  NEURST_CHECK_ARG(wide * page_size <= INT32_MAX - 4096, name ": a sequence is limited to 2^31 - 4097 positions");          \
  NEURST_CHECK_ARG(dtype == NEURST_F32 || dtype == NEURST_BF16, name ": dtype must be fp32 or bf16");                       \
  NEURST_CHECK_ARG(dh > 0 && dh <= 256 && dh % 8 == 0, name ": dh must be a multiple of 8 up to 256")

static inline PagedIndex paged_index(const int32_t* table, const int32_t* cu, const int32_t* ctx, int64_t tokens, int64_t batch, int64_t wide,
                                     int64_t ld_table, int64_t page_size, int64_t n_pages, bool own) {
  PagedIndex x;
  x.table = table; x.cu = cu; x.ctx = ctx; x.tokens = tokens; x.ld_table = ld_table;
  x.batch = (int)batch; x.wide = (int)wide; x.n_pages = (int)n_pages;
  x.own = own;
  x.page_log2 = 0;
  while (((int64_t)1 << x.page_log2) < page_size) ++x.page_log2;
  return x;
}
