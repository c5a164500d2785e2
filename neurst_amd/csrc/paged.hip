// The write into the paged key/value cache: new keys (rotated on the way, rotary.h) and values go to their pages, new queries
// come back rotated, in one launch.  No reference counterpart: the reference's cache holds whole outputs of equal length
// (st/models/decoders/transformer_decoder.py:123-182).
//
// Layout: K [page][head][slot][dh], V TRANSPOSED [page][head][dh][slot].  The attention's second product contracts over the
// keys, so its matrix instructions want eight consecutive KEYS of one column per lane: stored like this they are one
// 16-byte load from the page, with no trip through shared memory.  The price is paid here, once per token: a chunk is
// transposed in registers eight slots at a time, a single token scatters dh elements of 2 bytes.
//
// Bound by memory (chunks: 37 sequences of up to 700 tokens, 8 heads of 64 columns, bf16, 30 to 33 us = 3.2 to 3.5 TB/s at pages of
// 32 slots and more, 36 at 16; fp32 47 us = 4.5 TB/s at any) or by the launch (64 single tokens of 96 columns: 5.0 us).  A tile is 64 positions aligned in the cache; its items - 16
// bytes of a query or key row with its partner of the pair, eight slots x eight columns of values - are dealt to
// gridDim.y workgroups.  Lanes of a value item run over the slot groups first, then over the columns: a wave reads whole
// 128-byte row pieces and writes whole 128-byte column pieces.
#include "paged.h"
#include "rotary.h"

struct AppendArgs {
  PagedIndex ix;
  const void *k, *v, *q;
  void *k_pages, *v_pages, *q_out;
  const double* freq;
  int32_t* status;
  int64_t ldk, ldv, ldq, ldqo;
  int hkv, hq, dh, hg;
  float mscale;
  RotShape sh;
};

constexpr int APPEND_TILE = 64;

template <typename T, int VEC> __global__ void __launch_bounds__(256) paged_append_kernel(AppendArgs a) {
  constexpr int E = 16 / sizeof(T);          // slots of a value item, and its columns
  if (blockIdx.x == gridDim.x - 1) {
    if (blockIdx.y == 0) paged_look_over(a.ix, a.status);
    return;
  }
  const int lane = threadIdx.x & 63;
  PagedSeq s;
  const int b = paged_locate(a.ix, blockIdx.x, 1, APPEND_TILE, 2, lane, s);
  if (b < 0) return;
  int p0, p1;                                                              // positions p0 .. p1 - 1
  if (!paged_tile_positions(s, blockIdx.x - paged_tile_start(s.cu, 1, APPEND_TILE, 2, b), APPEND_TILE, p0, p1)) return;
  const int first = s.ctx - s.new_tokens;                                  // position of the first new token
  const int page = 1 << a.ix.page_log2, mask = page - 1;
  const int nt = p1 - p0, heads = a.hkv + a.hq, hgs = (heads + a.hg - 1) / a.hg;
  const int k_items = nt * hgs * a.sh.chunks;
  const int g0 = p0 / E, ng = (p1 - 1) / E - g0 + 1, cb = a.dh / E;
  const int v_items = ng * cb * a.hkv;
  for (int i = blockIdx.y * 256 + threadIdx.x; i < k_items + v_items; i += gridDim.y * 256) {
    if (i < k_items) {
      const int c = i % a.sh.chunks, rest = i / a.sh.chunks, hgi = rest % hgs, p = p0 + rest / hgs;
      const int64_t row = s.row0 + (p - first);
      const int pg = paged_page(a.ix, b, p);
      if (pg < 0) paged_report(a.status, PAGED_BAD_PAGE);
      const int h0 = hgi * a.hg, h1 = h0 + a.hg < heads ? h0 + a.hg : heads;
      float cs[VEC], sn[VEC];
      const bool turn = c < a.sh.rot_chunks;
      if (turn) rot_angles<VEC>(a.sh, a.freq, c, p, a.mscale, 1.f, cs, sn);
      for (int h = h0; h < h1; ++h) {
        const T* src;
        T* dst;
        if (h < a.hkv) {
          if (pg < 0) continue;
          src = static_cast<const T*>(a.k) + row * a.ldk + (int64_t)h * a.dh;
          dst = static_cast<T*>(a.k_pages) + ((((int64_t)pg * a.hkv + h) << a.ix.page_log2) + (p & mask)) * a.dh;
        } else {
          src = static_cast<const T*>(a.q) + row * a.ldq + (int64_t)(h - a.hkv) * a.dh;
          dst = static_cast<T*>(a.q_out) + row * a.ldqo + (int64_t)(h - a.hkv) * a.dh;
        }
        if (turn) rot_apply<T, VEC>(a.sh, src, dst, c, cs, sn);
        else if (src != dst) rot_pass<T, VEC>(a.sh, src, dst, c);
      }
    } else {
      const int j = i - k_items;
      const int sg = j % ng, rest = j / ng, col = (rest % cb) * E, h = rest / cb;
      const int ps = (g0 + sg) * E;                                          // first position of the group
      const int pg = paged_page(a.ix, b, ps);
      if (pg < 0) {
        paged_report(a.status, PAGED_BAD_PAGE);
        continue;
      }
      const T* src = static_cast<const T*>(a.v) + (int64_t)h * a.dh + col;
      T* dst = static_cast<T*>(a.v_pages) + ((((int64_t)pg * a.hkv + h) * a.dh + col) << a.ix.page_log2) + (ps & mask);
      if (ps >= p0 && ps + E <= p1) {
        RotVec<T, E> in[E];
#pragma unroll
        for (int e = 0; e < E; ++e)
          __builtin_memcpy(&in[e], __builtin_assume_aligned(src + (s.row0 + (ps + e - first)) * a.ldv, 16), 16);
#pragma unroll
        for (int d = 0; d < E; ++d) {
          RotVec<T, E> out;
#pragma unroll
          for (int e = 0; e < E; ++e) out.v[e] = in[e].v[d];
          __builtin_memcpy(__builtin_assume_aligned(dst + ((int64_t)d << a.ix.page_log2), 16), &out, 16);
        }
      } else {
        for (int e = 0; e < E; ++e) {
          const int p = ps + e;
          if (p < p0 || p >= p1) continue;
          RotVec<T, E> in;
          __builtin_memcpy(&in, __builtin_assume_aligned(src + (s.row0 + (p - first)) * a.ldv, 16), 16);
#pragma unroll
          for (int d = 0; d < E; ++d) dst[((int64_t)d << a.ix.page_log2) + e] = in.v[d];
        }
      }
    }
  }
}

template <typename T> static int append_launch(AppendArgs a, int64_t pairs, int layout, hipStream_t s) {
  const int es = sizeof(T);
  int vec = 16 / es;                                      // rows are 16-byte aligned (checked by the caller)
  if (!rot_vec_fits(pairs, a.dh, layout, vec)) vec /= 2;
  if (!rot_vec_fits(pairs, a.dh, layout, vec)) vec = layout == ROT_HALF ? 1 : 2;
  a.sh = rot_shape(pairs, a.dh, layout, vec);
  const int64_t tiles = paged_tiles(a.ix.tokens, a.ix.batch, 1, APPEND_TILE, 2);
  // items of an average sequence's tile decide over how many workgroups a tile is dealt; the angles are shared by two heads
  // once two workgroups' worth of items for every CU are there (bf16, 8 + 8 heads of 64 columns, one head / two / four, us:
  // 64 sequences of one token 4.4 / 5.6 / 6.5, 8 of up to 200 5.7 / 6.3 / 8.0, 37 of up to 60 9.1 / 9.0 / 10.5, of up to 200
  // 15.0 / 12.6 / 14.7, of up to 700 35.3 / 30.4 / 30.3)
  int64_t per = cdiv64(a.ix.tokens, a.ix.batch);
  if (per > APPEND_TILE) per = APPEND_TILE;
  const int heads = a.hkv + a.hq;
  a.hg = a.ix.tokens * a.sh.chunks * heads >= 2 * 256 * 256 ? 2 : 1;
  const int64_t items = per * a.sh.chunks * cdiv64(heads, a.hg) + cdiv64(per, 16 / es) * (a.dh / (16 / es)) * a.hkv;
  int64_t gy = cdiv64(items, 256);      // one item a thread (37 sequences of up to 700: 30.5 us; two items 31.9, four 33.6)
  if (gy > 64) gy = 64;
  const dim3 grid((unsigned)tiles + 1, (unsigned)gy);      // the last one: paged_look_over
  switch (vec) {
    case 8: if constexpr (sizeof(T) == 2) paged_append_kernel<T, 8><<<grid, 256, 0, s>>>(a); break;
    case 4: paged_append_kernel<T, 4><<<grid, 256, 0, s>>>(a); break;
    case 2: paged_append_kernel<T, 2><<<grid, 256, 0, s>>>(a); break;
    default: paged_append_kernel<T, 1><<<grid, 256, 0, s>>>(a); break;
  }
  NEURST_CHECK_LAUNCH("paged_append");
  return NEURST_OK;
}

extern "C" int neurst_paged_append(const void* k, const void* v, const void* q, void* k_pages, void* v_pages, void* q_out,
                                   const int32_t* page_table, const int32_t* cu_new, const int32_t* ctx_len, const double* freq,
                                   int32_t* status, int64_t tokens, int64_t batch, int64_t wide, int64_t ld_table, int64_t n_pages,
                                   int64_t page_size, int64_t kv_heads, int64_t q_heads, int64_t dh, int64_t ldk, int64_t ldv, int64_t ldq,
                                   int64_t ldqo, int64_t pairs, int layout, float mscale, int dtype, void* stream) {
  NEURST_CHECK_ARG(k && v && k_pages && v_pages, "paged_append: null pointer");
  PAGED_CHECK_INDEX("paged_append");
  NEURST_CHECK_ARG((q == nullptr) == (q_out == nullptr), "paged_append: q and q_out go together");
  if (!q) q_heads = 0;
  NEURST_CHECK_ARG(kv_heads > 0 && q_heads >= 0 && kv_heads + q_heads <= 4096, "paged_append: bad head counts");
  NEURST_CHECK_ARG(ldk >= kv_heads * dh && ldv >= kv_heads * dh && (!q || (ldq >= q_heads * dh && ldqo >= q_heads * dh)),
                   "paged_append: a row stride is smaller than its heads");
  NEURST_CHECK_ARG(q != q_out || ldq == ldqo, "paged_append: in place needs equal row strides");
  NEURST_CHECK_ARG(freq ? (pairs > 0 && 2 * pairs <= dh) : pairs == 0, "paged_append: 2 * pairs must be in 2..dh with freq, 0 without");
  NEURST_CHECK_ARG(layout == ROT_HALF || layout == ROT_INTERLEAVED, "paged_append: layout must be 0 (half) or 1 (interleaved)");
  const int64_t es = (int64_t)dtype_size(dtype);
  const uintptr_t align = (uintptr_t)k | (uintptr_t)v | (uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)q_out |
                          (uintptr_t)(ldk * es) | (uintptr_t)(ldv * es) | (q ? (uintptr_t)(ldq * es) | (uintptr_t)(ldqo * es) : 0);
  NEURST_CHECK_ARG(align % 16 == 0, "paged_append: pointers and row strides must be 16-byte aligned");
  if (tokens == 0 || batch == 0) return NEURST_OK;
  const Rows rk = {k, kv_heads * dh * es, ldk * es, tokens}, rv = {v, kv_heads * dh * es, ldv * es, tokens}, rq = {q, q_heads * dh * es, ldq * es, tokens},
             ro = {q_out, q_heads * dh * es, ldqo * es, tokens}, kp = {k_pages, n_pages * page_size * kv_heads * dh * es, 0, 1}, vp = {v_pages, kp.width, 0, 1};
  NEURST_CHECK_ARG(!rows_meet(ro, rk) && !rows_meet(ro, rv) && (q == q_out || !rows_meet(ro, rq)),
                   "paged_append: q_out must be q itself or apart from it, and apart from k and v");
  NEURST_CHECK_ARG(!rows_meet(kp, vp) && !rows_meet(kp, rk) && !rows_meet(kp, rv) && !rows_meet(kp, rq) && !rows_meet(kp, ro) && !rows_meet(vp, rk) &&
                       !rows_meet(vp, rv) && !rows_meet(vp, rq) && !rows_meet(vp, ro),
                   "paged_append: k_pages and v_pages must be apart from each other and from k, v, q and q_out");
  AppendArgs a;
  a.ix = paged_index(page_table, cu_new, ctx_len, tokens, batch, wide, ld_table, page_size, n_pages, true);
  a.k = k; a.v = v; a.q = q; a.k_pages = k_pages; a.v_pages = v_pages; a.q_out = q_out; a.freq = freq; a.status = status;
  a.ldk = ldk; a.ldv = ldv; a.ldq = ldq; a.ldqo = ldqo;
  a.hkv = (int)kv_heads; a.hq = (int)q_heads; a.dh = (int)dh; a.hg = 1; a.mscale = mscale;
  return dtype == NEURST_BF16 ? append_launch<bf16_t>(a, pairs, layout, as_stream(stream)) : append_launch<float>(a, pairs, layout, as_stream(stream));
}
