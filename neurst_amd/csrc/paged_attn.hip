// Attention of a chunk of new tokens over the paged key/value cache (paged.hip has the layout):
//
//   o[i, h] = sum_j softmax_j(scale q[i, h] . k[j, h / group]) v[j, h / group],   j = 0 .. p_i (causal) or 0 .. ctx - 1
//
// over all new tokens i of all sequences, p_i the token's position.  One pass with the running maximum and sum; the table of
// weights never exists.  A token that sees nothing gets zeros.  No reference counterpart in this form: decoding there re-runs
// st/layers/common_attention_v1.py:325-365 on dense caches of equal length.
//
// paged_attn_rows: few rows (single tokens, short chunks).  A workgroup owns 16 rows - tokens x the query heads that share a
// key/value head - and its waves take tiles of 32 keys (fp32: 16) in turn, straight from the pages to the matrix
// instructions.  The first product is taken transposed, S^T = K Q^T, with the keys of a tile dealt to the rows of the
// instruction such that a lane's results are eight CONSECUTIVE keys of one query: after exp2 and the rounding to bf16 they
// are, in place, the operand of O^T = V^T P^T, whose other operand is one 16-byte load from the transposed value pages.  No
// shared memory and no barrier until the waves join their partial results.  Bound by the cache's bytes: 32 sequences of up to
// 32000 keys, 32 heads on 8 of 128 columns, bf16, 396 to 411 us = 5.0 to 5.2 TB/s (a large copy here: 4.8).  Short ones by the chain lengths -
// page - keys - exponentials - values - join: 8 sequences of up to 500 keys, 8 heads of 64 columns, 6.9 us; 13 chunks of up to
// 75 tokens over 611 keys in fp32 24 us.
//
// paged_attn_tiles: many rows, bf16.  A wave owns 32 rows, a workgroup NW of them; tiles of 64 keys go from the pages to shared
// memory by direct loads, one tile ahead of the one in use, and all waves read them from there.  The same transposed
// products with the 32 x 32 x 16 instruction; the key that sits in row r of a 32-key block is chosen again so that a lane's
// results are runs of eight consecutive keys.  The first product of a tile runs beside the exponentials of the tile before,
// the second beside the next maximum.  Bound by what a CU's matrix, vector and shared-memory pipes do not overlap: three
// sequences of up to 4096 rows over 9000 keys, 16 heads on 4 of 128 columns, 500 to 526 us = 806 to 848 TFLOP/s (a large
// product: 1673); the first twenty calls after a pause take 550 to 610 us, until the card's clocks have settled.
// With any one of them left out it would still take four fifths: without the loads 78 %, without reading shared memory 83 %,
// without the exponentials 87 %.
#include "paged.h"

struct PagedAttnArgs {
  PagedIndex ix;
  const void *q, *k_pages, *v_pages;
  void* o;
  float *ws_o, *ws_ml;      // parts > 1: partial results [part][row][dh padded], [part][row][2]
  int32_t* status;
  int64_t ldq, ldo;
  int hkv, group, dh, causal;
  int parts, part_keys;     // the keys in parts of part_keys, one workgroup each
  int32_t* order;           // tiles in the order of their work, most first (null: as they come)
  int64_t tiles;            // of rows, an upper bound
  float scale_log2;         // scale * log2(e): exp(x) = exp2(x log2(e))
};

template <typename T> struct PagedMma;
template <> struct PagedMma<bf16_t> {
  static constexpr int E = 8, KT = 32, NSUB = 2;      // elements of a 16-byte load, keys of a tile, 16-key halves
  typedef bf16x8 V;
  static __device__ __forceinline__ f32x4 mma(V a, V b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct PagedMma<float> {
  static constexpr int E = 4, KT = 16, NSUB = 1;
  typedef f32x4 V;
  static __device__ __forceinline__ f32x4 mma(V a, V b, f32x4 c) {      // four steps of the 4-deep instruction
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
};

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
// exp2(m_old - m_new) where -inf stands for "nothing yet"
__device__ __forceinline__ float safe_max(float m) { return m == -INFINITY ? 0.f : m; }

// what a workgroup of `tile` works on; false: nothing
struct RowTile {
  int b, first_token, last_token, n_rows, kv_end, min_vis;   // keys 0 .. kv_end - 1 are visible to some row, 0 .. min_vis - 1 to every row
  int64_t row0;
  int shift;                                                  // position of token 0
  int row_begin;                                              // first of the tile's rows within the sequence
};
template <int ROWS> __device__ __forceinline__ bool row_tile(const PagedAttnArgs& a, int64_t tile, int lane, RowTile& t) {
  PagedSeq s;
  t.b = paged_locate(a.ix, tile, a.group, ROWS, 1, lane, s);
  if (t.b < 0) return false;
  if (!paged_tile_rows(s, tile - paged_tile_start(s.cu, a.group, ROWS, 1, t.b), a.group, ROWS, t.row_begin, t.n_rows)) return false;
  t.row0 = s.row0;
  t.first_token = t.row_begin / a.group;
  t.last_token = (t.row_begin + t.n_rows - 1) / a.group;
  t.shift = s.ctx - s.new_tokens;
  if (s.ctx == 0) { t.kv_end = t.min_vis = 0; t.shift = -1; }
  else if (a.causal) { t.kv_end = t.shift + t.last_token + 1; t.min_vis = t.shift + t.first_token + 1; }
  else t.kv_end = t.min_vis = s.ctx;
  return true;
}

// a part in which a row sees no key: no sum, and no partial result to read
__device__ __forceinline__ void part_nothing(const PagedAttnArgs& a, const RowTile& t, int kvh, int z, int row) {
  const int64_t wrow = ((int64_t)z * a.ix.tokens + t.row0 + row / a.group) * (a.hkv * a.group) + kvh * a.group + row % a.group;
  a.ws_ml[2 * wrow] = -INFINITY;
  a.ws_ml[2 * wrow + 1] = 0.f;
}

template <typename T, int DH, bool EXACT, int NW>
__global__ void __launch_bounds__(NW * 64, DH <= 64 ? 4 : DH <= 96 ? 3 : DH <= 128 ? 2 : 1) paged_attn_rows(PagedAttnArgs a) {
  typedef PagedMma<T> A;
  typedef typename A::V V;
  constexpr int E = A::E, KT = A::KT, NSUB = A::NSUB, KC = DH / (4 * E), ND = DH / 16;
  constexpr int NDP = ND < 8 ? ND : 8, LD = NDP * 16 + 4;      // dims joined at a time through LDS
  __shared__ float red[NW][16][LD];
  __shared__ float ml[NW][16][2];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, m = lane & 15, g = lane >> 4;
  // heads first: with a multiple of eight of them, or a divisor, an XCD sees few heads' keys through its L2
  const int kvh = (int)(blockIdx.x % (unsigned)a.hkv), z = blockIdx.y;
  if (blockIdx.x / (unsigned)a.hkv == a.tiles) {
    if (kvh == 0 && z == 0) paged_look_over(a.ix, a.status);
    return;
  }
  RowTile t;
  if (!row_tile<16>(a, blockIdx.x / (unsigned)a.hkv, lane, t)) return;
  const int dh = EXACT ? DH : a.dh;
  const int page = 1 << a.ix.page_log2, pmask = page - 1;
  // this lane's query: row m of the tile
  const bool valid = m < t.n_rows;
  const int r = t.row_begin + (valid ? m : 0), token = r / a.group, head = kvh * a.group + r % a.group;
  const T* qp = static_cast<const T*>(a.q) + (t.row0 + token) * a.ldq + (int64_t)head * dh;
  V qf[KC];
#pragma unroll
  for (int c = 0; c < KC; ++c) {
    const int d = c * 4 * E + E * g;
    if (EXACT || d < dh) qf[c] = *reinterpret_cast<const V*>(qp + d);
    else
#pragma unroll
      for (int e = 0; e < E; ++e) qf[c][e] = (T)0.f;
  }
  const int vis = a.causal ? (t.kv_end ? t.shift + token + 1 : 0) : t.kv_end;
  // this part's tiles
  const int nt = (t.kv_end + KT - 1) / KT, per = a.part_keys / KT;
  const int t0 = z * per, t1 = t0 + per < nt ? t0 + per : nt;
  if (t0 >= t1 && a.parts > 1) {
    if (tid < t.n_rows) part_nothing(a, t, kvh, z, t.row_begin + tid);
    return;
  }

  f32x4 acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  float mx = -INFINITY, l = 0.f;
  // Pages of the E-key groups this lane reads of a tile: keys of group m >> 2 for the first product, of group g for the
  // second; -1 refused, or beyond the last key.
  auto page_at = [&](int k) { return k < t.kv_end ? paged_page(a.ix, t.b, k) : -1; };
  auto load_k = [&](int ti, int id, V (&kf)[NSUB][KC]) {
    const int slot = ((ti * KT + E * (m >> 2)) & pmask) + (m & 3);
    const T* kb = static_cast<const T*>(a.k_pages) + ((((int64_t)(id < 0 ? 0 : id) * a.hkv + kvh) << a.ix.page_log2) + slot) * dh;
#pragma unroll
    for (int s = 0; s < NSUB; ++s)
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const int d = c * 4 * E + E * g;
        kf[s][c] = *reinterpret_cast<const V*>(kb + 4 * s * dh + (EXACT || d < dh ? d : 0));
      }
  };
  auto load_v = [&](int ti, int id, V (&vf)[ND]) {
    const T* vb = static_cast<const T*>(a.v_pages) + ((((int64_t)(id < 0 ? 0 : id) * a.hkv + kvh) * dh << a.ix.page_log2) + ((ti * KT + E * g) & pmask));
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const int dim = 16 * d + m;
      vf[d] = *reinterpret_cast<const V*>(vb + ((int64_t)(EXACT || dim < dh ? dim : 0) << a.ix.page_log2));
    }
  };
  // The loads of a wave's next tile go out as soon as the products have taken the registers of this one - the keys' after the
  // first, the values' after the second - and its pages are looked up one tile earlier still, so that the memory always has
  // most of a tile per wave to work on.
  V kf[NSUB][KC], vf[ND];
  int vp = -1, kp1 = -1, vp1 = -1;
  if (t0 + w < t1) {
    const int ti = t0 + w;
    const int kp = page_at(ti * KT + E * (m >> 2));
    vp = page_at(ti * KT + E * g);
    if (ti + NW < t1) {
      kp1 = page_at((ti + NW) * KT + E * (m >> 2));
      vp1 = page_at((ti + NW) * KT + E * g);
    }
    load_k(ti, kp, kf);
    load_v(ti, vp, vf);
  }
  for (int ti = t0 + w; ti < t1; ti += NW) {
    const int base = ti * KT, vg = base + E * g;
    const bool more = ti + NW < t1;
    if (vp < 0 && vg < t.kv_end) paged_report(a.status, PAGED_BAD_PAGE);
    const bool full = base + KT <= t.min_vis && __all(vp >= 0);
    f32x4 sc[NSUB];
#pragma unroll
    for (int s = 0; s < NSUB; ++s) {
      sc[s] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        V k = kf[s][c];
        if (!EXACT && c * 4 * E + E * g >= dh)
#pragma unroll
          for (int e = 0; e < E; ++e) k[e] = (T)0.f;
        sc[s] = A::mma(k, qf[c], sc[s]);
      }
    }
    int kp2 = -1, vp2 = -1;
    if (more) {
      load_k(ti + NW, kp1, kf);
      if (ti + 2 * NW < t1) {
        kp2 = page_at((ti + 2 * NW) * KT + E * (m >> 2));
        vp2 = page_at((ti + 2 * NW) * KT + E * g);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    float x[E];
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = sc[e >> 2][e & 3] * a.scale_log2;     // keys vg + e of query m
    if (!full) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (vp < 0 || vg + e >= vis) x[e] = -INFINITY;
    }
    float tm = x[0];
#pragma unroll
    for (int e = 1; e < E; ++e) tm = fmaxf(tm, x[e]);
    tm = fmaxf(tm, __shfl_xor(tm, 16, 64));
    tm = fmaxf(tm, __shfl_xor(tm, 32, 64));
    const float mn = fmaxf(mx, tm), mu = safe_max(mn);
    if (__any(mn > mx)) {
      const float al = fast_exp2(mx - mu);       // 0 while mx is -inf
      l *= al;
#pragma unroll
      for (int d = 0; d < ND; ++d) acc[d] *= al;
      mx = mn;
    }
    // the weights are rounded to the values' type for the second product (bf16: a relative 2^-8 of each at most, the plain form's
    // own rounding of the output is as large); their sum is taken before that, in fp32
    V p;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float pe = fast_exp2(x[e] - mu);
      l += pe;
      p[e] = (T)pe;
    }
    if (!full) {
      // slots no row sees - unwritten ones, a refused page's - may hold anything, NaN too
      bool odd = false;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          if (vp < 0 || vg + e >= t.kv_end || (!EXACT && 16 * d + m >= dh)) vf[d][e] = (T)0.f;
          odd |= !(fabsf((float)vf[d][e]) <= 3.4028235e38f);
        }
      if (__any(odd)) {
        // values that are not finite, in a tile that some rows see only in part (0 x NaN must not reach those that do not):
        // they are taken out of the product, and added to the rows that see one
        V seen;
#pragma unroll
        for (int e = 0; e < E; ++e) seen[e] = (T)(vp >= 0 && vg + e < vis ? 1.f : 0.f);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          V up, down;
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const float v = (float)vf[d][e];
            up[e] = (T)(v < INFINITY ? 0.f : 1.f);          // +inf and NaN
            down[e] = (T)(v > -INFINITY ? 0.f : 1.f);       // -inf and NaN
            if (!(fabsf(v) <= 3.4028235e38f)) vf[d][e] = (T)0.f;
          }
          const f32x4 zero = f32x4{0.f, 0.f, 0.f, 0.f}, nu = A::mma(up, seen, zero), nd = A::mma(down, seen, zero);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (nu[i] > 0.f) acc[d][i] += INFINITY;
            if (nd[i] > 0.f) acc[d][i] -= INFINITY;
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] = A::mma(vf[d], p, acc[d]);
    if (more) load_v(ti + NW, vp1, vf);
    __builtin_amdgcn_sched_barrier(0);
    vp = vp1;
    kp1 = kp2;
    vp1 = vp2;
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);

  // join the waves: thread (row, part) sums its share of the columns
  if (g == 0) { ml[w][m][0] = mx; ml[w][m][1] = l; }
  const int orow = tid / (4 * NW), part = tid % (4 * NW);
  float M = -INFINITY, L = 0.f, f[NW];
#pragma unroll
  for (int p0 = 0; p0 < ND; p0 += NDP) {
    if (p0) __syncthreads();
#pragma unroll
    for (int d = 0; d < NDP; ++d)
      if (p0 + d < ND) *reinterpret_cast<f32x4*>(&red[w][m][16 * d + 4 * g]) = acc[p0 + d];
    __syncthreads();
    if (p0 == 0) {
#pragma unroll
      for (int i = 0; i < NW; ++i) M = fmaxf(M, ml[i][orow][0]);
      const float mu = safe_max(M);
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        f[i] = fast_exp2(ml[i][orow][0] - mu);
        L += f[i] * ml[i][orow][1];
      }
    }
    if (orow < t.n_rows) {
      const int rr = t.row_begin + orow, tok = rr / a.group, hd = kvh * a.group + rr % a.group;
      const int64_t grow = t.row0 + tok;
      const float inv = L > 0.f ? 1.f / L : (L == L ? 0.f : L);
      for (int c = part * 4; c < NDP * 16; c += 16 * NW) {
        const int dim = p0 * 16 + c;
        if (dim >= dh) break;
        f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NW; ++i) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(&red[i][orow][c]);
          v += x * f[i];
        }
        if (a.parts == 1) {
          T* op = static_cast<T*>(a.o) + grow * a.ldo + (int64_t)hd * dh + dim;
          T out[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) out[j] = from_f32<T>(v[j] * inv);
          __builtin_memcpy(__builtin_assume_aligned(op, 4 * sizeof(T)), out, sizeof(out));
        } else {
          const int64_t wrow = ((int64_t)z * a.ix.tokens + grow) * (a.hkv * a.group) + hd;
          *reinterpret_cast<f32x4*>(a.ws_o + wrow * DH + dim) = v;
        }
      }
      if (a.parts > 1 && p0 == 0 && part == 0) {
        const int64_t wrow = ((int64_t)z * a.ix.tokens + grow) * (a.hkv * a.group) + hd;
        a.ws_ml[2 * wrow] = M;
        a.ws_ml[2 * wrow + 1] = L;
      }
    }
  }
}

// ---- many rows ---------------------------------------------------------------------------------------------------------
typedef __attribute__((ext_vector_type(16))) float f32x16;
constexpr int TILE_WAVES = 4;      // 32 rows each; two waves took longer at most sizes this kernel is chosen for (32 sequences of 204
                                   // rows over 8000 keys: 252 against 209 us)
constexpr int AHEAD = 4;      // fragments read from shared memory ahead of their product

// An image of rows of NC 16-byte chunks: chunk c of row r lies at another place of the row, chosen by r / PER - PER being the
// rows after which the 256 bytes of all banks come round again - so that the lanes of a read, neighbouring rows with one
// chunk, spread over the banks.  The direct loads write places in order and fetch the chunk that belongs there.
template <int NC> struct Image {
  static constexpr int PER = NC % 16 == 0 ? 1 : NC % 8 == 0 ? 2 : 4;
  static constexpr bool XOR = (NC & (NC - 1)) == 0;
  // (of 32 rows more the same where XOR)
  static __device__ __forceinline__ int place(int r, int c) {
    if constexpr (XOR) return c ^ ((r / PER) & (NC - 1));
    const int x = c + (r / PER) % NC;
    return x >= NC ? x - NC : x;
  }
  static __device__ __forceinline__ int chunk(int r, int at) {
    if constexpr (XOR) return at ^ ((r / PER) & (NC - 1));
    const int x = at - (r / PER) % NC;
    return x < 0 ? x + NC : x;
  }
};
// key of row r of the key image (32-key blocks), see above: bits 0, 1 stay, 2 -> 3, 3 -> 2, 4 stays
__device__ __forceinline__ int image_key(int r) { return (r & ~12) | ((r & 4) << 1) | ((r & 8) >> 1); }

__device__ __forceinline__ void load_to_lds(const void* src, char* dst) {      // 16 bytes a lane to dst + 16 * lane
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src, (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}

template <int DH, bool EXACT>
__global__ void __launch_bounds__(TILE_WAVES * 64, DH <= 128 ? 2 : 1) paged_attn_tiles(PagedAttnArgs a) {
  constexpr int NW = TILE_WAVES, ROWS = 32 * NW, KT = 64, NC = DH / 8, STEPS = DH / 16, ND = DH / 32, IMG = KT * DH * 2;
  typedef Image<NC> KI;
  typedef Image<8> VI;
  extern __shared__ __attribute__((aligned(1024))) char smem[];                 // keys [2], values [2], what `clean` notes
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), m = lane & 31, h = lane >> 5;
  const int kvh = (int)(blockIdx.x % (unsigned)a.hkv), z = blockIdx.y;
  if (blockIdx.x / (unsigned)a.hkv == a.tiles) {
    if (kvh == 0 && z == 0) paged_look_over(a.ix, a.status);
    return;
  }
  RowTile t;
  int64_t tile = blockIdx.x / (unsigned)a.hkv;
  if (a.order) tile = a.order[tile];
  if (!row_tile<ROWS>(a, tile, lane, t)) return;
  const int dh = EXACT ? DH : a.dh;
  const int page = 1 << a.ix.page_log2, pmask = page - 1;
  const int row = 32 * w + m;
  const bool valid = row < t.n_rows;
  const int r = t.row_begin + (valid ? row : 0), token = r / a.group, head = kvh * a.group + r % a.group;
  const bf16_t* qp = static_cast<const bf16_t*>(a.q) + (t.row0 + token) * a.ldq + (int64_t)head * dh;
  const float c_abs = fabsf(a.scale_log2);
  bf16x8 qf[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int d = 16 * s + 8 * h;
    u32x4 x = u32x4{0, 0, 0, 0};
    if (EXACT || d < dh) x = *reinterpret_cast<const u32x4*>(qp + d);
    if (a.scale_log2 < 0.f) x ^= 0x80008000u;       // the sign of the scale goes to the queries: the maximum is one of s |scale|
    qf[s] = __builtin_bit_cast(bf16x8, x);
  }
  const int vis = a.causal ? (t.kv_end ? t.shift + token + 1 : 0) : t.kv_end;
  // keys some row of this wave sees, keys all its rows see
  const int w_rows = t.n_rows - 32 * w;
  int w_end = 0, w_min = 0;
  if (w_rows > 0) {
    w_end = t.kv_end;
    w_min = t.min_vis;
    if (a.causal && t.kv_end) {
      w_end = t.shift + (t.row_begin + 32 * w + (w_rows < 32 ? w_rows : 32) - 1) / a.group + 1;
      w_min = t.shift + (t.row_begin + 32 * w) / a.group + 1;
    }
    w_end = __builtin_amdgcn_readfirstlane(w_end);
    w_min = __builtin_amdgcn_readfirstlane(w_min);
  }
  const int nt = (t.kv_end + KT - 1) / KT, per = a.part_keys / KT;
  const int t0 = z * per, t1 = t0 + per < nt ? t0 + per : nt;
  if (t0 >= t1 && a.parts > 1) {
    if (valid && h == 0) part_nothing(a, t, kvh, z, r);
    return;
  }

  // pages of the four 16-key groups of a tile, in lanes 0..3 of every quad: -1 refused, or beyond the last key
  auto pages_of = [&](int ti) {
    const int k = ti * KT + 16 * (lane & 3);
    const int id = ti < t1 && k < t.kv_end ? paged_page(a.ix, t.b, k) : -1;
    if (id < 0 && ti < t1 && k < t.kv_end && lane < 4 && w == 0) paged_report(a.status, PAGED_BAD_PAGE);
    return id;
  };
  // A wave's load moves a piece of 64 chunks.  A piece of the key image lies within 16 keys, so within one page: its base is a
  // scalar and the lanes' offsets are the same for every tile.  A piece of the value image is 8 columns x 64 keys: a lane's
  // 16-key group is one of two, by the piece's parity.
  constexpr int NP = (NC + NW - 1) / NW;
  const char* kpool = static_cast<const char*>(a.k_pages);
  const char* vpool = static_cast<const char*>(a.v_pages);
  int koff[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int n = (i * NW + w) * 64 + lane, rr = n / NC, c = KI::chunk(rr, n % NC);
    koff[i] = ((image_key(rr & 31) & 15 & pmask) * dh + (EXACT || 8 * c < dh ? 8 * c : 0)) * 2;
  }
  const int vc = VI::chunk(lane >> 3, lane & 7);           // chunk of an even piece; of an odd one: vc ^ 4
  const int64_t vrow = (int64_t)(lane >> 3) << (a.ix.page_log2 + 1);
  const int voff0 = vc * 16, voff1 = (vc ^ 4) * 16;        // pages of 64 slots or more hold a tile's keys in one piece
  auto issue_k = [&](int i, int ti, int ids) __attribute__((always_inline)) {      // this wave's piece i of a key image
    const int piece = i * NW + w, grp = piece * 4 / NC;    // the 16-key group
    if (NC % NW == 0 || piece < NC) {
      int id = __builtin_amdgcn_readlane(ids, grp);
      id = id < 0 ? 0 : id;
      const char* src = kpool + (((((int64_t)id * a.hkv + kvh) << a.ix.page_log2) + ((ti * KT + 16 * grp) & pmask)) * dh) * 2;
      load_to_lds(src + koff[i], smem + (ti & 1) * IMG + piece * 1024);
    }
  };
  const char* vsrc[2];                                     // where the value pieces of the next tile come from
  auto aim_v = [&](int ti, int ids) __attribute__((always_inline)) {
    if (page >= 64) {
      int id = __builtin_amdgcn_readlane(ids, 0);
      id = id < 0 ? 0 : id;
      const char* at = vpool + (((((int64_t)id * a.hkv + kvh) * dh) << a.ix.page_log2) + ((ti * KT) & pmask)) * 2;
      vsrc[0] = at + vrow + voff0;
      vsrc[1] = at + vrow + voff1;
    } else {
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        const int c = vc ^ (4 * o);
        int id = __shfl(ids, c >> 1, 64);
        id = id < 0 ? 0 : id;
        vsrc[o] = vpool + (((((int64_t)id * a.hkv + kvh) * dh) << a.ix.page_log2) + ((8 * c) & pmask)) * 2 + vrow;
      }
    }
  };
  auto issue_v = [&](int i, int ti) __attribute__((always_inline)) {
    const int piece = i * NW + w;
    if ((NC % NW == 0 || piece < NC) && (EXACT || piece * 8 < dh))
      load_to_lds(vsrc[piece & 1] + ((int64_t)piece << (a.ix.page_log2 + 4)), smem + (2 + (ti & 1)) * IMG + piece * 1024);
  };

  f32x16 acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;
  float mx = -INFINITY, l = 0.f;      // maximum in units of log2, sum of this lane's half
  auto okay_of = [&](int ids) { return (unsigned)(__ballot(ids >= 0) & 0xf); };
  auto full_of = [&](int ti, unsigned okay) { return ti * KT + KT <= w_min && okay == 0xf; };
  auto key_of = [&](int ti, int b, int st, int mm) __attribute__((always_inline)) {
    const char* img = smem + (ti & 1) * IMG;
    bf16x8 k = *reinterpret_cast<const bf16x8*>(img + 32 * b * NC * 16 + (mm * NC + KI::place(KI::XOR ? mm : 32 * b + mm, 2 * st + h)) * 16);
    if (!EXACT && 16 * st + 8 * h >= dh) k = bf16x8{};
    return k;
  };
  auto value_of = [&](int ti, int ks, int d, int mm) __attribute__((always_inline)) {
    return *reinterpret_cast<const bf16x8*>(smem + (2 + (ti & 1)) * IMG + 32 * d * 128 + (mm * 8 + VI::place(mm, 2 * ks + h)) * 16);
  };
  auto mask = [&](int ti, unsigned okay, f32x16 (&s)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = 32 * b + 16 * (i >> 3) + 8 * h + (i & 7);
        if (ti * KT + key >= vis || !(okay >> (2 * b + (i >> 3)) & 1)) s[b][i] = -INFINITY;
      }
  };
  auto max_of = [&](const f32x16 (&s)[2]) __attribute__((always_inline)) {
    float tm = s[0][0];
#pragma unroll
    for (int i = 1; i < 32; ++i) tm = fmaxf(tm, s[i >> 4][i & 15]);
    return tm;
  };
  // The maximum moves only when it has grown by 8 (a factor of 256 in the weights, which fp32 sums and bf16 weights hold as
  // well as 1): the accumulators are rescaled a few times a row instead of every tile.
  auto raise_max = [&](float tm) __attribute__((always_inline)) {
    tm = fmaxf(tm, __shfl_xor(tm, 32, 64)) * c_abs;
    if (__any(tm > mx + 8.f || (mx == -INFINITY && tm > -INFINITY))) {
      const float mn = fmaxf(mx, tm), al = fast_exp2(mx - safe_max(mn));
      l *= al;
#pragma unroll
      for (int d = 0; d < ND; ++d) acc[d] *= al;
      mx = mn;
    }
  };
  auto weight = [&](const f32x16 (&s)[2], int i, float mu, float& sum, bf16x8 (&p)[4]) __attribute__((always_inline)) {
    const float pe = fast_exp2(fmaf(s[i >> 4][i & 15], c_abs, -mu));
    sum += pe;
    p[i >> 3][i & 7] = (bf16_t)pe;         // rounded for the second product only, as in the other kernel
  };

  // Software pipeline, a tile t at a time: the first product of tile t + 1 runs while the vector unit makes the weights of
  // tile t, the second product of t while it finds the maximum of t + 1.  The keys of t + 2 and the values of t + 1 are loaded on the
  // way: both are used in the next turn, which begins with waiting for them.
  const int t1w = (w_end + KT - 1) / KT < t1 ? (w_end + KT - 1) / KT : t1;      // the wave's own end
  int id0 = pages_of(t0), id1 = pages_of(t0 + 1), id2 = pages_of(t0 + 2);
  f32x16 s[2];
  if (tid == 0) *reinterpret_cast<volatile int*>(smem + 4 * IMG + 16 * DH) = 0;
  if (t0 < t1) {
    aim_v(t0, id0);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      issue_k(i, t0, id0);
      issue_v(i, t0);
      if (t0 + 1 < t1) issue_k(i, t0 + 1, id1);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (t0 < t1w) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int st = 0; st < STEPS; ++st) s[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(key_of(t0, b, st, m), qf[st], st ? s[b] : f32x16{}, 0, 0, 0);
      const unsigned okay = okay_of(id0);
      if (!full_of(t0, okay)) mask(t0, okay, s);
      raise_max(max_of(s));
    }
  }
  // Values in a tile that some rows see only in part: slots nobody sees - unwritten ones, a refused page's - may hold anything
  // and become 0, and so do values that are not finite, whose product with a weight of 0 would be NaN; those are noted by
  // column and key and added to the rows that see them.
  uint8_t* noted = reinterpret_cast<uint8_t*>(smem + 4 * IMG);         // [+inf or NaN, -inf or NaN][column][key / 8]: a bit a key
  volatile int* noted_tile = reinterpret_cast<volatile int*>(smem + 4 * IMG + 16 * DH);
  auto clean = [&](int ti, unsigned okay) __attribute__((always_inline)) {
#pragma unroll 1
    for (int n = tid; n < DH * 8; n += NW * 64) {
      const int dim = n >> 3, c = VI::chunk(dim, n & 7), key = ti * KT + 8 * c;
      bf16x8* at = reinterpret_cast<bf16x8*>(smem + (2 + (ti & 1)) * IMG) + n;
      bf16x8 v = *at;
      unsigned up = 0, down = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = (float)v[e];
        if (!(okay >> (c >> 1) & 1) || key + e >= t.kv_end || (!EXACT && dim >= dh)) v[e] = (bf16_t)0.f;
        else if (!(fabsf(x) <= 3.4028235e38f) && key + e >= t.min_vis) {
          up |= x < INFINITY ? 0u : 1u << e;
          down |= x > -INFINITY ? 0u : 1u << e;
          v[e] = (bf16_t)0.f;
        }
      }
      *at = v;
      noted[dim * 8 + c] = (uint8_t)up;
      noted[(DH + dim) * 8 + c] = (uint8_t)down;
      if (up | down) *noted_tile = ti + 1;
    }
  };
  for (int ti = t0; ti < t1; ++ti) {
    if (ti > t0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // this wave's pieces of keys ti + 1 and values ti have landed
    __syncthreads();                                                   // everyone's have, and everyone has left the buffers of ti - 1
    const bool next = ti + 1 < t1, after = ti + 2 < t1;
    if (next) aim_v(ti + 1, id1);
    const int id3 = pages_of(ti + 3);
    const unsigned okay = okay_of(id0);
    const bool part = ti * KT + KT > t.min_vis || okay != 0xf;         // the same for the whole workgroup
    if (part) {
      clean(ti, okay);
      __syncthreads();
    }
    if (ti < t1w) {
      int mm = m;
      asm volatile("" : "+v"(mm));                         // image addresses are made here, not kept over the loop
      mm &= 31;
      const float mu = safe_max(mx);
      bf16x8 p[4];
      float sum = 0.f;
      __builtin_amdgcn_sched_barrier(0);
      // (of no use after the wave's last tile)
      f32x16 n[2];
      {
        constexpr int N = 2 * STEPS;
        bf16x8 k[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) k[i] = key_of(ti + 1, i / STEPS, i % STEPS, mm);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          n[i / STEPS] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[i % AHEAD], qf[i % STEPS], i % STEPS ? n[i / STEPS] : f32x16{}, 0, 0, 0);
          if (i + AHEAD < N) k[i % AHEAD] = key_of(ti + 1, (i + AHEAD) / STEPS, (i + AHEAD) % STEPS, mm);
#pragma unroll
          for (int e = 32 * i / N; e < 32 * (i + 1) / N; ++e) weight(s, e, mu, sum, p);
          // a load's way into the memory pipe takes as long as some of these steps: they are spread over them
          if (i * NP / N != (i + 1) * NP / N && after) issue_k(i * NP / N, ti + 2, id2);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      // made here, beside the products, and not where they are used
      asm volatile("" : "+v"(p[0]), "+v"(p[1]), "+v"(p[2]), "+v"(p[3]), "+v"(sum));
      l += sum;
      s[0] = n[0];
      s[1] = n[1];
      const unsigned ok1 = okay_of(id1);
      if (!full_of(ti + 1, ok1)) mask(ti + 1, ok1, s);
      __builtin_amdgcn_sched_barrier(0);
      float tm = s[0][0];
      {
        constexpr int N = 4 * ND;
        bf16x8 v[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) v[i] = value_of(ti, i / ND, i % ND, mm);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          acc[i % ND] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[i % AHEAD], p[i / ND], acc[i % ND], 0, 0, 0);
          if (i + AHEAD < N) v[i % AHEAD] = value_of(ti, (i + AHEAD) / ND, (i + AHEAD) % ND, mm);
#pragma unroll
          for (int e = 32 * i / N; e < 32 * (i + 1) / N; ++e) tm = fmaxf(tm, s[e >> 4][e & 15]);
          if (i * NP / N != (i + 1) * NP / N && next) issue_v(i * NP / N, ti + 1);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      asm volatile("" : "+v"(tm));
      if (part && *noted_tile == ti + 1) {
        uint64_t sees = 0;
#pragma unroll
        for (int k = 0; k < KT; ++k)
          if (ti * KT + k < vis && (okay >> (k >> 4) & 1)) sees |= 1ull << k;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int dim = 32 * d + (i & 3) + 8 * (i >> 2) + 4 * h;
            if (*reinterpret_cast<const uint64_t*>(noted + dim * 8) & sees) acc[d][i] += INFINITY;
            if (*reinterpret_cast<const uint64_t*>(noted + (DH + dim) * 8) & sees) acc[d][i] -= INFINITY;
          }
      }
      if (ti + 1 < t1w) raise_max(tm);
    } else {                                               // this wave's rows see no more, but others' do
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        if (after) issue_k(i, ti + 2, id2);
        if (next) issue_v(i, ti + 1);
      }
    }
    id0 = id1;
    id1 = id2;
    id2 = id3;
  }
  l += __shfl_xor(l, 32, 64);
  if (!valid) return;
  const int64_t grow = t.row0 + token;
  if (a.parts == 1) {
    const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
    bf16_t* op = static_cast<bf16_t*>(a.o) + grow * a.ldo + (int64_t)head * dh;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int dim = 32 * d + 2 * i + 4 * h;
        bf16x4 x;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = (bf16_t)(acc[d][i + j] * inv);
        if (EXACT || dim < dh) *reinterpret_cast<bf16x4*>(op + dim) = x;
      }
  } else {
    const int64_t wrow = ((int64_t)z * a.ix.tokens + grow) * (a.hkv * a.group) + head;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int dim = 32 * d + 2 * i + 4 * h;
        *reinterpret_cast<f32x4*>(a.ws_o + wrow * DH + dim) = f32x4{acc[d][i], acc[d][i + 1], acc[d][i + 2], acc[d][i + 3]};
      }
    if (h == 0) {
      a.ws_ml[2 * wrow] = mx;
      a.ws_ml[2 * wrow + 1] = l;
    }
  }
}

// Tiles by the keys their rows see, most first, so that the last workgroups to start are short ones: a causal batch of three
// sequences of 3600 to 9000 tokens leaves a quarter of the chip's time idle in the order it comes, a twentieth like this.
// One workgroup, a counting sort over 1024 classes; which of two tiles of a class comes first does not matter.
__global__ void __launch_bounds__(1024) paged_attn_order(PagedAttnArgs a, int rows) {
  __shared__ uint32_t first[1024];
  __shared__ uint32_t sums[16];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  first[tid] = 0;
  __syncthreads();
  const int64_t most = (((int64_t)a.ix.wide << a.ix.page_log2) + 1023) >> 10;      // keys of a class
  auto class_of = [&](int64_t tile) {
    int lo = 0, hi = a.ix.batch;                            // the last sequence that starts at or before the tile
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (paged_tile_start(a.ix.cu[mid], a.group, rows, 1, mid) <= tile) lo = mid;
      else hi = mid;
    }
    const PagedSeq s = paged_seq(a.ix, lo);
    const int64_t own = tile - paged_tile_start(a.ix.cu[lo], a.group, rows, 1, lo), total = (int64_t)s.new_tokens * a.group;
    if (own < 0 || own * rows >= total) return 1023;        // nothing to do
    const int64_t last = (own + 1) * rows < total ? ((own + 1) * rows - 1) / a.group : s.new_tokens - 1;
    const int64_t keys = a.causal && s.ctx ? s.ctx - s.new_tokens + last + 1 : s.ctx;
    const int64_t c = keys / most;
    return 1023 - (int)(c < 1023 ? c : 1023);
  };
  for (int64_t i = tid; i < a.tiles; i += 1024) atomicAdd(&first[class_of(i)], 1u);
  __syncthreads();
  const uint32_t mine = first[tid];
  uint32_t inc = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t x = (uint32_t)__shfl((int)inc, (lane - o) & 63, 64);
    if (lane >= o) inc += x;
  }
  if (lane == 63) sums[w] = inc;
  __syncthreads();
  uint32_t before = inc - mine;
  for (int i = 0; i < w; ++i) before += sums[i];
  first[tid] = before;
  __syncthreads();
  for (int64_t i = tid; i < a.tiles; i += 1024) a.order[atomicAdd(&first[class_of(i)], 1u)] = (int32_t)i;
}

// Joins the parts: one wave a row (token x head).  The rows are found by the tiles that wrote the parts, so that rows no
// sequence owns - behind the last one, or of lengths that were refused - are left as they were, like those of whole keys (2100
// rows of 8 heads in five parts: 10.3 us; over the tensors' rows, which does not tell them, 8.4).
template <typename T, int ROWS>
__global__ void __launch_bounds__(256) paged_attn_join(PagedAttnArgs a, int ldw, int64_t rows) {
  const int lane = threadIdx.x & 63, heads = a.hkv * a.group;
  const int kvh = (int)(blockIdx.x % (unsigned)a.hkv), own = blockIdx.y * 4 + (threadIdx.x >> 6);
  RowTile t;
  if (!row_tile<ROWS>(a, blockIdx.x / (unsigned)a.hkv, lane, t) || own >= t.n_rows) return;
  const int r = t.row_begin + own;
  const int head = kvh * a.group + r % a.group;
  const int64_t token = t.row0 + r / a.group, row = token * heads + head;
  // lane z holds part z's maximum and sum (at most 64 parts), and what its partial result counts
  float pm = -INFINITY, pl = 0.f;
  if (lane < a.parts) {
    const int64_t at = 2 * (lane * rows + row);
    pm = a.ws_ml[at];
    pl = a.ws_ml[at + 1];
  }
  const float M = wave_max(pm), f = fast_exp2(pm - safe_max(M)), L = wave_sum(f * pl);
  f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
  const int dim = lane * 4;
  for (int z = 0; z < a.parts; ++z) {
    const float fz = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), z));
    // a sum of 0: the row sees nothing there and no partial result was written; one that counts for nothing (fz 0) is added all
    // the same, as a NaN of it has to reach the result
    if (__builtin_amdgcn_readlane(__builtin_bit_cast(int, pl), z) != 0 && dim < a.dh)
      v += *reinterpret_cast<const f32x4*>(a.ws_o + (z * rows + row) * ldw + dim) * fz;
  }
  if (dim >= a.dh) return;
  const float inv = L > 0.f ? 1.f / L : (L == L ? 0.f : L);
  T out[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) out[j] = from_f32<T>(v[j] * inv);
  T* op = static_cast<T*>(a.o) + token * a.ldo + (int64_t)head * a.dh + dim;
  __builtin_memcpy(__builtin_assume_aligned(op, 4 * sizeof(T)), out, sizeof(out));
}

static int padded_dh(int64_t dh) {
  for (int d : {32, 64, 96, 128, 192, 256})
    if (dh <= d) return d;
  return 0;
}

// What a call launches, from its sizes alone (the lengths are on the device): the kernel, and into how many parts the keys are
// split so that the chip is filled.  Times below are bf16 with causal masks, ragged sequences of up to the stated sizes.
struct AttnPlan { int tiles, waves, parts, part_keys, order; };
static int plan_rows(const AttnPlan& p) { return p.tiles ? 32 * TILE_WAVES : 16; }
static AttnPlan attn_plan(int64_t tokens, int64_t batch, int64_t wide, int64_t page_size, int64_t kv_heads, int64_t group, int64_t dh, int dtype,
                          bool scaled) {
  AttnPlan p;
  const int64_t rows = cdiv64(tokens, batch) * group, keys = wide * page_size;      // rows of an average sequence to a key/value head
  // paged_attn_tiles reads a key once for 128 rows, but a workgroup walks its keys alone; in paged_attn_rows the waves share
  // them.  So the first needs rows to fill it and work to fill the chip - here from 2/3 G products (rows / tiles in us, 8
  // key/value heads of 64 columns: 1 x 204 rows x 500 keys 8.6 / 20.7, 8 x 102 x 500 10.4 / 19.9, 32 x 102 x 500 21 / 25,
  // 1 x 102 x 8000 29 / 26, 32 x 204 x 500 32 / 25, 8 x 204 x 8000 81 / 45, 32 x 25 x 8000 90 / 120, 32 x 409 x 8000 662 / 231)
  p.tiles = dtype == NEURST_BF16 && scaled && rows > 32 && (double)(batch * kv_heads) * (double)(rows * keys) * (double)dh >= 5.0 * (1 << 27);
  const int64_t wgs = batch * cdiv64(rows, plan_rows(p)) * kv_heads;
  // Parts of equal length, not of equal number a sequence: the workgroups of a ragged batch then take equally long.  At least
  // 512 keys each (tiles, 128 rows over 4 x 8000 keys of 128 columns: 45 us, with 1024 keys 58).
  // Tiles: as many parts as all run at once, two workgroups a CU up to 128 columns, then one.  One part more than that costs a
  // second turn (3 x 700 rows x 16000 keys: 199 against 152 us; whole, 2 x 1000 x 30000: 945 against 257).
  // Rows: a second launch joins the parts (4 to 10 us), so up to 1024 keys stay whole (4 sequences of one row, 1000 keys: 12.4 us, in
  // two parts 11.5 and a launch more; 2000 keys: 22 against 13, 16000 keys: 157 against 36); up to 4096 workgroups even out
  // ragged lengths (32 sequences, 32 heads on 8 of 128 columns, 32000 keys: 476 us, with 512 or 1024 workgroups 560).
  const int64_t at_once = dh <= 128 ? 512 : 256, least = 512;
  int64_t part = p.tiles ? cdiv64(keys, wgs < at_once ? at_once / wgs : 1) : cdiv64(keys * wgs, 4096);
  part = cdiv64(part, p.tiles ? 64 : least) * (p.tiles ? 64 : least);
  if (part < least) part = least;
  if (part * 64 < keys) part = cdiv64(keys, 64);
  if (part >= keys || keys <= 1024) part = keys;
  p.part_keys = (int)(cdiv64(cdiv64(keys, cdiv64(keys, part)), 64) * 64);
  p.parts = (int)cdiv64(keys, p.part_keys);
  // waves of a row workgroup: eight where few workgroups run (one row, 8 heads of 64 columns, 500 keys: 8 sequences 8.0 us
  // against 8.4 with four, 32 sequences 10.3 / 11.0; 64 sequences 14.9 / 13.8, 128 sequences 24.8 / 22.4)
  p.waves = p.tiles ? TILE_WAVES : wgs * p.parts <= 256 ? 8 : 4;
  // tiles sorted by work (by one workgroup, so up to 2^16 of them) where more workgroups are launched than run at once (three
  // sequences of up to 4096 rows over 9000 keys, 16 heads on 4 of 128 columns: 519 us, as they come 548)
  p.order = p.tiles && p.parts == 1 && wgs > at_once && paged_tiles(tokens, batch, group, plan_rows(p), 1) <= (1 << 16);
  return p;
}
static int64_t plan_bytes(const AttnPlan& p, int64_t tokens, int64_t batch, int64_t q_heads, int64_t group, int64_t dh) {
  if (p.order) return paged_tiles(tokens, batch, group, plan_rows(p), 1) * 4;
  return p.parts <= 1 ? 0 : (int64_t)p.parts * tokens * q_heads * (padded_dh(dh) + 2) * 4;
}

extern "C" int64_t neurst_paged_attention_workspace_bytes(int64_t tokens, int64_t batch, int64_t wide, int64_t page_size, int64_t q_heads,
                                                          int64_t kv_heads, int64_t dh, int dtype) {
  if (tokens <= 0 || batch <= 0 || wide <= 0 || page_size <= 0 || q_heads <= 0 || kv_heads <= 0 || dh <= 0 || dh > 256) return 0;
  const int64_t group = q_heads / kv_heads;
  const int64_t a = plan_bytes(attn_plan(tokens, batch, wide, page_size, kv_heads, group, dh, dtype, true), tokens, batch, q_heads, group, dh);
  const int64_t b = plan_bytes(attn_plan(tokens, batch, wide, page_size, kv_heads, group, dh, dtype, false), tokens, batch, q_heads, group, dh);
  return a > b ? a : b;
}

template <int DH> static int tiles_launch(const PagedAttnArgs& a, dim3 grid, hipStream_t s) {
  constexpr int LDS = 2 * 2 * 64 * DH * 2 + 16 * DH + 16;
  auto kernel = a.dh == DH ? paged_attn_tiles<DH, true> : paged_attn_tiles<DH, false>;
  if (LDS > 64 * 1024) {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (e != hipSuccess) { neurst_set_error("paged_attention: cannot reserve %d B of LDS: %s", LDS, hipGetErrorString(e)); return NEURST_E_LAUNCH; }
  }
  kernel<<<grid, TILE_WAVES * 64, LDS, s>>>(a);
  return NEURST_OK;
}

template <typename T> static int attn_launch(PagedAttnArgs a, AttnPlan plan, void* ws, hipStream_t s) {
  const int pd = padded_dh(a.dh);
  const int64_t rows = a.ix.tokens * a.hkv * a.group;
  if (a.parts > 1) {
    a.ws_o = static_cast<float*>(ws);
    a.ws_ml = a.ws_o + a.parts * rows * pd;
  }
  const int per = plan_rows(plan);
  a.tiles = paged_tiles(a.ix.tokens, a.ix.batch, a.group, per, 1);
  // behind the tiles one more workgroup for paged_look_over: a whole tile's, so that a head stays with its XCD in every part
  // (three sequences of up to 700 rows over 16000 keys in five parts: 98 us, with a single one 104)
  const dim3 grid((unsigned)((a.tiles + 1) * a.hkv), (unsigned)a.parts);
  if (plan.order) {
    a.order = static_cast<int32_t*>(ws);
    paged_attn_order<<<1, 1024, 0, s>>>(a, per);
    NEURST_CHECK_LAUNCH("paged_attention order");
  }
  if (plan.tiles) {
    if constexpr (sizeof(T) == 2) {
      switch (pd) {
        case 32: if (int e = tiles_launch<32>(a, grid, s)) return e; break;
        case 64: if (int e = tiles_launch<64>(a, grid, s)) return e; break;
        case 96: if (int e = tiles_launch<96>(a, grid, s)) return e; break;
        case 128: if (int e = tiles_launch<128>(a, grid, s)) return e; break;
        case 192: if (int e = tiles_launch<192>(a, grid, s)) return e; break;
        case 256: if (int e = tiles_launch<256>(a, grid, s)) return e; break;
      }
    }
  } else {
#define ROWS_CASE(D)                                                                       \
  case D:                                                                                  \
    if (plan.waves == 8) {                                                                 \
      if (a.dh == D) paged_attn_rows<T, D, true, 8><<<grid, 512, 0, s>>>(a);                \
      else paged_attn_rows<T, D, false, 8><<<grid, 512, 0, s>>>(a);                         \
    } else {                                                                               \
      if (a.dh == D) paged_attn_rows<T, D, true, 4><<<grid, 256, 0, s>>>(a);                \
      else paged_attn_rows<T, D, false, 4><<<grid, 256, 0, s>>>(a);                         \
    }                                                                                      \
    break;
    switch (pd) {
      ROWS_CASE(32) ROWS_CASE(64) ROWS_CASE(96) ROWS_CASE(128) ROWS_CASE(192) ROWS_CASE(256)
    }
#undef ROWS_CASE
  }
  NEURST_CHECK_LAUNCH("paged_attention");
  if (a.parts > 1) {
    const dim3 joins((unsigned)(a.tiles * a.hkv), (unsigned)(per / 4));
    if constexpr (sizeof(T) == 2) {
      if (plan.tiles) paged_attn_join<T, 32 * TILE_WAVES><<<joins, 256, 0, s>>>(a, pd, rows);
    }
    if (!plan.tiles) paged_attn_join<T, 16><<<joins, 256, 0, s>>>(a, pd, rows);
    NEURST_CHECK_LAUNCH("paged_attention join");
  }
  return NEURST_OK;
}

extern "C" int neurst_paged_attention(const void* q, const void* k_pages, const void* v_pages, void* o, const int32_t* page_table,
                                      const int32_t* cu_new, const int32_t* ctx_len, int32_t* status, int64_t tokens, int64_t batch,
                                      int64_t wide, int64_t ld_table, int64_t n_pages, int64_t page_size, int64_t q_heads, int64_t kv_heads,
                                      int64_t dh, int64_t ldq, int64_t ldo, float scale, int causal, int dtype, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
  NEURST_CHECK_ARG(q && k_pages && v_pages && o, "paged_attention: null pointer");
  PAGED_CHECK_INDEX("paged_attention");
  NEURST_CHECK_ARG(kv_heads > 0 && kv_heads <= 4096 && q_heads > 0 && q_heads <= 65536 && q_heads % kv_heads == 0,
                   "paged_attention: q_heads must be a multiple of kv_heads");
  NEURST_CHECK_ARG((tokens * (q_heads / kv_heads) / 16 + batch) * kv_heads <= INT32_MAX && tokens * (q_heads / kv_heads) <= INT32_MAX,
                   "paged_attention: too many rows");
  NEURST_CHECK_ARG(ldq >= q_heads * dh && ldo >= q_heads * dh, "paged_attention: a row stride is smaller than its heads");
  NEURST_CHECK_ARG(fabsf(scale) <= 2.3e38f, "paged_attention: scale must be finite, and so must scale * log2(e)");
  const int64_t es = (int64_t)dtype_size(dtype);
  const uintptr_t align = (uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)o | (uintptr_t)(ldq * es) | (uintptr_t)(ldo * es);
  NEURST_CHECK_ARG(align % 16 == 0, "paged_attention: pointers and row strides must be 16-byte aligned");
  if (tokens == 0 || batch == 0) return NEURST_OK;
  PagedAttnArgs a;
  a.ix = paged_index(page_table, cu_new, ctx_len, tokens, batch, wide, ld_table, page_size, n_pages, causal != 0);
  a.q = q; a.k_pages = k_pages; a.v_pages = v_pages; a.o = o; a.status = status;
  a.ws_o = a.ws_ml = nullptr;
  a.order = nullptr;
  a.ldq = ldq; a.ldo = ldo; a.hkv = (int)kv_heads; a.group = (int)(q_heads / kv_heads); a.dh = (int)dh; a.causal = causal ? 1 : 0;
  const AttnPlan plan = attn_plan(tokens, batch, wide, page_size, kv_heads, a.group, dh, dtype, scale != 0.f);
  a.parts = plan.parts;
  a.part_keys = plan.part_keys;
  a.scale_log2 = scale * 1.44269504088896340736f;
  const int64_t need = neurst_paged_attention_workspace_bytes(tokens, batch, wide, page_size, q_heads, kv_heads, dh, dtype);
  NEURST_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
                   "paged_attention: the workspace must hold neurst_paged_attention_workspace_bytes() bytes, 16-byte aligned");
  const int64_t pool = n_pages * page_size * kv_heads * dh * es;
  const Rows ro = {o, q_heads * dh * es, ldo * es, tokens}, rq = {q, q_heads * dh * es, ldq * es, tokens}, kp = {k_pages, pool, 0, 1}, vp = {v_pages, pool, 0, 1},
             ws = {workspace, need, 0, 1};
  NEURST_CHECK_ARG(!rows_meet(ro, rq) && !rows_meet(ro, kp) && !rows_meet(ro, vp), "paged_attention: o must be apart from q and the pages");
  NEURST_CHECK_ARG(!rows_meet(ws, ro) && !rows_meet(ws, rq) && !rows_meet(ws, kp) && !rows_meet(ws, vp),
                   "paged_attention: the workspace must be apart from q, o and the pages");
  return dtype == NEURST_BF16 ? attn_launch<bf16_t>(a, plan, workspace, as_stream(stream)) : attn_launch<float>(a, plan, workspace, as_stream(stream));
}
