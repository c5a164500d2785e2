// Rotary positions over rows of heads (rotary.h has the mathematics).  No reference counterpart: the reference's positions
// are the added sinusoids of st/layers/common_attention_v1.py:28-70; this is the other form of them, applied to the
// queries and keys of st/models/tools/utils.py:479-554.
//
// Bound by memory: 2 * sizeof(T) bytes an element.  A thread turns one 16-byte chunk of one head and its partner;
// neighbouring threads hold neighbouring chunks of a head, so a wave reads whole lines.  Computing the angles once for four
// heads a thread was slower at every size but one: the loads of the heads wait for each other (bf16, 16 heads of 96 columns:
// 512 rows 4.3 against 3.1 us, 4000 rows 7.7 / 7.5, 8000 rows 10.6 / 11.0, 16000 rows 21.3 / 19.2 = 5.1 TB/s).  Computing them
// once a row into shared memory gains a tenth with 16 heads (16000 rows 18.7) and loses as much with nine (fp32, 4099 rows of
// 96 columns, half of them turned: 7.9 against 7.0) or two.
#include "rotary.h"

struct RotArgs {
  const void* x;
  void* y;
  const double* freq;
  const int32_t* pos;
  int64_t ldx, ldy, row0;
  uint32_t rows, period, base;      // base: row0 modulo period
  int heads, pos0;
  float mscale, sign;
  RotShape sh;
};

template <typename T, int VEC> __global__ void __launch_bounds__(256) rotary_kernel(RotArgs a) {
  const uint32_t idx = blockIdx.x * 256u + threadIdx.x;
  const uint32_t c = idx % (uint32_t)a.sh.chunks, rest = idx / (uint32_t)a.sh.chunks;
  const uint32_t h = rest % (uint32_t)a.heads, r = rest / (uint32_t)a.heads;
  if (r >= a.rows) return;
  const int64_t row = a.row0 + r;
  const T* src = static_cast<const T*>(a.x) + row * a.ldx + (int64_t)h * a.sh.dh;
  T* dst = static_cast<T*>(a.y) + row * a.ldy + (int64_t)h * a.sh.dh;
  if ((int)c >= a.sh.rot_chunks) {
    if (src != dst) rot_pass<T, VEC>(a.sh, src, dst, (int)c);
    return;
  }
  const int p = a.pos ? a.pos[row] : a.pos0 + (int)(a.period ? (a.base + r) % a.period : (uint32_t)row);
  float cs[VEC], sn[VEC];
  rot_angles<VEC>(a.sh, a.freq, (int)c, p, a.mscale, a.sign, cs, sn);
  rot_apply<T, VEC>(a.sh, src, dst, (int)c, cs, sn);
}

template <typename T> static int rotary_launch(RotArgs a, int64_t rows, hipStream_t s) {
  const int64_t es = sizeof(T);
  const uintptr_t align = (uintptr_t)a.x | (uintptr_t)a.y | (uintptr_t)(a.ldx * es) | (uintptr_t)(a.ldy * es) | (uintptr_t)(a.sh.dh * es);
  int vec = 1;
  for (int v : {(int)(16 / es), (int)(8 / es), 2})
    if (align % (v * es) == 0 && rot_vec_fits(a.sh.n, a.sh.dh, a.sh.layout, v)) { vec = v; break; }
  // interleaved pairs that are not aligned to two elements: element-wise vectors of 2 read as T[2] need 2 * es alignment, so
  // such a tensor is refused by the caller's check
  a.sh = rot_shape(a.sh.n, a.sh.dh, a.sh.layout, vec);
  const int64_t per_row = (int64_t)a.sh.chunks * a.heads;
  const int64_t slice = ((int64_t)1 << 31) / per_row;          // the index of a launch fits 32 bits
  for (int64_t r0 = 0; r0 < rows; r0 += slice) {
    a.row0 = r0;
    a.base = a.period ? (uint32_t)(r0 % a.period) : 0u;
    a.rows = (uint32_t)(rows - r0 < slice ? rows - r0 : slice);
    const dim3 grid((unsigned)cdiv64((int64_t)a.rows * per_row, 256));
    switch (vec) {
      case 8: if constexpr (sizeof(T) == 2) rotary_kernel<T, 8><<<grid, 256, 0, s>>>(a); break;
      case 4: rotary_kernel<T, 4><<<grid, 256, 0, s>>>(a); break;
      case 2: rotary_kernel<T, 2><<<grid, 256, 0, s>>>(a); break;
      default: rotary_kernel<T, 1><<<grid, 256, 0, s>>>(a); break;
    }
    NEURST_CHECK_LAUNCH("rotary");
  }
  return NEURST_OK;
}

extern "C" int neurst_rotary(const void* x, void* y, const double* freq, const int32_t* positions, int64_t rows, int64_t heads, int64_t dh,
                             int64_t pairs, int64_t ldx, int64_t ldy, int64_t pos0, int64_t period, int layout, int inverse, float mscale,
                             int dtype, void* stream) {
  NEURST_CHECK_ARG(x && y && freq, "rotary: null pointer");
  NEURST_CHECK_ARG(dtype == NEURST_F32 || dtype == NEURST_BF16, "rotary: dtype must be fp32 or bf16");
  NEURST_CHECK_ARG(rows >= 0 && heads > 0 && heads <= 65536 && dh > 0 && dh <= 65536, "rotary: bad sizes");
  NEURST_CHECK_ARG(pairs > 0 && 2 * pairs <= dh, "rotary: 2 * pairs must be in 2..dh");
  NEURST_CHECK_ARG(ldx >= heads * dh && ldy >= heads * dh, "rotary: a row stride is smaller than its heads");
  NEURST_CHECK_ARG(layout == ROT_HALF || layout == ROT_INTERLEAVED, "rotary: layout must be 0 (half) or 1 (interleaved)");
  NEURST_CHECK_ARG(x != y || ldx == ldy, "rotary: in place needs equal row strides");
  NEURST_CHECK_ARG(period >= 0 && period <= INT32_MAX, "rotary: bad period");
  NEURST_CHECK_ARG(heads * dh <= INT32_MAX, "rotary: rows are limited to 2^31 - 1 columns");
  NEURST_CHECK_ARG(positions || (pos0 >= INT32_MIN && pos0 <= INT32_MAX && pos0 <= INT32_MAX - (period ? period : rows)),
                   "rotary: positions must fit 32 bits");
  const int64_t es = (int64_t)dtype_size(dtype);
  if (layout == ROT_INTERLEAVED)
    NEURST_CHECK_ARG((((uintptr_t)x | (uintptr_t)y | (uintptr_t)(ldx * es) | (uintptr_t)(ldy * es) | (uintptr_t)(dh * es)) % (2 * es)) == 0,
                     "rotary: interleaved pairs must be aligned to two elements");
  if (rows == 0) return NEURST_OK;
  NEURST_CHECK_ARG(x == y || !rows_meet(Rows{x, heads * dh * es, ldx * es, rows}, Rows{y, heads * dh * es, ldy * es, rows}),
                   "rotary: y must be x or apart from it");
  RotArgs a;
  a.x = x; a.y = y; a.freq = freq; a.pos = positions;
  a.ldx = ldx; a.ldy = ldy; a.period = (uint32_t)period; a.heads = (int)heads; a.pos0 = (int)pos0;
  a.mscale = mscale; a.sign = inverse ? -1.f : 1.f;
  a.sh = rot_shape(pairs, dh, layout, 2);
  return dtype == NEURST_BF16 ? rotary_launch<bf16_t>(a, rows, as_stream(stream)) : rotary_launch<float>(a, rows, as_stream(stream));
}
