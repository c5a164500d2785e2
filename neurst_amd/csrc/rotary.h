// Rotation of column pairs by position, shared by rotary.hip and the cache write of paged.hip.
//
// Pair i of a head at position p turns by a = p * freq[i]: u' = m (u cos a - v sin a), v' = m (v cos a + u sin a).
// The angle is counted in TURNS: t = p * (freq / 2 pi) in fp64, its nearest integer taken off there, and only the rest,
// |r| <= 1/2, goes on in fp32.  In fp32 the product alone is 0.06 rad off at position 2^20; in fp64 three roundings (freq / 2 pi:
// the constant and the product; the angle) leave it within |a| 2^-54 turns: 2^-34 for |a| = 2^20 rad, 2^-23 for 2^31 (over 64
// frequencies from 1 to 10^-4 it is 2^-35.4 and 2^-24.7 at the worst).  The rest in fp32 adds 2^-26.
#pragma once
#include "common.h"

enum { ROT_HALF = 0, ROT_INTERLEAVED = 1 };

// sin and cos of r turns, |r| <= 1/2: quarter turns off (q = nearest integer to 4 r), then |a| <= pi / 4 and the Taylor
// polynomials up to a^9 and a^10 (first terms left out: pi/4^11 / 11! = 2e-9 and pi/4^12 / 12! = 1e-10, below half an fp32 step)
__device__ __forceinline__ void sincos_turns(float r, float& s, float& c) {
  const float q = rintf(4.f * r);
  const float a = 6.28318530717958648f * fmaf(-0.25f, q, r);
  const float a2 = a * a;
  const float sp = fmaf(a2, fmaf(a2, fmaf(a2, fmaf(a2, 2.75573192e-6f, -1.98412698e-4f), 8.33333333e-3f), -1.66666667e-1f), 1.f) * a;
  const float cp = fmaf(a2, fmaf(a2, fmaf(a2, fmaf(a2, fmaf(a2, -2.75573192e-7f, 2.48015873e-5f), -1.38888889e-3f), 4.16666667e-2f), -0.5f), 1.f);
  const int qi = (int)q & 3;
  const float x = (qi & 1) ? cp : sp, y = (qi & 1) ? sp : cp;
  s = (qi & 2) ? -x : x;
  c = ((qi + 1) & 2) ? -y : y;
}

__device__ __forceinline__ void rotation(double pos, double freq, float mscale, float sign, float& s, float& c) {
  const double t = pos * (freq * 0.15915494309189533577);
  sincos_turns((float)(t - rint(t)), s, c);
  s *= mscale * sign;
  c *= mscale;
}

template <typename T, int VEC> struct RotVec { T v[VEC]; };
template <typename T, int VEC> __device__ __forceinline__ void rot_load(const T* p, float* f) {
  RotVec<T, VEC> r;
  __builtin_memcpy(&r, __builtin_assume_aligned(p, VEC * sizeof(T)), sizeof(r));
#pragma unroll
  for (int j = 0; j < VEC; ++j) f[j] = to_f32<T>(r.v[j]);
}
template <typename T, int VEC> __device__ __forceinline__ void rot_store(T* p, const float* f) {
  RotVec<T, VEC> r;
#pragma unroll
  for (int j = 0; j < VEC; ++j) r.v[j] = from_f32<T>(f[j]);      // the one rounding of the result to its type
  __builtin_memcpy(__builtin_assume_aligned(p, VEC * sizeof(T)), &r, sizeof(r));
}

// Chunks of one head, VEC elements a vector: `half` takes pairs (i, n + i), so a chunk is VEC pairs from two places;
// `interleaved` takes pairs (2 i, 2 i + 1), so a chunk is VEC / 2 pairs (VEC >= 2); columns from 2 n on pass through.
struct RotShape {
  int n, dh, layout, vec;          // pairs, columns of a head, layout, elements per vector
  int rot_chunks, chunks;          // chunks that turn, all chunks
};
static inline RotShape rot_shape(int64_t n, int64_t dh, int layout, int vec) {
  RotShape s;
  s.n = (int)n; s.dh = (int)dh; s.layout = layout; s.vec = vec;
  s.rot_chunks = (int)(layout == ROT_HALF ? n / vec : 2 * n / vec);
  s.chunks = s.rot_chunks + (int)((dh - 2 * n) / vec);
  return s;
}
static inline bool rot_vec_fits(int64_t n, int64_t dh, int layout, int vec) {
  if (vec == 1) return layout == ROT_HALF;
  return (layout == ROT_HALF ? n % vec == 0 : (2 * n) % vec == 0) && (dh - 2 * n) % vec == 0;
}

// cos / sin of the pairs of chunk c (< rot_chunks); interleaved fills VEC / 2 of them
template <int VEC> __device__ __forceinline__ void rot_angles(const RotShape& sh, const double* __restrict__ freq, int c, int pos, float mscale,
                                                              float sign, float* cs, float* sn) {
  const int np = sh.layout == ROT_HALF ? VEC : VEC / 2;
#pragma unroll
  for (int j = 0; j < VEC; ++j)
    if (j < np) rotation((double)pos, freq[c * np + j], mscale, sign, sn[j], cs[j]);
}

// one head's chunk: src and dst point at the head's first column and may be the same
template <typename T, int VEC> __device__ __forceinline__ void rot_apply(const RotShape& sh, const T* src, T* dst, int c, const float* cs,
                                                                         const float* sn) {
  float a[VEC], b[VEC];
  if (sh.layout == ROT_HALF) {
    rot_load<T, VEC>(src + c * VEC, a);
    rot_load<T, VEC>(src + sh.n + c * VEC, b);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float u = a[j], v = b[j];
      a[j] = u * cs[j] - v * sn[j];
      b[j] = v * cs[j] + u * sn[j];
    }
    rot_store<T, VEC>(dst + c * VEC, a);
    rot_store<T, VEC>(dst + sh.n + c * VEC, b);
  } else {
    rot_load<T, VEC>(src + c * VEC, a);
#pragma unroll
    for (int j = 0; j < VEC / 2; ++j) {
      const float u = a[2 * j], v = a[2 * j + 1];
      a[2 * j] = u * cs[j] - v * sn[j];
      a[2 * j + 1] = v * cs[j] + u * sn[j];
    }
    rot_store<T, VEC>(dst + c * VEC, a);
  }
}
template <typename T, int VEC> __device__ __forceinline__ void rot_pass(const RotShape& sh, const T* src, T* dst, int c) {
  const int at = 2 * sh.n + (c - sh.rot_chunks) * VEC;
  RotVec<T, VEC> r;
  __builtin_memcpy(&r, __builtin_assume_aligned(src + at, VEC * sizeof(T)), sizeof(r));
  __builtin_memcpy(__builtin_assume_aligned(dst + at, VEC * sizeof(T)), &r, sizeof(r));
}
