// Sampling of the next token from a row of logits with temperature, top-k, top-p and min-p and a given random number, beside
// the arg-max of greedy_step and the top-k of beam_topk.  No reference counterpart: the reference decodes by arg-max
// (st/models/decoders/transformer_decoder.py:83-90) or beam search.
//
//   w_i = exp((l_i - max l) / T);   keep the top_k largest (equal ones: lower index first), of these the shortest leading run
//   in descending order whose sum reaches top_p of theirs, of these the ones with w_i >= min_p;
//   id = the first kept index, in index order, whose running sum exceeds u times the kept sum;  logp = log(w_id / kept sum).
//
// Weights are INTEGERS, round(w 2^44), from an fp64 exponential: sums over up to 2^19 words stay below 2^63 and are the same
// in whatever order the lanes and the atomics add them, so a draw never depends on the launch, and a border falls within
// 1e-11 of where real numbers put it (fp32 sums would move it by 1e-6, past a word in one draw of thirty).  Words below
// 2^-45 of the best have weight 0 and are never drawn.
//
// The kept set is {key > K} and the words with key == K up to a place, keys being the logits in an order-preserving integer
// form.  First the words that can be kept at all are told from a bound (the top_k-th of the threads' own maxima; for top_p the
// step in which the row's sum passes it; min_p itself) and, up to 1024 of them, listed in index order; the rest of the work
// runs on that list, a word a thread.  K is found by counting, not by sorting: a histogram over 1024 equal steps of
// (max - l) / T in [0, 32) - all that can have weight - finds the step where the count passes top_k or the sum passes top_p,
// and the words of that one step, a dozen as a rule, are ranked among each other.  (Without the list every pass ran over the
// row: the 256 rows below took 86 us.)
//
// One workgroup a row; a row of up to 132 KB is read once, into shared memory, and every later pass runs on that.  Bound by
// the chain of passes and barriers: one row of 10000 words with top_p takes 13 us (its arg-max alone 4.0), 256 rows of 32003
// words with every filter, a CU each, 22 us = 1.5 TB/s (the arg-max 9.4 = 3.5 TB/s); without top_k by the fp64 exponentials,
// some 26 instructions a word: 256 rows of 32003 with top_p alone 28 us.  Longer rows are read from memory again by every pass:
// one row of 128000 words takes 41 us for the arg-max, 71 with every filter, 137 with top_p alone; 256 of them 116, 180, 289.
#include "common.h"

struct SampleArgs {
  const void* logits;
  const float* u;
  const float *temperature_rows, *top_p_rows, *min_p_rows;
  const int32_t* top_k_rows;
  int32_t* ids;
  float* logp;
  // bookkeeping of a decoding step (all null for a plain draw)
  int32_t *preds, *finished, *len_decoded, *n_unfinished, *status;
  float* scores;
  int64_t ld, step, max_steps;
  int V, top_k, eos;
  float temperature, top_p, min_p;
};

typedef unsigned long long u64;
constexpr int SAMPLE_BINS = 1024;
constexpr int SAMPLE_NOTHING = 4;                    // status: beside the paged cache's 1 and 2
constexpr double SAMPLE_ONE = 17592186044416.0;      // 2^44
constexpr float SAMPLE_SPAN = 32.f;                   // e^-32 < 2^-45: rounds to 0

__device__ __forceinline__ uint32_t logit_key(float l) {
  const uint32_t b = __builtin_bit_cast(uint32_t, l);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

// round(2^44 exp(x)), x in [-32, 0]: exp(x) = 2^(n / 16) exp(y), |y| <= ln2 / 32, with 2^(j / 16) from a table (sixteen values
// of 2^(j/16), each the double next to it) and the Taylor polynomial to y^6 (the next term is 4e-16).  Its coefficients come
// in scalar registers: as literals each would cost two moves an evaluation.
__device__ const double SAMPLE_ROOTS[16] = {
    1.0, 1.0442737824274138403, 1.0905077326652576592, 1.1387886347566916537, 1.1892071150027210667, 1.2418578120734840486,
    1.2968395546510096659, 1.3542555469368927283, 1.4142135623730950488, 1.4768261459394993114, 1.5422108254079408236,
    1.6104903319492543081, 1.6817928305074290861, 1.7562521603732994831, 1.8340080864093424635, 1.9152065613971472939};
struct SampleExp {
  double c6, c5, c4, c3;
  const double* roots;       // in shared memory
  __device__ __forceinline__ void init(const double* r) {
    roots = r;
    c6 = 1.38888888888888888889e-03;
    c5 = 8.33333333333333333333e-03;
    c4 = 4.16666666666666666667e-02;
    c3 = 1.66666666666666666667e-01;
    asm volatile("" : "+s"(c6), "+s"(c5), "+s"(c4), "+s"(c3));
  }
  __device__ __forceinline__ u64 operator()(double x) const {
    const double t = x * 23.083120654223414519, n = rint(t), y = (t - n) * 0.043321698784996581838;
    const int i = (int)n;
    double p = fma(c6, y, c5);
    p = fma(p, y, c4);
    p = fma(p, y, c3);
    p = fma(p, y, 0.5);
    p = fma(p, y, 1.0);
    p = fma(p, y, 1.0);
    // the sum with 2^52 holds the rounded integer in its low 52 bits
    const double v = ldexp(p * roots[i & 15], (i >> 4) + 44) + 4503599627370496.0;
    return __builtin_bit_cast(u64, v) & 0xFFFFFFFFFFFFFull;
  }
};

// ---- 64-lane scans through the DPP network (all lanes active) and sums over the waves of a workgroup ------------------------
template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS> __device__ __forceinline__ u64 dpp_u64(u64 v) {
  return (u64)dpp_u32<CTRL, ROWS>((uint32_t)v) | ((u64)dpp_u32<CTRL, ROWS>((uint32_t)(v >> 32)) << 32);
}
__device__ __forceinline__ u64 row_scan_u64(u64 v) {        // inclusive, within 16 lanes: shifts by 1, 2, 4, 8
  v += dpp_u64<0x111, 0xF>(v);
  v += dpp_u64<0x112, 0xF>(v);
  v += dpp_u64<0x114, 0xF>(v);
  v += dpp_u64<0x118, 0xF>(v);
  return v;
}
__device__ __forceinline__ u64 wave_scan_u64(u64 v) {       // inclusive: then the rows' last lanes on to the rows behind them
  v = row_scan_u64(v);
  v += dpp_u64<0x142, 0xA>(v);
  v += dpp_u64<0x143, 0xC>(v);
  return v;
}
__device__ __forceinline__ u64 readlane_u64(u64 v, int lane) {
  return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane) | ((u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane) << 32);
}

constexpr int SAMPLE_CAND = 256, SAMPLE_LIST = 1024;
struct SampleCand { u64 w; uint32_t key; int at; };

template <typename T, int NT> struct SampleShared {
  u64 hw[SAMPLE_BINS];
  SampleCand cand[SAMPLE_CAND];
  u64 ww[5][16], above, bin_w, drawn;
  double roots[16];
  uint32_t hc[SAMPLE_BINS];
  int list_at[SAMPLE_LIST];
  uint32_t wa[16], wb[16], bin_c, found_key, count;
  float wf[16];              // maxima of the waves
  int bin, found_at, place;
  T list[SAMPLE_LIST];
};

// sum over the waves before this one and over all, from each wave's own sum (the same in all its lanes); one barrier; each
// use has a slot of its own, so that it need not wait for the last one's readers
template <typename S, int NW> __device__ __forceinline__ void waves_sum(S& s, int slot, u64 mine, int w, int lane, u64& before, u64& all) {
  if (lane == 0) s.ww[slot][w] = mine;
  __syncthreads();
  const u64 inc = row_scan_u64(lane < NW ? s.ww[slot][lane] : 0);
  all = readlane_u64(inc, NW - 1);
  before = w ? readlane_u64(inc, w - 1) : 0;
}

// NaN is never drawn; -0 counts as +0
template <typename T> __device__ __forceinline__ float sample_word(T v) {
  const float x = to_f32<T>(v);
  return x == x ? x + 0.f : -INFINITY;
}

// A sequence of words: place i of step and lane, in index order wave by wave, step by step, lane by lane.  CLEAN: in shared
// memory, gone through sample_word and padded with -inf to whole steps.  AT_ONCE: words whose chains run side by side.
template <typename T, int NT, bool CLEAN, int AT_ONCE> struct SampleView {
  const T* p;                // [n]
  int n, base, steps;
  __device__ __forceinline__ void init(const T* p_, int n_, int tid) {
    p = p_;
    n = n_;
    steps = (n + NT - 1) / NT;
    base = (tid >> 6) * steps * 64 + (tid & 63);
  }
  __device__ __forceinline__ float at(int place) const {
    if constexpr (CLEAN) return to_f32<T>(p[place]);
    return place < n ? sample_word<T>(p[place]) : -INFINITY;
  }
  // f(word, place) for this lane's words; past the last step f sees -inf, which has no weight
  template <typename F> __device__ __forceinline__ void each(F f) const {
    for (int i = 0; i < steps; i += AT_ONCE) {
      float v[AT_ONCE];
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) v[j] = i + j < steps ? at(base + (i + j) * 64) : -INFINITY;
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) f(v[j], base + (i + j) * 64);
    }
  }
};

struct SampleRule {
  SampleExp exp44;
  float mx, bin_scale;
  double inv_t;
  u64 lowest;                // min_p as a weight
  // no branch: several words' chains of fp64 instructions run side by side
  __device__ __forceinline__ u64 weight(float l) const {
    const double x = ((double)l - (double)mx) * inv_t;
    return exp44(l == mx ? 0.0 : fmax(x, -(double)SAMPLE_SPAN));       // -32: rounds to 0
  }
  // step of the histogram: grows as l falls, 0 for the best; SAMPLE_BINS: no weight
  __device__ __forceinline__ int step_of(float l) const {
    const float x = (mx - l) * bin_scale;
    return l == mx ? 0 : (x < (float)SAMPLE_BINS ? (int)x : SAMPLE_BINS);
  }
};

// what the sum of the words kept by top_p has to reach
__device__ __forceinline__ u64 sample_need(float top_p, u64 total) {
  const u64 need = (u64)ceil((double)top_p * (double)total);
  return need < 1 ? 1 : need;
}

struct SampleLimit {         // words with key > K, and with key == K up to place `cut`
  uint32_t K;
  int cut;
  __device__ __forceinline__ bool holds(uint32_t key, int place) const { return key > K || (key == K && place <= cut); }
};

// the bin at which the running count (BY_WEIGHT: the running sum) reaches `want`, into s.bin, with what lies before it and in it
template <bool BY_WEIGHT, typename T, int NT> __device__ __forceinline__ void sample_cross(SampleShared<T, NT>& s, u64 want, int tid) {
  constexpr int NW = NT / 64, PER = SAMPLE_BINS / NT;
  const int lane = tid & 63, w = tid >> 6;
  auto part = [&](int i) -> u64 { return BY_WEIGHT ? s.hw[i] : (u64)s.hc[i]; };
  u64 x = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) x += part(tid * PER + j);
  const u64 inc = wave_scan_u64(x);
  u64 before, all;
  waves_sum<SampleShared<T, NT>, NW>(s, 1, readlane_u64(inc, 63), w, lane, before, all);
  u64 b = before + inc - x;
  if (b < want && b + x >= want) {
    for (int j = 0; j < PER; ++j) {
      const u64 y = part(tid * PER + j);
      if (b + y >= want) {
        s.bin = tid * PER + j;
        s.above = b;
        s.bin_c = s.hc[tid * PER + j];
        s.bin_w = y;
        break;
      }
      b += y;
    }
  }
  if (tid == 0) s.count = 0;
  __syncthreads();
}
template <typename T, int NT> __device__ __forceinline__ void sample_clear(SampleShared<T, NT>& s, int tid) {
  __syncthreads();
  for (int i = tid; i < SAMPLE_BINS; i += NT) { s.hc[i] = 0; s.hw[i] = 0; }
  __syncthreads();
}

// The word at which the running count (by_weight: the running sum), in descending order, reaches `need`: the new limit.
// sample_cross has found its step in the histogram over the words that `lim` holds.
template <bool BY_WEIGHT, typename T, int NT, typename View>
__device__ __forceinline__ SampleLimit sample_select(SampleShared<T, NT>& s, const View& r, const SampleRule& rule, SampleLimit lim, u64 need, int tid) {
  constexpr int NW = NT / 64;
  const int lane = tid & 63, w = tid >> 6;
  const int bin = s.bin;
  if (s.bin_c <= SAMPLE_CAND) {
    // its words, ranked among each other
    r.each([&](float l, int place) {
      if (rule.step_of(l) == bin && l > -INFINITY) {
        const uint32_t key = logit_key(l);
        const u64 x = BY_WEIGHT ? rule.weight(l) : 1;
        if (lim.holds(key, place) && x) {
          const uint32_t at = atomicAdd(&s.count, 1u);       // the order does not matter
          if (at < SAMPLE_CAND) s.cand[at] = SampleCand{x, key, place};
        }
      }
    });
    __syncthreads();
    const int n = (int)s.bin_c;
    if (tid < n) {
      const SampleCand me = s.cand[tid];
      u64 b = s.above;
      for (int j = 0; j < n; ++j) {
        const SampleCand c = s.cand[j];
        if (c.key > me.key || (c.key == me.key && c.at < me.at)) b += c.w;
      }
      if (b < need && b + me.w >= need) {
        s.found_key = me.key;
        s.found_at = me.at;
      }
    }
    __syncthreads();
    return SampleLimit{s.found_key, s.found_at};
  }
  // very many words in one step (ties, or logits closer than 1 / 32 of the temperature): counted again over the range of
  // their keys until one key is left, and that key's words by place
  u64 above = s.above;
  uint32_t lo = 0xffffffffu, hi = 0;
  r.each([&](float l, int place) {
    if (rule.step_of(l) == bin && l > -INFINITY) {
      const uint32_t k = logit_key(l);
      if (lim.holds(k, place)) {
        lo = k < lo ? k : lo;
        hi = k > hi ? k : hi;
      }
    }
  });
  for (int o = 32; o > 0; o >>= 1) {
    const uint32_t x = (uint32_t)__shfl_xor((int)lo, o, 64), y = (uint32_t)__shfl_xor((int)hi, o, 64);
    lo = x < lo ? x : lo;
    hi = y > hi ? y : hi;
  }
  if (lane == 0) { s.wa[w] = lo; s.wb[w] = hi; }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    lo = s.wa[i] < lo ? s.wa[i] : lo;
    hi = s.wb[i] > hi ? s.wb[i] : hi;
  }
  while (lo < hi) {
    const int bits = 32 - __builtin_clz(hi - lo), shift = bits > 10 ? bits - 10 : 0;      // 1024 bins
    sample_clear(s, tid);
    r.each([&](float l, int place) {
      const uint32_t k = logit_key(l);
      if (k >= lo && k <= hi && lim.holds(k, place)) {
        const u64 x = rule.weight(l);
        if (x || !BY_WEIGHT) {
          atomicAdd(&s.hc[(hi - k) >> shift], 1u);
          if (BY_WEIGHT) atomicAdd(&s.hw[(hi - k) >> shift], x);
        }
      }
    });
    __syncthreads();
    sample_cross<BY_WEIGHT>(s, need - above, tid);
    above += s.above;
    hi -= (uint32_t)s.bin << shift;
    const uint32_t span = (1u << shift) - 1u;
    if (hi - lo > span) lo = hi - span;
  }
  const uint32_t K = hi, ties = s.bin_c;
  const u64 one = BY_WEIGHT ? s.bin_w / ties : 1;
  const uint32_t m = (uint32_t)((need - above + one - 1) / one);      // of `ties` equal words the first m
  uint32_t c = 0;
  r.each([&](float l, int place) { c += logit_key(l) == K && place <= (lim.K == K ? lim.cut : 0x7fffffff) ? 1u : 0u; });
  u64 before, all;
  waves_sum<SampleShared<T, NT>, NW>(s, 0, readlane_u64(wave_scan_u64(c), 63), w, lane, before, all);
  uint32_t seen = (uint32_t)before;
  if (seen < m)
    r.each([&](float l, int place) {
      const u64 eq = __ballot(logit_key(l) == K);
      const uint32_t here = (uint32_t)__popcll(eq);
      if (seen < m && seen + here >= m && ((eq >> lane) & 1) && seen + (uint32_t)__popcll(eq & ((2ull << lane) - 1)) == m) s.found_at = place;
      seen += here;
    });
  __syncthreads();
  return SampleLimit{K, s.found_at};
}

// top_k, top-p and min-p over a view that holds every word that can be kept, and the draw: the place drawn in s.place, its
// weight in s.drawn; returns the sum of the words kept.  k: 0 for none; then, where top_p < 1, `all` is the sum over the row
// (the view may lack words) and sample_cross has found the step in which it is passed.  Words behind step `far` are not
// looked at.
template <typename T, int NT, typename View>
__device__ __forceinline__ u64 sample_draw(SampleShared<T, NT>& s, const View& r, const SampleRule& rule, uint32_t k, float top_p, float u, u64 all,
                                           int far, int tid) {
  constexpr int NW = NT / 64;
  typedef SampleShared<T, NT> S;
  const int lane = tid & 63, w = tid >> 6;
  SampleLimit lim = {0u, 0x7fffffff};
  u64 before, total;
  if (k) {
    sample_clear(s, tid);
    uint32_t mine = 0;
    r.each([&](float l, int) {
      const int b = rule.step_of(l);
      if (b <= far && b < SAMPLE_BINS) {
        atomicAdd(&s.hc[b], 1u);
        ++mine;
      }
    });
    waves_sum<S, NW>(s, 0, readlane_u64(wave_scan_u64(mine), 63), w, lane, before, total);
    // Else every word with weight stays.  With a bound `far` the words counted are those above it, k at least, and the words
    // behind it are in the view all the same (too many for the list): the limit is set even where the count is k exactly.
    if (total > (u64)k || far < SAMPLE_BINS) {
      sample_cross<false>(s, (u64)k, tid);
      lim = sample_select<false>(s, r, rule, lim, (u64)k, tid);
    }
  }
  if (top_p < 1.f) {
    total = all;
    if (k) {
      u64 mine = 0;
      r.each([&](float l, int place) {
        const u64 x = rule.weight(l);
        mine += lim.holds(logit_key(l), place) ? x : 0;
      });
      waves_sum<S, NW>(s, 3, readlane_u64(wave_scan_u64(mine), 63), w, lane, before, total);
    }
    const u64 need = sample_need(top_p, total);
    if (need < total) {
      if (k) {
        sample_clear(s, tid);
        r.each([&](float l, int place) {
          const int b = rule.step_of(l);
          if (b <= far && b < SAMPLE_BINS && lim.holds(logit_key(l), place)) {
            const u64 x = rule.weight(l);
            if (x) {
              atomicAdd(&s.hc[b], 1u);
              atomicAdd(&s.hw[b], x);
            }
          }
        });
        __syncthreads();
        sample_cross<true>(s, need, tid);
      }
      lim = sample_select<true>(s, r, rule, lim, need, tid);
    }
  }
  auto kept = [&](float l, int place) -> u64 {
    const u64 x = lim.holds(logit_key(l), place) ? rule.weight(l) : 0;
    return x >= rule.lowest ? x : 0;
  };
  u64 mine = 0;
  r.each([&](float l, int place) { mine += kept(l, place); });
  const u64 inc = wave_scan_u64(mine), own = readlane_u64(inc, 63);
  waves_sum<S, NW>(s, 4, own, w, lane, before, total);
  u64 thr = (u64)((double)u * (double)total);
  if (thr >= total) thr = total - 1;
  if (r.steps == 1) {                                        // a word a lane
    const u64 c = before + inc;
    if (c > thr && c - mine <= thr) {
      s.place = r.base;
      s.drawn = mine;
    }
    __syncthreads();
    return total;
  }
  if (before <= thr && thr < before + own && lane == 0) {    // this wave's words hold the draw
    s.bin = w;
    s.above = before;
  }
  __syncthreads();
  // its steps' sums, dealt to all waves
  const int first = s.bin * r.steps * 64 + lane;
  for (int i = w; i < r.steps; i += NW) {
    const u64 x = wave_scan_u64(kept(r.at(first + i * 64), first + i * 64));
    if (lane == 63) s.hw[i] = x;
  }
  __syncthreads();
  if (w == 0) {
    u64 run = s.above;
    int at = 0;
    for (int j = 0; j < r.steps; j += 64) {                  // 64 steps at a time
      const u64 x = j + lane < r.steps ? s.hw[j + lane] : 0, inc = run + wave_scan_u64(x);
      const u64 over = __ballot(inc > thr);
      if (over) {
        at = j + __builtin_ctzll(over);
        run = readlane_u64(inc - x, at - j);
        break;
      }
      run = readlane_u64(inc, 63);
    }
    const int place = first + at * 64;
    const u64 x = kept(r.at(place), place), c = run + wave_scan_u64(x);
    if (c > thr && c - x <= thr) {
      s.place = place;
      s.drawn = x;
    }
  }
  __syncthreads();
  return total;
}

template <typename T, int NT, bool CACHED> __global__ void __launch_bounds__(NT) sample_kernel(SampleArgs a) {
  constexpr int NW = NT / 64;
  typedef SampleShared<T, NT> S;
  __shared__ S s;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t row = blockIdx.x;
  extern __shared__ __attribute__((aligned(16))) char row_lds[];
  const T* src = static_cast<const T*>(a.logits) + row * a.ld;
  SampleView<T, NT, CACHED, 4> r;
  r.init(CACHED ? reinterpret_cast<const T*>(row_lds) : src, a.V, tid);
  float mx = -INFINITY;
  if constexpr (CACHED) {
    // 16 bytes a lane (rows need not be aligned to that), four loads before the first is used; a wave reads its own words
    constexpr int E = 16 / sizeof(T), STRIDE = 64 * E;
    struct Words { T v[E]; };
    T* dst = reinterpret_cast<T*>(row_lds);
    const int own = r.steps * 64, w0 = w * own;
    for (int i = lane * E; i < own; i += 4 * STRIDE) {
      Words x[4];
      if (a.V >= E) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int at = w0 + i + j * STRIDE;
          __builtin_memcpy(&x[j], src + (i + j * STRIDE < own && at + E <= a.V ? at : 0), sizeof(Words));
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = w0 + i + j * STRIDE;
        if (i + j * STRIDE >= own) continue;
        if (at + E > a.V)                                   // the end of the row, padded to whole steps
          for (int e = 0; e < E; ++e) x[j].v[e] = at + e < a.V ? src[at + e] : (T)-INFINITY;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float l = sample_word<T>(x[j].v[e]);
          x[j].v[e] = (T)l;
          mx = fmaxf(mx, l);
        }
        __builtin_memcpy(__builtin_assume_aligned(dst + at, 16), &x[j], 16);
      }
    }
  } else {
    r.each([&](float l, int) { mx = fmaxf(mx, l); });
  }
  float temp = a.temperature_rows ? a.temperature_rows[row] : a.temperature;
  float top_p = a.top_p_rows ? a.top_p_rows[row] : a.top_p;
  float min_p = a.min_p_rows ? a.min_p_rows[row] : a.min_p;
  int top_k = a.top_k_rows ? a.top_k_rows[row] : a.top_k;
  if (!(temp > 0.f)) { temp = 1.f; top_k = 1; }
  if (!(top_p > 0.f)) top_p = 0.f;
  if (!(min_p > 0.f)) min_p = 0.f;
  if (min_p > 1.f) min_p = 1.f;
  if (top_k <= 0 || top_k > a.V) top_k = a.V;
  float u = a.u[row];
  u = u > 0.f ? (u < 1.f ? u : 1.f) : 0.f;
  for (int i = tid; i < SAMPLE_BINS; i += NT) { s.hc[i] = 0; s.hw[i] = 0; }
  const float own_max = mx;
  mx = wave_max(mx);
  if (lane == 0) s.wf[w] = mx;
  if (tid < 16) s.roots[tid] = SAMPLE_ROOTS[tid];
  __syncthreads();
  mx = wave_max(lane < NW ? s.wf[lane] : -INFINITY);

  int id = -1;
  float logp = -INFINITY;
  if (mx > -INFINITY && top_k == 1) {                       // the first maximum
    int best = 0x7fffffff;
    r.each([&](float l, int place) { best = l == mx && place < best ? place : best; });
    for (int o = 32; o > 0; o >>= 1) {
      const int x = __shfl_xor(best, o, 64);
      best = x < best ? x : best;
    }
    if (lane == 0) s.wa[w] = (uint32_t)best;
    __syncthreads();
    id = (int)s.wa[0];
    for (int i = 1; i < NW; ++i) id = (int)s.wa[i] < id ? (int)s.wa[i] : id;
    logp = 0.f;
  } else if (mx > -INFINITY) {
    SampleRule rule;
    rule.mx = mx;
    rule.exp44.init(s.roots);
    rule.inv_t = 1.0 / (double)temp;
    rule.bin_scale = (float)fmin(SAMPLE_BINS / SAMPLE_SPAN * rule.inv_t, 3e38);      // finite: wider steps do no harm
    rule.lowest = (u64)ceil((double)min_p * SAMPLE_ONE);
    const bool by_k = top_k < a.V, by_p = top_p < 1.f;
    u64 before, n, all = 0;
    // How far down a kept word can lie, as a step of the histogram; as a rule that leaves a few per cent of the words.
    int far = SAMPLE_BINS;
    if (min_p > 0.f) {
      const float steps = (SAMPLE_BINS / SAMPLE_SPAN) * -logf(min_p) + 2.f;
      far = steps < (float)SAMPLE_BINS ? (int)steps : SAMPLE_BINS;
    }
    if (by_k && top_k <= NT) {
      // the top_k-th of the threads' own maxima bounds the top_k-th of all words
      const int b = rule.step_of(own_max);
      if (b < SAMPLE_BINS) atomicAdd(&s.hc[b], 1u);
      waves_sum<S, NW>(s, 0, (u64)__popcll(__ballot(b < SAMPLE_BINS)), w, lane, before, n);
      if (n >= (u64)top_k) {
        sample_cross<false>(s, (u64)top_k, tid);
        far = s.bin;             // (min_p comes after top_k: its words may be fewer, never others)
      } else {
        far = SAMPLE_BINS;
      }
    } else if (by_k) {
      far = SAMPLE_BINS;
    } else if (by_p) {
      // the histogram over the row tells the step in which the sum passes top_p
      u64 mine = 0;
      r.each([&](float l, int) {
        const u64 x = rule.weight(l);
        const int b = rule.step_of(l);
        if (x && b < SAMPLE_BINS) {
          atomicAdd(&s.hc[b], 1u);
          atomicAdd(&s.hw[b], x);
          mine += x;
        }
      });
      waves_sum<S, NW>(s, 0, readlane_u64(wave_scan_u64(mine), 63), w, lane, before, all);
      const u64 need = sample_need(top_p, all);
      if (need < all) {
        sample_cross<true>(s, need, tid);
        far = s.bin;
      } else {
        far = SAMPLE_BINS;
      }
    }
    n = (u64)a.V;
    if (far < SAMPLE_BINS) {
      // They go to a list, in index order, and the rest of the work runs on that.  Told by a logit a step below the bound: more
      // words do no harm.
      const float least = fminf(mx, mx - (float)(far + 2) / rule.bin_scale);
      uint32_t mine = 0;
      r.each([&](float l, int) { mine += (uint32_t)__popcll(__ballot(l >= least)); });
      waves_sum<S, NW>(s, 2, (u64)mine, w, lane, before, n);
      if (n <= SAMPLE_LIST) {
        int at = (int)before;
        r.each([&](float l, int place) {
          const u64 in = __ballot(l >= least);
          if (in) {
            if ((in >> lane) & 1) {
              const int i = at + __popcll(in & ((1ull << lane) - 1));
              s.list[i] = (T)l;
              s.list_at[i] = place;
            }
            at += __popcll(in);
          }
        });
        const int padded = ((int)n + NT - 1) / NT * NT;
        for (int i = (int)n + tid; i < padded; i += NT) s.list[i] = (T)-INFINITY;
      }
    }
    u64 total;
    if (n <= SAMPLE_LIST && far < SAMPLE_BINS) {
      __syncthreads();
      SampleView<T, NT, true, 1> few;
      few.init(s.list, (int)n, tid);
      total = sample_draw(s, few, rule, by_k ? (uint32_t)top_k : 0u, top_p, u, all, SAMPLE_BINS, tid);
      id = s.list_at[s.place];
    } else {
      total = sample_draw(s, r, rule, by_k ? (uint32_t)top_k : 0u, top_p, u, all, far, tid);
      id = s.place;
    }
    logp = (float)log((double)s.drawn / (double)total);
  }
  if (tid == 0) {
    if (!a.preds) {
      a.ids[row] = id;
      a.logp[row] = logp;
    } else {
      const int was = a.finished[row];
      const int tok = was || id < 0 ? a.eos : id;
      const int fin = was | (tok == a.eos ? 1 : 0);
      a.preds[row * a.max_steps + a.step] = tok;
      a.finished[row] = fin;
      if (!fin) {
        a.len_decoded[row] += 1;
        atomicAdd(a.n_unfinished, 1);      // a count: whole numbers, any order
      }
      if (!was && id >= 0) a.scores[row] += logp;
      if (!was && id < 0 && a.status) atomicOr(a.status, SAMPLE_NOTHING);
      a.ids[row] = tok;
    }
  }
}

template <typename T> static int sample_launch(const SampleArgs& a, int64_t rows, hipStream_t s) {
  // Threads of a row, 256 / 1024 in us without filters and with top_k 50, top_p 0.95: one row of 2000 words 6.0 / 6.9 and
  // 10.3 / 12.4, of 6000 9.5 / 8.3 and 11.9 / 12.6, of 16000 18.6 / 10.9 and 16.1 / 13.6; where rows share CUs (2048 of them)
  // 4000 words 27 / 49 and 37 / 95, 8000 words 52 / 63 and 56 / 100, 16000 words 151 / 93 and 134 / 114.
  // 132 KB of shared memory hold a row beside the histogram.
  const int nt = a.V > (rows > 512 ? 8192 : 4096) ? 1024 : 256;
  const int64_t padded = cdiv64(a.V, nt) * nt, bytes = padded * (int64_t)sizeof(T);
  const bool cached = bytes <= 132 * 1024;
  static_assert(sizeof(SampleShared<T, 1024>) + 132 * 1024 <= 160 * 1024, "shared memory of a CU");
#define SAMPLE_CASE(N, C)                                                                                              \
  do {                                                                                                                 \
    if (C && bytes > 32 * 1024) {                                                                                      \
      hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&sample_kernel<T, N, C>),                       \
                                         hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);                      \
      if (e != hipSuccess) {                                                                                           \
        neurst_set_error("sample: %s", hipGetErrorString(e));                                                          \
        return NEURST_E_LAUNCH;                                                                                        \
      }                                                                                                                \
    }                                                                                                                  \
    sample_kernel<T, N, C><<<(unsigned)rows, N, C ? bytes : 0, s>>>(a);                                                \
  } while (0)
  if (nt == 256) SAMPLE_CASE(256, true);
  else if (cached) SAMPLE_CASE(1024, true);
  else SAMPLE_CASE(1024, false);
#undef SAMPLE_CASE
  NEURST_CHECK_LAUNCH("sample");
  return NEURST_OK;
}

static int sample_call(SampleArgs a, int64_t rows, int64_t V, int dtype, void* stream, const char* name) {
  NEURST_CHECK_ARG(a.logits && a.u, "%s: null pointer", name);
  NEURST_CHECK_ARG(dtype == NEURST_F32 || dtype == NEURST_BF16, "%s: logits must be fp32 or bf16", name);
  NEURST_CHECK_ARG(rows >= 0 && rows <= INT32_MAX && V > 0 && V <= (1 << 19) && a.ld >= V, "%s: rows of 1..524288 words", name);
  NEURST_CHECK_ARG(a.temperature_rows || (a.temperature >= 0.f && a.temperature <= 3.4e38f), "%s: temperature must be finite and >= 0", name);
  NEURST_CHECK_ARG(a.top_p_rows || (a.top_p > 0.f && a.top_p <= 1.f), "%s: top_p must be in (0, 1]", name);
  NEURST_CHECK_ARG(a.min_p_rows || (a.min_p >= 0.f && a.min_p <= 1.f), "%s: min_p must be in [0, 1]", name);
  NEURST_CHECK_ARG(a.top_k_rows || a.top_k >= 0, "%s: top_k must be >= 0 (0: all)", name);
  if (rows == 0) return NEURST_OK;
  a.V = (int)V;
  return dtype == NEURST_BF16 ? sample_launch<bf16_t>(a, rows, as_stream(stream)) : sample_launch<float>(a, rows, as_stream(stream));
}

extern "C" int neurst_sample(const void* logits, const float* u, int32_t* ids, float* logp, const float* temperature_rows,
                             const int32_t* top_k_rows, const float* top_p_rows, const float* min_p_rows, float temperature, int top_k,
                             float top_p, float min_p, int64_t rows, int64_t V, int64_t ld, int dtype, void* stream) {
  NEURST_CHECK_ARG(ids && logp, "sample: null pointer");
  SampleArgs a = {};
  a.logits = logits; a.u = u; a.ids = ids; a.logp = logp;
  a.temperature_rows = temperature_rows; a.top_k_rows = top_k_rows; a.top_p_rows = top_p_rows; a.min_p_rows = min_p_rows;
  a.temperature = temperature; a.top_k = top_k; a.top_p = top_p; a.min_p = min_p; a.ld = ld;
  return sample_call(a, rows, V, dtype, stream, "sample");
}

extern "C" int neurst_sample_step_checked(const void* logits, const float* u, int32_t* tokens, int32_t* preds, int32_t* finished,
                                          int32_t* len_decoded, int32_t* n_unfinished, float* scores, int32_t* status,
                                          const float* temperature_rows, const int32_t* top_k_rows, const float* top_p_rows,
                                          const float* min_p_rows, float temperature, int top_k, float top_p, float min_p, int64_t rows, int64_t V,
                                          int64_t ld, int64_t step, int64_t max_steps, int eos, int dtype, void* stream) {
  NEURST_CHECK_ARG(tokens && preds && finished && len_decoded && n_unfinished && scores, "sample_step: null pointer");
  NEURST_CHECK_ARG(step >= 0 && step < max_steps, "sample_step: step out of range");
  SampleArgs a = {};
  a.logits = logits; a.u = u; a.ids = tokens; a.preds = preds; a.finished = finished; a.len_decoded = len_decoded;
  a.n_unfinished = n_unfinished; a.scores = scores; a.status = status;
  a.temperature_rows = temperature_rows; a.top_k_rows = top_k_rows; a.top_p_rows = top_p_rows; a.min_p_rows = min_p_rows;
  a.temperature = temperature; a.top_k = top_k; a.top_p = top_p; a.min_p = min_p; a.ld = ld;
  a.step = step; a.max_steps = max_steps; a.eos = eos;
  return sample_call(a, rows, V, dtype, stream, "sample_step");
}

extern "C" int neurst_sample_step(const void* logits, const float* u, int32_t* tokens, int32_t* preds, int32_t* finished, int32_t* len_decoded,
                                  int32_t* n_unfinished, float* scores, const float* temperature_rows, const int32_t* top_k_rows,
                                  const float* top_p_rows, const float* min_p_rows, float temperature, int top_k, float top_p, float min_p,
                                  int64_t rows, int64_t V, int64_t ld, int64_t step, int64_t max_steps, int eos, int dtype, void* stream) {
  return neurst_sample_step_checked(logits, u, tokens, preds, finished, len_decoded, n_unfinished, scores, nullptr, temperature_rows, top_k_rows,
                                    top_p_rows, min_p_rows, temperature, top_k, top_p, min_p, rows, V, ld, step, max_steps, eos, dtype, stream);
}
