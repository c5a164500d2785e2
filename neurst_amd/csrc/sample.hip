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
// The kept set is {key > K} and the first m words (by index) with key == K, keys being the logits in an order-preserving
// integer form.  K is found by counting, not by sorting: a histogram over 2048 equal steps of (max - l) / T in [0, 32) - all
// that can have weight - finds the step where the count passes top_k or the sum passes top_p, then the words of that one step
// are counted again over the range of their keys until one key is left.
//
// One workgroup a row; a row of up to 128 KB is read once, into shared memory, and every later pass runs on that.  Bound by
// the chain of passes and barriers for few rows, by the fp64 exponentials (~25 instructions a word) for many.
#include "common.h"

struct SampleArgs {
  const void* logits;
  const float* u;
  const float *temperature_rows, *top_p_rows, *min_p_rows;
  const int32_t* top_k_rows;
  int32_t* ids;
  float* logp;
  // bookkeeping of a decoding step (all null for a plain draw)
  int32_t *preds, *finished, *len_decoded, *n_unfinished;
  float* scores;
  int64_t ld, step, max_steps;
  int V, top_k, eos;
  float temperature, top_p, min_p;
};

typedef unsigned long long u64;
constexpr int SAMPLE_BINS = 2048;
constexpr double SAMPLE_ONE = 17592186044416.0;      // 2^44
constexpr float SAMPLE_SPAN = 32.f;                   // e^-32 < 2^-45: rounds to 0

__device__ __forceinline__ uint32_t logit_key(float l) {
  const uint32_t b = __builtin_bit_cast(uint32_t, l);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

// round(2^44 exp(x)), x in [-32, 0]: exp(x) = 2^n exp(y), |y| <= ln2 / 2, Taylor polynomial to y^11 (the next term is 6e-15)
__device__ __forceinline__ u64 sample_weight(double x) {
  const double t = x * 1.4426950408889634074, n = rint(t), y = (t - n) * 0.69314718055994530942;
  double p = 2.50521083854417187751e-08;
  p = fma(p, y, 2.75573192239858906526e-07);
  p = fma(p, y, 2.75573192239858906526e-06);
  p = fma(p, y, 2.48015873015873015873e-05);
  p = fma(p, y, 1.98412698412698412698e-04);
  p = fma(p, y, 1.38888888888888888889e-03);
  p = fma(p, y, 8.33333333333333333333e-03);
  p = fma(p, y, 4.16666666666666666667e-02);
  p = fma(p, y, 1.66666666666666666667e-01);
  p = fma(p, y, 0.5);
  p = fma(p, y, 1.0);
  p = fma(p, y, 1.0);
  // the sum with 2^52 holds the rounded integer in its low 52 bits
  const double v = ldexp(p, (int)n + 44) + 4503599627370496.0;
  return __builtin_bit_cast(u64, v) & 0xFFFFFFFFFFFFFull;
}

__device__ __forceinline__ u64 shfl_u64(u64 v, int src) {
  return (u64)(uint32_t)__shfl((int)(uint32_t)v, src, 64) | ((u64)(uint32_t)__shfl((int)(uint32_t)(v >> 32), src, 64) << 32);
}
__device__ __forceinline__ u64 wave_scan_u64(u64 v, int lane) {      // inclusive
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 x = shfl_u64(v, (lane - o) & 63);
    if (lane >= o) v += x;
  }
  return v;
}
__device__ __forceinline__ uint32_t wave_scan_u32(uint32_t v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t x = (uint32_t)__shfl((int)v, (lane - o) & 63, 64);
    if (lane >= o) v += x;
  }
  return v;
}

template <int NT> struct SampleShared {
  u64 hw[SAMPLE_BINS];
  uint32_t hc[SAMPLE_BINS];
  u64 ww[16];
  uint32_t wc[16], wa[16], wb[16];
  float wf[16];
  int bin;
  uint32_t above_c, bin_c;
  u64 above_w, bin_w;
  u64 seg[512];
  int cut;
};

// The row, in shared memory (CACHED) or read again on every pass.  Wave w owns the words [w * span, (w + 1) * span), 64
// neighbours at a time, so index order is wave, step, lane.
template <typename T, int NT, bool CACHED> struct SampleRow {
  const T* p;
  int V, base, steps;
  __device__ __forceinline__ float fetch(int i) const {
    const int idx = base + i * 64;
    const float x = CACHED || idx < V ? to_f32<T>(p[idx]) : -INFINITY;
    return x == x ? x + 0.f : -INFINITY;           // NaN is never drawn; -0 counts as +0
  }
  __device__ __forceinline__ void init(const T* row, T* lds, int V_, int tid) {
    V = V_;
    steps = (V + NT - 1) / NT;
    base = (tid >> 6) * steps * 64 + (tid & 63);
    if constexpr (CACHED) {                        // every lane keeps to its own words: no barrier needed
#pragma unroll 8
      for (int i = 0; i < steps; ++i) {
        const int idx = base + i * 64;
        lds[idx] = idx < V ? row[idx] : (T)-INFINITY;
      }
      p = lds;
    } else {
      p = row;
    }
  }
  template <int UNROLL = 4, typename F> __device__ __forceinline__ void each(F f) const {
#pragma unroll UNROLL
    for (int i = 0; i < steps; ++i) f(fetch(i), base + i * 64, i);
  }
};

// first bin at which the running count (or, by_weight, the running sum) reaches `need`, into s.bin / above_* / bin_*
template <int NT> __device__ __forceinline__ void sample_cross(SampleShared<NT>& s, bool by_weight, u64 need, int tid) {
  constexpr int PER = SAMPLE_BINS / NT;
  const int lane = tid & 63, w = tid >> 6;
  uint32_t c = 0;
  u64 x = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) { c += s.hc[tid * PER + j]; x += s.hw[tid * PER + j]; }
  const uint32_t ci = wave_scan_u32(c, lane);
  const u64 xi = wave_scan_u64(x, lane);
  if (lane == 63) { s.wc[w] = ci; s.ww[w] = xi; }
  __syncthreads();
  uint32_t cb = ci - c;
  u64 xb = xi - x;
  for (int i = 0; i < w; ++i) { cb += s.wc[i]; xb += s.ww[i]; }
  if (by_weight ? (xb < need && xb + x >= need) : ((u64)cb < need && (u64)cb + c >= need)) {
    for (int j = 0; j < PER; ++j) {
      const uint32_t bc = s.hc[tid * PER + j];
      const u64 bw = s.hw[tid * PER + j];
      if (by_weight ? xb + bw >= need : (u64)cb + bc >= need) {
        s.bin = tid * PER + j;
        s.above_c = cb; s.above_w = xb;
        s.bin_c = bc; s.bin_w = bw;
        break;
      }
      cb += bc;
      xb += bw;
    }
  }
  __syncthreads();
}

template <typename T, int NT, bool CACHED> __global__ void __launch_bounds__(NT) sample_kernel(SampleArgs a) {
  constexpr int NW = NT / 64;
  __shared__ SampleShared<NT> s;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t row = blockIdx.x;
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

  extern __shared__ __attribute__((aligned(16))) char row_lds[];
  SampleRow<T, NT, CACHED> r;
  r.init(static_cast<const T*>(a.logits) + row * a.ld, reinterpret_cast<T*>(row_lds), a.V, tid);
  for (int i = tid; i < SAMPLE_BINS; i += NT) { s.hc[i] = 0; s.hw[i] = 0; }
  float mx = -INFINITY;
  r.each([&](float l, int, int) { mx = fmaxf(mx, l); });
  mx = wave_max(mx);
  if (lane == 0) s.wf[w] = mx;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NW; ++i) mx = fmaxf(mx, s.wf[i]);

  int id = -1;
  float logp = -INFINITY;
  if (mx > -INFINITY) {
    const double inv_t = 1.0 / (double)temp;
    const float bin_scale = (float)(SAMPLE_BINS / SAMPLE_SPAN * inv_t);
    auto weight = [&](float l) -> u64 {
      if (l == mx) return (u64)SAMPLE_ONE;
      const double x = ((double)l - (double)mx) * inv_t;
      return x >= -SAMPLE_SPAN ? sample_weight(x) : 0;
    };
    // step of the histogram: monotone in l, 0 for the best; words of the last step and below share it
    auto step_of = [&](float l) -> int {
      const float x = (mx - l) * bin_scale;
      return l == mx ? 0 : (x < (float)(SAMPLE_BINS - 1) ? (int)x : SAMPLE_BINS - 1);
    };
    uint32_t K = 0;            // kept: key > K, or key == K and index <= cut
    int cut = 0x7fffffff;
    bool limited = false;
    u64 kept_in_k = 0;         // the sum over the words top_k keeps
    const bool by_k = top_k < a.V, by_p = top_p < 1.f;
    uint32_t m = 0, ties = 0;  // of the words with key == K the first m are kept, there are `ties`
    if (top_k == 1) {
      uint32_t c = 0;
      r.each([&](float l, int, int) { c += l == mx ? 1u : 0u; });
      c = wave_scan_u32(c, lane);
      if (lane == 63) s.wa[w] = c;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NW; ++i) ties += s.wa[i];
      K = logit_key(mx);
      m = 1;
      limited = true;
    } else {
      // phase 0: the count reaches top_k; phase 1: the sum reaches top_p of what phase 0 kept
      for (int phase = by_k ? 0 : 1; phase < (by_p ? 2 : 1); ++phase) {
        u64 mine = 0;
        uint32_t count = 0;
        if (phase && by_k) {
          __syncthreads();
          for (int i = tid; i < SAMPLE_BINS; i += NT) { s.hc[i] = 0; s.hw[i] = 0; }
          __syncthreads();
        }
        r.each([&](float l, int, int) {
          const u64 x = logit_key(l) >= K ? weight(l) : 0;
          if (x) {
            const int b = step_of(l);
            atomicAdd(&s.hc[b], 1u);
            atomicAdd(&s.hw[b], x);
            mine += x;
            ++count;
          }
        });
        mine = wave_scan_u64(mine, lane);
        count = wave_scan_u32(count, lane);
        if (lane == 63) { s.ww[w] = mine; s.wa[w] = count; }
        __syncthreads();
        u64 need = 0, n = 0;
        if (phase == 0 || !by_k) kept_in_k = 0;
#pragma unroll
        for (int i = 0; i < NW; ++i) {
          if (phase == 0 || !by_k) kept_in_k += s.ww[i];
          n += s.wa[i];
        }
        __syncthreads();
        if (phase == 0) {
          if (n <= (u64)top_k) continue;       // every word with weight stays
          need = (u64)top_k;
        } else {
          need = (u64)ceil((double)top_p * (double)kept_in_k);
          if (need < 1) need = 1;
          if (need >= kept_in_k) continue;
        }
        // down to one key: ac / aw = words and sum before it, s.bin_c / s.bin_w = those that equal it
        sample_cross<NT>(s, phase == 1, need, tid);
        const int bin = s.bin;
        uint32_t ac = s.above_c;
        u64 aw = s.above_w;
        uint32_t lo = 0xffffffffu, hi = 0;
        r.each([&](float l, int, int) {
          if (l > -INFINITY && step_of(l) == bin && weight(l)) {
            const uint32_t k = logit_key(l);
            lo = k < lo ? k : lo;
            hi = k > hi ? k : hi;
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
          const int bits = 32 - __builtin_clz(hi - lo), shift = bits > 11 ? bits - 11 : 0;
          for (int i = tid; i < SAMPLE_BINS; i += NT) { s.hc[i] = 0; s.hw[i] = 0; }
          __syncthreads();
          r.each([&](float l, int, int) {
            const uint32_t k = logit_key(l);
            if (k >= lo && k <= hi) {
              const u64 x = weight(l);
              if (x) {
                atomicAdd(&s.hc[(hi - k) >> shift], 1u);
                atomicAdd(&s.hw[(hi - k) >> shift], x);
              }
            }
          });
          __syncthreads();
          sample_cross<NT>(s, phase == 1, need - (phase == 1 ? aw : (u64)ac), tid);
          ac += s.above_c;
          aw += s.above_w;
          hi -= (uint32_t)s.bin << shift;
          const uint32_t span = (1u << shift) - 1u;
          if (hi - lo > span) lo = hi - span;
          __syncthreads();
        }
        K = hi;
        ties = s.bin_c;
        const u64 each = s.bin_w / ties;
        if (phase == 0) {
          m = (uint32_t)top_k - ac;
          kept_in_k = aw + (u64)m * each;
        } else {
          m = (uint32_t)((need - aw + each - 1) / each);
        }
        limited = true;
      }
    }
    __syncthreads();
    if (limited && m < ties) {      // equal words: the first m by index
      uint32_t c = 0;
      r.each([&](float l, int, int) { c += logit_key(l) == K ? 1u : 0u; });
      c = wave_scan_u32(c, lane);
      if (lane == 63) s.wc[w] = c;
      __syncthreads();
      uint32_t before = 0;
      for (int i = 0; i < w; ++i) before += s.wc[i];
      if (before < m && before + s.wc[w] >= m) {
        uint32_t seen = before;
        r.template each<1>([&](float l, int idx, int) {
          const u64 eq = __ballot(logit_key(l) == K);
          const uint32_t here = (uint32_t)__popcll(eq);
          if (seen < m && seen + here >= m) {
            const bool mine_last = ((eq >> lane) & 1) && seen + (uint32_t)__popcll(eq & ((2ull << lane) - 1)) == m;
            if (mine_last) s.cut = idx;
          }
          seen += here;
        });
      }
      __syncthreads();
      cut = s.cut;
    }
    const u64 lowest = (u64)ceil((double)min_p * SAMPLE_ONE);
    auto kept = [&](float l, int idx) -> u64 {
      const uint32_t k = logit_key(l);
      if (limited && (k < K || (k == K && idx > cut))) return 0;
      const u64 x = weight(l);
      return x >= lowest ? x : 0;
    };
    u64 mine = 0;
    r.each([&](float l, int idx, int) { mine += kept(l, idx); });
    const u64 incl = wave_scan_u64(mine, lane);
    if (lane == 63) s.ww[w] = incl;
    for (int i = tid; i < 512; i += NT) s.seg[i] = 0;
    __syncthreads();
    u64 total = 0, before = 0;
    for (int i = 0; i < NW; ++i) {
      if (i < w) before += s.ww[i];
      total += s.ww[i];
    }
    u64 thr = (u64)((double)u * (double)total);
    if (thr >= total) thr = total - 1;
    if (before <= thr && thr < before + s.ww[w]) {      // this wave holds the word: its step, then its lane
      r.each([&](float l, int idx, int i) {
        const u64 x = kept(l, idx);
        if (x) atomicAdd(&s.seg[i], x);
      });
      __threadfence_block();
      u64 run = before;
      int at = 0;
      for (int j = 0; j < r.steps; j += 64) {           // 64 steps at a time
        const u64 x = *(volatile u64*)&s.seg[j + lane], inc = run + wave_scan_u64(x, lane);
        const u64 over = __ballot(inc > thr);
        if (over) {
          const int k = __builtin_ctzll(over);
          at = j + k;
          run = shfl_u64(inc - x, k);
          break;
        }
        run = shfl_u64(inc, 63);
      }
      const int idx = r.base + at * 64;
      const float l = r.fetch(at);
      const u64 x = kept(l, idx);
      const u64 c = run + wave_scan_u64(x, lane);
      if (c > thr && c - x <= thr) {
        s.cut = idx;
        s.above_w = x;
      }
    }
    __syncthreads();
    id = s.cut;
    logp = (float)log((double)s.above_w / (double)total);
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
      a.ids[row] = tok;
    }
  }
}

template <typename T> static int sample_launch(const SampleArgs& a, int64_t rows, hipStream_t s) {
  // 1024 threads once a row gives each of them four words; 128 KB of shared memory hold the row beside the histogram
  const int nt = a.V > 4096 ? 1024 : 256;
  const int64_t padded = cdiv64(a.V, nt) * nt, bytes = padded * (int64_t)sizeof(T);
  const bool cached = bytes <= 128 * 1024;
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

extern "C" int neurst_sample_step(const void* logits, const float* u, int32_t* tokens, int32_t* preds, int32_t* finished, int32_t* len_decoded,
                                  int32_t* n_unfinished, float* scores, const float* temperature_rows, const int32_t* top_k_rows,
                                  const float* top_p_rows, const float* min_p_rows, float temperature, int top_k, float top_p, float min_p,
                                  int64_t rows, int64_t V, int64_t ld, int64_t step, int64_t max_steps, int eos, int dtype, void* stream) {
  NEURST_CHECK_ARG(tokens && preds && finished && len_decoded && n_unfinished && scores, "sample_step: null pointer");
  NEURST_CHECK_ARG(step >= 0 && step < max_steps, "sample_step: step out of range");
  SampleArgs a = {};
  a.logits = logits; a.u = u; a.ids = tokens; a.preds = preds; a.finished = finished; a.len_decoded = len_decoded;
  a.n_unfinished = n_unfinished; a.scores = scores;
  a.temperature_rows = temperature_rows; a.top_k_rows = top_k_rows; a.top_p_rows = top_p_rows; a.min_p_rows = min_p_rows;
  a.temperature = temperature; a.top_k = top_k; a.top_p = top_p; a.min_p = min_p; a.ld = ld;
  a.step = step; a.max_steps = max_steps; a.eos = eos;
  return sample_call(a, rows, V, dtype, stream, "sample_step");
}
