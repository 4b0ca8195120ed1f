// Draws a token from each row of logits: temperature, top-k, top-p and min-p, from given uniform numbers (gfx950).
//
//   w_j = exp((l_j - max) / T).  Kept: the top_k largest; of those the shortest prefix, largest first, that holds top_p of
//   their mass; of those the ones with w_j >= min_p.  The answer is the lowest index at which the running sum of the kept
//   w, by index, exceeds u times their sum.  Ties go to the lowest index.
//
// The answer is an index that a sum decides, so the sums are exact: every w is rounded once to a multiple of 2^-F (F = 44
// for rows of up to 2^18 logits) and added as a 64-bit integer.  The order of additions then changes nothing, and the
// answer is the real numbers' unless u lies within about 2^-40 of a border.
#include <limits.h>
#include <math.h>

#include "common.h"

namespace {

typedef unsigned long long u64;

// ordered key of a logit: larger logit, larger key; -inf and NaN (never drawn) get 0; both zeros the same
__device__ __forceinline__ uint32_t key_of(float l) {
  if (!(l > -INFINITY)) return 0u;
  const uint32_t b = __builtin_bit_cast(uint32_t, l + 0.f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __builtin_bit_cast(float, key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
}

// log2 of w: (l - max) log2(e) / T
struct Scale {
  float m;          // the row's largest logit
  double c;         // log2(e) / T
  int F;            // weights are multiples of 2^-F
};
__device__ __forceinline__ double log2_weight(const Scale& s, float l) { return l == s.m ? 0.0 : ((double)l - (double)s.m) * s.c; }
__device__ __forceinline__ u64 fixed_weight(const Scale& s, double t) {
  if (!(t > -64.0)) return 0;                       // (NaN: -inf / inf)
  return (u64)(ldexp(exp2(t), s.F) + 0.5);
}
__device__ __forceinline__ u64 weight_of(const Scale& s, float l) {
  return l > -INFINITY ? fixed_weight(s, log2_weight(s, l)) : 0ull;
}

struct Settings {
  double T, p, minp;
  int64_t k;
  const float *Tr, *pr, *mr;
  const int32_t* kr;
};

template <int NT>
struct RowState {
  u64 mass[256];
  uint32_t cnt[256];
  u64 wsum[NT / 64];
  uint32_t wcnt[NT / 64];
  uint32_t key;         // what the last descent found
  u64 above;            // mass above that key
  uint32_t n_above;     // number above that key
  u64 total;
  int64_t answer;
};

// exclusive scan of a thread's value over the workgroup; total to *sum
template <int NT, typename I>
__device__ I block_scan(I v, I* s, I* sum) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  I inc = v;
  for (int o = 1; o < 64; o <<= 1) {
    const I up = __shfl_up(inc, o);
    if (lane >= o) inc += up;
  }
  __syncthreads();
  if (lane == 63) s[wave] = inc;
  __syncthreads();
  I before = 0, all = 0;
  for (int w = 0; w < NT / 64; ++w) {
    if (w < wave) before += s[w];
    all += s[w];
  }
  *sum = all;
  return before + inc - v;
}

// One workgroup per row; the ordered keys are searched byte by byte, the row read once for each byte.
template <typename T, int NT>
__global__ __launch_bounds__(NT) void sample_row_kernel(int64_t rows, int64_t V, const T* __restrict__ logits, int64_t ld, Settings st, int F,
                                                        const float* __restrict__ u, int64_t* __restrict__ out) {
  __shared__ RowState<NT> S;
  const int tid = threadIdx.x;
  const int64_t r = blockIdx.x;
  const T* x = logits + r * ld;
  const double temp = st.Tr ? (double)st.Tr[r] : st.T;
  const int64_t kk = st.kr ? (int64_t)st.kr[r] : st.k;
  const double p = st.pr ? (double)st.pr[r] : st.p;
  const double mp = st.mr ? (double)st.mr[r] : st.minp;

  // the largest logit, and its lowest index
  u64 best = 0;
  for (int64_t j = tid; j < V; j += NT) {
    const u64 b = ((u64)key_of((float)x[j]) << 32) | (uint32_t)~(uint32_t)j;
    best = b > best ? b : best;
  }
  for (int o = 32; o > 0; o >>= 1) {
    const u64 b = __shfl_xor(best, o);
    best = b > best ? b : best;
  }
  if ((tid & 63) == 0) S.wsum[tid >> 6] = best;
  __syncthreads();
  for (int w = 0; w < NT / 64; ++w) best = S.wsum[w] > best ? S.wsum[w] : best;
  const uint32_t kmax = (uint32_t)(best >> 32);
  if (kmax == 0 || !(temp > 0.0)) {
    if (tid == 0) out[r] = kmax == 0 ? -1 : (int64_t)(uint32_t)~(uint32_t)best;
    return;
  }
  const Scale sc = {logit_of(kmax), 1.4426950408889634074 / temp, F};
  const bool by_k = kk > 0 && kk < V, by_p = p < 1.0;
  const double tmin = mp > 0.0 ? log2(mp < 1.0 ? mp : 1.0) : -INFINITY;

  // a cut: every key above `cut`, and the first `ties` (by index) that equal it
  uint32_t cut = 1, ties = UINT_MAX;
  u64 whole = 0;                        // mass of what top-k keeps
  for (int stage = by_k ? 0 : 1; stage < (by_p ? 2 : 1); ++stage) {
    // stage 0: the kk-th largest key; stage 1: the key at which the mass, from above, reaches p of the whole
    u64 need = 0;
    if (stage == 1) {
      if (!by_k) {
        u64 w = 0;
        for (int64_t j = tid; j < V; j += NT) w += weight_of(sc, (float)x[j]);
        block_scan<NT>(w, S.wsum, &whole);
      }
      const double d = ceil((p > 0.0 ? p : 0.0) * (double)whole);
      need = d >= 1.0 ? (u64)d : 1;
      if (need > whole) need = whole;
    }
    uint32_t prefix = 0;
    u64 above = 0;
    uint32_t n_above = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      for (int b = tid; b < 256; b += NT) { S.mass[b] = 0; S.cnt[b] = 0; }
      __syncthreads();
      for (int64_t j = tid; j < V; j += NT) {
        const uint32_t key = key_of((float)x[j]);
        if (key == 0 || key < cut) continue;
        if (shift < 24 && (key >> (shift + 8)) != (prefix >> (shift + 8))) continue;
        const uint32_t b = key >> shift & 255;
        atomicAdd(&S.cnt[b], 1u);
        if (stage == 1 && key > cut) atomicAdd(&S.mass[b], weight_of(sc, (float)x[j]));
      }
      __syncthreads();
      if (tid == 0) {
        // the ties at top-k's own cut count only `ties` times
        if (stage == 1 && ties != UINT_MAX && (shift == 24 || (cut >> (shift + 8)) == (prefix >> (shift + 8))))
          S.mass[cut >> shift & 255] += ties * weight_of(sc, logit_of(cut));
        u64 m = above;
        uint32_t n = n_above;
        int b = 255;
        for (; b > 0; --b) {
          if (stage == 0 ? n + S.cnt[b] >= (u64)kk : m + S.mass[b] >= need) break;
          m += S.mass[b];
          n += S.cnt[b];
        }
        S.key = prefix | (uint32_t)b << shift;
        S.above = m;
        S.n_above = n;
      }
      __syncthreads();
      prefix = S.key;
      above = S.above;
      n_above = S.n_above;
    }
    if (stage == 0) {
      // fewer than kk logits that can be drawn: the descent ends at key 0 and everything is kept
      cut = prefix > 0 ? prefix : 1;
      ties = prefix > 0 ? (uint32_t)(kk - n_above) : UINT_MAX;
      u64 w = 0;
      if (by_p) {
        for (int64_t j = tid; j < V; j += NT)
          if (key_of((float)x[j]) > cut) w += weight_of(sc, (float)x[j]);
        if (prefix == 0)
          for (int64_t j = tid; j < V; j += NT)
            if (key_of((float)x[j]) == cut) w += weight_of(sc, (float)x[j]);
        block_scan<NT>(w, S.wsum, &whole);
        if (prefix > 0) whole += ties * weight_of(sc, logit_of(cut));
      }
    } else {
      const u64 w = weight_of(sc, logit_of(prefix));
      const u64 c = w ? (need - above + w - 1) / w : 1;
      if (prefix > cut) {
        cut = prefix;
        ties = c < UINT_MAX ? (uint32_t)c : UINT_MAX;
      } else if (c < ties) {
        ties = (uint32_t)c;
      }
    }
  }

  // by index: every thread a contiguous piece; ties first, then mass, then the piece in which the sum passes
  const int64_t seg = (V + NT - 1) / NT, lo = tid * seg < V ? tid * seg : V, hi = lo + seg < V ? lo + seg : V;
  uint32_t eq = 0, all_eq;
  for (int64_t j = lo; j < hi; ++j) eq += key_of((float)x[j]) == cut;
  const uint32_t eq0 = block_scan<NT>(eq, S.wcnt, &all_eq);
  u64 mass = 0, all;
  uint32_t e = eq0;
  for (int64_t j = lo; j < hi; ++j) {
    const float l = (float)x[j];
    const uint32_t key = key_of(l);
    if (key < cut || key == 0 || (key == cut && e++ >= ties)) continue;
    const double t = log2_weight(sc, l);
    if (t >= tmin) mass += fixed_weight(sc, t);
  }
  const u64 m0 = block_scan<NT>(mass, S.wsum, &all);
  const float uu = u[r];
  u64 target = uu > 0.f ? (u64)((double)uu * (double)all) : 0;
  if (target >= all) target = all - 1;
  if (m0 <= target && target < m0 + mass) {
    u64 run = m0;
    e = eq0;
    for (int64_t j = lo; j < hi; ++j) {
      const float l = (float)x[j];
      const uint32_t key = key_of(l);
      if (key < cut || key == 0 || (key == cut && e++ >= ties)) continue;
      const double t = log2_weight(sc, l);
      if (t >= tmin) run += fixed_weight(sc, t);
      if (run > target) {
        out[r] = j;
        break;
      }
    }
  }
}

}  // namespace

extern "C" int tad_sample_tokens(int64_t rows, int64_t V, const void* logits, int dtype, int64_t ld, double temperature, const float* temperature_rows,
                                 int64_t top_k, const int32_t* top_k_rows, double top_p, const float* top_p_rows, double min_p,
                                 const float* min_p_rows, const float* u, int64_t* out, tad_stream_t stream) {
  TAD_CHECK(rows >= 0 && rows <= INT_MAX && V >= 1 && V <= INT_MAX, "tad_sample_tokens: bad sizes");
  TAD_CHECK(dtype == TAD_F32 || dtype == TAD_BF16, "tad_sample_tokens: bad element type");
  TAD_CHECK(ld >= V, "tad_sample_tokens: bad leading dimension");
  TAD_CHECK(temperature_rows || temperature >= 0.0, "tad_sample_tokens: the temperature has to be 0 or more");
  TAD_CHECK(top_p_rows || top_p >= 0.0, "tad_sample_tokens: top_p has to be 0 or more");
  TAD_CHECK(min_p_rows || (min_p >= 0.0 && min_p <= 1.0), "tad_sample_tokens: min_p has to lie in [0, 1]");
  TAD_CHECK(top_k_rows || top_k >= 0, "tad_sample_tokens: top_k has to be 0 (off) or more");
  if (rows == 0) return TAD_OK;
  TAD_CHECK(logits && u && out, "tad_sample_tokens: null pointer");
  int lg = 0;
  while (((int64_t)1 << lg) < V) ++lg;
  const int F = 62 - lg < 44 ? 62 - lg : 44;
  const Settings st = {temperature, top_p, min_p, top_k, temperature_rows, top_p_rows, min_p_rows, top_k_rows};
  hipStream_t s = (hipStream_t)stream;
  if (dtype == TAD_F32)
    hipLaunchKernelGGL((sample_row_kernel<float, 256>), dim3((unsigned)rows), dim3(256), 0, s, rows, V, (const float*)logits, ld, st, F, u, out);
  else
    hipLaunchKernelGGL((sample_row_kernel<bf16_t, 256>), dim3((unsigned)rows), dim3(256), 0, s, rows, V, (const bf16_t*)logits, ld, st, F, u, out);
  TAD_LAUNCH_CHECK();
  return TAD_OK;
}
