// Draws a token from each row of logits: temperature, top-k, top-p and min-p, from given uniform numbers (gfx950).
//
//   w_j = exp((l_j - max) / T).  Kept: the top_k largest; of those the shortest prefix, largest first, that holds top_p of
//   their mass; of those the ones with w_j >= min_p.  The answer is the lowest index at which the running sum of the kept
//   w, by index, exceeds u times their sum.  Ties go to the lowest index.
//
// The answer is an index that a sum decides, so the sums are exact: every w is rounded once to a multiple of 2^-F (F = 44
// for rows of up to 2^18 logits) and added as a 64-bit integer.  The order of additions then changes nothing, and the
// answer is the real numbers' unless u lies within about 2^-40 of a border.  Float64 fused multiply-adds issue at the rate
// of float32 ones here, so such a weight costs about 20 instructions.
//
// Every filter keeps a prefix of the row in falling order (ties by index), so their conjunction is the shortest of the
// prefixes: one cut (a key, and how many of those that equal it).
#include <limits.h>
#include <math.h>

#include "row_pieces.h"

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

struct Scale {
  float m;          // the row's largest logit
  double c;         // log2(e) / T
  int F;            // weights are multiples of 2^-F
};
// log2 of w
__device__ __forceinline__ double log2_weight(const Scale& s, float l) { return l == s.m ? 0.0 : ((double)l - (double)s.m) * s.c; }
// 2^t in units of 2^-F, rounded: 2^n times the series of e^z, z = ln 2 (t - n), |z| <= 0.347, whose first term left out is below
// 2^-47; the last bits come out of the addition of 2^52
__device__ __forceinline__ u64 fixed_weight(const Scale& s, double t) {
  if (!(t > -48.0)) return 0;                       // (NaN: -inf / inf)
  const double n = rint(t), z = (t - n) * 0.6931471805599453094;
  double p = 1.0 / 479001600;
  p = __builtin_fma(p, z, 1.0 / 39916800);
  p = __builtin_fma(p, z, 1.0 / 3628800);
  p = __builtin_fma(p, z, 1.0 / 362880);
  p = __builtin_fma(p, z, 1.0 / 40320);
  p = __builtin_fma(p, z, 1.0 / 5040);
  p = __builtin_fma(p, z, 1.0 / 720);
  p = __builtin_fma(p, z, 1.0 / 120);
  p = __builtin_fma(p, z, 1.0 / 24);
  p = __builtin_fma(p, z, 1.0 / 6);
  p = __builtin_fma(p, z, 0.5);
  p = __builtin_fma(p, z, 1.0);
  p = __builtin_fma(p, z, 1.0);
  return __builtin_bit_cast(u64, __builtin_amdgcn_ldexp(p, (int)n + s.F) + 4503599627370496.0) & 0xfffffffffffffull;
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
struct RowSettings {
  double T, p, tmin;       // tmin: log2 of min_p
  int64_t k;
  __device__ RowSettings(const Settings& st, int64_t r) {
    T = st.Tr ? (double)st.Tr[r] : st.T;
    k = st.kr ? (int64_t)st.kr[r] : st.k;
    p = st.pr ? (double)st.pr[r] : st.p;
    const double m = st.mr ? (double)st.mr[r] : st.minp;
    tmin = m > 0.0 ? log2(m < 1.0 ? m : 1.0) : -INFINITY;
  }
};
// the mass that a prefix has to reach, and the sum that has to be exceeded
__device__ __forceinline__ u64 mass_needed(double p, u64 whole) {
  const double d = ceil((p > 0.0 ? p : 0.0) * (double)whole);
  const u64 n = d >= 1.0 ? (u64)d : 1;
  return n < whole ? n : whole;
}
__device__ __forceinline__ u64 target_of(float u, u64 all) {
  const u64 t = u > 0.f ? (u >= 1.f ? all : (u64)((double)u * (double)all)) : 0;
  return t < all ? t : all - 1;
}

// ---------------------------------------------------------------- rows of up to 2048 logits: G lanes of a wave per row
// The row and its weights stay in registers, a contiguous piece of E logits or fewer a lane; what the lanes share goes
// across with DPP moves.  A cut is searched for by bisection: on the logits' values (their weights are exponential in them,
// so a few steps separate neighbours), then, where a value does not lie between its neighbours any more, on the ordered
// keys, so that it ends after at most 48 steps whatever the logits are.
template <int CTRL, typename V>
__device__ __forceinline__ V dpp(V v) {
  if constexpr (sizeof(V) == 8) {
    const u64 b = __builtin_bit_cast(u64, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xf, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xf, 0xf, false);
    return __builtin_bit_cast(V, (u64)hi << 32 | lo);
  } else {
    return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
  }
}
template <typename V>
__device__ __forceinline__ V lane_value(V v, int l) {
  if constexpr (sizeof(V) == 8) {
    const u64 b = __builtin_bit_cast(u64, v);
    return __builtin_bit_cast(V, (u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), l) << 32 |
                                     (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, l));
  } else {
    return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l));
  }
}
struct Add {
  template <typename V> __device__ __forceinline__ V operator()(V a, V b) const { return a + b; }
};
struct Max {
  template <typename V> __device__ __forceinline__ V operator()(V a, V b) const { return a > b ? a : b; }
};
struct Min {
  template <typename V> __device__ __forceinline__ V operator()(V a, V b) const { return a < b ? a : b; }
};
template <int G, typename Op, typename V>
__device__ __forceinline__ V across(V v) {
  const Op op;
  v = op(v, dpp<0xB1>(v));                    // quad_perm [1,0,3,2]
  v = op(v, dpp<0x4E>(v));                    // quad_perm [2,3,0,1]
  if constexpr (G >= 16) {
    v = op(v, dpp<0x141>(v));                 // row_half_mirror
    v = op(v, dpp<0x140>(v));                 // row_mirror
  }
  if constexpr (G == 64) v = op(op(lane_value(v, 0), lane_value(v, 16)), op(lane_value(v, 32), lane_value(v, 48)));
  return v;
}
// what the lanes before this one hold together
template <int G, typename V>
__device__ __forceinline__ V lanes_before(V v, int lane) {
  V inc = v;
#pragma unroll
  for (int o = 1; o < G; o <<= 1) {
    const V up = __shfl_up(inc, o, G);
    if (lane >= o) inc += up;
  }
  return inc - v;
}

template <typename T, int G, int E>
__global__ __launch_bounds__(256) void sample_group_kernel(int64_t rows, int V, int per, const T* __restrict__ logits, int64_t ld, Settings st, int F,
                                                           const float* __restrict__ u, int64_t* __restrict__ out) {
  const int lane = threadIdx.x & (G - 1), j0 = lane * per;
  const int64_t r = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
  if (r >= rows) return;
  const T* x = logits + r * ld;
#define EACH(...)                        \
  _Pragma("unroll") for (int e = 0; e < E; ++e) { \
    if (e >= per) break;                 \
    __VA_ARGS__                          \
  }
  float v[E];
  EACH(v[e] = j0 + e < V ? (float)x[j0 + e] : -INFINITY;)
  const RowSettings rs(st, r);
  float m = -INFINITY;
  EACH(v[e] = v[e] > -INFINITY ? v[e] : -INFINITY; m = fmaxf(m, v[e]);)
  m = across<G, Max>(m);
  if (m == -INFINITY || !(rs.T > 0.0)) {
    int at = V;
    EACH(at = v[e] == m && e < at - j0 ? j0 + e : at;)
    at = across<G, Min>(at);
    if (lane == 0) out[r] = m == -INFINITY ? -1 : at;
    return;
  }
  const Scale sc = {m, 1.4426950408889634074 / rs.T, F};
  const bool by_k = rs.k > 0 && rs.k < V, by_p = rs.p < 1.0;
  u64 w[E];
  uint32_t low = 0;                           // the ones below min_p
  EACH(const double t = log2_weight(sc, v[e]); w[e] = v[e] > -INFINITY ? fixed_weight(sc, t) : 0ull; low |= t >= rs.tmin ? 0u : 1u << e;)

  // halves the distance between two keys: by value as long as that lies between them
  const auto between = [](uint32_t lo, uint32_t hi, int step) {
    const uint32_t b = key_of(0.5f * logit_of(lo) + 0.5f * logit_of(hi));
    return step < 16 && b > lo && b <= hi ? b : lo + (hi - lo + 1) / 2;
  };
  // drops what lies below `cut`, and of its equals (n of them) all but the first `ties`
  const auto drop = [&](float cut, uint32_t ties, uint32_t n) {
    uint32_t rank = 0;
    if (ties < n) {
      uint32_t mine = 0;
      EACH(mine += v[e] == cut;)
      rank = lanes_before<G>(mine, lane);
    }
    EACH(const bool gone = v[e] < cut || (ties < n && v[e] == cut && rank++ >= ties); v[e] = gone ? -INFINITY : v[e]; w[e] = gone ? 0 : w[e];)
  };

  if (by_k) {
    int n = 0;
    uint32_t lo = UINT_MAX, hi = key_of(m);
    EACH(n += v[e] > -INFINITY; const uint32_t k = key_of(v[e]); lo = k && k < lo ? k : lo;)
    n = across<G, Add>(n);
    lo = across<G, Min>(lo);
    if (n > rs.k) {
      const int want = (int)rs.k;
      int c = n;                              // that many reach `lo`
      for (int step = 0; lo < hi && c != want; ++step) {
        const uint32_t b = between(lo, hi, step);
        const float f = logit_of(b);
        int k = 0;
        EACH(k += v[e] >= f;)
        k = across<G, Add>(k);
        if (k >= want) { lo = b; c = k; } else hi = b - 1;
      }
      const float cut = logit_of(lo);
      uint32_t eq = 0;
      EACH(eq += v[e] == cut;)
      eq = across<G, Add>(eq);
      drop(cut, eq - (uint32_t)(c - want), eq);
    }
  }
  if (by_p) {
    u64 whole = 0;
    int n = 0;
    uint32_t lo = UINT_MAX, hi = key_of(m);
    EACH(whole += w[e]; n += w[e] != 0; const uint32_t k = key_of(v[e]); lo = w[e] && k < lo ? k : lo;)
    whole = across<G, Add>(whole);
    n = across<G, Add>(n);
    lo = across<G, Min>(lo);
    const u64 need = mass_needed(rs.p, whole);
    int above = 0;                            // n reach `lo`, `above` lie above `hi`
    for (int step = 0; lo < hi && n - above > 1; ++step) {
      const uint32_t b = between(lo, hi, step);
      const float f = logit_of(b);
      u64 mass = 0;
      int k = 0;
      EACH(const bool in = v[e] >= f; mass += in ? w[e] : 0ull; k += in;)
      mass = across<G, Add>(mass);
      k = across<G, Add>(k);
      if (mass >= need) { lo = b; n = k; } else { hi = b - 1; above = k; }
    }
    const float cut = logit_of(lo);
    uint32_t eq = (uint32_t)(n - above), ties = eq;
    if (eq > 1) {                             // (lo = hi: equals)
      u64 mass = 0, one = 0;
      EACH(mass += v[e] > cut ? w[e] : 0ull; one = v[e] == cut ? w[e] : one;)
      mass = across<G, Add>(mass);
      one = across<G, Max>(one);
      ties = (uint32_t)((need - mass + one - 1) / one);
    }
    drop(cut, ties, eq);
  }
  u64 mine = 0;
  EACH(w[e] = low >> e & 1 ? 0ull : w[e]; mine += w[e];)
  const u64 all = across<G, Add>(mine), target = target_of(u[r], all);
  u64 run = lanes_before<G>(mine, lane);
  if (run <= target && target < run + mine) {
    int at = 0;
    EACH(run += w[e]; at += run <= target;)
    out[r] = j0 + at;
  }
#undef EACH
}

// ---------------------------------------------------------------- longer rows: a workgroup per row
constexpr int BINS = 768;       // of log2 w, sixteen to the octave, down to 2^-48

template <int NT>
struct RowState {
  static constexpr int NW = NT / 64;
  static constexpr int CAP = NT < 256 ? 256 : NT;       // candidates
  u64 list[CAP];
  u64 mass[BINS];
  uint32_t cnt[256];
  u64 wsum[NW];
  uint32_t wcnt[NW];
  uint32_t n, key, n_above;
  u64 above;
};

template <int NT, typename I>
__device__ __forceinline__ I block_total(I v, I* s) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if constexpr (NT == 64) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  I all = 0;
  for (int w = 0; w < NT / 64; ++w) all += s[w];
  return all;
}
// exclusive scan of a thread's value over the workgroup; the total to *sum
template <int NT, typename I>
__device__ __forceinline__ I block_scan(I v, I* s, I* sum) {
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

// sorts list[0 .. P), P a power of two: falling, or rising
template <int NT>
__device__ void sort_list(u64* list, int P, bool falling) {
  for (int size = 2; size <= P; size <<= 1)
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < P / 2; i += NT) {
        const int lo = 2 * i - (i & (stride - 1)), hi = lo + stride;
        const u64 a = list[lo], b = list[hi];
        if ((a < b) == (((lo & size) == 0) == falling) && a != b) { list[lo] = b; list[hi] = a; }
      }
    }
  __syncthreads();
}
__device__ __forceinline__ int pow2_at_least(int n) {
  int P = 64;
  while (P < n) P <<= 1;
  return P;
}

template <typename T, int NT>
__global__ __launch_bounds__(NT) void sample_row_kernel(int64_t rows, int64_t V, const T* __restrict__ logits, int64_t ld, Settings st, int F,
                                                        const float* __restrict__ u, int64_t* __restrict__ out) {
  typedef RowState<NT> State;
  constexpr int VEC = RowPieces<T>::VEC, NW = State::NW, CAP = State::CAP;
  __shared__ State S;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t r = blockIdx.x;
  const RowPieces<T> row(logits + r * ld, V);
  const RowSettings rs(st, r);
  // a wave's own contiguous share of the pieces
  const int64_t seg = (row.np + NW - 1) / NW, lo = wave * seg < row.np ? wave * seg : row.np, hi = lo + seg < row.np ? lo + seg : row.np;

#define EACH_PIECE(...)                                   \
  _Pragma("unroll 4") for (int64_t i = lo + lane; i < hi; i += 64) { \
    float v[VEC];                                         \
    row.load(i, v);                                       \
    __VA_ARGS__                                           \
  }

  // the largest logit of the thread, then of the row
  float tm = -INFINITY;
  EACH_PIECE(_Pragma("unroll") for (int e = 0; e < VEC; ++e) tm = v[e] > tm ? v[e] : tm;)
  float m = tm;
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  if constexpr (NT > 64) {
    float* f = reinterpret_cast<float*>(S.wcnt);
    if (lane == 0) f[wave] = m;
    __syncthreads();
    for (int w = 0; w < NW; ++w) m = fmaxf(m, f[w]);
    __syncthreads();
  }
  if (m == -INFINITY) {
    if (tid == 0) out[r] = -1;
    return;
  }
  if (!(rs.T > 0.0)) {
    u64 at = ~0ull;                       // the lowest index of the largest
    EACH_PIECE(_Pragma("unroll") for (int e = 0; e < VEC; ++e) if (v[e] == m) {
      const u64 j = (u64)(row.first(i) + e);
      at = j < at ? j : at;
    })
    for (int o = 32; o > 0; o >>= 1) {
      const u64 b = __shfl_xor(at, o);
      at = b < at ? b : at;
    }
    if (lane == 0) S.wsum[wave] = at;
    __syncthreads();
    for (int w = 0; w < NW; ++w) at = S.wsum[w] < at ? S.wsum[w] : at;
    if (tid == 0) out[r] = (int64_t)at;
    return;
  }
  const Scale sc = {m, 1.4426950408889634074 / rs.T, F};
  const bool by_k = rs.k > 0 && rs.k < V, by_p = rs.p < 1.0;

  // ---- few candidates: all that top-k can keep fits the list
  if ((by_k && rs.k <= CAP / 2) || ((by_k || by_p) && V <= CAP)) {
    const int64_t kk = by_k ? rs.k : V;
    uint32_t thr = 0;
    if (V > CAP) {
      // kk threads whose largest is at least `thr`: so at least kk logits are; 16 bits of it are enough (NT < kk: no thread's
      // largest says anything, and the list runs over)
      const uint32_t mine = key_of(tm);
      for (int bit = 31; bit >= 16; --bit) {
        const uint32_t t = thr | 1u << bit;
        int n = __popcll(__ballot(mine >= t));
        if constexpr (NT > 64) n = __syncthreads_count(mine >= t);
        if (n >= kk) thr = t;
      }
    }
    if (thr == 0) thr = 1;
    if (tid == 0) S.n = 0;
    __syncthreads();
    EACH_PIECE(_Pragma("unroll") for (int e = 0; e < VEC; ++e) {
      const uint32_t key = key_of(v[e]);
      if (key >= thr) {
        const uint32_t at = atomicAdd(&S.n, 1u);
        if (at < CAP) S.list[at] = (u64)key << 32 | (uint32_t)~(uint32_t)(row.first(i) + e);
      }
    })
    __syncthreads();
    const uint32_t n = S.n;
    if (n <= CAP) {
      const int P = pow2_at_least((int)n);
      for (int i = n + tid; i < P; i += NT) S.list[i] = 0;
      sort_list<NT>(S.list, P, true);
      const int nk = kk < n ? (int)kk : (int)n;
      u64 whole = 0;
      if (by_p) {
        u64 w = 0;
        for (int i = tid; i < nk; i += NT) w += weight_of(sc, logit_of((uint32_t)(S.list[i] >> 32)));
        whole = block_total<NT>(w, S.wsum);
      }
      const u64 need = by_p ? mass_needed(rs.p, whole) : ~0ull;
      u64 above = 0, kept = 0;
      uint32_t nkept = 0;
      for (int base = 0; base < nk; base += NT) {
        const int i = base + tid;
        const double t = i < nk ? log2_weight(sc, logit_of((uint32_t)(S.list[i] >> 32))) : -INFINITY;
        const u64 w = i < nk ? fixed_weight(sc, t) : 0;
        u64 sum;
        const u64 before = above + block_scan<NT>(w, S.wsum, &sum);
        const bool keep = i < nk && before < need && t >= rs.tmin;
        nkept += block_total<NT>((uint32_t)keep, S.wcnt);
        kept += block_total<NT>(keep ? w : 0ull, S.wsum);
        above += sum;
      }
      // by index: index << 32 | key, rising
      const int Q = pow2_at_least((int)nkept);
      __syncthreads();
      for (int i = tid; i < Q; i += NT) {
        const u64 a = S.list[i];
        S.list[i] = i < (int)nkept ? (u64)(uint32_t)~(uint32_t)a << 32 | a >> 32 : ~0ull;
      }
      sort_list<NT>(S.list, Q, false);
      const u64 target = target_of(u[r], kept);
      u64 run = 0;
      for (int base = 0; base < (int)nkept; base += NT) {
        const int i = base + tid;
        const u64 w = i < (int)nkept ? weight_of(sc, logit_of((uint32_t)S.list[i])) : 0;
        u64 sum;
        const u64 before = run + block_scan<NT>(w, S.wsum, &sum);
        if (before <= target && target < before + w) out[r] = (int64_t)(S.list[i] >> 32);
        run += sum;
      }
      return;
    }
    __syncthreads();
  }

  // ---- the cut: every key above `cut`, and the first `ties` (by index) that equal it (ALL: no need to count them)
  constexpr uint32_t ALL = UINT_MAX;
  uint32_t cut = 0, ties = ALL;
  u64 whole = 0, need = 0;                 // mass of what top-k keeps, and top_p of it
  bool found = false;
  if (by_p && !by_k) {
    // masses by log2 w; the bin in which the sum from above reaches what is needed is looked at closely
    for (int b = tid; b < BINS; b += NT) S.mass[b] = 0;
    if (tid == 0) S.n = 0;
    __syncthreads();
    u64 sum = 0;
    EACH_PIECE(_Pragma("unroll") for (int e = 0; e < VEC; ++e) {
      const double t = log2_weight(sc, v[e]);
      if (v[e] > -INFINITY && t > -48.0) {
        const u64 w = fixed_weight(sc, t);
        sum += w;
        atomicAdd(&S.mass[(int)(t * -16.0)], w);
      }
    })
    whole = block_total<NT>(sum, S.wsum);
    need = mass_needed(rs.p, whole);
    __syncthreads();
    u64 above = 0;
    for (int base = 0; base < BINS; base += NT) {
      const int b = base + tid;
      const u64 w = b < BINS ? S.mass[b] : 0;
      u64 all;
      const u64 before = above + block_scan<NT>(w, S.wsum, &all);
      if (before < need && need <= before + w) { S.key = (uint32_t)b; S.above = before; }
      above += all;
    }
    __syncthreads();
    const int bin = (int)S.key;
    above = S.above;
    EACH_PIECE(_Pragma("unroll") for (int e = 0; e < VEC; ++e) {
      const double t = log2_weight(sc, v[e]);
      if (v[e] > -INFINITY && t > -48.0 && (int)(t * -16.0) == bin) {
        const uint32_t at = atomicAdd(&S.n, 1u);
        if (at < CAP) S.list[at] = (u64)key_of(v[e]) << 32 | (uint32_t)~(uint32_t)(row.first(i) + e);
      }
    })
    __syncthreads();
    const int n = (int)S.n;
    if (S.n <= CAP) {
      found = true;
      const int P = pow2_at_least(n);
      for (int i = n + tid; i < P; i += NT) S.list[i] = 0;
      sort_list<NT>(S.list, P, true);
      for (int base = 0; base < n; base += NT) {
        const int i = base + tid;
        const u64 w = i < n ? weight_of(sc, logit_of((uint32_t)(S.list[i] >> 32))) : 0;
        u64 all;
        const u64 before = above + block_scan<NT>(w, S.wsum, &all);
        if (before < need && need <= before + w) {
          // the last one kept; how many equal it, kept and at all
          const uint32_t key = (uint32_t)(S.list[i] >> 32);
          int f = i, l = i;
          while (f > 0 && (uint32_t)(S.list[f - 1] >> 32) == key) --f;
          while (l + 1 < n && (uint32_t)(S.list[l + 1] >> 32) == key) ++l;
          S.key = key;
          S.n_above = l == i ? ALL : (uint32_t)(i - f + 1);
        }
        above += all;
      }
      __syncthreads();
      cut = S.key;
      ties = S.n_above;
    }
    __syncthreads();
  }
  if (by_k || (by_p && !found)) {
    // many candidates, or a bin of many: the ordered keys are searched byte by byte, the row read once for each byte;
    // stage 0: the k-th largest key; stage 1: the key at which the mass, from above, reaches what is needed
    for (int stage = by_k ? 0 : 1; stage < (by_p ? 2 : 1); ++stage) {
      if (stage == 1) need = mass_needed(rs.p, whole);
      uint32_t prefix = 0, n_above = 0;
      u64 above = 0;
      for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        for (int b = tid; b < 256; b += NT) { S.mass[b] = 0; S.cnt[b] = 0; }
        __syncthreads();
        EACH_PIECE(_Pragma("unroll") for (int e = 0; e < VEC; ++e) {
          const uint32_t key = key_of(v[e]);
          if (key == 0 || key < cut || (shift < 24 && (key >> (shift + 8)) != (prefix >> (shift + 8)))) continue;
          const uint32_t b = key >> shift & 255;
          if (stage == 0) atomicAdd(&S.cnt[b], 1u);
          else if (key > cut) atomicAdd(&S.mass[b], weight_of(sc, v[e]));
        })
        __syncthreads();
        if (tid == 0) {
          // the ties at top-k's own cut count only `ties` times
          if (stage == 1 && ties != ALL && (shift == 24 || (cut >> (shift + 8)) == (prefix >> (shift + 8))))
            S.mass[cut >> shift & 255] += ties * weight_of(sc, logit_of(cut));
          u64 w = above;
          uint32_t n = n_above;
          int b = 255;
          for (; b > 0; --b) {
            if (stage == 0 ? n + S.cnt[b] >= (u64)rs.k : w + S.mass[b] >= need) break;
            w += S.mass[b];
            n += S.cnt[b];
          }
          S.key = prefix | (uint32_t)b << shift;
          S.above = w;
          S.n_above = n;
        }
        __syncthreads();
        prefix = S.key;
        above = S.above;
        n_above = S.n_above;
      }
      if (stage == 0) {
        // (fewer than k logits that can be drawn: the search ends at key 0 and all of them are kept)
        cut = prefix;
        ties = prefix > 0 ? (uint32_t)(rs.k - n_above) : ALL;
        if (by_p) {
          u64 w = 0;
          EACH_PIECE(_Pragma("unroll") for (int e = 0; e < VEC; ++e) if (key_of(v[e]) > cut) w += weight_of(sc, v[e]);)
          whole = block_total<NT>(w, S.wsum);
          if (prefix > 0) whole += ties * weight_of(sc, logit_of(cut));
        }
      } else {
        const u64 w = weight_of(sc, logit_of(prefix));
        const u64 c = w ? (need - above + w - 1) / w : 1;
        if (prefix > cut) {
          cut = prefix;
          ties = c < ALL ? (uint32_t)c : ALL;
        } else if (c < ties) {
          ties = (uint32_t)c;
        }
      }
    }
  }

  // ---- by index: the waves' shares of the ties, then of the mass; the wave in whose share the sum passes walks it again
  __syncthreads();
  uint32_t eq = 0;                         // ties before this wave's share
  if (ties != ALL) {
    uint32_t n = 0;
    EACH_PIECE(_Pragma("unroll") for (int e = 0; e < VEC; ++e) n += key_of(v[e]) == cut;)
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o);
    if (lane == 0) S.wcnt[wave] = n;
    __syncthreads();
    for (int w = 0; w < wave; ++w) eq += S.wcnt[w];
  }
  u64 mass = 0, target = 0, run = 0;
  for (int pass = 0; pass < 2; ++pass) {
    uint32_t e0 = eq;
    for (int64_t i0 = lo; i0 < hi; i0 += 64) {
      float v[VEC];
      const int64_t i = i0 + lane;
      if (i < hi) row.load(i, v);
      else
        for (int e = 0; e < VEC; ++e) v[e] = -INFINITY;
      uint32_t tie = 0;                    // ties before this lane's piece
      if (ties != ALL) {
        uint32_t n = 0;
#pragma unroll
        for (int e = 0; e < VEC; ++e) n += key_of(v[e]) == cut;
        uint32_t inc = n;
        for (int o = 1; o < 64; o <<= 1) {
          const uint32_t up = __shfl_up(inc, o);
          if (lane >= o) inc += up;
        }
        tie = e0 + inc - n;
        e0 += __shfl(inc, 63);
      }
      u64 w[VEC], sum = 0;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const uint32_t key = key_of(v[e]);
        w[e] = 0;
        if (key == 0 || key < cut || (key == cut && ties != ALL && tie++ >= ties)) continue;
        const double t = log2_weight(sc, v[e]);
        if (t >= rs.tmin) w[e] = fixed_weight(sc, t);
        sum += w[e];
      }
      if (pass == 0) {
        mass += sum;
        continue;
      }
      u64 inc = sum;
      for (int o = 1; o < 64; o <<= 1) {
        const u64 up = __shfl_up(inc, o);
        if (lane >= o) inc += up;
      }
      u64 before = run + inc - sum;
      if (before <= target && target < before + sum) {
        int at = 0;
        for (; at < VEC - 1 && before + w[at] <= target; ++at) before += w[at];
        out[r] = row.first(i) + at;
      }
      run += __shfl(inc, 63);
      if (run > target) return;
    }
    if (pass == 1) return;
    for (int o = 32; o > 0; o >>= 1) mass += __shfl_xor(mass, o);
    if (lane == 0) S.wsum[wave] = mass;
    __syncthreads();
    u64 all = 0;
    for (int w = 0; w < NW; ++w) {
      if (w < wave) run += S.wsum[w];
      all += S.wsum[w];
    }
    target = target_of(u[r], all);
    if (!(run <= target && target < run + mass)) return;
  }
#undef EACH_PIECE
}

template <typename T>
int launch_sample(int64_t rows, int64_t V, const void* logits, int64_t ld, const Settings& st, int F, const float* u, int64_t* out, hipStream_t s) {
  const T* x = (const T*)logits;
#define GROUP_(G, E)                                                                                                                             \
  hipLaunchKernelGGL((sample_group_kernel<T, G, E>), dim3((unsigned)cdiv64(rows, 256 / G)), dim3(256), 0, s, rows, (int)V, (int)cdiv64(V, G), x, ld, \
                     st, F, u, out)
  if (V <= 16) {
    GROUP_(4, 4);
  } else if (V <= 64) {
    GROUP_(4, 16);
  } else if (V <= 256) {
    GROUP_(16, 16);
  } else if (V <= 1024) {
    GROUP_(64, 16);
  } else if (V <= 2048) {
    GROUP_(64, 32);
#undef GROUP_
  } else if (V <= 16384) {
    hipLaunchKernelGGL((sample_row_kernel<T, 256>), dim3((unsigned)rows), dim3(256), 0, s, rows, V, x, ld, st, F, u, out);
  } else {
    hipLaunchKernelGGL((sample_row_kernel<T, 1024>), dim3((unsigned)rows), dim3(1024), 0, s, rows, V, x, ld, st, F, u, out);
  }
  TAD_LAUNCH_CHECK();
  return TAD_OK;
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
  return dtype == TAD_F32 ? launch_sample<float>(rows, V, logits, ld, st, F, u, out, s) : launch_sample<bf16_t>(rows, V, logits, ld, st, F, u, out, s);
}
