// Draws a token from each row of logits: temperature, top-k, top-p and min-p, from given uniform numbers (gfx950).
//
//   w_j = exp((l_j - max) / T).  Kept: the top_k largest; of those the shortest prefix, largest first, that holds top_p of
//   their mass; of those the ones with w_j >= min_p.  The answer is the lowest index at which the running sum of the kept
//   w, by index, exceeds u times their sum.  Ties go to the lowest index.
//
// The answer is an index that a sum decides, so the sums are exact: every w is rounded once to a whole multiple of 2^-F (F =
// 44 for rows of up to 512 logits and of 2049 to 2^17, else a few less) and added as a whole number, in float64 where all
// of a sum fits its 53 bits and in 64-bit integers beyond.  The order of additions then changes nothing.  What is left are the
// weights' own roundings, at most 2^-(F+1) of the largest each: the answer is the real numbers' unless u times the sum lies
// within V 2^-(F+1) of a border (2^-36 at 512 logits, 2^-32 at 2048, 2^-28 at 131072; about sqrt(V) / V of that where the
// roundings are of either sign; all of it where most logits are equal), next to which u itself is a multiple of 2^-24 or so.  A
// weight below half a unit is 0: a filter that counts keeps it, and it is never drawn.  Float64 fused multiply-adds issue at
// the rate of float32 ones here, so such a weight costs about 20 instructions.
//
// Every filter keeps a prefix of the row in falling order (ties by index), so their conjunction is the shortest of the
// prefixes: one cut (a key, and how many of those that equal it).
#include <limits.h>
#include <math.h>

#include "lanes.h"
#include "row_pieces.h"

namespace {

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
// log2 of w; NaN logits, and -inf whatever T is, count as 2^-100
__device__ __forceinline__ double log2_weight(const Scale& s, float l) { return fmax(((double)l - (double)s.m) * s.c, -100.0); }
// 2^t in units of 2^-F, rounded to a whole number (0 from about t = -F - 1 down): 2^n 2^f, n the whole number next to t, by an
// addition that leaves n + F in the low bits, and 2^f = 1 + f g(f), |f| <= 1/2, g the polynomial that meets (2^f - 1) / f at the
// ten Chebyshev points there: off by less than 2^-50
__device__ __forceinline__ double fixed_weight(const Scale& s, double t) {
  const double magic = 6755399441055744.0 + (double)s.F, r = t + magic, f = t - (r - magic);
  double p = 7.070977866508139e-09;
  p = __builtin_fma(p, f, 1.0205905413765595e-07);
  p = __builtin_fma(p, f, 1.3215451633221434e-06);
  p = __builtin_fma(p, f, 1.5252672924850737e-05);
  p = __builtin_fma(p, f, 0.00015403530424776529);
  p = __builtin_fma(p, f, 0.0013333558200794592);
  p = __builtin_fma(p, f, 0.009618129107618665);
  p = __builtin_fma(p, f, 0.05550410866465167);
  p = __builtin_fma(p, f, 0.24022650695910075);
  p = __builtin_fma(p, f, 0.6931471805599462);
  p = __builtin_fma(p, f, 1.0);
  const u64 b = __builtin_bit_cast(u64, p);
  const uint32_t hi = (uint32_t)(b >> 32) + ((uint32_t)__builtin_bit_cast(u64, r) << 20);
  return rint(__builtin_bit_cast(double, (u64)hi << 32 | (uint32_t)b));
}
// a whole number below 2^52 as an integer
__device__ __forceinline__ u64 whole_number(double w) { return __builtin_bit_cast(u64, w + 4503599627370496.0) & 0xfffffffffffffull; }
__device__ __forceinline__ double weight_of(const Scale& s, float l) { return fixed_weight(s, log2_weight(s, l)); }
// sum + w where `in`: one move and one multiply-add
__device__ __forceinline__ double add_if(bool in, double w, double sum) { return __builtin_fma(in ? 1.0 : 0.0, w, sum); }

struct Settings {
  double T, p, minp;
  int64_t k;
  const float *Tr, *pr, *mr;
  const int32_t* kr;
};
struct RowSettings {
  double T, c, p, tmin;    // c: log2(e) / T, finite (0 times it is 0); tmin: log2 of min_p
  int64_t k;
  __device__ RowSettings(const Settings& st, int64_t r) {
    T = st.Tr ? (double)st.Tr[r] : st.T;
    c = fmin(1.4426950408889634074 / T, 1e300);
    k = st.kr ? (int64_t)st.kr[r] : st.k;
    p = st.pr ? (double)st.pr[r] : st.p;
    const double m = st.mr ? (double)st.mr[r] : st.minp;
    tmin = m > 0.0 ? log2(m < 1.0 ? m : 1.0) : -INFINITY;
  }
};
// all in units of 2^-F: the mass that a prefix has to reach; how many weights `one` reach what is left of it; the sum that
// has to be exceeded
__device__ __forceinline__ u64 mass_needed(double p, u64 whole) {
  const double d = ceil((p > 0.0 ? p : 0.0) * (double)whole);
  const u64 n = d >= 1.0 ? (u64)d : 1;
  return n < whole ? n : whole;
}
__device__ __forceinline__ double mass_needed(double p, double whole) { return fmin(fmax(ceil(p * whole), 1.0), whole); }
__device__ __forceinline__ u64 ties_needed(u64 left, u64 one) { return one ? (left + one - 1) / one : 1; }
__device__ __forceinline__ u64 ties_needed(double left, double one) { return ties_needed((u64)left, (u64)one); }
__device__ __forceinline__ u64 target_of(float u, u64 all) {
  const u64 t = u > 0.f ? (u >= 1.f ? all : (u64)((double)u * (double)all)) : 0;
  return t < all ? t : all - 1;
}
__device__ __forceinline__ double target_of(float u, double all) { return fmin(floor((u > 0.f ? (double)u : 0.0) * all), all - 1.0); }

constexpr float LARGEST = 3.4028234663852886e38f;      // what +inf counts as

// ---------------------------------------------------------------- rows of up to 2048 logits: G lanes of a wave per row
// The row and its weights stay in registers, a contiguous piece of E logits or fewer a lane; what the lanes share goes
// across with DPP moves.  A cut is searched for by bisection: on the logits' values (their weights are exponential in them,
// so a few steps separate neighbours), then, where a value does not lie between its neighbours any more, on the ordered
// keys, so that it ends after at most 48 steps whatever the logits are (9 to 11 where they are spread like a normal's).  98304 x
// 48 float32, top-p: 24 us, bound by instructions (without a filter 11); a thread per row walking LDS: 167.
template <typename T, int G, int E>
__global__ __launch_bounds__(256) void sample_group_kernel(int64_t rows, int V, int per, const T* __restrict__ logits, int64_t ld, Settings st, int F,
                                                           const float* __restrict__ u, int64_t* __restrict__ out) {
  const int lane = threadIdx.x & (G - 1), j0 = lane * per;
  const int64_t r = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
  if (r >= rows) return;
  const T* x = logits + r * ld;
#define EACH(...)                        \
  _Pragma("unroll") for (int e = 0; e < E; ++e) { \
    __VA_ARGS__                          \
  }
  float v[E];
  EACH(v[e] = e < per && j0 + e < V ? (float)x[j0 + e] : -INFINITY;)
  const RowSettings rs(st, r);
  float m = -INFINITY;
  EACH(v[e] = v[e] > -INFINITY ? fminf(v[e], LARGEST) : -INFINITY; m = fmaxf(m, v[e]);)
  m = across<G, Max>(m);
  if (m == -INFINITY || !(rs.T > 0.0)) {
    int at = V;
    EACH(at = v[e] == m && e < at - j0 ? j0 + e : at;)
    at = across<G, Min>(at);
    if (lane == 0) out[r] = m == -INFINITY ? -1 : at;
    return;
  }
  const Scale sc = {m, rs.c, F};
  const bool by_k = rs.k > 0 && rs.k < V, by_p = rs.p < 1.0;
  double w[E];
  uint32_t low = 0;                           // the ones below min_p
  EACH(const double t = log2_weight(sc, v[e]); w[e] = fixed_weight(sc, t); low |= t >= rs.tmin ? 0u : 1u << e;)

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
    double whole = 0;
    int n = 0;
    uint32_t lo = UINT_MAX, hi = key_of(m);
    EACH(whole += w[e]; n += w[e] != 0; const uint32_t k = key_of(v[e]); lo = w[e] != 0 && k < lo ? k : lo;)
    whole = across<G, Add>(whole);
    n = across<G, Add>(n);
    lo = across<G, Min>(lo);
    const double need = mass_needed(rs.p, whole);
    int above = 0;                            // n reach `lo`, `above` lie above `hi`
    for (int step = 0; lo < hi && n - above > 1; ++step) {
      const uint32_t b = between(lo, hi, step);
      const float f = logit_of(b);
      double mass = 0;
      int k = 0;
      EACH(const bool in = v[e] >= f; mass = add_if(in, w[e], mass); k += in;)
      mass = across<G, Add>(mass);
      k = across<G, Add>(k);
      if (mass >= need) { lo = b; n = k; } else { hi = b - 1; above = k; }
    }
    const float cut = logit_of(lo);
    uint32_t eq = (uint32_t)(n - above), ties = eq;
    if (eq > 1) {                             // (lo = hi: equals)
      double mass = 0, one = 0;
      EACH(mass = add_if(v[e] > cut, w[e], mass); one = v[e] == cut ? w[e] : one;)
      mass = across<G, Add>(mass);
      one = across<G, Max>(one);
      ties = (uint32_t)ties_needed(need - mass, one);
    }
    drop(cut, ties, eq);
  }
  double mine = 0;
  EACH(w[e] = low >> e & 1 ? 0.0 : w[e]; mine += w[e];)
  const double all = across<G, Add>(mine), target = target_of(u[r], all);
  double run = lanes_before<G>(mine, lane);
  if (run <= target && target < run + mine) {
    int at = 0;
    EACH(run += w[e]; at += run <= target;)
    out[r] = j0 + at;
  }
#undef EACH
}

// ---------------------------------------------------------------- longer rows: a workgroup per row
constexpr int BINS = 512;                          // of log2 w, down to 2^-16

struct Candidate {
  u64 k;             // key << 32 | ~index: falling logits, equal ones by index
  double w;
};
template <int NT>
struct RowState {
  // CAP: candidates of a list.  PAIRS: those that are compared each with each, more are sorted first (1 x 32000 with top-k 200: 18 us,
  // up to 512 pairs 22; 1 x 131072 float32 with 256, 1024 threads: 40 up to 256 pairs, 31 up to 512).  FEW: top-k that such a
  // list is for; what a list for more takes, the histogram takes too (512 x 65536, 224: 93 us against 133; 1 x 4000: 17 against 16)
  static constexpr int NW = NT / 64, CAP = 1024, PAIRS = NT < 1024 ? 256 : 512, FEW = NT * 7 / 16;
  u64 list[CAP];
  union {
    u64 mass[NW][BINS];
    Candidate pair[PAIRS];
  };
  uint32_t cnt[BINS];
  uint32_t piece[NW][64];
  u64 reach[2][NW];
  u64 wsum[NW];
  uint32_t wcnt[NW];
  float wmax[NW], wmin[NW];
  uint32_t n, n_above, key, ties, at;
  u64 above, upto;
  double total;
};

template <int NT, typename I>
__device__ __forceinline__ I block_total(I v, I* s) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
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

// Sorts list[0 .. n), entries that all differ: falling, or rising.  Up to a thread's worth (and 512) every entry's place is
// counted, all pairs compared; more (up to the next power of two, which the list has to hold) are sorted by exchanges, a barrier
// for each step.  1 x 4000 with top-k 300: 16 us (exchanges alone 22, up to 128 of them by one wave 20); 4096 x 8000: 168 (191, 185).
template <int NT>
__device__ void sort_list(u64* list, int n, bool falling) {
  constexpr int RANKED = NT < 512 ? NT : 512;
  const u64 flip = falling ? 0 : ~0ull;
  const int tid = threadIdx.x;
  __syncthreads();
  if (n <= RANKED) {
    const u64 mine = tid < n ? list[tid] ^ flip : 0;
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += (list[j] ^ flip) > mine;
    __syncthreads();
    if (tid < n) list[rank] = mine ^ flip;
    __syncthreads();
    return;
  }
  int P = RANKED;
  while (P < n) P <<= 1;
  for (int i = n + tid; i < P; i += NT) list[i] = flip;
  __syncthreads();
  for (int size = 2; size <= P; size <<= 1)
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      for (int i = tid; i < P / 2; i += NT) {
        const int lo = 2 * i - (i & (stride - 1)), hi = lo + stride;
        const u64 a = list[lo], b = list[hi];
        if ((a < b) == (((lo & size) == 0) == falling) && a != b) { list[lo] = b; list[hi] = a; }
      }
      __syncthreads();
    }
}

// A row with a small top-k takes two looks: the largest of every thread and piece, then the pieces that can hold a candidate;
// top-p alone adds the exact sum of the row; all else the masses of the row by bins.  256 x 131072 bf16 with settings per row
// (top-k about 64): 27 us (its argmax alone: 15), 1 x 32000: 11 us, of which 2 are the load and the rest steps that wait for
// each other.
template <typename T, int NT>
__global__ __launch_bounds__(NT) void sample_row_kernel(int64_t rows, int64_t V, const T* __restrict__ logits, int64_t ld, Settings st, int F,
                                                        const float* __restrict__ u, int64_t* __restrict__ out) {
  typedef RowState<NT> State;
  constexpr int VEC = RowPieces<T>::VEC, NW = State::NW, CAP = State::CAP, PAIRS = State::PAIRS, FEW = State::FEW;
  __shared__ State S;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t r = blockIdx.x;
  const RowPieces<T> row(logits + r * ld, V);
  const RowSettings rs(st, r);
  const float uu = u[r];
  // a wave's own contiguous share of the pieces
  const int64_t seg = (row.np + NW - 1) / NW, lo = wave * seg < row.np ? wave * seg : row.np, hi = lo + seg < row.np ? lo + seg : row.np;
  bool infinite = false;                    // +inf among the logits

  // every piece of the share, and every element of the piece (v[e])
#define EACH_PIECE(...) _Pragma("unroll 2") ONE_BY_ONE(__VA_ARGS__)
#define ONE_BY_ONE(...)                                                                  \
  for (int64_t i = lo + lane; i < hi; i += 64) {                                         \
    float v[VEC];                                                                        \
    row.load(i, v);                                                                      \
    if (infinite) {                                                                      \
      _Pragma("unroll") for (int e = 0; e < VEC; ++e) v[e] = v[e] == INFINITY ? LARGEST : v[e]; \
    }                                                                                    \
    __VA_ARGS__                                                                          \
  }
#define EACH(...) _Pragma("unroll") for (int e = 0; e < VEC; ++e) { __VA_ARGS__ }

  // The first look: the thread's largest logit, the row's, and the smallest of the threads'; every thread sees every NT-th piece,
  // so that logits in falling order are spread too.  With top-p alone the sum of the weights as well, roughly (each thread's
  // relative to its own largest).
  const bool guess = rs.T > 0.0 && !(rs.k > 0 && rs.k < V) && rs.p < 1.0;
  const float rough = (float)rs.c;
  float tm = -INFINITY, tz = 0.f;
  const auto look = [&](const float (&v)[VEC]) {
    float b = tm;
    EACH(b = fmaxf(b, v[e]);)
    if (guess) {
      const float from = fmaxf(b, -LARGEST);
      tz *= __builtin_amdgcn_exp2f((tm - from) * rough);
      EACH(tz += __builtin_amdgcn_exp2f((v[e] - from) * rough);)
    }
    tm = b;
  };
  // (the largest of each of the thread's first H pieces stays in a register: which pieces a later look at the row needs)
  constexpr int H = 16;
  float most[H];
#pragma unroll
  for (int h = 0; h < H; ++h) {
    const int64_t i = tid + NT * h;
    most[h] = -INFINITY;
    if (i < row.np) {
      float v[VEC];
      row.load(i, v);
      look(v);
      EACH(most[h] = fmaxf(most[h], v[e]);)
    }
  }
  for (int64_t i = tid + NT * H; i < row.np; i += NT) {
    float v[VEC];
    row.load(i, v);
    look(v);
  }
  // The pieces that the wave has seen with an element that reaches f: S.piece[wave] has them in order, up to 64; returns how many
  // there are.
  const auto pieces_from = [&](float f) {
    int n = 0;
    const auto take = [&](bool in, int64_t i) {
      const u64 b = __ballot(in);
      const int at = n + __popcll(b & ((1ull << lane) - 1));
      if (in && at < 64) S.piece[wave][at] = (uint32_t)i;
      n += __popcll(b);
    };
#pragma unroll
    for (int h = 0; h < H; ++h) {
      if (NT * h >= row.np) break;
      take(most[h] >= f, tid + NT * h);
    }
    for (int64_t i0 = NT * H; i0 < row.np; i0 += NT) {
      float v[VEC], b = -INFINITY;
      if (i0 + tid < row.np) {
        row.load(i0 + tid, v);
        EACH(b = fmaxf(b, v[e]);)
      }
      take(b >= f, i0 + tid);
    }
    lds_in_order();
    return n;
  };
  float m = across<64, Max>(tm), least = across<64, Min>(tm > -INFINITY ? tm : INFINITY);
  if (lane == 0) {
    S.wmax[wave] = m;
    S.wmin[wave] = least;
  }
  if (tid == 0) S.n = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    m = fmaxf(m, S.wmax[w]);
    least = fminf(least, S.wmin[w]);
  }
  if (m == -INFINITY) {
    if (tid == 0) out[r] = -1;
    return;
  }
  if (!(rs.T > 0.0)) {
    u64 at = ~0ull;                         // the lowest index of the largest (pieces come in order: the first that has it)
    const float top = fminf(m, LARGEST);
    if (pieces_from(top) > 0) {
      const int64_t i = S.piece[wave][0];
      float v[VEC];
      row.load(i, v);
      EACH(if (v[VEC - 1 - e] >= top) at = (u64)(row.first(i) + VEC - 1 - e);)
    }
    at = across<64, Min>(at);
    if (lane == 0) S.wsum[wave] = at;
    __syncthreads();
    for (int w = 0; w < NW; ++w) at = S.wsum[w] < at ? S.wsum[w] : at;
    if (tid == 0) out[r] = (int64_t)at;
    return;
  }
  infinite = m == INFINITY;
  m = fminf(m, LARGEST);
  tm = fminf(tm, LARGEST);
  const Scale sc = {m, rs.c, F};
  const bool by_k = rs.k > 0 && rs.k < V, by_p = rs.p < 1.0;
  // halves the distance between two keys: by value as long as that lies between them
  const auto between = [](uint32_t a, uint32_t b, int step) {
    const uint32_t k = key_of(0.5f * logit_of(a) + 0.5f * logit_of(b));
    return step < 16 && k > a && k <= b ? k : a + (b - a + 1) / 2;
  };

  // ---- few candidates: all that top-k can keep fits the list; or, with top-p alone, a guess: that the largest GUESS logits
  // hold top_p of the mass, as they do where a model is sure of its answers
  constexpr int GUESS = 160;
  if ((by_k && rs.k <= FEW) || guess) {
    const int64_t kk = by_k ? rs.k : GUESS;
    // where kk threads' largest reach `floor`, at least kk logits do; not many more than kk are wanted
    // (the numbers of three values at a time, one barrier a step)
    float floor = -LARGEST;
    int step = 0;
    const auto reach = [&](float f1, float f2, float f3) {        // 16 bits each
      const u64 mine = (u64)__popcll(__ballot(tm >= f1)) | (u64)__popcll(__ballot(tm >= f2)) << 16 | (u64)__popcll(__ballot(tm >= f3)) << 32;
      if (lane == 0) S.reach[step & 1][wave] = mine;
      __syncthreads();
      u64 all = 0;
#pragma unroll
      for (int w = 0; w < NW; ++w) all += S.reach[step & 1][w];
      ++step;
      return all;
    };
    if ((int64_t)(reach(least, least, least) & 0xffff) >= kk) {
      uint32_t a = key_of(least), b = key_of(m);
      while (a < b && step < 16) {
        const uint32_t k2 = between(a, b, step), k1 = between(a, k2, step), k3 = between(k2, b, step);
        const u64 all = reach(logit_of(k1), logit_of(k2), logit_of(k3));
        const int n1 = (int)(all & 0xffff), n2 = (int)(all >> 16 & 0xffff), n3 = (int)(all >> 32);
        int n = 0;
        if (n3 >= kk) { a = k3; n = n3; }
        else if (n2 >= kk) { a = k2; b = k3 - 1; n = n2; }
        else if (n1 >= kk) { a = k1; b = k2 - 1; n = n1; }
        else b = k1 - 1;
        if (n && n <= kk + kk / 4 + 8) break;
      }
      floor = logit_of(a);
    }
    // every lane takes one of the wave's pieces that reach it
    {
      const int np = pieces_from(floor);
      const bool on = lane < np && np <= 64;
      const int64_t i = on ? S.piece[wave][lane] : 0;
      float v[VEC];
      int n = 0;
      if (on) {
        row.load(i, v);
        EACH(v[e] = infinite && v[e] == INFINITY ? LARGEST : v[e]; n += v[e] >= floor;)
      }
      int at = lanes_before<64>(n, lane);
      int base = 0;
      if (lane == 63) base = (int)atomicAdd(&S.n, (uint32_t)(np <= 64 ? at + n : CAP + 1));
      at += __builtin_amdgcn_readlane(base, 63);
      if (on) EACH(if (v[e] >= floor) {
        if (at < CAP) S.list[at] = (u64)key_of(v[e]) << 32 | (uint32_t)~(uint32_t)(row.first(i) + e);
        ++at;
      })
    }
    __syncthreads();
    int n = S.n < CAP + 1 ? (int)S.n : CAP + 1;
    const int nk = kk < n && !guess ? (int)kk : n;
    u64 whole_row = 0;
    if (guess) {
      // (weighed roughly first: only a guess that holds is worth the exact sum of the row; a NaN or an infinity: it does not)
      bool good = n <= PAIRS;
      if (good) {
        const float some = tid < n ? __builtin_amdgcn_exp2f((logit_of((uint32_t)(S.list[tid] >> 32)) - m) * rough) : 0.f;
        const float all = block_total<NT>(tz * __builtin_amdgcn_exp2f((tm - m) * rough), S.wmax);
        good = block_total<NT>(some, S.wmin) > 1.001f * (float)rs.p * all;
      }
      if (good) {
        double w = 0;
        ONE_BY_ONE(EACH(w += weight_of(sc, v[e]);))
        whole_row = block_total<NT>((u64)w, S.wsum);
      } else {
        n = CAP + 1;
      }
    }
    if (n <= PAIRS) {
      // each with each: its place and the mass above it in falling order, then the kept mass below it by index
      const bool on = tid < n;
      const u64 mine = on ? S.list[tid] : 0;
      const double t = on ? log2_weight(sc, logit_of((uint32_t)(mine >> 32))) : -100.0, w = fixed_weight(sc, t);
      if (on) S.pair[tid] = {mine, w};
      __syncthreads();
      double above = 0;
      int rank = 0;
      if (on) {
#pragma unroll 8
        for (int j = 0; j < n; ++j) {
          const Candidate c = S.pair[j];
          const bool in = c.k > mine;
          rank += in;
          above = add_if(in, c.w, above);
        }
        if (rank == nk - 1) S.total = above + w;
      }
      __syncthreads();
      const double need = guess ? (double)mass_needed(rs.p, whole_row) : mass_needed(rs.p, S.total);
      if (need <= S.total) {                   // (always, but for a guess)
        const bool keep = on && rank < nk && (!by_p || above < need) && t >= rs.tmin;
        if (on) S.pair[tid].w = keep ? w : 0.0;
        __syncthreads();
        if (!keep) return;
        double before = 0, all = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) {
          const Candidate c = S.pair[j];
          before = add_if((uint32_t)c.k > (uint32_t)mine, c.w, before);
          all += c.w;
        }
        const double target = target_of(uu, all);
        if (before <= target && target < before + w) out[r] = (int64_t)(uint32_t)~(uint32_t)mine;
        return;
      }
      n = CAP + 1;
    }
    if (n <= CAP) {
      // sorted: by logit for the cut, the kept ones by index for the answer
      sort_list<NT>(S.list, n, true);
      u64 whole = 0;
      if (by_p) {
        u64 w = 0;
        for (int i = tid; i < nk; i += NT) w += whole_number(weight_of(sc, logit_of((uint32_t)(S.list[i] >> 32))));
        whole = block_total<NT>(w, S.wsum);
      }
      const u64 need = by_p ? mass_needed(rs.p, whole) : ~0ull;
      u64 above = 0, kept = 0;
      uint32_t nkept = 0;
      for (int base = 0; base < nk; base += NT) {
        const int i = base + tid;
        const double t = i < nk ? log2_weight(sc, logit_of((uint32_t)(S.list[i] >> 32))) : -100.0;
        const u64 w = i < nk ? whole_number(fixed_weight(sc, t)) : 0;
        u64 sum;
        const u64 before = above + block_scan<NT>(w, S.wsum, &sum);
        const bool keep = i < nk && before < need && t >= rs.tmin;
        nkept += block_total<NT>((uint32_t)keep, S.wcnt);
        kept += block_total<NT>(keep ? w : 0ull, S.wsum);
        above += sum;
      }
      // index << 32 | key, rising
      __syncthreads();
      for (int i = tid; i < (int)nkept; i += NT) {
        const u64 a = S.list[i];
        S.list[i] = (u64)(uint32_t)~(uint32_t)a << 32 | a >> 32;
      }
      sort_list<NT>(S.list, (int)nkept, false);
      const u64 target = target_of(uu, kept);
      u64 run = 0;
      for (int base = 0; base < (int)nkept; base += NT) {
        const int i = base + tid;
        const u64 w = i < (int)nkept ? whole_number(weight_of(sc, logit_of((uint32_t)S.list[i]))) : 0;
        u64 sum;
        const u64 before = run + block_scan<NT>(w, S.wsum, &sum);
        if (before <= target && target < before + w) out[r] = (int64_t)(S.list[i] >> 32);
        run += sum;
      }
      return;
    }
    __syncthreads();
  }

  // ---- the cut: every logit above `cut`, and the first `ties` (by index) that equal it (ALL: no need to count them)
  constexpr uint32_t ALL = UINT_MAX;
  float cut = -LARGEST;
  uint32_t ties = ALL;
  bool shares = false;                       // S.wsum holds the kept mass of every wave's share
  if (by_k || by_p) {
    // masses, and for top-k numbers, by log2 w: the bin in which what is wanted is reached is gathered, sorted and searched.
    // (Top-k may reach further down: to the smallest of the threads' largest; never to 2^-100, where what is not drawn stands)
    const double depth = by_k ? fmin(fmax(-log2_weight(sc, least), 16.0), 90.0) : 16.0, per_octave = BINS / depth;
    const auto bin_of = [&](double t) { return (int)(t * -per_octave); };
    for (int b = tid; b < NW * BINS; b += NT) S.mass[0][b] = 0;
    for (int b = tid; b < BINS; b += NT) S.cnt[b] = 0;
    __syncthreads();
    double sum = 0;
    uint32_t number = 0;
    ONE_BY_ONE(EACH(const double t = log2_weight(sc, v[e]), w = fixed_weight(sc, t); sum += w; number += v[e] > -INFINITY;
                    const int bin = bin_of(t);
                    if (bin < BINS) {
                      atomicAdd(&S.mass[wave][bin], whole_number(w));
                      if (by_k) atomicAdd(&S.cnt[bin], 1u);
                    }))
    u64 whole = block_total<NT>((u64)sum, S.wsum);
    const uint32_t drawable = block_total<NT>(number, S.wcnt);
    // the bin where the running number (or mass) reaches what is wanted, with what lies above it; BINS: none does
    const auto find = [&](bool by_number, u64 want) {
      u64 above = 0;
      uint32_t n_above = 0;
      __syncthreads();
      if (tid == 0) S.key = BINS;
      for (int base = 0; base < BINS; base += NT) {
        const int b = base + tid;
        u64 w = 0, all;
        uint32_t n = 0, n_all;
        if (b < BINS) {
          for (int i = 0; i < NW; ++i) w += S.mass[i][b];
          n = S.cnt[b];
        }
        const u64 before = above + block_scan<NT>(w, S.wsum, &all);
        const uint32_t n_before = n_above + block_scan<NT>(n, S.wcnt, &n_all);
        if (by_number ? n_before < want && want <= n_before + n : before < want && want <= before + w) {
          S.key = (uint32_t)b;
          S.above = before;
          S.n_above = n_before;
        }
        above += all;
        n_above += n_all;
      }
      __syncthreads();
      return (int)S.key;
    };
    // the logits of a bin, falling; false if they are too many
    const auto gather = [&](int bin) {
      if (tid == 0) S.n = 0;
      __syncthreads();
      EACH_PIECE(EACH(if (bin_of(log2_weight(sc, v[e])) == bin) {
        const uint32_t at = atomicAdd(&S.n, 1u);
        if (at < CAP) S.list[at] = (u64)key_of(v[e]) << 32 | (uint32_t)~(uint32_t)(row.first(i) + e);
      }))
      __syncthreads();
      if (S.n > CAP) return false;
      sort_list<NT>(S.list, (int)S.n, true);
      return true;
    };
    // the cut at the list's entry at which the number (or the mass, S.above of it above the list) reaches `want`
    const auto cut_in_list = [&](bool by_number, u64 want) {
      const int n = (int)S.n;
      u64 above = S.above;
      const uint32_t n_above = S.n_above;
      for (int base = 0; base < n; base += NT) {
        const int i = base + tid;
        const u64 w = i < n ? whole_number(weight_of(sc, logit_of((uint32_t)(S.list[i] >> 32)))) : 0;
        u64 all;
        const u64 before = above + block_scan<NT>(w, S.wsum, &all);
        if (i < n && (by_number ? n_above + i + 1 == want : before < want && want <= before + w)) {
          const uint32_t key = (uint32_t)(S.list[i] >> 32);
          int f = i;
          while (f > 0 && (uint32_t)(S.list[f - 1] >> 32) == key) --f;
          S.key = key;
          S.ties = i + 1 < n && (uint32_t)(S.list[i + 1] >> 32) == key ? (uint32_t)(i - f + 1) : ALL;
          S.at = (uint32_t)i;
          S.upto = before + w;
        }
        above += all;
      }
      __syncthreads();
      cut = logit_of(S.key);
      ties = S.ties;
    };
    int bin = BINS;
    bool found = true;
    if (by_k && drawable > rs.k) {
      bin = find(true, (u64)rs.k);
      found = bin < BINS && gather(bin);
      if (found) {
        cut_in_list(true, (u64)rs.k);
        whole = S.upto;
      }
    }
    if (by_p && found) {
      const u64 need = mass_needed(rs.p, whole);
      const int kbin = bin;
      bin = find(false, need);          // (top-k's own bin again: the list is there)
      found = bin < BINS && (bin == kbin || gather(bin));
      if (found) cut_in_list(false, need);
    }
    if (found && bin < BINS && rs.tmin == -INFINITY) {
      // the shares' kept masses: whole bins above the cut's, and the list up to it
      shares = true;
      u64 w = 0;
      for (int b = lane; b < bin; b += 64) w += S.mass[wave][b];
      w = across<64, Add>(w);
      __syncthreads();
      if (lane == 0) S.wsum[wave] = w;
      __syncthreads();
      for (int i = tid; i <= (int)S.at; i += NT) {
        const int64_t piece = (int64_t)(uint32_t)~(uint32_t)S.list[i] / VEC;
        atomicAdd(&S.wsum[piece / seg], whole_number(weight_of(sc, logit_of((uint32_t)(S.list[i] >> 32)))));
      }
    }
    if (!found) {
      // a bin of many, or none: bisection over the row
      cut = -LARGEST;
      ties = ALL;
      const auto above_of = [](float f) { return logit_of(key_of(f) + 1); };      // the next larger value
      const auto count = [&](float f) {
        uint32_t n = 0;
        EACH_PIECE(EACH(n += v[e] >= f;))
        return block_total<NT>(n, S.wcnt);
      };
      const auto mass_from = [&](float f) {
        double w = 0;
        ONE_BY_ONE(float b = -INFINITY; EACH(b = fmaxf(b, v[e]);) if (__any(b >= f)) EACH(w = add_if(v[e] >= f, weight_of(sc, v[e]), w);))
        return block_total<NT>((u64)w, S.wsum);
      };
      if (by_k && drawable > rs.k) {
        const uint32_t want = (uint32_t)rs.k;
        uint32_t a = key_of(-LARGEST), b = key_of(m), c = drawable;
        for (int step = 0; a < b && c != want; ++step) {
          const uint32_t k = between(a, b, step), got = count(logit_of(k));
          if (got >= want) { a = k; c = got; } else b = k - 1;
        }
        cut = logit_of(a);
        if (c != want) ties = want - (cut < m ? count(above_of(cut)) : 0);
      }
      if (by_p) {
        // what reaches top-k's cut has the mass of its ties there
        const u64 tied = ties != ALL ? ties * whole_number(weight_of(sc, cut)) : 0;
        const auto mass = [&](float f) { return ties == ALL || f > cut ? mass_from(f) : (cut < m ? mass_from(above_of(cut)) : 0) + tied; };
        const u64 need = mass_needed(rs.p, mass(cut));
        uint32_t a = key_of(cut), b = key_of(m);
        for (int step = 0; a < b; ++step) {
          const uint32_t k = between(a, b, step);
          if (mass(logit_of(k)) >= need) a = k; else b = k - 1;
        }
        const float f = logit_of(a);
        const u64 c = ties_needed(need - (f < m ? mass_from(above_of(f)) : 0), whole_number(weight_of(sc, f)));
        if (f > cut || ties == ALL || c < ties) ties = c < ALL ? (uint32_t)c : ALL;
        cut = f;
      }
    }
  }

  // ---- by index: the waves' masses, then the share in which the sum passes divided among the waves element by element, until
  // the lanes of a wave hold it
  const int64_t width = seg * VEC;           // elements of a wave's share
  int64_t A = 0, B = V;
  u64 base = 0, target = 0;
  uint32_t tie = 0;                          // ties before A
  const auto clean = [&](float l) { return infinite && l == INFINITY ? LARGEST : l; };
  // the share in which the sum passes (S.wsum: masses, S.wcnt: ties)
  const auto choose = [&](int64_t share) {
    int w = 0;
    for (; w < NW - 1 && base + S.wsum[w] <= target; ++w) {
      base += S.wsum[w];
      if (ties != ALL) tie += S.wcnt[w];
    }
    A += w * share;
    B = A + share < B ? A + share : B;
  };
  uint32_t eq = 0;
  __syncthreads();
  if (ties != ALL) {
    ONE_BY_ONE(EACH(eq += v[e] == cut;))
    eq = across<64, Add>(eq);
    if (lane == 0) S.wcnt[wave] = eq;
    __syncthreads();
    eq = 0;
    for (int w = 0; w < wave; ++w) eq += S.wcnt[w];
  }
  if (!shares) {
    double mass = 0;
    if (cut == -LARGEST && rs.tmin == -INFINITY) {
      ONE_BY_ONE(EACH(mass += weight_of(sc, v[e]);))
    } else if (ties == ALL) {
      ONE_BY_ONE(float b = -INFINITY; EACH(b = fmaxf(b, v[e]);) if (__any(b >= cut))
                     EACH(const double t = log2_weight(sc, v[e]); mass = add_if(v[e] >= cut && t >= rs.tmin, fixed_weight(sc, t), mass);))
    } else {
      for (int64_t i0 = lo; i0 < hi; i0 += 64) {
        float v[VEC];
        if (i0 + lane < hi) row.load(i0 + lane, v);
        else EACH(v[e] = -INFINITY;)
        uint32_t n = 0;
        EACH(v[e] = clean(v[e]); n += v[e] == cut;)
        uint32_t before = eq + lanes_before<64>(n, lane);
        eq += across<64, Add>(n);
        EACH(const double t = log2_weight(sc, v[e]); const bool in = (v[e] > cut || (v[e] == cut && before++ < ties)) && t >= rs.tmin;
             mass = add_if(in, fixed_weight(sc, t), mass);)
      }
    }
    const u64 all = across<64, Add>((u64)mass);
    if (lane == 0) S.wsum[wave] = all;
    __syncthreads();
  }
  {
    u64 all = 0;
    for (int w = 0; w < NW; ++w) all += S.wsum[w];
    target = target_of(uu, all);
  }
  choose(width);
  // a lane's element of 64 neighbours from j0 on: its kept weight; ties: before j0, moved on
  const auto kept = [&](int64_t j0, int64_t end, uint32_t& before) {
    const float l = j0 + lane < end ? clean((float)row.x[j0 + lane]) : -INFINITY;
    const double t = log2_weight(sc, l);
    bool in = l >= cut && t >= rs.tmin;
    if (ties != ALL) {
      const u64 b = __ballot(l == cut);
      in = in && (l > cut || before + __popcll(b & ((1ull << lane) - 1)) < ties);
      before += __popcll(b);
    }
    return in ? fixed_weight(sc, t) : 0.0;
  };
  while (B - A > 64) {
    const int64_t share = ((B - A + NW - 1) / NW + 63) / 64 * 64, a = A + wave * share < B ? A + wave * share : B, b = a + share < B ? a + share : B;
    uint32_t before = tie;
    __syncthreads();
    if (ties != ALL) {
      uint32_t n = 0;
      for (int64_t j = a + lane; j < b; j += 64) n += clean((float)row.x[j]) == cut;
      n = across<64, Add>(n);
      if (lane == 0) S.wcnt[wave] = n;
      __syncthreads();
      for (int w = 0; w < wave; ++w) before += S.wcnt[w];
    }
    double mass = 0;
#pragma unroll 1
    for (int64_t j0 = a; j0 < b; j0 += 64) mass += kept(j0, b, before);
    const u64 all = across<64, Add>((u64)mass);
    if (lane == 0) S.wsum[wave] = all;
    __syncthreads();
    choose(share);
  }
  if (wave != 0) return;
  const u64 w = (u64)kept(A, B, tie), before = base + lanes_before<64>(w, lane);
  if (before <= target && target < before + w) out[r] = A + lane;
#undef EACH_PIECE
#undef ONE_BY_ONE
#undef EACH
}

template <typename T>
int launch_sample(int64_t rows, int64_t V, const void* logits, int64_t ld, const Settings& st, int F, const float* u, int64_t* out, hipStream_t s) {
  const T* x = (const T*)logits;
#define GROUP_(G, E)                                                                                                                             \
  hipLaunchKernelGGL((sample_group_kernel<T, G, E>), dim3((unsigned)cdiv64(rows, 256 / G)), dim3(256), 0, s, rows, (int)V, (int)cdiv64(V, G), x, ld, \
                     st, F, u, out)
  // as few lanes as leave a lane at most 16 logits (98304 x 120 bf16: 87 us with 16 lanes of 8, 89 with 4 of 32, but 300 rows 14
  // against 34; 65536 x 500: 167 with 64 lanes of 8, 161 with 16 of 32, but one row 8 against 17); up to 32 of them before a
  // workgroup per row, whose barriers cost more than that (16384 x 2000 float32: 172 us against 312)
  if (V <= 16) GROUP_(4, 4);
  else if (V <= 32) GROUP_(4, 8);
  else if (V <= 48) GROUP_(4, 12);
  else if (V <= 64) GROUP_(4, 16);
  else if (V <= 128) GROUP_(16, 8);
  else if (V <= 256) GROUP_(16, 16);
  else if (V <= 512) GROUP_(64, 8);
  else if (V <= 1024) GROUP_(64, 16);
  else if (V <= 1536) GROUP_(64, 24);
  else if (V <= 2048) GROUP_(64, 32);
#undef GROUP_
  else {
    // One workgroup per row.  Up to a row for every CU the largest that the row feeds is the fastest (top-k 50, 64 x 131072 bf16:
    // 44 / 26 / 20 us with 256 / 512 / 1024 threads; 1 x 32000: 13 / 11 / 13); with more rows small workgroups wait for each
    // other's barriers less (4096 x 8000 bf16: 49 / 81 / 171 us; 1024 x 32000: 23 / 30 / 54; 512 x 65536: 30 / 22 / 35).
    const int64_t bytes = V * (int64_t)sizeof(T);
    const bool many = rows > 256;
    int nt = many && bytes <= 98304 ? 256 : bytes <= (many ? 1 << 20 : 131072) ? 512 : 1024;
    // The next larger one where its list of candidates has room for a top-k that this one's has not, up to 160 and (rows that feed
    // it) 320 (4096 x 8000 float32, top-k 160: 150 us against 189, 200: 230 against 163; 1024 x 32000 bf16, 160: 49 against
    // 115; 512 x 65536, 256: 69 against 133; 2000 x 65536 float32, 320: 367 against 480; 1 x 32000, 256: 25 against 41).
    // Settings per row are not known here.
    const int64_t k = st.kr || st.k >= V ? 0 : st.k;
    if (nt == 256 && k > RowState<256>::FEW && k <= 160) nt = 512;
    if (nt == 512 && k > RowState<512>::FEW && k <= 320 && bytes > (many ? 98304 : 49152)) nt = 1024;
#define ROW_(NT) hipLaunchKernelGGL((sample_row_kernel<T, NT>), dim3((unsigned)rows), dim3(NT), 0, s, rows, V, x, ld, st, F, u, out)
    if (nt == 256) ROW_(256);
    else if (nt == 512) ROW_(512);
    else ROW_(1024);
#undef ROW_
  }
  TAD_LAUNCH_CHECK();
  return TAD_OK;
}

}  // namespace

extern "C" int tad_sample_tokens(int64_t rows, int64_t V, const void* logits, int dtype, int64_t ld, double temperature, const float* temperature_rows,
                                 int64_t top_k, const int32_t* top_k_rows, double top_p, const float* top_p_rows, double min_p,
                                 const float* min_p_rows, const float* u, int64_t* out, tad_stream_t stream) {
  TAD_CHECK(rows >= 0 && V >= 1 && V <= INT_MAX, "tad_sample_tokens: bad sizes");
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
  const int whole = V <= 2048 ? 53 : 61, F = whole - lg < 44 ? whole - lg : 44;       // bits of the row's largest sum (a thread's: 53)
  const Settings st = {temperature, top_p, min_p, top_k, temperature_rows, top_p_rows, min_p_rows, top_k_rows};
  hipStream_t s = (hipStream_t)stream;
  // at most 2^22 rows a launch: a grid holds fewer than 2^32 threads
  const int64_t step = (int64_t)1 << 22;
  for (int64_t r = 0; r < rows; r += step) {
    const int64_t part = rows - r < step ? rows - r : step;
    const Settings at = {st.T, st.p, st.minp, st.k, st.Tr ? st.Tr + r : nullptr, st.pr ? st.pr + r : nullptr, st.mr ? st.mr + r : nullptr,
                         st.kr ? st.kr + r : nullptr};
    const int rc = dtype == TAD_F32 ? launch_sample<float>(part, V, (const float*)logits + r * ld, ld, at, F, u + r, out + r, s)
                                    : launch_sample<bf16_t>(part, V, (const bf16_t*)logits + r * ld, ld, at, F, u + r, out + r, s);
    if (rc != TAD_OK) return rc;
  }
  return TAD_OK;
}
