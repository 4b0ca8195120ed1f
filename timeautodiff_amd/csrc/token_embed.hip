// Embedding lookup by integer tokens, with scaling, and its gradient over sorted tokens (gfx950).
//
//   forward:   out[i, :] = scale * table[tok[i], :]
//   gradient:  dtable[v, :] (+)= scale * sum over the i with tok[i] = v of dout[i, :]
//
// A token outside [0, vocab) is padding: a row of zeros forward, no share in any gradient.  Both move bytes and compute
// nothing to speak of: HBM bounds them (each row of dout read once, each row of dtable written once), and at a few
// thousand tokens the launches do.
//
// The gradient sums in a fixed order (the tokens sorted, equal ones by position; fp32), so it is the same bits every time,
// and its work is cut by sorted POSITION, not by row of the table: one token that fills the whole batch costs what any
// other batch costs.
#include <limits.h>
#include <math.h>

#include "common.h"

namespace {

typedef unsigned long long u64;

// ---------------------------------------------------------------- element packs
template <typename T, int VEC> struct Pack;
template <int VEC> struct Pack<float, VEC> { typedef float type __attribute__((ext_vector_type(VEC), aligned(VEC < 4 ? 4 * VEC : 16))); };
template <int VEC> struct Pack<bf16_t, VEC> { typedef __bf16 type __attribute__((ext_vector_type(VEC), aligned(2 * VEC))); };
template <> struct Pack<float, 1> { typedef float type; };
template <> struct Pack<bf16_t, 1> { typedef bf16_t type; };

template <typename T, int VEC>
__device__ __forceinline__ void load_pack(const T* p, float (&v)[VEC]) {
  typedef typename Pack<T, VEC>::type P;
  const P x = *reinterpret_cast<const P*>(p);
  if constexpr (VEC == 1) {
    v[0] = (float)x;
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = (float)x[i];
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_pack(T* p, const float (&v)[VEC]) {
  typedef typename Pack<T, VEC>::type P;
  P x;
  if constexpr (VEC == 1) {
    x = (T)v[0];
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[i] = (T)v[i];
  }
  *reinterpret_cast<P*>(p) = x;
}

// 16 bytes a lane, side by side, past the caches: rows of the table's gradient are not read again
template <int VEC>
__device__ __forceinline__ void stream_pack(float* p, const float (&v)[VEC]) {
  if constexpr (VEC == 4) {
    const f32x4 x = {v[0], v[1], v[2], v[3]};
    __builtin_nontemporal_store(x, reinterpret_cast<f32x4*>(p));
  } else {
    store_pack<float, VEC>(p, v);
  }
}

// ---------------------------------------------------------------- forward
// L lanes (a power of two, at most a wave) walk the columns of one row; a wave holds 64 / L rows side by side and U of them one
// after another, whose loads are all issued before the first is used.  32768 x 2048 bf16: 49 us, 5.5 TB/s; 98304 x 128 float32
// to bf16: 8.5 us, 3.1 TB/s (its waves wait once for a token and once for a row).
template <typename TI, typename TO, int VEC, int U>
__global__ __launch_bounds__(256) void token_embed_fwd_kernel(int64_t n, int nv, int lanes_log2, int64_t vocab, const int64_t* __restrict__ tok,
                                                              int64_t tstride, float scale, const TI* __restrict__ table, int64_t ldt,
                                                              TO* __restrict__ out, int64_t ldo) {
  const int L = 1 << lanes_log2;
  const int64_t group = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> lanes_log2;     // U rows each
  const int64_t ngroups = ((int64_t)gridDim.x * 256) >> lanes_log2;
  const int lane = threadIdx.x & (L - 1);
  int64_t row[U], t[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    row[u] = group + u * ngroups;
    t[u] = row[u] < n ? tok[row[u] * tstride] : -1;
  }
  for (int c = lane; c < nv; c += L) {
    float v[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[u][i] = 0.f;
      if ((uint64_t)t[u] < (uint64_t)vocab) load_pack<TI, VEC>(table + t[u] * ldt + (int64_t)c * VEC, v[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (row[u] < n) {
        const bool live = (uint64_t)t[u] < (uint64_t)vocab;
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[u][i] = live ? v[u][i] * scale : 0.f;
        store_pack<TO, VEC>(out + row[u] * ldo + (int64_t)c * VEC, v[u]);
      }
    }
  }
}

// ---------------------------------------------------------------- sorting the tokens
// key = token << 32 | position; padding gets the token `vocab`, behind every other.  Sorted by token, equal ones by position.
__device__ __forceinline__ u64 key_at(const int64_t* tok, int64_t tstride, int64_t vocab, int64_t i) {
  const int64_t t = tok[i * tstride];
  return ((u64)((uint64_t)t < (uint64_t)vocab ? t : vocab) << 32) | (u64)i;
}

// Up to RANK_N tokens: every token's place is counted directly, all pairs compared: a workgroup holds all tokens in LDS and
// counts for 64 of them, each of its 16 waves over a sixteenth of the others (two instructions a comparison of 64 lanes).  2400
// tokens: 6.7 us, most of it the wait for the tokens (a bitonic sort of them in one workgroup: 35).
constexpr int RANK_N = 8192;
__global__ __launch_bounds__(1024) void sort_rank_kernel(int n, int64_t vocab, const int64_t* __restrict__ tok, int64_t tstride, u64* __restrict__ keys) {
  __shared__ __attribute__((aligned(16))) uint32_t s[RANK_N];
  __shared__ uint32_t part[16][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int groups = (n + 63) >> 6, mine = blockIdx.x;
  for (int i = threadIdx.x; i < groups * 64; i += 1024) s[i] = i < n ? (uint32_t)(key_at(tok, tstride, vocab, i) >> 32) : UINT_MAX;
  __syncthreads();
  const uint32_t t = s[mine * 64 + lane];
  uint32_t rank = 0;
  for (int g = wave; g < groups; g += 16) {
    const uint4* p = reinterpret_cast<const uint4*>(s + g * 64);
    if (g != mine) {
      const uint32_t than = t + (g < mine);        // equal ones count where they come before
#pragma unroll
      for (int q = 0; q < 16; ++q) {
        const uint4 k = p[q];
        rank += k.x < than;
        rank += k.y < than;
        rank += k.z < than;
        rank += k.w < than;
      }
    } else {
      for (int q = 0; q < 64; ++q) rank += s[g * 64 + q] < t + (q < lane);
    }
  }
  part[wave][lane] = rank;
  __syncthreads();
  const int i = mine * 64 + lane;
  if (wave == 0 && i < n) {
    for (int w = 1; w < 16; ++w) rank += part[w][lane];
    keys[rank] = (u64)t << 32 | (u64)i;
  }
}

// More: by digits of up to 9 bits from the lowest, two launches a digit.  A workgroup has a tile of neighbouring keys, every
// wave a contiguous share of it, so that keys of one digit keep their order: the first launch counts digits by tile, the
// second adds up what comes before (lower digits; earlier tiles; earlier waves) and moves the keys.  No workgroup waits for
// another, and no distribution of tokens is worse than another.  98304 tokens of 9 bits: 3.2 + 9.5 us, latency of 96
// workgroups (fewer and larger tiles are slower, more of them read more counts).
constexpr int MAX_BINS = 512, MAX_TILES = 128, RWAVES = 8;

struct Digit {
  const int64_t* tok;       // the first digit's source
  int64_t tstride, vocab;
  const u64* in;            // the others'
  int64_t n;
  int tile, shift, bins;
  __device__ __forceinline__ u64 key(int64_t i) const { return in ? in[i] : key_at(tok, tstride, vocab, i); }
  __device__ __forceinline__ int of(u64 key) const { return (int)(key >> (32 + shift)) & (bins - 1); }
};

__global__ __launch_bounds__(512) void sort_count_kernel(Digit d, uint32_t* __restrict__ counts) {
  __shared__ uint32_t h[MAX_BINS];
  const int64_t base = (int64_t)blockIdx.x * d.tile;
  const int m = (int)(d.n - base < d.tile ? d.n - base : d.tile);
  h[threadIdx.x] = 0;
  __syncthreads();
#pragma unroll 4
  for (int i = threadIdx.x; i < m; i += 512) atomicAdd(&h[d.of(d.key(base + i))], 1u);
  __syncthreads();
  counts[blockIdx.x * MAX_BINS + threadIdx.x] = h[threadIdx.x];
}

__global__ __launch_bounds__(512) void sort_move_kernel(Digit d, int tiles, const uint32_t* __restrict__ counts, u64* __restrict__ out) {
  __shared__ uint32_t at[RWAVES][MAX_BINS];
  __shared__ uint32_t wsum[RWAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t base = (int64_t)blockIdx.x * d.tile;
  const int m = (int)(d.n - base < d.tile ? d.n - base : d.tile);
  const int share = d.tile / RWAVES, w0 = wave * share, w1 = w0 + share < m ? w0 + share : m;
#pragma unroll
  for (int w = 0; w < RWAVES; ++w) at[w][tid] = 0;
  __syncthreads();
#pragma unroll 4
  for (int i = w0 + lane; i < w1; i += 64) atomicAdd(&at[wave][d.of(d.key(base + i))], 1u);
  // this thread's digit: how many in all tiles, in the tiles before
  uint32_t all = 0, before = 0;
  for (int t0 = 0; t0 < tiles; t0 += 32) {
    uint32_t c[32];
#pragma unroll
    for (int t = 0; t < 32; ++t) c[t] = counts[(t0 + t < tiles ? t0 + t : 0) * MAX_BINS + tid];
#pragma unroll
    for (int t = 0; t < 32; ++t) {
      all += t0 + t < tiles ? c[t] : 0;
      before += t0 + t < (int)blockIdx.x ? c[t] : 0;
    }
  }
  uint32_t inc = all;
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t up = __shfl_up(inc, o);
    if (lane >= o) inc += up;
  }
  if (lane == 63) wsum[wave] = inc;
  __syncthreads();
  uint32_t place = before + inc - all;
  for (int w = 0; w < wave; ++w) place += wsum[w];
#pragma unroll
  for (int w = 0; w < RWAVES; ++w) {
    const uint32_t c = at[w][tid];
    at[w][tid] = place;
    place += c;
  }
  __syncthreads();
  volatile uint32_t* mine = at[wave];        // this wave's alone from here on
  constexpr int U = 4;                       // keys of 64 lanes in flight
  for (int i0 = w0; i0 < w1; i0 += 64 * U) {
    u64 key[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int i = i0 + 64 * k + lane;
      key[k] = d.key(base + (i < w1 ? i : w0));
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const bool on = i0 + 64 * k + lane < w1;
      const int g = d.of(key[k]);
      u64 same = __ballot(on);
      if (same == 0) break;
      for (int b = 1; b < d.bins; b <<= 1) {
        const u64 set = __ballot(g & b);
        same &= (g & b) ? set : ~set;
      }
      const int ahead = __popcll(same & ((1ull << lane) - 1));
      if (on) {
        const uint32_t p = mine[g];
        out[p + ahead] = key[k];
        if (ahead == 0) mine[g] = p + __popcll(same);
      }
    }
  }
}

// ---------------------------------------------------------------- sums over the sorted tokens
// A wave adds the rows of S <= 64 neighbouring sorted positions, 64 * VEC * M columns of them, GW waves (a chunk) side by side.
// A run of equal tokens inside a wave's share is a finished row of dtable.  What reaches over an edge between waves of the
// workgroup is added up in LDS, what reaches over its edges goes to the workspace (slot 0: the run that came in from the
// left; slot 1: one that begins here and goes on) and is added up by the launch behind, always in the order of positions.
// Eight rows are in flight a wave.  32768 x 2048 bf16 into 65536 rows, zeros included: 140 us, 4.8 TB/s; 98304 x 128 float32 into
// 500: 11.6 us, 4.4 TB/s.
constexpr int GW = 8;
constexpr int ZROWS = 8;      // rows of the table a wave of the zero part looks after

template <int VEC>
__device__ __forceinline__ void put_row(float* dt, const float (&acc)[VEC], float scale, int accumulate) {
  float v[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = acc[i] * scale;
  if (accumulate) {
    float o[VEC];
    load_pack<float, VEC>(dt, o);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] += o[i];
  }
  if (accumulate) store_pack<float, VEC>(dt, v);
  else stream_pack<VEC>(dt, v);
}

template <typename T, int VEC, int M>
__global__ __launch_bounds__(GW * 64) void embed_grad_sum_kernel(int64_t n, int D, int64_t vocab, int S, int64_t nchunks, int ctiles, float scale,
                                                                 int accumulate, const u64* __restrict__ keys, const T* __restrict__ dout, int64_t ldd,
                                                                 float* __restrict__ dtable, int64_t ldg, float* __restrict__ part) {
  constexpr int CT = 64 * VEC * M, U = 8;
  __shared__ __attribute__((aligned(16))) float edge[GW][2][CT];
  __shared__ uint32_t head_tok[GW], state[GW];       // state: 1 a run came in, 2 and ends here, 4 one goes on
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (blockIdx.x >= nchunks * ctiles) {
    // rows that no token names are zero (overwriting mode): a lane looks one row up in the sorted keys
    const int64_t v0 = ((blockIdx.x - nchunks * ctiles) * GW + wave) * ZROWS;
    if (v0 >= vocab) return;
    const int64_t v = v0 + (lane & (ZROWS - 1));
    int64_t lo = 0, hi = n;
    const u64 want = (u64)v << 32;
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (keys[mid] < want) lo = mid + 1; else hi = mid;
    }
    const bool absent = v < vocab && (lo == n || (keys[lo] >> 32) != (u64)v);
    const u64 todo = __ballot(absent);
    for (int r = 0; r < ZROWS; ++r) {
      if (!(todo >> r & 1)) continue;
      float* row = dtable + (v0 + r) * ldg;
      for (int c = lane * VEC; c < D; c += 64 * VEC) {
        float z[VEC] = {};
        stream_pack<VEC>(row + c, z);
      }
    }
    return;
  }
  const int64_t chunk = blockIdx.x / ctiles;
  const int c0 = (int)(blockIdx.x - chunk * ctiles) * CT, c = c0 + lane * VEC;
  const int64_t a = (chunk * GW + wave) * S;
  const int m = a < n ? (int)(n - a < S ? n - a : S) : 0;
  bool on[M];
#pragma unroll
  for (int p = 0; p < M; ++p) on[p] = c + p * 64 * VEC < D;
  uint32_t st = 0;
  if (m > 0) {
    const u64 key = keys[a + (lane < m ? lane : m - 1)];
    const uint32_t tok = (uint32_t)(key >> 32);
    const uint32_t left = a > 0 ? (uint32_t)(keys[a - 1] >> 32) : UINT_MAX;
    const uint32_t right = a + m < n ? (uint32_t)(keys[a + m] >> 32) : UINT_MAX;
    const int live = __popcll(__ballot(lane < m && tok < (uint64_t)vocab));      // padding lies behind everything else
    uint32_t next = (uint32_t)__shfl_down(tok, 1);
    if (lane == m - 1) next = right;
    const u64 ends = __ballot(lane < live && tok != next);
    const uint32_t tok0 = __builtin_amdgcn_readfirstlane(tok);
    bool came = live > 0 && tok0 == left;
    float acc[M][VEC] = {};
    for (int j0 = 0; j0 < live; j0 += U) {
      float v[U][M][VEC];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int j = j0 + k < live ? j0 + k : live - 1;             // (the last row again, not added: the loads need no branch)
        const uint32_t pos = __builtin_amdgcn_readlane((uint32_t)key, j);
#pragma unroll
        for (int p = 0; p < M; ++p)
          if (on[p]) load_pack<T, VEC>(dout + (int64_t)pos * ldd + c + p * 64 * VEC, v[k][p]);
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int j = j0 + k;
        if (j >= live) break;
#pragma unroll
        for (int p = 0; p < M; ++p)
#pragma unroll
          for (int i = 0; i < VEC; ++i) acc[p][i] += v[k][p][i];
        if (ends >> j & 1) {
          const int64_t row = (int64_t)__builtin_amdgcn_readlane(tok, j) * ldg + c;
#pragma unroll
          for (int p = 0; p < M; ++p) {
            if (came) store_pack<float, VEC>(&edge[wave][0][(p * 64 + lane) * VEC], acc[p]);
            else if (on[p]) put_row<VEC>(dtable + row + p * 64 * VEC, acc[p], scale, accumulate);
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[p][i] = 0.f;
          }
          if (came) st |= 3;
          came = false;
        }
      }
    }
    if (live > 0 && !(ends >> (live - 1) & 1)) {                     // goes on to the right
#pragma unroll
      for (int p = 0; p < M; ++p) store_pack<float, VEC>(&edge[wave][came ? 0 : 1][(p * 64 + lane) * VEC], acc[p]);
      st |= came ? 1 : 4;
    }
    if (lane == 0) head_tok[wave] = tok0;
  }
  if (lane == 0) state[wave] = st;
  __syncthreads();
  for (int cc = threadIdx.x; cc < CT && c0 + cc < D; cc += GW * 64) {
    float run = 0.f;
    bool outer = true, open = false;            // the run in hand began left of the workgroup; there is one
    for (int w = 0; w < GW; ++w) {
      const uint32_t f = state[w];
      if (f & 1) {
        run += edge[w][0][cc];
        open = true;
        if (f & 2) {
          if (outer) {
            part[(2 * chunk) * D + c0 + cc] = run;
          } else {
            float one[1] = {run};
            put_row<1>(dtable + (int64_t)head_tok[w] * ldg + c0 + cc, one, scale, accumulate);
          }
          open = false;
        }
      }
      if (f & 4) {
        run = edge[w][1][cc];
        outer = false;
        open = true;
      }
    }
    if (open) part[(2 * chunk + (outer ? 0 : 1)) * D + c0 + cc] = run;
  }
}

// Runs that reach over the edges of chunks: a workgroup for each chunk in which one begins (the others leave at once) and
// each 64 * VEC columns; its waves add every fourth part, and the four sums are added in order.  4.6 us, loads that wait for
// each other (5.3 with the parts asked for only when it is known which).
template <int VEC>
__global__ __launch_bounds__(256) void embed_grad_join_kernel(int64_t n, int D, int64_t vocab, int P, int64_t nchunks, int ctiles, float scale,
                                                              int accumulate, const u64* __restrict__ keys, const float* __restrict__ part,
                                                              float* __restrict__ dtable, int64_t ldg) {
  __shared__ __attribute__((aligned(16))) float s[4][64 * VEC];
  const int64_t chunk = blockIdx.x / ctiles;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = ((int)(blockIdx.x - chunk * ctiles) * 64 + lane) * VEC;
  const int64_t a = chunk * P, b = a + P;                       // (not the last chunk: nothing goes on from there)
  // the tokens that decide and the wave's first parts are asked for together (parts that turn out not to be are not used)
  const auto begins = [&](int64_t k) { return (uint32_t)(keys[(k < nchunks ? k : chunk) * P] >> 32); };
  const uint32_t t = (uint32_t)(keys[b] >> 32), at_end = (uint32_t)(keys[b - 1] >> 32), at_start = a > 0 ? (uint32_t)(keys[a - 1] >> 32) : UINT_MAX;
  uint32_t next = begins(chunk + 1 + lane);
  float own[VEC] = {}, one[VEC] = {};
  if (c < D) {
    if (wave == 0) load_pack<float, VEC>(part + (2 * chunk + 1) * D + c, own);
    if (chunk + 1 + wave < nchunks) load_pack<float, VEC>(part + (2 * (chunk + 1 + wave)) * D + c, one);
  }
  if (t >= (uint64_t)vocab || at_end != t || at_start == t) return;
  int64_t last = chunk;                                         // the last chunk that begins inside the run
  for (;;) {
    const u64 in = __ballot(last + 1 + lane < nchunks && next == t);
    last += in == ~0ull ? 64 : __ffsll((long long)~in) - 1;
    if (in != ~0ull) break;
    next = begins(last + 1 + lane);
  }
  float acc[VEC] = {};
  if (c < D) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = wave == 0 ? own[i] : 0.f;
    if (chunk + 1 + wave <= last) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] += one[i];
    }
#pragma unroll 8
    for (int64_t k = chunk + 5 + wave; k <= last; k += 4) {
      float v[VEC];
      load_pack<float, VEC>(part + (2 * k) * D + c, v);
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] += v[i];
    }
  }
  store_pack<float, VEC>(&s[wave][lane * VEC], acc);
  __syncthreads();
  if (wave == 0 && c < D) {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      acc[i] = ((s[0][lane * VEC + i] + s[1][lane * VEC + i]) + s[2][lane * VEC + i]) + s[3][lane * VEC + i];
    put_row<VEC>(dtable + (int64_t)t * ldg + c, acc, scale, accumulate);
  }
}

// Few tokens and few rows: a workgroup for each row of the table and each 64 * VEC columns looks through all tokens itself, each
// of its 16 waves through a sixteenth of them, and adds what it finds: one launch, where sorting takes three.  2400 x 128 into 50
// rows: 6.8 us (sorted: 15).
constexpr int DIRECT_N = 4096, DIRECT_WAVES = 16;

template <typename T, int VEC>
__global__ __launch_bounds__(DIRECT_WAVES * 64) void embed_grad_direct_kernel(int n, int D, int64_t vocab, int ctiles, float scale, int accumulate,
                                                                              const int64_t* __restrict__ tok, int64_t tstride,
                                                                              const T* __restrict__ dout, int64_t ldd, float* __restrict__ dtable,
                                                                              int64_t ldg) {
  constexpr int SLICE = DIRECT_N / DIRECT_WAVES, U = 8;
  __shared__ __attribute__((aligned(16))) float part[DIRECT_WAVES][64 * VEC];
  __shared__ uint16_t found[DIRECT_WAVES][SLICE];
  __shared__ int number[DIRECT_WAVES];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int v = blockIdx.x / ctiles, c = ((int)blockIdx.x - v * ctiles) * 64 * VEC + lane * VEC;
  const int slice = ((n + DIRECT_WAVES * 64 - 1) / (DIRECT_WAVES * 64)) * 64, lo = wave * slice, hi = lo + slice < n ? lo + slice : n;
  int count = 0;
#pragma unroll
  for (int k = 0; k < SLICE / 64; ++k) {
    const int i = lo + 64 * k + lane;
    const bool in = 64 * k < slice && i < hi && tok[i * tstride] == v;
    const u64 b = __ballot(in);
    if (in) found[wave][count + __popcll(b & ((1ull << lane) - 1))] = (uint16_t)i;
    count += __popcll(b);
  }
  if (lane == 0) number[wave] = count;
  float acc[VEC] = {};
  for (int j0 = 0; j0 < count; j0 += U) {
    float x[U][VEC];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int pos = found[wave][j0 + k < count ? j0 + k : count - 1];
      if (c < D) load_pack<T, VEC>(dout + pos * ldd + c, x[k]);
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (j0 + k >= count) break;
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] += x[k][i];
    }
  }
  store_pack<float, VEC>(&part[wave][lane * VEC], acc);
  __syncthreads();
  if (wave != 0 || c >= D) return;
  int total = 0;
#pragma unroll
  for (int w = 0; w < DIRECT_WAVES; ++w) total += number[w];
  if (accumulate && total == 0) return;
#pragma unroll
  for (int w = 1; w < DIRECT_WAVES; ++w)
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] += part[w][lane * VEC + i];
  put_row<VEC>(dtable + v * ldg + c, acc, scale, accumulate);
}

// ---------------------------------------------------------------- host side
// workgroups that write the rows which no token names (overwriting mode only)
inline int64_t zero_groups(int64_t vocab, int accumulate) { return accumulate ? 0 : cdiv64(vocab, ZROWS * GW); }

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

constexpr int64_t COUNT_BYTES = MAX_TILES * MAX_BINS * 4;
inline int64_t key_bytes(int64_t n) { return (n * 8 + 15) / 16 * 16; }

// How the gradient is cut: S positions a wave, `packs` packs of VEC columns a lane.
struct GradPlan {
  int vec, packs, S, ctiles;
  int64_t nchunks;
};
GradPlan grad_plan(int64_t n, int D, int dtype, bool wide) {
  GradPlan g;
  g.vec = 1;
  if (wide)
    while (g.vec < 4 && D >= 128 * g.vec) g.vec *= 2;
  g.packs = dtype == TAD_BF16 && g.vec == 4 && D >= 512 ? 2 : 1;
  g.ctiles = (int)cdiv64(D, 64 * g.vec * g.packs);
  g.S = 64;
  while (g.S > 8 && cdiv64(n, g.S) * g.ctiles < 4096) g.S /= 2;
  g.nchunks = cdiv64(n, g.S * GW);
  return g;
}

template <typename TI, typename TO>
int launch_fwd(int64_t n, int D, int64_t vocab, const int64_t* tok, int64_t tstride, float scale, const void* table, int64_t ldt, void* out,
               int64_t ldo, hipStream_t s) {
  constexpr int V = sizeof(TI) + sizeof(TO) < 8 ? 8 : 4;
  const bool wide = D % V == 0 && ldt % V == 0 && ldo % V == 0 && aligned16(table) && aligned16(out);
  const int nv = wide ? D / V : D;
  int ll = 0;
  while (ll < 6 && (1 << ll) < nv) ++ll;
  // four rows a lane where that still leaves every CU several waves
  const bool many = (cdiv64(n, 4) << ll) >= 256 * 1024;
  const int64_t grid = cdiv64(cdiv64(n, many ? 4 : 1) << ll, 256);
  TAD_CHECK(grid < (1 << 24), "tad_token_embed_fwd: too many tokens");          // (a grid holds fewer than 2^32 threads)
#define FWD_(VEC, U)                                                                                                                                   \
  hipLaunchKernelGGL((token_embed_fwd_kernel<TI, TO, VEC, U>), dim3((unsigned)grid), dim3(256), 0, s, n, nv, ll, vocab, tok, tstride, scale, (const TI*)table, \
                     ldt, (TO*)out, ldo)
  if (wide) {
    if (many) FWD_(V, 4); else FWD_(V, 1);
  } else {
    if (many) FWD_(1, 4); else FWD_(1, 1);
  }
#undef FWD_
  TAD_LAUNCH_CHECK();
  return TAD_OK;
}

template <typename T, int VEC>
void launch_direct(int64_t n, int D, int64_t vocab, const int64_t* tok, int64_t tstride, float scale, int accumulate, const void* dout, int64_t ldd,
                   float* dtable, int64_t ldg, hipStream_t s) {
  const int ct = (int)cdiv64(D, 64 * VEC);
  hipLaunchKernelGGL((embed_grad_direct_kernel<T, VEC>), dim3((unsigned)(vocab * ct)), dim3(DIRECT_WAVES * 64), 0, s, (int)n, D, vocab, ct, scale,
                     accumulate, tok, tstride, (const T*)dout, ldd, dtable, ldg);
}

template <typename T, int VEC, int M>
void launch_sum(const GradPlan& g, int64_t n, int D, int64_t vocab, float scale, int accumulate, const u64* keys, const void* dout, int64_t ldd,
                float* dtable, int64_t ldg, float* part, hipStream_t s) {
  const int64_t grid = g.nchunks * g.ctiles + zero_groups(vocab, accumulate);
  hipLaunchKernelGGL((embed_grad_sum_kernel<T, VEC, M>), dim3((unsigned)grid), dim3(GW * 64), 0, s, n, D, vocab, g.S, g.nchunks, g.ctiles, scale,
                     accumulate, keys, (const T*)dout, ldd, dtable, ldg, part);
}

}  // namespace

extern "C" int tad_token_embed_fwd(int64_t n, int D, int64_t vocab, const int64_t* tokens, int64_t tok_stride, float scale, const void* table,
                                   int table_dtype, int64_t ld_table, void* out, int out_dtype, int64_t ldo, tad_stream_t stream) {
  TAD_CHECK(n >= 0 && D >= 1 && vocab >= 0, "tad_token_embed_fwd: bad sizes");
  TAD_CHECK((table_dtype == TAD_F32 || table_dtype == TAD_BF16) && (out_dtype == TAD_F32 || out_dtype == TAD_BF16), "tad_token_embed_fwd: bad element type");
  TAD_CHECK(ld_table >= D && ldo >= D && tok_stride >= 0, "tad_token_embed_fwd: bad leading dimension");
  TAD_CHECK(n < (int64_t)1 << 40, "tad_token_embed_fwd: too many tokens");        // (the sizes of the launch are formed in 64 bits)
  if (n == 0) return TAD_OK;
  TAD_CHECK(tokens && out && (table || vocab == 0), "tad_token_embed_fwd: null pointer");
  hipStream_t s = (hipStream_t)stream;
  if (table_dtype == TAD_F32)
    return out_dtype == TAD_F32 ? launch_fwd<float, float>(n, D, vocab, tokens, tok_stride, scale, table, ld_table, out, ldo, s)
                                : launch_fwd<float, bf16_t>(n, D, vocab, tokens, tok_stride, scale, table, ld_table, out, ldo, s);
  return out_dtype == TAD_F32 ? launch_fwd<bf16_t, float>(n, D, vocab, tokens, tok_stride, scale, table, ld_table, out, ldo, s)
                              : launch_fwd<bf16_t, bf16_t>(n, D, vocab, tokens, tok_stride, scale, table, ld_table, out, ldo, s);
}

// the keys twice, the digits' counts, then the parts of runs over edges
extern "C" int64_t tad_token_embed_bwd_workspace_bytes(int64_t n, int D) {
  if (n <= 0 || D < 1) return 0;
  // the parts of the finest cut that any alignment or type of dout leads to
  int64_t part = 0;
  for (int dt = TAD_F32; dt <= TAD_BF16; ++dt)
    for (int wide = 0; wide < 2; ++wide) {
      const GradPlan g = grad_plan(n, D, dt, wide);
      if (2 * g.nchunks * D > part) part = 2 * g.nchunks * D;
    }
  return 2 * key_bytes(n) + COUNT_BYTES + part * 4;
}

extern "C" int tad_token_embed_bwd(int64_t n, int D, int64_t vocab, const int64_t* tokens, int64_t tok_stride, float scale, const void* dout,
                                   int dout_dtype, int64_t ld_dout, float* dtable, int64_t ld_dtable, int accumulate, void* workspace,
                                   int64_t workspace_bytes, tad_stream_t stream) {
  TAD_CHECK(n >= 0 && D >= 1 && vocab >= 0, "tad_token_embed_bwd: bad sizes");
  TAD_CHECK(n <= INT_MAX && vocab < INT_MAX, "tad_token_embed_bwd: more than 2^31 - 1 tokens or rows");
  TAD_CHECK(dout_dtype == TAD_F32 || dout_dtype == TAD_BF16, "tad_token_embed_bwd: bad element type");
  TAD_CHECK(ld_dout >= D && ld_dtable >= D && tok_stride >= 0, "tad_token_embed_bwd: bad leading dimension");
  if (vocab == 0 || (n == 0 && accumulate)) return TAD_OK;
  TAD_CHECK(dtable && (n == 0 || (tokens && dout)), "tad_token_embed_bwd: null pointer");
  hipStream_t s = (hipStream_t)stream;
  if (n == 0) return tad_zero_2d(vocab, (int64_t)D * 4, dtable, ld_dtable * 4, stream);
  const bool wide = D % 4 == 0 && ld_dtable % 4 == 0 && ld_dout % 4 == 0 && aligned16(dout) && aligned16(dtable);
  const GradPlan g = grad_plan(n, D, dout_dtype, wide);
  const int64_t kb = key_bytes(n);
  TAD_CHECK(workspace && aligned16(workspace) && workspace_bytes >= 2 * kb + COUNT_BYTES + 2 * g.nchunks * D * 4,
            "tad_token_embed_bwd: workspace of %lld bytes, 16-byte aligned, needed", (long long)tad_token_embed_bwd_workspace_bytes(n, D));
  TAD_CHECK(g.nchunks * g.ctiles + zero_groups(vocab, accumulate) < (1 << 23) && g.nchunks * cdiv64(D, wide ? 256 : 64) < (1 << 24),
            "tad_token_embed_bwd: too many tokens or rows");                        // (a grid holds fewer than 2^32 threads)
  // the direct form, where its workgroups are few (2048: two rounds of the chip), read the tokens few times (2^22: 32 MB from L2)
  // and a row of the table does not get so many tokens that the one workgroup's time is theirs (2400 tokens of 128 columns
  // into 50, 500, 1700 rows: 11 us against 15 sorted; 4096 into 2 rows: 24 against 17; 100 into 40000 rows: 99 against 15)
  const int64_t groups = vocab * cdiv64(D, 64 * g.vec);
  if (n <= DIRECT_N && vocab <= 2048 && groups <= 2048 && groups * n <= (1 << 22) && (n <= 1024 || n <= 128 * vocab)) {
#define DIRECT_(T, V) launch_direct<T, V>(n, D, vocab, tokens, tok_stride, scale, accumulate, dout, ld_dout, dtable, ld_dtable, s)
    if (dout_dtype == TAD_BF16) {
      if (g.vec == 4) DIRECT_(bf16_t, 4); else if (g.vec == 2) DIRECT_(bf16_t, 2); else DIRECT_(bf16_t, 1);
    } else {
      if (g.vec == 4) DIRECT_(float, 4); else if (g.vec == 2) DIRECT_(float, 2); else DIRECT_(float, 1);
    }
#undef DIRECT_
    TAD_LAUNCH_CHECK();
    return TAD_OK;
  }
  u64* a = (u64*)workspace;
  u64* b = (u64*)((char*)workspace + kb);
  uint32_t* counts = (uint32_t*)((char*)workspace + 2 * kb);
  float* part = (float*)((char*)workspace + 2 * kb + COUNT_BYTES);
  if (n <= RANK_N) {
    hipLaunchKernelGGL(sort_rank_kernel, dim3((unsigned)cdiv64(n, 64)), dim3(1024), 0, s, (int)n, vocab, tokens, tok_stride, a);
    TAD_LAUNCH_CHECK();
  } else {
    int bits = 1, tile = 512;
    while (vocab >> bits) ++bits;                      // tokens 0 .. vocab (padding)
    while (cdiv64(n, tile) > MAX_TILES) tile *= 2;
    const int digits = (bits + 8) / 9, width = (bits + digits - 1) / digits, tiles = (int)cdiv64(n, tile);
    Digit d = {tokens, tok_stride, vocab, nullptr, n, tile, 0, 1 << width};
    for (int k = 0; k < digits; ++k, d.shift += width) {
      hipLaunchKernelGGL(sort_count_kernel, dim3((unsigned)tiles), dim3(512), 0, s, d, counts);
      TAD_LAUNCH_CHECK();
      hipLaunchKernelGGL(sort_move_kernel, dim3((unsigned)tiles), dim3(512), 0, s, d, tiles, counts, a);
      TAD_LAUNCH_CHECK();
      d.in = a;
      u64* t = a; a = b; b = t;
    }
    a = b;
  }
#define SUM_(T, V, M) launch_sum<T, V, M>(g, n, D, vocab, scale, accumulate, a, dout, ld_dout, dtable, ld_dtable, part, s)
  if (dout_dtype == TAD_BF16) {
    if (g.packs == 2) SUM_(bf16_t, 4, 2); else if (g.vec == 4) SUM_(bf16_t, 4, 1); else if (g.vec == 2) SUM_(bf16_t, 2, 1); else SUM_(bf16_t, 1, 1);
  } else {
    if (g.vec == 4) SUM_(float, 4, 1); else if (g.vec == 2) SUM_(float, 2, 1); else SUM_(float, 1, 1);
  }
#undef SUM_
  TAD_LAUNCH_CHECK();
  if (g.nchunks > 1) {
    const int64_t most = g.nchunks - 1;
    const int ct = (int)cdiv64(D, wide ? 256 : 64);
    if (wide)
      hipLaunchKernelGGL((embed_grad_join_kernel<4>), dim3((unsigned)(most * ct)), dim3(256), 0, s, n, D, vocab, g.S * GW, g.nchunks, ct, scale, accumulate,
                         a, part, dtable, ld_dtable);
    else
      hipLaunchKernelGGL((embed_grad_join_kernel<1>), dim3((unsigned)(most * ct)), dim3(256), 0, s, n, D, vocab, g.S * GW, g.nchunks, ct, scale, accumulate,
                         a, part, dtable, ld_dtable);
    TAD_LAUNCH_CHECK();
  }
  return TAD_OK;
}
